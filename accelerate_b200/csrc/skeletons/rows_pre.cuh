// Helpers of the row operators (log probabilities, distillation, layer norm): 16-byte blocks of Half or
// Float values, conversions, warp sums.  Included in front of every rows_*.cuh skeleton.
//
//   ROW_F16      1: the row's elements are Half, 0: Float
//   ROW_THREADS  threads per CTA

#if ROW_F16
typedef u16 row_t;
#else
typedef f32 row_t;
#endif
constexpr int ROW_E = 16 / (int)sizeof(row_t);   // elements per 16-byte block

#define ROW_INF __int_as_float(0x7f800000)
#define ROW_NAN __int_as_float(0x7fc00000)
#define ROW_LOG2E 1.44269504088896341f
#define ROW_LN2 0.693147180559945309f

__device__ __forceinline__ f32 row_h2f(u16 h) { f32 r; asm("cvt.f32.f16 %0, %1;" : "=f"(r) : "h"(h)); return r; }
__device__ __forceinline__ u16 row_f2h(f32 v) { u16 r; asm("cvt.rn.f16.f32 %0, %1;" : "=h"(r) : "f"(v)); return r; }
__device__ __forceinline__ f32 row_wide(u16 h) { return row_h2f(h); }
__device__ __forceinline__ f32 row_wide(f32 v) { return v; }
__device__ __forceinline__ void row_narrow(f32 v, u16& o) { o = row_f2h(v); }
__device__ __forceinline__ void row_narrow(f32 v, f32& o) { o = v; }
// 2^x, relative error 2^-22 (0 for -inf, NaN for NaN); one instruction of the special-function unit
__device__ __forceinline__ f32 row_ex2(f32 x) { f32 r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
__device__ __forceinline__ f32 row_max_nan(f32 a, f32 b) { f32 r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ u32 row_max_nan2(u32 a, u32 b) { u32 r; asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
__device__ __forceinline__ void row_h2x2(u32 w, f32& lo, f32& hi) {
  asm("{ .reg .b16 l, h; mov.b32 {l, h}, %2; cvt.f32.f16 %0, l; cvt.f32.f16 %1, h; }" : "=f"(lo), "=f"(hi) : "r"(w));
}
__device__ __forceinline__ u32 row_x2h2(f32 lo, f32 hi) { u32 r; asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo)); return r; }

// Two Floats in one 64-bit register: an instruction does both (each rounded as if alone).  The statistics with
// alternatives are bound by instructions issued, and this saves half the additions' and products' slots (4096 x 131072
// Halves, k = 20: 221 -> 212 us).  The norms and distillation's gradient gain nothing from it and do without.
typedef u64 row_two;
__device__ __forceinline__ row_two row_pair(f32 a, f32 b) { row_two r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ void row_split(row_two v, f32& a, f32& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ row_two row_fma2(row_two a, row_two b, row_two c) { row_two r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ row_two row_mul2(row_two a, row_two b) { row_two r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ row_two row_add2(row_two a, row_two b) { row_two r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }

// The elements of a 16-byte block as Floats, and back (rounded to nearest even).
__device__ __forceinline__ void row_unpack(const uint4& b, f32 (&v)[ROW_E]) {
  const u32 w[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#if ROW_F16
    row_h2x2(w[i], v[2 * i], v[2 * i + 1]);
#else
    v[i] = __uint_as_float(w[i]);
#endif
  }
}
__device__ __forceinline__ uint4 row_pack(const f32 (&v)[ROW_E]) {
  u32 w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#if ROW_F16
    w[i] = row_x2h2(v[2 * i], v[2 * i + 1]);
#else
    w[i] = __float_as_uint(v[i]);
#endif
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
#if ROW_F16
#define ROW_PAD 0xfc00fc00u      /* two Halves of -inf */
#else
#define ROW_PAD 0xff800000u      /* -inf */
#endif

// A row that may start anywhere: the aligned 16-byte blocks that touch it.  Block i holds the elements
// [i*E - shift, i*E - shift + E); only the first and the last may reach over the row's ends.
struct row_span {
  const row_t* x;      // the row's first element
  int n, shift, blocks;
  __device__ __forceinline__ row_span(const row_t* x_, int n_) : x(x_), n(n_) {
    shift = (int)(((u64)x_ & 15) / sizeof(row_t));
    blocks = n_ > 0 ? (shift + n_ + ROW_E - 1) / ROW_E : 0;
  }
  __device__ __forceinline__ int first(int i) const { return i * ROW_E - shift; }
  // Block i; elements outside the row read as -inf, which no statistic counts.  Nothing outside the row is touched.
  __device__ __forceinline__ uint4 load(int i) const {
    const int j = first(i);
    if (j >= 0 && j + ROW_E <= n) return __ldcs(reinterpret_cast<const uint4*>(x + j));
    u64 w[2] = {(u64)ROW_PAD << 32 | ROW_PAD, (u64)ROW_PAD << 32 | ROW_PAD};
    constexpr int BITS = 8 * (int)sizeof(row_t);
    const int e0 = j < 0 ? -j : 0, e1 = min(ROW_E, n - j);
#pragma unroll 1
    for (int e = e0; e < e1; ++e) {
#if ROW_F16
      const u64 h = x[j + e];
#else
      const u64 h = __float_as_uint(x[j + e]);
#endif
      const int at = e * BITS & 63;
      const u64 mask = (((u64)1 << BITS) - 1) << at;
      if (e * BITS < 64) w[0] = (w[0] & ~mask) | (h << at);
      else w[1] = (w[1] & ~mask) | (h << at);
    }
    return make_uint4((u32)w[0], (u32)(w[0] >> 32), (u32)w[1], (u32)(w[1] >> 32));
  }
  // The blocks that lie wholly inside the row: [inner0, inner1)
  __device__ __forceinline__ int inner0() const { return shift ? 1 : 0; }
  __device__ __forceinline__ int inner1() const { return (shift + n) / ROW_E; }
  // Block i of those
  __device__ __forceinline__ uint4 load_inner(int i) const { return __ldcs(reinterpret_cast<const uint4*>(x - shift) + i); }
  // U blocks per thread, THREADS apart, from block t on; blocks from `end` on read as -inf
  template <int U> __device__ __forceinline__ void load_tile(uint4 (&b)[U], int t, int end) const {
    const int i = t + (int)threadIdx.x;
    if (t >= inner0() && t + U * ROW_THREADS <= min(end, inner1())) {
#pragma unroll
      for (int u = 0; u < U; ++u) b[u] = load_inner(i + u * ROW_THREADS);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) b[u] = i + u * ROW_THREADS < end ? load(i + u * ROW_THREADS) : make_uint4(ROW_PAD, ROW_PAD, ROW_PAD, ROW_PAD);
    }
  }
};

// ---- warp sums and maxima (every lane gets the result; the order of the additions is fixed) ----
__device__ __forceinline__ f32 row_warp_sum(f32 v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(ACC_FULL_MASK, v, d);
  return v;
}
__device__ __forceinline__ f32 row_warp_max(f32 v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor_sync(ACC_FULL_MASK, v, d));
  return v;
}
