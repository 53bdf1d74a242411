// What the layer norm kernels share: a row spread over NORM_WARPS warps (NORM_GROUP lanes), NORM_U accesses of
// NORM_VE elements per lane.  Lane g holds the elements [(u * NORM_GROUP + g) * NORM_VE, + NORM_VE).
//
//   NORM_VE     elements per access, a power of two: the widest access, up to 16 bytes, on whose boundary every row
//               and both parameter vectors start; neighbouring lanes hold neighbouring accesses, so that narrow ones
//               still cover whole sectors
//   NORM_WARPS  warps per row, a power of two; NORM_ROWS rows per CTA at a time
//   NORM_U      accesses per lane;  NORM_GROUP * NORM_U * NORM_VE >= n

#define NORM_GROUP (NORM_WARPS * 32)
#define NORM_ROWS (ROW_THREADS / NORM_GROUP)

template <int N> struct __align__(2 * N) norm_bits16 { u16 v[N]; };
template <int N> struct __align__(4 * N) norm_bits32 { f32 v[N]; };
template <class T, int N> struct norm_vec;
template <int N> struct norm_vec<u16, N> { typedef norm_bits16<N> type; };
template <int N> struct norm_vec<f32, N> { typedef norm_bits32<N> type; };
#if ROW_F16
#define NORM_BYTES (2 * NORM_VE)
#else
#define NORM_BYTES (4 * NORM_VE)
#endif
template <int B> struct norm_raw;
template <> struct norm_raw<16> { typedef uint4 type; };
template <> struct norm_raw<8> { typedef uint2 type; };
template <> struct norm_raw<4> { typedef u32 type; };
template <> struct norm_raw<2> { typedef u16 type; };
typedef norm_raw<NORM_BYTES>::type norm_word;
// What came with one access.  Halves stay in the words they came in; Floats are kept as Floats (as words, the
// compiler's schedule cost the forward kernel 6 to 10 %).
#if ROW_F16
typedef norm_word norm_x;
#else
typedef norm_vec<f32, NORM_VE>::type norm_x;
#endif

// One access of x or dy: read once, so it takes no place in L1 (gamma and beta live there).
__device__ __forceinline__ norm_x norm_load(const row_t* p) {
  norm_word w;
#if NORM_BYTES == 16
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "l"(p));
#else
  w = __ldcs(reinterpret_cast<const norm_word*>(p));
#endif
  norm_x r;
  memcpy(&r, &w, NORM_BYTES);
  return r;
}
// the same from shared memory
__device__ __forceinline__ norm_x norm_shared(const norm_x* p) {
  const norm_word w = *reinterpret_cast<const norm_word*>(p);
  norm_x r;
  memcpy(&r, &w, NORM_BYTES);
  return r;
}
__device__ __forceinline__ void norm_wide(const norm_x& b, f32 (&v)[NORM_VE]) {
#if ROW_F16 && NORM_VE > 1
  u32 w[NORM_VE / 2];
  memcpy(w, &b, NORM_BYTES);
#pragma unroll
  for (int i = 0; i < NORM_VE / 2; ++i) row_h2x2(w[i], v[2 * i], v[2 * i + 1]);
#elif ROW_F16
  v[0] = row_h2f(b);
#else
#pragma unroll
  for (int e = 0; e < NORM_VE; ++e) v[e] = b.v[e];
#endif
}
__device__ __forceinline__ void norm_store(row_t* p, const f32 (&v)[NORM_VE]) {
#if ROW_F16 && NORM_VE > 1
  u32 w[NORM_VE / 2];
#pragma unroll
  for (int i = 0; i < NORM_VE / 2; ++i) w[i] = row_x2h2(v[2 * i], v[2 * i + 1]);
#elif ROW_F16
  const u16 w = row_f2h(v[0]);
#else
  norm_x w;
#pragma unroll
  for (int e = 0; e < NORM_VE; ++e) w.v[e] = v[e];
#endif
  norm_word o;
  memcpy(&o, &w, NORM_BYTES);
  __stcs(reinterpret_cast<norm_word*>(p), o);
}
// NORM_VE parameters (gamma, beta) from j on
__device__ __forceinline__ void norm_params(const param_t* p, f32 (&v)[NORM_VE]) {
  constexpr int PER = (int)(16 / sizeof(param_t)) < NORM_VE ? (int)(16 / sizeof(param_t)) : NORM_VE;
#pragma unroll
  for (int h = 0; h < NORM_VE; h += PER) {
    typedef typename norm_vec<param_t, PER>::type vec;
    const vec b = *reinterpret_cast<const vec*>(p + h);
#pragma unroll
    for (int e = 0; e < PER; ++e) v[h + e] = row_wide(b.v[e]);
  }
}

// NORM_VE of them as Floats from shared memory
__device__ __forceinline__ void norm_gamma(const f32* p, f32 (&v)[NORM_VE]) {
#pragma unroll
  for (int e = 0; e < NORM_VE; e += 4) {
    if (NORM_VE >= 4) {
      const float4 q = *reinterpret_cast<const float4*>(p + e);
      v[e] = q.x;
      v[(e + 1) % NORM_VE] = q.y;
      v[(e + 2) % NORM_VE] = q.z;
      v[(e + 3) % NORM_VE] = q.w;
    } else {
      for (int i = 0; i < NORM_VE; ++i) v[i] = p[i];
    }
  }
}
#if NORM_BYTES >= 4
// One access to shared memory without registers in between
__device__ __forceinline__ void norm_copy(norm_x* to, const row_t* from) {
  const u32 at = (u32)__cvta_generic_to_shared(to);
#if NORM_BYTES == 16
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
#else
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(at), "l"(from), "n"(NORM_BYTES) : "memory");
#endif
}
#endif

// Sums of a group's lanes, the same in every lane.  With several warps per row the warps' sums meet in shared memory;
// `slot` alternates between calls, so that one barrier per call is enough.
template <int N> __device__ __forceinline__ void norm_sum(f32 (&s)[N], f32 (*red)[ROW_THREADS / 32][N], int slot) {
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] = row_warp_sum(s[i]);
#if NORM_WARPS > 1
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) red[slot][warp][i] = s[i];
  __syncthreads();
  const int w0 = warp / NORM_WARPS * NORM_WARPS;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    s[i] = red[slot][w0][i];
#pragma unroll
    for (int w = 1; w < NORM_WARPS; ++w) s[i] += red[slot][w0 + w][i];
  }
#endif
}
