// What the layer norm kernels share: a row spread over NORM_WARPS warps (NORM_GROUP lanes), NORM_U accesses of
// NORM_VE elements per lane.  Lane g holds the elements [(u * NORM_GROUP + g) * NORM_VE, + NORM_VE).
//
//   NORM_VE     elements per access: 16 bytes' worth if every row and both parameter vectors start on 16-byte
//               boundaries, else 1; neighbouring lanes then hold neighbouring elements, so the narrow accesses of a
//               warp still cover whole sectors
//   NORM_WARPS  warps per row, a power of two; NORM_ROWS rows per CTA at a time
//   NORM_U      accesses per lane;  NORM_GROUP * NORM_U * NORM_VE >= n

#define NORM_GROUP (NORM_WARPS * 32)
#define NORM_ROWS (ROW_THREADS / NORM_GROUP)

template <int N> struct __align__(2 * N) norm_bits16 { u16 v[N]; };
template <int N> struct __align__(4 * N) norm_bits32 { f32 v[N]; };
template <class T, int N> struct norm_vec;
template <int N> struct norm_vec<u16, N> { typedef norm_bits16<N> type; };
template <int N> struct norm_vec<f32, N> { typedef norm_bits32<N> type; };
typedef norm_vec<row_t, NORM_VE>::type norm_x;

// One access of x or dy: read once, so it takes no place in L1 (gamma and beta live there).
__device__ __forceinline__ norm_x norm_load(const row_t* p) {
  norm_x r;
#if NORM_VE > 1
  uint4 b;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w) : "l"(p));
  memcpy(&r, &b, 16);
#else
  r.v[0] = __ldcs(p);
#endif
  return r;
}
__device__ __forceinline__ void norm_wide(const norm_x& b, f32 (&v)[NORM_VE]) {
#if ROW_F16 && NORM_VE > 1
  uint4 w;
  memcpy(&w, &b, 16);
  row_unpack(w, v);
#else
#pragma unroll
  for (int e = 0; e < NORM_VE; ++e) v[e] = row_wide(b.v[e]);
#endif
}
__device__ __forceinline__ void norm_store(row_t* p, const f32 (&v)[NORM_VE]) {
#if NORM_VE > 1
  __stcs(reinterpret_cast<uint4*>(p), row_pack(v));
#else
  row_t o;
  row_narrow(v[0], o);
  __stcs(p, o);
#endif
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

#if NORM_VE > 1
// NORM_VE of them as Floats from shared memory
__device__ __forceinline__ void norm_gamma(const f32* p, f32 (&v)[NORM_VE]) {
#pragma unroll
  for (int h = 0; h < NORM_VE; h += 4) {
    const float4 q = *reinterpret_cast<const float4*>(p + h);
    v[h] = q.x;
    v[h + 1] = q.y;
    v[h + 2] = q.z;
    v[h + 3] = q.w;
  }
}
// 16 bytes to shared memory without registers in between
__device__ __forceinline__ void norm_copy(uint4* to, const row_t* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((u32)__cvta_generic_to_shared(to)), "l"(from) : "memory");
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
