// Gradient of the distillation loss (rows_stats.cuh) with respect to the student's logits:
//   ds_j = g tau (p_j - sum of q_k over the entries k with id_k = j),   p_j = e^(s_j/tau - lse),
// 0 for a row without teacher entries.  One read and one write of the row; the normaliser comes from the forward
// pass.  It is one Float: half a step of it, 2^-24 of its size, is a relative error of every p_j (2^-11 at 2^14).  From
// there on every CTA reads its row twice more, for the maximum m and Z = sum e^((s - m)/tau), and takes
// p_j = e^((s_j - m)/tau) / Z, if these give the normaliser it got, up to three of its steps.  ROW_C CTAs share a row,
// each with a stretch of its blocks; once a CTA has written its stretch it rewrites the elements in it that have
// teacher entries (an id that occurs twice is written once, with the sum).

struct Params { i64 x, ids, teacher, lse, g, out, rows, n, k, tau, err; };

constexpr int DG_TILE = ROW_THREADS * ROW_U;
constexpr int DG_WARPS = ROW_THREADS / 32;

extern "C" __global__ void __launch_bounds__(ROW_THREADS, ROW_MIN_BLOCKS) acc_rows_distill_grad(const __grid_constant__ Params p) {
  __shared__ f32 red[2][DG_WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const i64 row = blockIdx.x / ROW_C;
  const int part = (int)(blockIdx.x % ROW_C);
  const int n = (int)p.n, k = (int)p.k;
  const row_span span(reinterpret_cast<const row_t*>(p.x) + row * p.n, n);
  row_t* const out = reinterpret_cast<row_t*>(p.out) + row * p.n;
  // (blocks of input and output are aligned alike when the two arrays are)
  const bool vec = (((u64)out ^ (u64)span.x) & 15) == 0;
  const int per = (span.blocks + ROW_C - 1) / ROW_C;
  const int b0 = min(part * per, span.blocks), b1 = min(b0 + per, span.blocks);
  const f32 tau = __uint_as_float((u32)p.tau);
  const f32 c = ROW_LOG2E / tau;
  const i32* ids = reinterpret_cast<const i32*>(p.ids) + row * p.k;
  const teacher_t* ts = reinterpret_cast<const teacher_t*>(p.teacher) + row * p.k;

  uint4 nxt[ROW_U];
#pragma unroll
  for (int u = 0; u < ROW_U; ++u) {
    const int i = b0 + u * ROW_THREADS + tid;
    if (i < b1) nxt[u] = span.load(i);
  }
  const f32 lse = reinterpret_cast<const f32*>(p.lse)[row];
  f32 scale = reinterpret_cast<const f32*>(p.g)[row] * tau;
  // the teacher's distribution: maximum and sum over the entries that are there
  f32 mt = -ROW_INF;
  bool bad = false;
  for (int i = tid; i < k; i += ROW_THREADS) {
    const int id = ids[i];
    bad = bad || id >= n;
    if (id >= 0 && id < n) mt = row_max_nan(mt, row_wide(ts[i]));
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) mt = row_max_nan(mt, __shfl_xor_sync(ACC_FULL_MASK, mt, d));
  if (lane == 0) red[0][warp] = mt;
  bad = __syncthreads_or(bad) != 0;
  mt = red[0][0];
#pragma unroll
  for (int w = 1; w < DG_WARPS; ++w) mt = row_max_nan(mt, red[0][w]);
  f32 es = 0.0f;
  if (mt != -ROW_INF)
    for (int i = tid; i < k; i += ROW_THREADS) {
      const int id = ids[i];
      if (id >= 0 && id < n) es += row_ex2((row_wide(ts[i]) - mt) * c);
    }
  es = row_warp_sum(es);
  if (lane == 0) red[1][warp] = es;
  __syncthreads();
  es = 0.0f;
#pragma unroll
  for (int w = 0; w < DG_WARPS; ++w) es += red[1][w];
  const bool has = es != 0.0f;
  if (es != es) scale = es;              // a NaN among the teacher's logits: no gradient is a number
  if (bad && tid == 0 && part == 0) acc_fail(p.err, 1003);

  // p_j g tau = 2^(c (s - tau lse)) g tau: the product tau lse is not rounded before the subtraction, so the exponent
  // is right to half a step for the lse that was given.  A row without an element above -inf comes with lse = -inf:
  // the type's lowest value in its place lets its -inf elements yield 0.
  f32 from = lse == -ROW_INF ? -3.402823466e38f : lse, by = tau, p_scale = scale;
  if (has && fabsf(lse) >= 16384.0f) {
    f32 m = -ROW_INF, z = 0.0f;
    for (int i = tid; i < span.blocks; i += ROW_THREADS) {
      f32 v[ROW_E];
      row_unpack(span.load(i), v);
#pragma unroll
      for (int e = 0; e < ROW_E; ++e) m = fmaxf(m, v[e]);
    }
    m = row_warp_max(m);
    if (lane == 0) red[0][warp] = m;     // (everybody has read what was there: a barrier lies between)
    __syncthreads();
#pragma unroll
    for (int w = 0; w < DG_WARPS; ++w) m = fmaxf(m, red[0][w]);
    if (m != -ROW_INF)
      for (int i = tid; i < span.blocks; i += ROW_THREADS) {
        f32 v[ROW_E], sum = 0.0f;
        row_unpack(span.load(i), v);
#pragma unroll
        for (int e = 0; e < ROW_E; ++e) sum += row_ex2((v[e] - m) * c);
        z += sum;
      }
    z = row_warp_sum(z);
    if (lane == 0) red[1][warp] = z;
    __syncthreads();
    z = 0.0f;
#pragma unroll
    for (int w = 0; w < DG_WARPS; ++w) z += red[1][w];
    const f32 own = m / tau + logf(z);
    if (z > 0.0f && (own == lse || fabsf(own - lse) <= fabsf(lse) * (3.0f / 8388608.0f))) {
      from = m;
      by = 1.0f;
      p_scale = scale / z;
    }
  }
#define DG_P(s) (row_ex2(fmaf(-from, by, s) * c) * p_scale)
  for (int t = b0; t < b1; t += DG_TILE) {
    uint4 cur[ROW_U];
#pragma unroll
    for (int u = 0; u < ROW_U; ++u) cur[u] = nxt[u];
    if (t + DG_TILE < b1) {
#pragma unroll
      for (int u = 0; u < ROW_U; ++u) {
        const int i = t + DG_TILE + u * ROW_THREADS + tid;
        if (i < b1) nxt[u] = span.load(i);
      }
    }
#pragma unroll
    for (int u = 0; u < ROW_U; ++u) {
      const int i = t + u * ROW_THREADS + tid;
      if (i >= b1) continue;
      f32 v[ROW_E];
      row_unpack(cur[u], v);
#pragma unroll
      for (int e = 0; e < ROW_E; ++e) v[e] = has ? DG_P(v[e]) : 0.0f;
      const int j = span.first(i);
      if (vec && j >= 0 && j + ROW_E <= n) {
        *reinterpret_cast<uint4*>(out + j) = row_pack(v);   // (a streaming store: 4 % more time for the largest case, 348 us with this one)
      } else {
#pragma unroll
        for (int e = 0; e < ROW_E; ++e)
          if (j + e >= 0 && j + e < n) row_narrow(v[e], out[j + e]);
      }
    }
  }
  if (!has) return;
  __syncthreads();                       // this CTA's stretch is written
  const int j0 = max(span.first(b0), 0), j1 = min(span.first(b1), n);
  for (int i = tid; i < k; i += ROW_THREADS) {
    const int id = ids[i];
    if (id < j0 || id >= j1) continue;
    f32 q = 0.0f;
    bool first = true;
    for (int o = 0; o < k; ++o)
      if (ids[o] == id) {
        if (o < i) first = false;
        q += row_ex2((row_wide(ts[o]) - mt) * c);
      }
    if (first) row_narrow(DG_P(row_wide(span.x[id])) - scale * (q / es), out[id]);
  }
}
