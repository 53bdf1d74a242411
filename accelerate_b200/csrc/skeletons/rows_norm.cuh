// Layer norm along the innermost dimension:
//   mu = sum x / n,  var = sum (x - mu)^2 / n,  r = 1 / sqrt(var + eps),  y = (x - mu) r gamma + beta.
// The row is read once and stays in registers as it came; both sums run over the kept values (the second around the
// mean, so that nothing cancels), in Float.  Bound by HBM: one read and one write of the row; gamma and beta come
// from L1 and L2.  NORM_LONG: rows longer than the registers of a CTA hold; it reads the row three times, which L2 keeps.

struct Params { i64 x, gamma, beta, y, mean, rstd, rows, n, eps; };

extern "C" __global__ void __launch_bounds__(ROW_THREADS) acc_rows_norm(const __grid_constant__ Params p) {
#if NORM_WARPS > 1
  __shared__ f32 red[2][ROW_THREADS / 32][1];
#else
  f32(*red)[ROW_THREADS / 32][1] = nullptr;
#endif
  const int g = threadIdx.x % NORM_GROUP;
  const i64 row = (i64)blockIdx.x * NORM_ROWS + threadIdx.x / NORM_GROUP;
  // (groups behind the last row go through the barriers with an empty row)
  const int n = row < p.rows ? (int)p.n : 0;
  const f32 eps = __uint_as_float((u32)p.eps), len = (f32)p.n;
  const row_t* x = reinterpret_cast<const row_t*>(p.x) + row * p.n;
  row_t* y = reinterpret_cast<row_t*>(p.y) + row * p.n;
  const param_t* gamma = reinterpret_cast<const param_t*>(p.gamma);
  const param_t* beta = reinterpret_cast<const param_t*>(p.beta);
  constexpr int STEP = NORM_GROUP * NORM_VE;

  f32 s[1] = {0.0f};
#if NORM_LONG
  for (int j = g * NORM_VE; j < n; j += STEP) {
    f32 v[NORM_VE];
    norm_wide(norm_load(x + j), v);
#pragma unroll
    for (int e = 0; e < NORM_VE; ++e) s[0] += v[e];
  }
#else
  norm_x b[NORM_U];
#pragma unroll
  for (int u = 0; u < NORM_U; ++u)
    if (u * STEP + g * NORM_VE < n) b[u] = norm_load(x + u * STEP + g * NORM_VE);
#pragma unroll
  for (int u = 0; u < NORM_U; ++u)
    if (u * STEP + g * NORM_VE < n) {
      f32 v[NORM_VE];
      norm_wide(b[u], v);
#pragma unroll
      for (int e = 0; e < NORM_VE; ++e) s[0] += v[e];
    }
#endif
  norm_sum(s, red, 0);
  const f32 mean = s[0] / len;
  s[0] = 0.0f;
#if NORM_LONG
  for (int j = g * NORM_VE; j < n; j += STEP) {
    f32 v[NORM_VE];
    norm_wide(norm_load(x + j), v);
#pragma unroll
    for (int e = 0; e < NORM_VE; ++e) s[0] = fmaf(v[e] - mean, v[e] - mean, s[0]);
  }
#else
#pragma unroll
  for (int u = 0; u < NORM_U; ++u)
    if (u * STEP + g * NORM_VE < n) {
      f32 v[NORM_VE];
      norm_wide(b[u], v);
#pragma unroll
      for (int e = 0; e < NORM_VE; ++e) s[0] = fmaf(v[e] - mean, v[e] - mean, s[0]);
    }
#endif
  norm_sum(s, red, 1);
  const f32 rstd = 1.0f / sqrtf(s[0] / len + eps);
  if (g == 0 && row < p.rows) {
    reinterpret_cast<f32*>(p.mean)[row] = mean;
    reinterpret_cast<f32*>(p.rstd)[row] = rstd;
  }
#if NORM_LONG
  for (int j = g * NORM_VE; j < n; j += STEP) {
    const norm_x bu = norm_load(x + j);
#else
#pragma unroll
  for (int u = 0; u < NORM_U; ++u) {
    const int j = u * STEP + g * NORM_VE;
    if (j >= n) continue;
    const norm_x bu = b[u];
#endif
    f32 v[NORM_VE], ga[NORM_VE], be[NORM_VE];
    norm_wide(bu, v);
    norm_params(gamma + j, ga);
    norm_params(beta + j, be);
#pragma unroll
    for (int e = 0; e < NORM_VE; ++e) v[e] = fmaf((v[e] - mean) * rstd, ga[e], be[e]);
    norm_store(y + j, v);
  }
}
