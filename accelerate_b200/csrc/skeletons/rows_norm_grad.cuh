// Gradients of layer norm (rows_norm.cuh).  With xh = (x - mu) r and a = dy gamma:
//   dx = r (a - mean a - xh mean(a xh)),   dgamma = sum over rows of dy xh,   dbeta = sum over rows of dy.
// Bound by HBM: x and dy are read once, dx is written once.  A CTA walks over rows NORM_ROWS at a time; a lane holds
// the same columns of every row, so that the sums over rows stay in its registers.  At the end the CTA's sums go to
// `partial` (one line of 2 n Floats per CTA) and acc_rows_norm_sums adds the lines in their order: the same
// numbers every time, whatever order the CTAs ran in.
//
//   NORM_STAGES  rows of x and dy on their way while one is worked on: every lane copies its own elements to shared
//                memory (cp.async) and reads them back itself, so the ring needs no barrier and no flag.  0: rows of
//                Halves that start on odd elements (no such copy of 2 bytes exists) are loaded directly.
//   NORM_KEEP    1: xh and a stay in registers between the two passes (up to 16 elements per lane); 0: the row is
//                read from the ring twice (32 elements per lane, whose sums alone take 64 registers)
//   NORM_LONG    rows longer than that: dx alone (x and dy read twice), the sums over rows by acc_rows_norm_cols

struct Params { i64 x, gamma, mean, rstd, dy, dx, partial, dgamma, dbeta, rows, n, lines, chunk; };

extern __shared__ uint4 norm_memory[];

#if NORM_SUMS
// Lines of partial sums -> dgamma, dbeta.  32 columns per CTA, the warps take lines in turn.
extern "C" __global__ void __launch_bounds__(ROW_THREADS) acc_rows_norm_sums(const __grid_constant__ Params p) {
  __shared__ f32 part[2][ROW_THREADS / 32][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int W = ROW_THREADS / 32;
  const i64 j = (i64)blockIdx.x * 32 + lane;
  f32 sg = 0.0f, sb = 0.0f;
  if (j < p.n) {
    const f32* q = reinterpret_cast<const f32*>(p.partial) + j;
#pragma unroll 4
    for (i64 l = warp; l < p.lines; l += W) {
      sg += q[l * 2 * p.n];
      sb += q[l * 2 * p.n + p.n];
    }
  }
  part[0][warp][lane] = sg;
  part[1][warp][lane] = sb;
  __syncthreads();
  if (warp < 2 && j < p.n) {
    f32 s = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) s += part[warp][w][lane];
    row_narrow(s, reinterpret_cast<param_t*>(warp == 0 ? p.dgamma : p.dbeta)[j]);
  }
}
#elif NORM_COLS
// Sums over `chunk` rows of 32 columns per CTA (rows too long for acc_rows_norm_grad's registers).
extern "C" __global__ void __launch_bounds__(ROW_THREADS) acc_rows_norm_cols(const __grid_constant__ Params p) {
  __shared__ f32 part[2][ROW_THREADS / 32][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int W = ROW_THREADS / 32;
  const i64 cols = (p.n + 31) / 32;
  const i64 j = (blockIdx.x % cols) * 32 + lane, line = blockIdx.x / cols;
  const i64 r1 = (line + 1) * p.chunk < p.rows ? (line + 1) * p.chunk : p.rows;
  f32 sg = 0.0f, sb = 0.0f;
  if (j < p.n)
#pragma unroll 4
    for (i64 r = line * p.chunk + warp; r < r1; r += W) {
      const f32 d = row_wide(reinterpret_cast<const row_t*>(p.dy)[r * p.n + j]);
      const f32 xh = (row_wide(reinterpret_cast<const row_t*>(p.x)[r * p.n + j]) - reinterpret_cast<const f32*>(p.mean)[r]) *
                     reinterpret_cast<const f32*>(p.rstd)[r];
      sg = fmaf(d, xh, sg);
      sb += d;
    }
  part[0][warp][lane] = sg;
  part[1][warp][lane] = sb;
  __syncthreads();
  if (warp < 2 && j < p.n) {
    f32 s = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) s += part[warp][w][lane];
    reinterpret_cast<f32*>(p.partial)[line * 2 * p.n + warp * p.n + j] = s;
  }
}
#else
extern "C" __global__ void __launch_bounds__(ROW_THREADS, ROW_THREADS > 256 ? 1 : 2) acc_rows_norm_grad(const __grid_constant__ Params p) {
#if NORM_WARPS > 1
  __shared__ f32 red[2][ROW_THREADS / 32][2];
#else
  f32(*red)[ROW_THREADS / 32][2] = nullptr;
#endif
  const int g = threadIdx.x % NORM_GROUP, sub = threadIdx.x / NORM_GROUP;
  const int n = (int)p.n;
  const f32 len = (f32)p.n;
  constexpr int STEP = NORM_GROUP * NORM_VE;
  const param_t* gamma = reinterpret_cast<const param_t*>(p.gamma);
#if NORM_LONG
  for (i64 row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const row_t* x = reinterpret_cast<const row_t*>(p.x) + row * p.n;
    const row_t* dy = reinterpret_cast<const row_t*>(p.dy) + row * p.n;
    row_t* dx = reinterpret_cast<row_t*>(p.dx) + row * p.n;
    const f32 mean = reinterpret_cast<const f32*>(p.mean)[row], rstd = reinterpret_cast<const f32*>(p.rstd)[row];
    f32 s[2] = {0.0f, 0.0f};
    for (int j = g * NORM_VE; j < n; j += STEP) {
      f32 v[NORM_VE], d[NORM_VE], ga[NORM_VE];
      norm_wide(norm_load(x + j), v);
      norm_wide(norm_load(dy + j), d);
      norm_params(gamma + j, ga);
#pragma unroll
      for (int e = 0; e < NORM_VE; ++e) {
        const f32 a = d[e] * ga[e];
        s[0] += a;
        s[1] = fmaf(a, (v[e] - mean) * rstd, s[1]);
      }
    }
    norm_sum(s, red, 0);
    const f32 ma = s[0] / len, mb = s[1] / len;
    for (int j = g * NORM_VE; j < n; j += STEP) {
      f32 v[NORM_VE], d[NORM_VE], ga[NORM_VE];
      norm_wide(norm_load(x + j), v);
      norm_wide(norm_load(dy + j), d);
      norm_params(gamma + j, ga);
#pragma unroll
      for (int e = 0; e < NORM_VE; ++e) v[e] = rstd * (fmaf(-((v[e] - mean) * rstd), mb, fmaf(d[e], ga[e], -ma)));
      norm_store(dx + j, v);
    }
    __syncthreads();                     // the next row writes the same slot
  }
#else
  f32 sg[NORM_U * NORM_VE], sb[NORM_U * NORM_VE];
#pragma unroll
  for (int i = 0; i < NORM_U * NORM_VE; ++i) sg[i] = sb[i] = 0.0f;
  i64 row = (i64)blockIdx.x * NORM_ROWS + sub;
  const i64 stride = (i64)gridDim.x * NORM_ROWS;
#if NORM_STAGES
  // the ring: [stage][x, dy][access][thread], behind it gamma
  norm_x* const mine = reinterpret_cast<norm_x*>(norm_memory) + threadIdx.x;
  constexpr int PLANE = NORM_U * ROW_THREADS;
  auto fetch = [&](i64 r, int stage) {
    if (r < p.rows) {
      const row_t* x = reinterpret_cast<const row_t*>(p.x) + r * p.n;
      const row_t* dy = reinterpret_cast<const row_t*>(p.dy) + r * p.n;
#pragma unroll
      for (int u = 0; u < NORM_U; ++u) {
        const int j = u * STEP + g * NORM_VE;
        if (j < n) {
          norm_copy(mine + (2 * stage) * PLANE + u * ROW_THREADS, x + j);
          norm_copy(mine + (2 * stage + 1) * PLANE + u * ROW_THREADS, dy + j);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < NORM_STAGES - 1; ++s) fetch(row + s * stride, s);
  int stage = 0;
#endif
#if NORM_STAGES
  f32* const gs = reinterpret_cast<f32*>(reinterpret_cast<norm_x*>(norm_memory) + 2 * NORM_STAGES * PLANE);
  for (int j = threadIdx.x; j < n; j += ROW_THREADS) gs[j] = row_wide(gamma[j]);
  __syncthreads();
#endif
  f32 mean = 0.0f, rstd = 0.0f, mean_next = 0.0f, rstd_next = 0.0f;
  if (row < p.rows) {
    mean_next = reinterpret_cast<const f32*>(p.mean)[row];
    rstd_next = reinterpret_cast<const f32*>(p.rstd)[row];
  }
  int slot = 0;
  // (a CTA's groups make the same number of trips: they share the barriers)
  for (i64 first = (i64)blockIdx.x * NORM_ROWS; first < p.rows; first += stride, row += stride) {
    const bool there = row < p.rows;
    mean = mean_next;
    rstd = rstd_next;
    if (row + stride < p.rows) {
      mean_next = reinterpret_cast<const f32*>(p.mean)[row + stride];
      rstd_next = reinterpret_cast<const f32*>(p.rstd)[row + stride];
    }
#if NORM_STAGES
    // (the stage fetched into now was read in the trip before, by this thread)
    fetch(row + (NORM_STAGES - 1) * stride, (stage + NORM_STAGES - 1) % NORM_STAGES);
    asm volatile("cp.async.wait_group %0;" ::"n"(NORM_STAGES - 1) : "memory");
    const norm_x* const bx = mine + (2 * stage) * PLANE;
    const norm_x* const bd = mine + (2 * stage + 1) * PLANE;
    stage = (stage + 1) % NORM_STAGES;
#endif
#if NORM_STAGES
#define NORM_TAKE(u)                                 \
  norm_wide(norm_shared(bx + (u) * ROW_THREADS), v); \
  norm_wide(norm_shared(bd + (u) * ROW_THREADS), d); \
  norm_gamma(gs + j, ga);
#else
    norm_x kx[NORM_U], kd[NORM_U];
#pragma unroll
    for (int u = 0; u < NORM_U; ++u) {
      const int j = u * STEP + g * NORM_VE;
      if (there && j < n) {
        kx[u] = norm_load(reinterpret_cast<const row_t*>(p.x) + row * p.n + j);
        kd[u] = norm_load(reinterpret_cast<const row_t*>(p.dy) + row * p.n + j);
      }
    }
#define NORM_TAKE(u)   \
  norm_wide(kx[u], v); \
  norm_wide(kd[u], d); \
  norm_params(gamma + j, ga);
#endif
#if NORM_KEEP
    f32 xh_kept[NORM_U][NORM_VE], a_kept[NORM_U][NORM_VE];
#endif
    f32 s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < NORM_U; ++u) {
      const int j = u * STEP + g * NORM_VE;
      if (there && j < n) {
        f32 v[NORM_VE], d[NORM_VE], ga[NORM_VE];
        NORM_TAKE(u)
#pragma unroll
        for (int e = 0; e < NORM_VE; ++e) {
          const f32 xh = (v[e] - mean) * rstd, a = d[e] * ga[e];
          s[0] += a;
          s[1] = fmaf(a, xh, s[1]);
          sg[u * NORM_VE + e] = fmaf(d[e], xh, sg[u * NORM_VE + e]);
          sb[u * NORM_VE + e] += d[e];
#if NORM_KEEP
          xh_kept[u][e] = xh;
          a_kept[u][e] = a;
#endif
        }
      }
    }
    norm_sum(s, red, slot);
    slot ^= 1;
    const f32 ma = s[0] / len, mb = s[1] / len;
    row_t* dx = reinterpret_cast<row_t*>(p.dx) + row * p.n;
#pragma unroll
    for (int u = 0; u < NORM_U; ++u) {
      const int j = u * STEP + g * NORM_VE;
      if (there && j < n) {
        f32 v[NORM_VE];
#if NORM_KEEP
#pragma unroll
        for (int e = 0; e < NORM_VE; ++e) v[e] = rstd * fmaf(-xh_kept[u][e], mb, a_kept[u][e] - ma);
#else
        f32 d[NORM_VE], ga[NORM_VE];
        NORM_TAKE(u)
#pragma unroll
        for (int e = 0; e < NORM_VE; ++e) v[e] = rstd * fmaf(-((v[e] - mean) * rstd), mb, d[e] * ga[e] - ma);
#endif
        norm_store(dx + j, v);
      }
    }
  }
  // this CTA's line: the groups' sums one after the other
  f32* line = reinterpret_cast<f32*>(p.partial) + (i64)blockIdx.x * 2 * p.n;
#if NORM_ROWS > 1
  f32* const sums = reinterpret_cast<f32*>(norm_memory);   // 2 n Floats, where the ring was
#if NORM_STAGES
  asm volatile("cp.async.wait_all;" ::: "memory");
#endif
  __syncthreads();
#pragma unroll 1
  for (int q = 0; q < NORM_ROWS; ++q) {
    if (q == sub) {
#pragma unroll
      for (int u = 0; u < NORM_U; ++u)
#pragma unroll
        for (int e = 0; e < NORM_VE; ++e) {
          const int j = u * STEP + g * NORM_VE + e;
          if (j < n) {
            sums[j] = q == 0 ? sg[u * NORM_VE + e] : sums[j] + sg[u * NORM_VE + e];
            sums[n + j] = q == 0 ? sb[u * NORM_VE + e] : sums[n + j] + sb[u * NORM_VE + e];
          }
        }
    }
    __syncthreads();
  }
  for (int j = threadIdx.x; j < 2 * n; j += ROW_THREADS) line[j] = sums[j];
#else
#pragma unroll
  for (int u = 0; u < NORM_U; ++u)
#pragma unroll
    for (int e = 0; e < NORM_VE; ++e) {
      const int j = u * STEP + g * NORM_VE + e;
      if (j < n) {
        line[j] = sg[u * NORM_VE + e];
        line[n + j] = sb[u * NORM_VE + e];
      }
    }
#endif
#endif
}
#endif
