// Statistics of a row of logits in one pass over it: the normaliser ln sum e^(x/tau), and behind it either
//   log probabilities (ROW_DISTILL 0): the given token's log probability, the entropy, and the ROW_TOPK
//     k largest logits with their indices; or
//   a distillation loss (ROW_DISTILL 1): tau^2 sum q (ln q - ln p) against a teacher's few entries.
//
// Mathematics.  With c = log2(e)/tau and m the running maximum, every thread keeps Z = sum 2^t and
// W = sum 2^t t over its elements, t = c (x - m), and moves both to a new maximum m' by Z' = s Z,
// W' = s (W + d Z), d = c (m - m'), s = 2^d.  Threads, warps and CTAs join by the same rule.  Then
//   lse = m/tau + ln Z,     entropy = ln Z - ln 2 W / Z,     ln p_j = (x_j - m)/tau - ln Z.
// (not x_j/tau - lse: one Float holds lse to half a step of its own size, which for a row around 1e6 is 0.03, and a row
// of nothing but the type's lowest value would come out with a probability of 1 for each of its elements)
// Half: t = c x - M with M = c m rounded, one instruction; what the rounding shifts is known exactly and comes
// off the end (M - c m).  Float: the subtraction first, since c m can leave the range (rows masked with the
// type's lowest value); a Float element has twice the bytes to pay for the second instruction.
// Sums are Float; products with 2^t = 0 are 0, so masked (-inf) elements count for nothing.
//
// A cluster of ROW_C CTAs shares a row (ROW_C > 1 when there are few rows) and joins through distributed
// shared memory: no scratch in global memory, nothing that two launches could share.

//   x, tok or ids: arrays; the outputs; n = row length; k = alternatives, or teacher entries per row
struct Params { i64 x, tok, teacher, out0, out1, out2, out3, out4, rows, n, k, tau, err; };

constexpr int ST_TILE = ROW_THREADS * ROW_U;     // blocks per tile
constexpr int ST_WARPS = ROW_THREADS / 32;
constexpr int ST_CAP = 1024;                     // candidate keys held in shared memory
constexpr int ST_BATCH = ST_CAP / 2;             // elements looked at between two looks at the list
constexpr int ST_HOT = 512;                      // listed blocks

struct row_stat { f32 m, z, w; };
struct st_shared {
#if ROW_TOPK
  __align__(16) u64 cand[ST_CAP];
  uint4 hot[ST_HOT];        // blocks that may hold candidates,
  int hot_block[ST_HOT];    // and their numbers
  int hot_count[2];         // of this list and the next
  int count;                // candidates, while they are being appended
  int kept;                 // candidates of this CTA at the end (read by the cluster's first CTA)
  u64 key[ST_WARPS];
#endif
  row_stat part[ST_WARPS];
  row_stat cta;
  int warp_count[ST_WARPS];
};

extern __shared__ uint4 st_memory[];
static_assert(sizeof(st_shared) <= ROW_SMEM, "the host asks for less shared memory than the kernel uses");
#define sh (*reinterpret_cast<st_shared*>(st_memory))

// (a maximum of -inf, "nothing yet", stands at 0: its sums are 0)
__device__ __forceinline__ f32 st_base(f32 m) { return m == -ROW_INF ? 0.0f : m; }
__device__ __forceinline__ f32 st_shift(f32 from, f32 to, f32 c) {
  if (from == -ROW_INF) return 0.0f;
#if ROW_F16
  return from * c - to * c;            // both rounded, as the elements saw them (--fmad=false)
#else
  return (from - to) * c;
#endif
}
__device__ __forceinline__ row_stat st_join(const row_stat& a, const row_stat& b, f32 c) {
  row_stat r;
  r.m = fmaxf(a.m, b.m);
  const f32 da = st_shift(a.m, r.m, c), db = st_shift(b.m, r.m, c);
  const f32 sa = row_ex2(da), sb = row_ex2(db);
  r.z = sa * a.z + sb * b.z;
  // (d z is 0 times infinity when the other maximum is out of reach: that part is then 0)
  r.w = (sa == 0.0f ? 0.0f : sa * fmaf(da, a.z, a.w)) + (sb == 0.0f ? 0.0f : sb * fmaf(db, b.z, b.w));
  return r;
}

// Order of the alternatives in one whole number: the value (NaN above +inf, -0 equal to 0) in the upper 32 bits,
// the complement of the index below it.  Larger is better, no two elements of a row are equal.
__device__ __forceinline__ u32 st_order(f32 v) {
  if (v != v) return 0xffffffffu;
  const u32 u = __float_as_uint(v + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ f32 st_value(u32 o) {
  if (o == 0xffffffffu) return ROW_NAN;
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ u64 st_key(f32 v, int j) { return ((u64)st_order(v) << 32) | (u32)~j; }
__device__ __forceinline__ int st_index(u64 key) { return (int)~(u32)key; }
#if ROW_F16
__device__ __forceinline__ f32 st_block_max(u32 m) { f32 lo, hi; row_h2x2(m, lo, hi); return row_max_nan(lo, hi); }
#else
__device__ __forceinline__ f32 st_block_max(f32 m) { return m; }
#endif
#define ST_NONE ((u64)0x007fffffffffffffull)     /* the best key of a -inf element: candidates lie above it */

#if ROW_TOPK
// Every candidate to its place in falling order, as long as that is one of the first k; `sorted` of the n candidates are
// in order already, at the front.  A thread counts, for Q candidates, those among the unsorted ones that are better;
// among the sorted ones a search finds the place.
template <int Q> __device__ __forceinline__ void st_rank(int sorted, int n, int k) {
  const int tid = threadIdx.x;
  u64 key[Q];
  int rank[Q];
  if (sorted <= 32) sorted = 0;          // (counting through them is no slower than the search)
  if ((tid & ~31) < n) {
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int i = q * ROW_THREADS + tid;
      key[q] = i < n ? sh.cand[i] : 0;
      rank[q] = i < sorted ? i : 0;
      if (i >= sorted) {
        int lo = 0, hi = sorted;         // better ones: [0, lo), worse ones: [hi, sorted)
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          if (sh.cand[mid] > key[q]) lo = mid + 1; else hi = mid;
        }
        rank[q] = lo;
      }
    }
    int i = sorted;
    if ((i & 1) && i < n) {
#pragma unroll
      for (int q = 0; q < Q; ++q) rank[q] += sh.cand[i] > key[q];
      ++i;
    }
#pragma unroll 4
    for (; i + 1 < n; i += 2) {
      const ulonglong2 c = *reinterpret_cast<const ulonglong2*>(&sh.cand[i]);
#pragma unroll
      for (int q = 0; q < Q; ++q) rank[q] += (c.x > key[q]) + (c.y > key[q]);
    }
    if (i < n)
#pragma unroll
      for (int q = 0; q < Q; ++q) rank[q] += sh.cand[i] > key[q];
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < Q; ++q)
    if (q * ROW_THREADS + tid < n && rank[q] < k) sh.cand[rank[q]] = key[q];
  if (tid == 0) sh.count = n < k ? n : k;
  __syncthreads();
}
// The same for so few candidates that 2^SPLIT threads can share the counting for each: what a drain waits for is the
// length of that loop.
template <int SPLIT> __device__ __forceinline__ void st_rank_few(int n, int k) {
  const int tid = threadIdx.x, i = tid >> SPLIT;
  const u64 key = i < n ? sh.cand[i] : 0;
  int rank = 0;
#pragma unroll 4
  for (int j = tid & ((1 << SPLIT) - 1); j < n; j += 1 << SPLIT) rank += sh.cand[j] > key;
#pragma unroll
  for (int d = 1; d < (1 << SPLIT); d <<= 1) rank += __shfl_xor_sync(ACC_FULL_MASK, rank, d);
  __syncthreads();
  if (i < n && (tid & ((1 << SPLIT) - 1)) == 0 && rank < k) sh.cand[rank] = key;
  if (tid == 0) sh.count = n < k ? n : k;
  __syncthreads();
}
// The best k of the n candidates, in falling order, to the front of the list, and their number.  Long lists
// (rows in an unusual order): a bitonic sort.
__device__ __forceinline__ int st_compact(int sorted, int n, int k) {
  const int tid = threadIdx.x;
  if (n <= ROW_THREADS / 4) {
    st_rank_few<2>(n, k);
  } else if (n <= ROW_THREADS / 2) {
    st_rank_few<1>(n, k);
  } else if (n <= ROW_THREADS) {
    st_rank<1>(sorted, n, k);
  } else if (n <= 2 * ROW_THREADS) {
    st_rank<2>(sorted, n, k);
  } else {
    for (int i = n + tid; i < ST_CAP; i += ROW_THREADS) sh.cand[i] = 0;
    __syncthreads();
    for (int len = 2; len <= ST_CAP; len <<= 1)
      for (int d = len >> 1; d > 0; d >>= 1) {
        for (int i = tid; i < ST_CAP / 2; i += ROW_THREADS) {
          const int lo = 2 * i - (i & (d - 1)), hi = lo + d;
          const u64 a = sh.cand[lo], b = sh.cand[hi];
          const bool falling = (lo & len) == 0;
          if (falling ? a < b : a > b) { sh.cand[lo] = b; sh.cand[hi] = a; }
        }
        __syncthreads();
      }
    if (tid == 0) sh.count = n < k ? n : k;
    __syncthreads();
  }
  return n < k ? n : k;
}

// The candidate list of a CTA, the same in every thread
struct st_list {
  int held = 0;                  // candidates
  int sorted = 0;                // so many of them, at the front, are in order
  bool overflow = false;
  int phase = 0;                 // which count the blocks listed now go to
  u64 thr_key = ST_NONE;         // only elements above this key are candidates
  f32 thr = -ROW_INF;            // its value: a quick test for all elements of a thread
#if ROW_F16
  u32 thr2 = ROW_PAD;            // the same as two Halves (every threshold is an element, so this is exact)
#endif
};
// Whether a block's maximum is above the threshold's value, or NaN
#if ROW_F16
__device__ __forceinline__ bool st_above(u32 most, const st_list& l) { return row_max_nan2(most, l.thr2) != l.thr2; }
#else
__device__ __forceinline__ bool st_above(f32 most, const st_list& l) { return !(most <= l.thr); }
#endif
// A block that may hold a candidate goes to the list of blocks.  Its best possible key: the block's maximum at the
// block's first element.
__device__ __forceinline__ void st_push(const st_list& l, const uint4& block, f32 most, int i, int first) {
  if (st_key(most, max(first, 0)) > l.thr_key) {
    const int slot = atomicAdd(&sh.hot_count[l.phase], 1);
    if (slot < ST_HOT) {
      sh.hot[slot] = block;
      sh.hot_block[slot] = i;
    }
  }
}
// The threads share the listed blocks' elements; those above the threshold become candidates, and the best k of them
// the new list.  `overflow`, and nothing done, if more blocks came than the list holds.
__device__ __forceinline__ st_list st_drain(st_list l, int shift, int k) {
  const int tid = threadIdx.x;
  __syncthreads();
  // (the other count is 0: it was cleared a drain ago, with barriers since)
  const int blocks = sh.hot_count[l.phase];
  l.phase ^= 1;
  l.overflow = blocks > ST_HOT;
  if (blocks == 0) return l;
  if (l.overflow) {
    __syncthreads();
    if (tid == 0) sh.hot_count[l.phase ^ 1] = 0;
    return l;
  }
  const int n = blocks * ROW_E;
  for (int base = 0; base < n; base += ST_BATCH) {
    const int end = min(base + ST_BATCH, n);
    for (int i = base + tid; i < end; i += ROW_THREADS) {
      const int slot = i / ROW_E, e = i % ROW_E;
      const f32 v = row_wide(reinterpret_cast<const row_t*>(&sh.hot[slot])[e]);
      const u64 key = st_key(v, sh.hot_block[slot] * ROW_E - shift + e);
      if (key > l.thr_key) sh.cand[atomicAdd(&sh.count, 1)] = key;
    }
    __syncthreads();
    l.held = sh.count;
    if (base + ST_BATCH < n) {
      if (l.held > ST_CAP - ST_BATCH) l.held = l.sorted = st_compact(l.sorted, l.held, k);
      else __syncthreads();              // (everybody has read the count)
    } else {
      if (tid == 0) sh.hot_count[l.phase ^ 1] = 0;
      l.held = l.sorted = st_compact(l.sorted, l.held, k);
    }
    if (l.sorted == k && l.held == k) {
      l.thr_key = sh.cand[k - 1];
      const f32 v = st_value((u32)(l.thr_key >> 32));
      l.thr = v != v ? ROW_INF : v;
#if ROW_F16
      l.thr2 = row_x2h2(l.thr, l.thr);
#endif
    }
  }
  return l;
}
#endif

__device__ __forceinline__ u32 st_cluster_addr(const void* p, int rank) {
  u32 a, r;
  asm("{ .reg .u64 t; cvta.to.shared.u64 t, %1; cvt.u32.u64 %0, t; }" : "=r"(a) : "l"(p));
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  return r;
}
__device__ __forceinline__ void st_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

extern "C" __global__ void __launch_bounds__(ROW_THREADS, ROW_MIN_BLOCKS)
#if ROW_C > 1
__cluster_dims__(ROW_C, 1, 1)
#endif
acc_rows_stats(const __grid_constant__ Params p) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const i64 row = blockIdx.x / ROW_C;
  const int part = (int)(blockIdx.x % ROW_C);
  const int n = (int)p.n, k = (int)p.k;
  const row_span span(reinterpret_cast<const row_t*>(p.x) + row * p.n, n);
  const int per = (span.blocks + ROW_C - 1) / ROW_C;
  const int b0 = min(part * per, span.blocks), b1 = min(b0 + per, span.blocks);
  const f32 tau = __uint_as_float((u32)p.tau);
  const f32 c = ROW_LOG2E / tau;

  row_stat st = {-ROW_INF, 0.0f, 0.0f};
#if ROW_TOPK
  st_list list;
  int drained = b0, due = b0;            // blocks from `drained` on are not in the list of candidates yet; the next drain is behind tile `due`
  if (tid == 0) sh.count = sh.hot_count[0] = sh.hot_count[1] = 0;
  __syncthreads();
#endif

  for (int t = b0; t < b1; t += ST_TILE) {
    uint4 cur[ROW_U];
    span.load_tile(cur, t, b1);
    // maxima: of each block and of the chunk (a NaN stays visible)
    f32 mc;
#if ROW_F16
    u32 mb[ROW_U], mp;
#pragma unroll
    for (int u = 0; u < ROW_U; ++u) {
      mb[u] = row_max_nan2(row_max_nan2(cur[u].x, cur[u].y), row_max_nan2(cur[u].z, cur[u].w));
      mp = u == 0 ? mb[0] : row_max_nan2(mp, mb[u]);
    }
    mc = st_block_max(mp);
#else
    f32 mb[ROW_U];
#pragma unroll
    for (int u = 0; u < ROW_U; ++u) {
      f32 v[ROW_E];
      row_unpack(cur[u], v);
      mb[u] = row_max_nan(row_max_nan(v[0], v[1]), row_max_nan(v[2], v[3]));
      mc = u == 0 ? mb[0] : row_max_nan(mc, mb[u]);
    }
#endif
#if ROW_TOPK
    if (t == b0) {
      // The first tile sets the threshold, a key that at least k elements of the tile reach.  Every warp
      // answers for its share of the k: with T the largest 16-bit prefix that so many of its lanes' maxima reach, it
      // takes all maxima above T and, lane by lane, as many at T as are missing; the least key among those (rounded
      // down to the end of its block).  Few more than k reach it as long as the share is a small part of the 32 lanes; at
      // k = 128 every lane's maximum has to, and so do about 500 of the tile's 1024 blocks.
      const int share = (k + ST_WARPS - 1) / ST_WARPS;
      const u32 pre = mc == -ROW_INF ? 0u : (st_order(mc) >> 16);
      u32 T = 0;
#pragma unroll 1
      for (u32 bit = 1u << 15; bit != 0; bit >>= 1)
        if (__popc(__ballot_sync(ACC_FULL_MASK, pre >= (T | bit))) >= share) T |= bit;
      u64 least = ST_NONE + 1;           // (fewer maxima than its share: no bound but -inf)
      if (T != 0) {
        const int above = __popc(__ballot_sync(ACC_FULL_MASK, pre > T));
        const u32 ties = __ballot_sync(ACC_FULL_MASK, pre == T);
        least = ~(u64)0;
        if (pre == T && __popc(ties & ((1u << lane) - 1)) < share - above) {
          int last = 0;
#pragma unroll
          for (int u = ROW_U - 1; u >= 0; --u)
            if (st_block_max(mb[u]) == mc || mc != mc) last = span.first(t + u * ROW_THREADS + tid) + ROW_E - 1;
          if (mc != mc) last = 0x7fffffff;
          least = st_key(mc, last);
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
          const u64 o = __shfl_xor_sync(ACC_FULL_MASK, least, d);
          least = o < least ? o : least;
        }
      }
      if (lane == 0) sh.key[warp] = least;
      __syncthreads();
      for (int w = 0; w < ST_WARPS; ++w) least = sh.key[w] < least ? sh.key[w] : least;
      list.thr_key = least - 1;
    }
    // (later elements of the threshold's own value stand behind it: their indices are higher)
    if (t == b0) {
#pragma unroll
      for (int u = 0; u < ROW_U; ++u) {
        const int i = t + u * ROW_THREADS + tid;
        st_push(list, cur[u], st_block_max(mb[u]), i, span.first(i));
      }
    } else if (!(mc <= list.thr) && !list.overflow) {
#pragma unroll
      for (int u = 0; u < ROW_U; ++u)
        if (st_above(mb[u], list)) {
          const int slot = atomicAdd(&sh.hot_count[list.phase], 1);
          if (slot < ST_HOT) {
            sh.hot[slot] = cur[u];
            sh.hot_block[slot] = t + u * ROW_THREADS + tid;
          }
        }
    }
#endif
    // statistics
    const f32 mn = fmaxf(st.m, mc);
    if (mn > st.m) {
      if (st.m != -ROW_INF) {
        const f32 d = st_shift(st.m, mn, c), s = row_ex2(d);
        st.w = s == 0.0f ? 0.0f : s * fmaf(d, st.z, st.w);
        st.z *= s;
      }
      st.m = mn;
    }
    const row_two cc = row_pair(c, c);
#if ROW_F16
    const f32 neg = -(st_base(st.m) * c);
    const row_two nn = row_pair(neg, neg);
#define ST_T(x) row_fma2(x, cc, nn)
#else
    const f32 neg = -st_base(st.m);
    const row_two nn = row_pair(neg, neg);
#define ST_T(x) row_mul2(row_add2(x, nn), cc)
#endif
    row_two z0 = 0, z1 = 0, w0 = 0, w1 = 0;          // (pairs of +0)
#pragma unroll
    for (int u = 0; u < ROW_U; ++u) {
      f32 v[ROW_E];
      row_unpack(cur[u], v);
#pragma unroll
      for (int e = 0; e < ROW_E; e += 2) {
        f32 ta, tb;
        row_split(ST_T(row_pair(v[e], v[e + 1])), ta, tb);
        const row_two ex = row_pair(row_ex2(ta), row_ex2(tb));
        row_two& z = e & 2 ? z1 : z0;
        z = row_add2(z, ex);
#if !ROW_DISTILL
        // (a masked element has t = -inf and 2^t = 0: the bound keeps their product at 0)
        row_two& w = e & 2 ? w1 : w0;
        w = row_fma2(ex, row_pair(fmaxf(ta, -1000.0f), fmaxf(tb, -1000.0f)), w);
#endif
      }
    }
    f32 za, zb, wa, wb;
    row_split(row_add2(z0, z1), za, zb);
    row_split(row_add2(w0, w1), wa, wb);
    st.z += za + zb;
    st.w += wa + wb;

#if ROW_TOPK
    // The list is drained behind the first tile and whenever the part of the row seen since has doubled: each time
    // about k elements are expected above the old threshold.  Warps run on their own in between.
    if (t >= due || t + ST_TILE >= b1) {
      if (!list.overflow) list = st_drain(list, span.shift, k);
      if (!list.overflow) drained = t + ST_TILE;
      due = t + ST_TILE + (t - b0);
    }
#endif
  }
#if ROW_TOPK
  if (list.overflow)
    // More blocks came than the list holds: once more over the tiles since, with the list drained as often as it may
    // fill up.  That takes a row in rising order, or more than 120 alternatives: the first tile of ordinary rows then lists
    // nearly as many blocks as there is room for (k = 128: a third of the CTAs come here, and read their whole part twice).
    // 4096 x 131072 Halves: k = 20 212 us, 64 276, 100 363, 112 442, 120 542, 124 637, 128 781.
    for (int s = drained; s < b1; s += ST_HOT) {
#pragma unroll 1
      for (int u = 0; u < ST_HOT / ROW_THREADS; ++u) {
        const int i = s + u * ROW_THREADS + tid;
        if (i < b1) {
          const uint4 block = span.load(i);
          f32 v[ROW_E], most;
          row_unpack(block, v);
          most = v[0];
#pragma unroll
          for (int e = 1; e < ROW_E; ++e) most = row_max_nan(most, v[e]);
          st_push(list, block, most, i, span.first(i));
        }
      }
      list = st_drain(list, span.shift, k);
    }
#endif
#if ROW_TOPK
  int held = list.held;                  // (sorted by the last drain)
  if (tid == 0) sh.kept = held;
#endif
  // join the statistics: lanes, warps, CTAs of the cluster
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    row_stat o;
    o.m = __shfl_xor_sync(ACC_FULL_MASK, st.m, d);
    o.z = __shfl_xor_sync(ACC_FULL_MASK, st.z, d);
    o.w = __shfl_xor_sync(ACC_FULL_MASK, st.w, d);
    st = st_join(st, o, c);
  }
  if (lane == 0) sh.part[warp] = st;
  __syncthreads();
  st = sh.part[0];
#pragma unroll
  for (int w = 1; w < ST_WARPS; ++w) st = st_join(st, sh.part[w], c);
#if ROW_C > 1
  if (tid == 0) sh.cta = st;
  st_cluster_sync();
  if (part == 0) {
    row_stat o[ROW_C];
#pragma unroll
    for (int r = 1; r < ROW_C; ++r)
      asm volatile("ld.shared::cluster.f32 %0, [%3];\n ld.shared::cluster.f32 %1, [%3 + 4];\n ld.shared::cluster.f32 %2, [%3 + 8];"
                   : "=f"(o[r].m), "=f"(o[r].z), "=f"(o[r].w) : "r"(st_cluster_addr(&sh.cta, r)));
#pragma unroll
    for (int r = 1; r < ROW_C; ++r) st = st_join(st, o[r], c);
#if ROW_TOPK
    const int own = held;
    int more[ROW_C];
    u64 key[ROW_C];
#pragma unroll
    for (int r = 1; r < ROW_C; ++r)
      asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(more[r]) : "r"(st_cluster_addr(&sh.kept, r)));
#pragma unroll
    for (int r = 1; r < ROW_C; ++r)      // (at most k <= 128 of them: one per thread)
      if (tid < more[r]) asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(key[r]) : "r"(st_cluster_addr(&sh.cand[tid], r)));
#pragma unroll
    for (int r = 1; r < ROW_C; ++r) {
      if (tid < more[r]) sh.cand[held + tid] = key[r];
      held += more[r];
    }
    __syncthreads();
    held = st_compact(own, held, k);
#endif
  }
  st_cluster_sync();                     // nobody leaves while its shared memory is being read
  if (part != 0) return;
#endif

  // a row without an element above -inf has no distribution: its normaliser is -inf
  const bool none = st.m == -ROW_INF && st.z == 0.0f;
  const f32 base = st_base(st.m);
  f32 ln_z = -ROW_INF;                   // ln sum e^((x - m) / tau)
  if (!none) {
    ln_z = logf(st.z);
#if ROW_F16
    ln_z += ROW_LN2 * fmaf(-base, c, base * c);
#endif
  }
  const f32 lse = base / tau + ln_z;
#if ROW_DISTILL
  // The teacher's entries, one warp: with e_i = exp((t_i - max t)/tau) and E their sum, q_i = e_i / E and
  // loss = tau^2 (sum e_i ((t_i - max t) - (s_i - m)) / (tau E) - ln E + ln Z).
  if (warp == 0) {
    const i32* ids = reinterpret_cast<const i32*>(p.tok) + row * p.k;
    const teacher_t* ts = reinterpret_cast<const teacher_t*>(p.teacher) + row * p.k;
    f32 mt = -ROW_INF;
    bool bad = false;
    for (int i = lane; i < k; i += 32) {
      const int id = ids[i];
      bad = bad || id >= n;
      if (id >= 0 && id < n) mt = row_max_nan(mt, row_wide(ts[i]));
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) mt = row_max_nan(mt, __shfl_xor_sync(ACC_FULL_MASK, mt, d));
    f32 es = 0.0f, as = 0.0f;
    for (int i = lane; i < k; i += 32) {
      const int id = ids[i];
      if (id >= 0 && id < n) {
        const f32 dt = mt == -ROW_INF ? -ROW_INF : row_wide(ts[i]) - mt;
        const f32 e = row_ex2(dt * c);
        if (e != 0.0f) {
          es += e;
          as += e * ((dt - (row_wide(span.x[id]) - base)) / tau);
        }
      }
    }
    es = row_warp_sum(es);
    as = row_warp_sum(as);
    bad = __any_sync(ACC_FULL_MASK, bad);
    if (lane == 0) {
      f32 loss = 0.0f;                   // no entry, no loss
      if (es != 0.0f) loss = none ? ROW_INF : tau * tau * (as / es - logf(es) + ln_z);
      if (bad) {
        acc_fail(p.err, 1003);           // "index out of bounds", reported by the next download or b200_sync
        loss = ROW_NAN;
      }
      reinterpret_cast<f32*>(p.out0)[row] = loss;
      reinterpret_cast<f32*>(p.out1)[row] = lse;
    }
  }
#else
  if (tid == 0) {
    const i64 tok = (i64) reinterpret_cast<const token_t*>(p.tok)[row];
    f32 logp = 0.0f;                     // no given token
    if (tok >= n) {
      acc_fail(p.err, 1003);
      logp = ROW_NAN;
    } else if (tok >= 0) {
      logp = none ? -ROW_INF : row_wide(span.x[tok]) - base - ln_z;
    }
    reinterpret_cast<f32*>(p.out0)[row] = logp;
    reinterpret_cast<f32*>(p.out1)[row] = lse;
    reinterpret_cast<f32*>(p.out2)[row] = none ? 0.0f : logf(st.z) - ROW_LN2 * (st.w / st.z);
  }
#if ROW_TOPK
  __syncthreads();
  if (held < k) {
    // All elements above -inf are in the list.  The places behind them go to -inf elements, lowest index first: they
    // are among the row's first 2k - 1 elements.
    const int finite = held;
    for (int base = 0; base < 2 * k; base += ROW_THREADS) {
      const int j = base + tid;
      bool free_one = j < n && j < 2 * k;
      for (int i = 0; i < finite; ++i) free_one = free_one && st_index(sh.cand[i]) != j;
      const u32 ones = __ballot_sync(ACC_FULL_MASK, free_one);
      __syncthreads();
      if (lane == 0) sh.warp_count[warp] = __popc(ones);
      __syncthreads();
      int at = held + __popc(ones & ((1u << lane) - 1)), all = held;
      for (int w = 0; w < ST_WARPS; ++w) {
        if (w < warp) at += sh.warp_count[w];
        all += sh.warp_count[w];
      }
      if (free_one && at < k) sh.cand[at] = st_key(-ROW_INF, j);
      held = all < k ? all : k;
    }
    __syncthreads();
  }
  if (tid < k) {
    int id = -1;                         // a row shorter than k ends in (-1, -inf)
    f32 logp = -ROW_INF;
    if (tid < held) {
      const u64 key = sh.cand[tid];
      id = st_index(key);
      if (!none) logp = st_value((u32)(key >> 32)) - base - ln_z;
    }
    reinterpret_cast<i32*>(p.out3)[row * p.k + tid] = id;
    reinterpret_cast<f32*>(p.out4)[row * p.k + tid] = logp;
  }
#endif
#endif
}
