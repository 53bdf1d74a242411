// Foreign array functions of this backend (Aforeign, AST.hs:307-316; the reference's way to put hand-written code
// behind an array function, with a definition in array code beside it): the row operators.
//
// Names, constants, arguments and results (sh: any outer shape, the same for all arguments of a call; t: Half or Float):
//   b200.logProbs       (consts k)    tokens (sh, Int32 or Int), logits (sh:.n, t)
//                                     -> (sh, (log probability, normaliser, entropy) Floats), (sh:.k, (Int32 index, Float))
//   b200.distill        (consts tau)  ids (sh:.k, Int32; k <= 4096), teacher (sh:.k, t'), student (sh:.n, t) -> (sh, loss), (sh, normaliser)
//   b200.distillGrad    (consts tau)  ids, teacher, student, normaliser (sh, Float), gradient (sh, Float) -> (sh:.n, t)
//   b200.layerNorm      (consts eps)  gamma, beta (Vector of t or Float), xs (sh:.n, t) -> (sh:.n, t), (sh, (mean, rstd) Floats)
//   b200.layerNormGrad  (consts)      gamma, xs, (sh, (mean, rstd)), dys (sh:.n, t) -> (sh:.n, t), dgamma, dbeta (gamma's type)
#include <algorithm>
#include <cmath>
#include <cstring>

#include "runtime.hpp"

namespace accb200 {

namespace {

const struct { const char* name; Foreign op; } kForeign[] = {
    {"b200.logProbs", F_LOG_PROBS},   {"b200.distill", F_DISTILL},           {"b200.distillGrad", F_DISTILL_GRAD},
    {"b200.layerNorm", F_LAYER_NORM}, {"b200.layerNormGrad", F_LAYER_NORM_GRAD},
};
// the alternatives of logProbs: the list is selected and merged by one thread per entry
constexpr int kMostAlternatives = 128;
// a teacher's entries per row: distillGrad looks for equal ids pair by pair
constexpr int64_t kMostEntries = 4096;
// indices inside a row are 32 bits (rows of a tile's width below 2^31)
constexpr int64_t kMostColumns = (1LL << 31) - (1LL << 20);

typedef std::map<std::string, std::string> Variant;

bool is(const ArrayInfo& a, int rank, Ty t) { return a.rank == rank && !a.elt.tuple && a.elt.s == t; }
bool is_real(const ArrayInfo& a) { return !a.elt.tuple && (a.elt.s == F16 || a.elt.s == F32); }
bool is_floats(const ArrayInfo& a, int rank, size_t n) {
  if (a.rank != rank || !a.elt.tuple || a.elt.e.size() != n) return false;
  for (auto& c : a.elt.e)
    if (c.tuple || c.s != F32) return false;
  return true;
}
// the array of logits, or the rows to be normalised
const ArrayInfo& rows_arg(const Node& n) {
  switch (n.foreign) {
    case F_LOG_PROBS: case F_LAYER_NORM_GRAD: return n.arg_info[1];
    default: return n.arg_info[2];
  }
}
std::string ctype(Ty t) { return t == F16 ? "u16" : t == F32 ? "f32" : t == I64 ? "i64" : "i32"; }
std::string str(int64_t v) { return std::to_string(v); }

// what the kernel's st_shared takes (rows_stats.cuh): candidates and listed blocks, and the warps' statistics
size_t stats_smem(bool topk) { return (topk ? 1024 * 8 + 512 * 20 : 0) + 512; }

}  // namespace

Foreign foreign_named(const std::string& name) {
  for (auto& f : kForeign)
    if (name == f.name) return f.op;
  return F_NONE;
}

void foreign_check(const Node& n, const std::vector<ArrayInfo>& outs) {
  std::string name;
  for (auto& f : kForeign)
    if (f.op == n.foreign) name = f.name;
  auto need = [&](bool ok, const std::string& what) { if (!ok) throw Error(B200_ERR_TYPE, name + ": " + what); };
  const std::vector<ArrayInfo>& a = n.arg_info;
  const size_t nargs[] = {0, 2, 3, 5, 3, 4}, nouts[] = {0, 2, 2, 1, 2, 3}, nconsts[] = {0, 1, 1, 1, 1, 0};
  need(a.size() == nargs[n.foreign], "takes " + std::to_string(nargs[n.foreign]) + " arrays");
  need(n.consts.size() == nconsts[n.foreign], "takes " + std::to_string(nconsts[n.foreign]) + " constants");
  const ArrayInfo& x = rows_arg(n);
  need(x.rank >= 1 && is_real(x), "the rows must be an array of Half or Float of rank 1 or more");
  const int r = x.rank;
  need(outs.size() == nouts[n.foreign], "the function yields another number of arrays");
  switch (n.foreign) {
    case F_LOG_PROBS: {
      const double k = n.consts[0];
      if (!(k >= 0 && k <= kMostAlternatives && k == std::floor(k)))
        throw Error(B200_ERR_UNSUPPORTED, name + ": the number of alternatives must be a whole number from 0 to " + str(kMostAlternatives));
      need(is(a[0], r - 1, I32) || is(a[0], r - 1, I64), "the given tokens must be Int32 or Int, one per row");
      need(is_floats(outs[0], r - 1, 3) && outs[1].rank == r && outs[1].elt == Type::tup({Type::scalar(I32), Type::scalar(F32)}), "the function yields other arrays");
      break;
    }
    case F_DISTILL: case F_DISTILL_GRAD: {
      const double tau = n.consts[0];
      // (outside this range products of the temperature and a Float logit leave the type's range)
      if (!(tau >= 1e-4 && tau <= 1e4)) throw Error(B200_ERR_ARG, name + ": the temperature must lie between 1e-4 and 1e4");
      need(is(a[0], r, I32), "the teacher's tokens must be Int32, one list per row");
      need(a[1].rank == r && is_real(a[1]), "the teacher's logits must be Half or Float, one list per row");
      if (n.foreign == F_DISTILL) {
        need(is(outs[0], r - 1, F32) && is(outs[1], r - 1, F32), "the function yields other arrays");
      } else {
        need(is(a[3], r - 1, F32) && is(a[4], r - 1, F32), "normaliser and gradient must be Float, one per row");
        need(is(outs[0], r, x.elt.s), "the function yields other arrays");
      }
      break;
    }
    case F_LAYER_NORM: {
      if (!(n.consts[0] >= 0 && n.consts[0] <= 3.4e38)) throw Error(B200_ERR_ARG, name + ": epsilon must be finite and not negative");
      need((is(a[0], 1, x.elt.s) || is(a[0], 1, F32)) && is(a[1], 1, a[0].elt.s), "gamma and beta must be vectors of the rows' type or of Float");
      need(is(outs[0], r, x.elt.s) && is_floats(outs[1], r - 1, 2), "the function yields other arrays");
      break;
    }
    case F_LAYER_NORM_GRAD:
      need(is(a[0], 1, x.elt.s) || is(a[0], 1, F32), "gamma must be a vector of the rows' type or of Float");
      need(is_floats(a[2], r - 1, 2), "the statistics must be pairs of Floats, one per row");
      need(is(a[3], r, x.elt.s), "the gradient must have the rows' type and rank");
      need(is(outs[0], r, x.elt.s) && is(outs[1], 1, a[0].elt.s) && is(outs[2], 1, a[0].elt.s), "the function yields other arrays");
      break;
    case F_NONE: break;
  }
}

Glue foreign_glue(const Node& n) {
  Glue g;
  g.defines["ROW_F16"] = rows_arg(n).elt.s == F16 ? "1" : "0";
  switch (n.foreign) {
    case F_LOG_PROBS:
      g.defines["ROW_DISTILL"] = "0";
      g.defines["ROW_TOPK"] = n.consts[0] > 0 ? "1" : "0";
      g.defines["ROW_SMEM"] = str((int64_t)stats_smem(n.consts[0] > 0));
      g.code = "typedef " + ctype(n.arg_info[0].elt.s) + " token_t;\n";
      break;
    case F_DISTILL:
      g.defines["ROW_DISTILL"] = "1";
      g.defines["ROW_TOPK"] = "0";
      g.defines["ROW_SMEM"] = str((int64_t)stats_smem(false));
      g.code = "typedef " + ctype(n.arg_info[1].elt.s) + " teacher_t;\n";
      break;
    case F_DISTILL_GRAD: g.code = "typedef " + ctype(n.arg_info[1].elt.s) + " teacher_t;\n"; break;
    case F_LAYER_NORM: case F_LAYER_NORM_GRAD: g.code = "typedef " + ctype(n.arg_info[0].elt.s) + " param_t;\n"; break;
    case F_NONE: break;
  }
  return g;
}

// ---- launch shapes ------------------------------------------------------------------------------------
namespace {

constexpr int kThreads = 256, kStatsThreads = 128;

Variant stats_variant(int ctas) { return {{"ROW_THREADS", str(kStatsThreads)}, {"ROW_U", "8"}, {"ROW_MIN_BLOCKS", "7"}, {"ROW_C", str(ctas)}}; }
Variant distill_grad_variant(int ctas) { return {{"ROW_THREADS", str(kThreads)}, {"ROW_U", "4"}, {"ROW_MIN_BLOCKS", "4"}, {"ROW_C", str(ctas)}}; }

// CTAs that share a row: at least `least`, and enough to give every SM `several`, as long as each has a tile of its own.
// The statistics take as few as fill the machine (500 rows of 50257 Floats, k = 5: 1 CTA per row 29.8 us, 2 CTAs 28.0,
// 4 CTAs 40.8: every CTA finds a threshold of its own); the gradient, whose CTAs are independent, four (4096 rows of
// 131072 Halves: 363 us with one CTA per row, 348 with four, 515 with sixteen).
int ctas_per_row(int64_t rows, int64_t n, int elt_bytes, int sms, int least, int several, int most) {
  const int64_t tiles = (n * elt_bytes + 16 * kThreads * 4 - 1) / (16 * kThreads * 4);
  int c = 1;
  while (c < most && (c < least || rows * c < several * (int64_t)sms) && 2 * c <= tiles) c *= 2;
  return c;
}

// A row over warps and registers (rows_norm_pre.cuh)
struct NormShape {
  int ve, warps, u, threads;
  bool whole;              // the row fits the registers
  int stages = 0;          // gradients: rows in flight through shared memory
  bool keep = true;        // gradients: a row's values stay in registers between the passes
  Variant variant() const {
    return {{"ROW_THREADS", str(threads)}, {"NORM_VE", str(ve)},         {"NORM_WARPS", str(warps)},         {"NORM_U", str(u)},
            {"NORM_LONG", whole ? "0" : "1"}, {"NORM_STAGES", str(stages)}, {"NORM_KEEP", keep ? "1" : "0"}};
  }
  uint64_t key() const {
    return (uint64_t)ve << 40 | (uint64_t)warps << 32 | (uint64_t)u << 16 | (uint64_t)(threads / 32) << 8 | (uint64_t)stages << 4 | (keep ? 2 : 0) | (whole ? 1 : 0);
  }
  int rows() const { return threads / 32 / warps; }
};
// the next size of the list 1 2 3 4 6 8 12 16 ...: few kernels for all lengths
int round_up_u(int64_t u) {
  int v = 1;
  while (v < u) v = (v & (v - 1)) == 0 && v > 1 ? v + v / 2 : (v == 1 ? 2 : v / 3 * 4);
  return v;
}
// As few warps per row as hold it at `most_elems` elements per lane: long per-lane runs leave fewer shuffles, barriers and
// addresses per element (forward, 65536 x 2048 Halves: 32 elements 89 us, 16 elements 97, 8 elements 134).
NormShape norm_shape(int64_t n, int ve, int most_elems, int most_warps, int64_t rows, int sms) {
  NormShape s{ve, 1, 1, kThreads, true};
  const int64_t units = std::max<int64_t>((n + ve - 1) / ve, 1);
  const int most_u = std::max(1, most_elems / ve);
  auto need = [&](int w) { return (units + w * 32 - 1) / (w * 32); };
  while (s.warps < most_warps && need(s.warps) > most_u) s.warps *= 2;
  // few rows: more warps on each, so that the machine has something to do (8 x 4096 Halves 4.2 us instead of 5.2,
  // 300 x 1024 Floats 4.2 instead of 6.2)
  while (s.warps < 8 && need(s.warps) > 1 && rows * s.warps < 16 * (int64_t)sms) s.warps *= 2;
  if (need(s.warps) > most_u) {
    s.whole = false;
    s.warps = 16;
    s.u = 1;
  } else {
    s.u = round_up_u(need(s.warps));
  }
  s.threads = std::max(kThreads, s.warps * 32);
  return s;
}
constexpr int kNormElems = 32, kNormWarps = 32;          // forward: elements per thread, warps per row
// Elements per access: the widest, up to 16 bytes, on whose boundary all rows and the parameters start.
int norm_access(const std::vector<const DevArray*>& rows_like, const std::vector<const DevArray*>& params, int64_t cols, int elt_bytes, int param_bytes) {
  uint64_t at = (uint64_t)cols * elt_bytes, pat = 0;
  for (auto* a : rows_like) at |= (uint64_t)(uintptr_t)a->leaf[0]->ptr;
  for (auto* a : params) pat |= (uint64_t)(uintptr_t)a->leaf[0]->ptr;
  int ve = 16 / elt_bytes;
  while (ve > 1 && (at % (ve * elt_bytes) != 0 || pat % std::min(16, ve * param_bytes) != 0)) ve /= 2;
  return ve;
}
// (single elements per access: eight per lane, 50000 x 1001 Halves 80 us; sixteen 86)
NormShape norm_forward_shape(int64_t n, int ve, int64_t rows, int sms) {
  const NormShape s = norm_shape(n, ve, ve <= 2 ? 8 * ve : 32, 8, rows, sms);
  return s.whole ? s : norm_shape(n, ve, kNormElems, kNormWarps, rows, sms);
}
constexpr int kNormGradElems = 16, kNormGradWarps = 16;  // gradients; twice the elements where they pass through shared memory
// Shared memory per CTA for rows in flight: two CTAs of 256 threads per SM, or one of 512 (32768 x 4096 Halves: 155 us;
// three CTAs with fewer rows in flight 189, loads without the ring 222)
constexpr int64_t kRingBytes = 112 << 10, kRingBytesAlone = 208 << 10;
// gamma as Floats, for any length that comes to a shape
int64_t norm_gamma_bytes(const NormShape& s) { return 4LL * s.u * s.warps * 32 * s.ve; }
NormShape norm_grad_shape(int64_t n, int ve, int elt_bytes, int64_t rows, int sms) {
  const int bytes = ve * elt_bytes;
  // (accesses of one element: eight per lane, which leave registers for more rows at a time, as long as the row fits:
  // 50000 x 1001 Floats 139 us, with sixteen 169)
  NormShape s = norm_shape(n, ve, std::min(kNormGradElems, 8 * ve), kNormGradWarps, rows, sms);
  if (!s.whole) s = norm_shape(n, ve, kNormGradElems, kNormGradWarps, rows, sms);
  if (bytes == 2) return s;
  const NormShape reread = s;
  if (!s.whole) {
    if (bytes < 16) return reread;
    s = norm_shape(n, ve, 2 * kNormGradElems, kNormGradWarps, rows, sms);
    if (!s.whole) return s;
    s.keep = false;
  }
  const int64_t stage = 2LL * bytes * s.u * s.threads, room = (s.threads > kThreads ? kRingBytesAlone : kRingBytes) - norm_gamma_bytes(s);
  s.stages = (int)std::min<int64_t>(4, room / stage);
  return s.stages < 2 ? reread : s;
}
size_t norm_grad_smem(const NormShape& s, int elt_bytes, int64_t n) {
  if (!s.whole) return 0;
  const size_t ring = 2u * s.ve * elt_bytes * s.u * s.threads * s.stages + (s.stages ? norm_gamma_bytes(s) : 0), sums = s.rows() > 1 ? (size_t)n * 8 : 0;
  return std::max(ring, sums);
}

}  // namespace

std::vector<std::pair<std::string, Variant>> foreign_variants(const Node& n) {
  std::vector<std::pair<std::string, Variant>> v;
  const int ve = rows_arg(n).elt.s == F16 ? 8 : 4;
  auto with = [](Variant a, const char* key) { a["NORM_SUMS"] = a["NORM_COLS"] = "0"; if (*key) a[key] = "1"; return a; };
  auto add = [&](const char* skeleton, Variant a) {
    for (auto& b : v)
      if (b.second == a) return;
    v.push_back({skeleton, std::move(a)});
  };
  switch (n.foreign) {
    case F_LOG_PROBS: case F_DISTILL:    // (what ctas_per_row can give)
      for (int c : {1, 2, 4, 8}) add("rows_stats", stats_variant(c));
      break;
    case F_DISTILL_GRAD:
      for (int c : {1, 2, 4, 8, 16}) add("rows_distill_grad", distill_grad_variant(c));
      break;
    case F_LAYER_NORM:                   // (short rows to long ones, few and many)
      for (int64_t rows : {1 << 20, 1})
        for (int64_t len : {1024, 4096, 1 << 20})
          for (int w : {ve, 2, 1}) add("rows_norm", norm_forward_shape(len, w, rows, 148).variant());
      break;
    case F_LAYER_NORM_GRAD:
      for (int64_t rows : {1 << 20, 1})
        for (int64_t len : {1024, 4096, 12000, 1 << 20})
          for (int w : {ve, 2, 1}) add("rows_norm_grad", with(norm_grad_shape(len, w, 16 / ve, rows, 148).variant(), ""));
      add("rows_norm_grad", with(NormShape{1, 1, 1, 1024, true}.variant(), "NORM_SUMS"));
      add("rows_norm_grad", with(NormShape{1, 1, 1, kThreads, true}.variant(), "NORM_COLS"));
      break;
    case F_NONE: break;
  }
  return v;
}

// ---- execution -------------------------------------------------------------------------------------------
namespace {

uint64_t ptr_of(const DevArray& a, int leaf = 0) { return (uint64_t)(uintptr_t)a.leaf[leaf]->ptr; }
uint64_t float_bits(double v) {
  const float f = (float)v;
  uint32_t b;
  memcpy(&b, &f, 4);
  return b;
}
// The kernel of a foreign node for a launch shape: `key` identifies the shape, `variant` spells it out, once.
template <class V> CompiledKernel& shape_kernel(Ctx& c, NodeState& st, uint64_t key, const char* skeleton, V variant, const char* entry, int threads, size_t smem) {
  auto it = st.shape_memo.find(key);
  if (it != st.shape_memo.end()) {
    c.mem_hits++;
    return *it->second;
  }
  CompiledKernel& k = node_kernel(c, st, skeleton, variant(), entry, threads, smem);
  st.shape_memo[key] = &k;
  return k;
}
void launch(Ctx& c, CompiledKernel& k, int64_t grid, int threads, size_t smem, std::vector<uint64_t> params) {
  if (grid <= 0) return;
  if (grid > 2147483647LL) throw Error(B200_ERR_UNSUPPORTED, "grid too large");
  void* args[1] = {params.data()};
  c.check(c.drv.LaunchKernel(k.fn, (unsigned)grid, 1, 1, (unsigned)threads, 1, 1, (unsigned)smem, (CUstream)c.stream, args, nullptr), "cuLaunchKernel");
  c.launches++;
}

}  // namespace

void Program::exec_foreign(const Node& n, Env& env) {
  Ctx& c = *ctx;
  // Results and scratch come from the context's pool and go back to it when the caller frees them: a captured graph
  // would keep writing to memory that belongs to somebody else by the time it is replayed.
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  c.check(cudaStreamIsCapturing(c.stream, &capture), "cudaStreamIsCapturing");
  if (capture != cudaStreamCaptureStatusNone) throw Error(B200_ERR_UNSUPPORTED, "a row operator cannot be captured into a CUDA graph");
  NodeState& st = nodes[n.id];
  std::vector<DevArrayP> a;
  for (auto& name : n.args) a.push_back(env.at(name));
  const DevArray& x = *a[n.foreign == F_LOG_PROBS || n.foreign == F_LAYER_NORM_GRAD ? 1 : 2];
  const std::vector<int64_t> outer(x.shape.begin(), x.shape.end() - 1);
  for (auto& b : a)
    for (size_t l = 0; l < b->leaf.size(); ++l)
      if ((uintptr_t)b->leaf[l]->ptr % ty_bytes[b->leaf_ty[l]]) throw Error(B200_ERR_ARG, "an array does not start on a boundary of its elements");
  const int64_t cols = std::max<int64_t>(x.shape.back(), 0);
  int64_t rows = 1;
  for (int64_t d : outer) rows *= std::max<int64_t>(d, 0);
  if (cols > kMostColumns) throw Error(B200_ERR_UNSUPPORTED, "rows of " + str(cols) + " elements are too long");
  auto outer_is = [&](const DevArray& b, bool list) {
    if (std::vector<int64_t>(b.shape.begin(), b.shape.end() - (list ? 1 : 0)) != outer) throw Error(B200_ERR_BOUNDS, "shape mismatch");
  };
  const int elt_bytes = ty_bytes[x.elt.s];
  const uint64_t err = (uint64_t)(uintptr_t)(c.d_words + 0);
  switch (n.foreign) {
    case F_LOG_PROBS: {
      outer_is(*a[0], false);
      const int64_t k = (int64_t)n.consts[0];
      std::vector<int64_t> list = outer;
      list.push_back(k);
      DevArrayP stats = c.new_array(n.out_info[0].elt, outer), top = c.new_array(n.out_info[1].elt, list);
      env[n.outs[0]] = stats;
      env[n.outs[1]] = top;
      if (rows == 0) break;
      const int ctas = ctas_per_row(rows, cols, elt_bytes, c.sm_count, 1, 4, 8);
      const size_t smem = stats_smem(k > 0);
      CompiledKernel& ker = shape_kernel(c, st, (uint64_t)ctas, "rows_stats", [&] { return stats_variant(ctas); }, "acc_rows_stats", kStatsThreads, smem);
      launch(c, ker, rows * ctas, kStatsThreads, smem,
             {ptr_of(x), ptr_of(*a[0]), 0, ptr_of(*stats, 0), ptr_of(*stats, 1), ptr_of(*stats, 2), ptr_of(*top, 0), ptr_of(*top, 1),
              (uint64_t)rows, (uint64_t)cols, (uint64_t)k, float_bits(1.0), err});
      break;
    }
    case F_DISTILL: case F_DISTILL_GRAD: {
      outer_is(*a[0], true);
      outer_is(*a[1], true);
      if (a[0]->shape != a[1]->shape) throw Error(B200_ERR_BOUNDS, "shape mismatch");
      const int64_t k = std::max<int64_t>(a[0]->shape.back(), 0);
      if (k > kMostEntries) throw Error(B200_ERR_UNSUPPORTED, "more than " + str(kMostEntries) + " teacher entries per row");
      if (n.foreign == F_DISTILL) {
        DevArrayP loss = c.new_array(n.out_info[0].elt, outer), lse = c.new_array(n.out_info[1].elt, outer);
        env[n.outs[0]] = loss;
        env[n.outs[1]] = lse;
        if (rows == 0) break;
        const int ctas = ctas_per_row(rows, cols, elt_bytes, c.sm_count, 1, 4, 8);
        const size_t smem = stats_smem(false);
        CompiledKernel& ker = shape_kernel(c, st, (uint64_t)ctas, "rows_stats", [&] { return stats_variant(ctas); }, "acc_rows_stats", kStatsThreads, smem);
        launch(c, ker, rows * ctas, kStatsThreads, smem,
               {ptr_of(x), ptr_of(*a[0]), ptr_of(*a[1]), ptr_of(*loss), ptr_of(*lse), 0, 0, 0, (uint64_t)rows, (uint64_t)cols, (uint64_t)k,
                float_bits(n.consts[0]), err});
      } else {
        outer_is(*a[3], false);
        outer_is(*a[4], false);
        DevArrayP dx = c.new_array(n.out_info[0].elt, x.shape);
        env[n.outs[0]] = dx;
        if (rows == 0 || cols == 0) break;
        const int ctas = ctas_per_row(rows, cols, elt_bytes, c.sm_count, 4, 8, 16);
        CompiledKernel& ker = shape_kernel(c, st, (uint64_t)ctas, "rows_distill_grad", [&] { return distill_grad_variant(ctas); }, "acc_rows_distill_grad", kThreads, 0);
        launch(c, ker, rows * ctas, kThreads, 0,
               {ptr_of(x), ptr_of(*a[0]), ptr_of(*a[1]), ptr_of(*a[3]), ptr_of(*a[4]), ptr_of(*dx), (uint64_t)rows, (uint64_t)cols, (uint64_t)k,
                float_bits(n.consts[0]), err});
      }
      break;
    }
    case F_LAYER_NORM: {
      if (a[0]->shape[0] != x.shape.back() || a[1]->shape[0] != x.shape.back()) throw Error(B200_ERR_BOUNDS, "shape mismatch");
      DevArrayP y = c.new_array(n.out_info[0].elt, x.shape), stats = c.new_array(n.out_info[1].elt, outer);
      env[n.outs[0]] = y;
      env[n.outs[1]] = stats;
      if (rows == 0) break;
      const int ve = norm_access({&x, y.get()}, {a[0].get(), a[1].get()}, cols, elt_bytes, ty_bytes[a[0]->elt.s]);
      const NormShape s = norm_forward_shape(cols, ve, rows, c.sm_count);
      CompiledKernel& ker = shape_kernel(c, st, s.key(), "rows_norm", [&] { return s.variant(); }, "acc_rows_norm", s.threads, 0);
      launch(c, ker, (rows + s.rows() - 1) / s.rows(), s.threads, 0,
             {ptr_of(x), ptr_of(*a[0]), ptr_of(*a[1]), ptr_of(*y), ptr_of(*stats, 0), ptr_of(*stats, 1), (uint64_t)rows, (uint64_t)cols, float_bits(n.consts[0])});
      break;
    }
    case F_LAYER_NORM_GRAD: {
      if (a[0]->shape[0] != x.shape.back() || a[3]->shape != x.shape) throw Error(B200_ERR_BOUNDS, "shape mismatch");
      outer_is(*a[2], false);
      DevArrayP dx = c.new_array(n.out_info[0].elt, x.shape);
      DevArrayP dgamma = c.new_array(n.out_info[1].elt, a[0]->shape), dbeta = c.new_array(n.out_info[2].elt, a[0]->shape);
      env[n.outs[0]] = dx;
      env[n.outs[1]] = dgamma;
      env[n.outs[2]] = dbeta;
      if (cols == 0) break;
      const int ve = norm_access({&x, dx.get(), a[3].get()}, {a[0].get()}, cols, elt_bytes, ty_bytes[a[0]->elt.s]);
      const NormShape s = norm_grad_shape(cols, ve, elt_bytes, rows, c.sm_count);
      // (one source for three kernels: which of them it compiles to)
      auto which = [&](bool sums, bool cols_) {
        return [&, sums, cols_] {
          Variant v = sums || cols_ ? NormShape{1, 1, 1, sums ? 1024 : kThreads, true}.variant() : s.variant();
          v["NORM_SUMS"] = sums ? "1" : "0";
          v["NORM_COLS"] = cols_ ? "1" : "0";
          return v;
        };
      };
      const size_t smem = norm_grad_smem(s, elt_bytes, cols);
      CompiledKernel& ker = shape_kernel(c, st, s.key(), "rows_norm_grad", which(false, false), "acc_rows_norm_grad", s.threads, smem);
      // as many CTAs as fit at once, and few enough for four trips each: a CTA costs a line of partial sums (2048 x 768
      // Floats: 16.5 us with 148 lines, 18.5 with 296)
      const int64_t groups = (rows + s.rows() - 1) / s.rows();
      const int64_t grid = std::min(groups, std::min<int64_t>((int64_t)c.sm_count * ker.max_blocks_per_sm, std::max<int64_t>(c.sm_count, groups / 4)));
      // lines of partial sums: one per CTA; for long rows one per `chunk` rows
      const int64_t tiles = (cols + 31) / 32;
      int64_t lines = grid, chunk = 0;
      if (!s.whole) {
        chunk = std::max<int64_t>(8, (rows * tiles + 8 * c.sm_count - 1) / (8 * c.sm_count));
        lines = (rows + chunk - 1) / chunk;
      }
      std::shared_ptr<Buffer> partial = c.alloc((size_t)lines * 2 * cols * 4);
      const std::vector<uint64_t> params = {ptr_of(x), ptr_of(*a[0]), ptr_of(*a[2], 0), ptr_of(*a[2], 1), ptr_of(*a[3]), ptr_of(*dx),
                                            (uint64_t)(uintptr_t)partial->ptr, ptr_of(*dgamma), ptr_of(*dbeta), (uint64_t)rows, (uint64_t)cols, (uint64_t)lines, (uint64_t)chunk};
      launch(c, ker, grid, s.threads, smem, params);
      if (!s.whole) {
        CompiledKernel& kc = shape_kernel(c, st, 1, "rows_norm_grad", which(false, true), "acc_rows_norm_cols", kThreads, 0);
        launch(c, kc, lines * tiles, kThreads, 0, params);
      }
      CompiledKernel& ks = shape_kernel(c, st, 2, "rows_norm_grad", which(true, false), "acc_rows_norm_sums", 1024, 0);
      launch(c, ks, tiles, 1024, 0, params);
      break;
    }
    case F_NONE: break;
  }
}

}  // namespace accb200
