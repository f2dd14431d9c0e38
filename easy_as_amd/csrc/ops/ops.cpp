// ops.cpp — the operators' entry points: their checks, their plans and their launches.
#include <cstdlib>
#include <cstring>

#include "ops.h"

namespace eas {
namespace {

#define OPS_CHECK(cond, message) \
  do {                           \
    if (!(cond)) return fail_status(EAS_HIP_ERR_INVALID, message); \
  } while (0)
#define OPS_HIP(call)                                                                               \
  do {                                                                                              \
    const hipError_t e_ = (call);                                                                   \
    if (e_ != hipSuccess) return fail_status(EAS_HIP_ERR_RUNTIME, hipGetErrorString(e_));           \
  } while (0)

#define OPS_TRY(call)      \
  do {                     \
    const int rc_ = (call); \
    if (rc_) return rc_;   \
  } while (0)

constexpr int kCus = 256;
constexpr int64_t kOneChunk = 1 << 21;  // most elements whose sums over rows are made in one stage
constexpr int64_t kMost = 0x7fffff00;  // rows and columns are 32-bit in the kernels

int elem(int dtype) { return dtype == EAS_HIP_F32 ? 4 : 2; }
bool is_dtype(int d) { return d == EAS_HIP_F16 || d == EAS_HIP_BF16 || d == EAS_HIP_F32; }
bool is_act(int a) { return a >= EAS_HIP_ACT_NONE && a <= EAS_HIP_ACT_SILU; }
bool size_ok(int64_t n) { return n >= 0 && n <= kMost; }
int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }
int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Scratch, laid out the same way when its size is asked for and when it is used.
struct Arena {
  char* base;      // null: only the size is wanted
  uint64_t used = 0;
  void* take(uint64_t bytes) {
    void* p = base ? base + used : nullptr;
    used += (uint64_t)up((int64_t)bytes, 256);
    return p;
  }
};

// A matrix as it lies in memory: rows of `cols` elements
struct Operand {
  const void* p;
  int64_t ld;
  int64_t rows, cols;
  bool along_k;  // its rows run along the reduction
};

// What the DMA takes: rows at any 4 bytes, and for rows along k whole 16-byte chunks of k (of others, what a chunk reads
// past a row's end goes to columns that are not stored).  Offsets within a tile are 32-bit: at up to 4 MB from row to row
// every tile has them (255 rows); rows further apart are copied closer, unless they are as long, when the plan has to
// find a tile that reaches them.
bool direct(const Operand& o, int dtype) {
  const int64_t e = elem(dtype);
  return (uint64_t)o.p % 4 == 0 && o.ld * e % 4 == 0 && (o.ld * e <= (4 << 20) || o.ld <= up(o.cols, 8)) &&
         (!o.along_k || o.cols * e % 16 == 0);
}

// Products of few rows read 16-bit operands that are not direct, or out of a tile's reach, through registers, at any
// alignment and length: a copy would move the weights, all their work, three times.  EAS_HIP_OPS_GEMM's tiles have no such form.
constexpr int64_t kFewRows = 64;
bool few_rows(int64_t m, int dtype) {
  const char* v = getenv("EAS_HIP_OPS_GEMM");
  return m <= kFewRows && dtype != EAS_HIP_F32 && !(v && !strncmp(v, "tile", 4));
}

// An operand that is not direct is copied to aligned rows first.
void realign(PrepareParams& p, Operand& o, int dtype, Arena& ws) {
  if (direct(o, dtype) || o.rows == 0 || o.cols == 0) return;
  const int i = p.copies++;
  p.src[i] = o.p;
  p.src_ld[i] = o.ld;
  p.rows[i] = (int)o.rows;
  p.cols[i] = (int)o.cols;
  p.dst_ld[i] = o.ld = up(o.cols, 8);
  o.p = p.dst[i] = ws.take((uint64_t)(o.rows * o.ld * elem(dtype)));
}

// bytes from row to row, the largest of `count` operands
int64_t row_bytes(const Operand* o, int count, int dtype) {
  int64_t ld = 0;
  for (int i = 0; i < count; ++i) ld = o[i].ld > ld ? o[i].ld : ld;
  return ld * elem(dtype);
}

// Whether two matrices share an element, by their address ranges; matrices of one row stride side by side in the same
// rows (halves of a wider one) do not.
struct Area {
  const void* p;
  int64_t ld, rows, cols;
  int elem;
};
bool shares(const Area& a, const Area& b) {
  if (!a.p || !b.p || !a.rows || !b.rows || !a.cols || !b.cols) return false;
  const char *pa = (const char*)a.p, *pb = (const char*)b.p;
  const int64_t la = ((a.rows - 1) * a.ld + a.cols) * a.elem, lb = ((b.rows - 1) * b.ld + b.cols) * b.elem;
  if (pa + la <= pb || pb + lb <= pa) return false;
  if (a.ld * a.elem != b.ld * b.elem) return true;
  const int64_t row = a.ld * a.elem;
  int64_t d = (pb - pa) % row;
  if (d < 0) d += row;
  return d < a.cols * a.elem || row - d < b.cols * b.elem;
}
bool same(const Area& a, const Area& b) { return a.p == b.p && a.elem == b.elem && (a.ld == b.ld || a.rows <= 1); }
// No output shares memory with another area, but those named as its input in place.
int check_apart(const Area* outs, int n_outs, const Area* ins, int n_ins, const Area* in_place, int n_in_place) {
  for (int i = 0; i < n_outs; ++i) {
    for (int j = i + 1; j < n_outs; ++j) OPS_CHECK(!shares(outs[i], outs[j]), "two outputs share memory");
    for (int j = 0; j < n_ins; ++j) OPS_CHECK(!shares(outs[i], ins[j]), "an output shares memory with an input");
    for (int j = 0; j < n_in_place; ++j)
      OPS_CHECK(!shares(outs[i], in_place[j]) || (i == 0 && same(outs[0], in_place[j])), "an output shares memory with an input");
  }
  return EAS_HIP_OK;
}

// ---- the product's plan -------------------------------------------------------------

// k per stage, rows and columns of a tile (gated: of each of its two halves)
struct GemmTile {
  int bk, bm, bn;
};
struct GemmPlan {
  GemmKernel kernel;
  int splits;
  double ns;  // by the model
};

GemmTile tile_of(GemmKernel k, const GemmForm& f) {
  const int e = elem(f.dtype);
  switch (k) {
    case kGemmTile64: return {128 / e, 64, 64};
    case kGemmTile128: return {128 / e, 128, f.gated ? 64 : 128};
    case kGemmTile256: return {64 / e, 256, f.gated ? 128 : 256};
    default:
      return {skinny_bytes(f.b_outer) / e, k == kGemmSkinny1 ? 16 : k == kGemmSkinny2 ? 32 : 64, skinny_columns(f.b_outer)};
  }
}

GemmKernel few_kernel(int64_t m) { return m <= 16 ? kGemmSkinny1 : m <= 32 ? kGemmSkinny2 : kGemmSkinny4; }

// Whether a tile's offsets reach its rows: those within the operand below the largest range of a buffer, 2^31 - 4 bytes,
// and rows past the end of k, which lie past that range, below 2^32, where the offsets would wrap.
bool reaches(GemmKernel kernel, const GemmForm& f, int64_t m, int64_t n, int64_t k) {
  if (f.any) return true;
  const GemmTile t = tile_of(kernel, f);
  const int64_t e = elem(f.dtype), range = (1ll << 31) - 4, wrap = 1ll << 32;
  auto along = [&](int64_t row, int64_t rows, int64_t high) {  // `high` rows along k, of bk each
    const int64_t last = (rows < high ? rows : high) - 1;
    return last <= 0 || row <= (range - t.bk * e) / last;
  };
  auto across = [&](int64_t row, int64_t wide) {  // bk rows of `wide`
    const int64_t last = (k < t.bk ? k : t.bk) - 1;
    return (last <= 0 || row <= (range - wide * e) / last) && row <= (wrap - wide * e) / (t.bk - 1);
  };
  return (f.a_outer ? across(f.a_row, t.bm) : along(f.a_row, m, t.bm)) && (f.b_outer ? across(f.b_row, t.bn) : along(f.b_row, n, t.bn));
}

// Nanoseconds of a launch by a model of its rounds: workgroups side by side on the card's CUs, a time per k of one
// round and a fixed part, and for a split k the parts' way through memory and the launch that joins them.  The times are
// those of launches of one round over k = 2048 to 14336: a 256 x 256 tile 21.5 ns per k on half the card's CUs and 26 on
// all, 128 x 128 8.3, 64 x 64 4.7 alone on a CU and 7.2 for two (gated 6.2: its ring leaves room for one).
double estimate(GemmKernel kernel, const GemmForm& f, int64_t m, int64_t n, int64_t k, int terms, int prods, int splits) {
  const GemmTile t = tile_of(kernel, f);
  const int64_t tiles = cdiv(m, t.bm) * cdiv(n, t.bn) * prods * splits;
  const double kk = (double)cdiv(cdiv(k, t.bk) * terms, splits) * t.bk;
  const bool f32 = f.dtype == EAS_HIP_F32;
  double ns;
  if (kernel == kGemmTile256) {
    ns = (double)cdiv(tiles, kCus) * (kk * (tiles > kCus * 3 / 4 ? 26 : 21.5) + 6000);
  } else if (kernel == kGemmTile128) {
    ns = (double)cdiv(tiles, kCus) * (kk * (f32 ? 61 : 8.3) + 3000);
  } else if (f.gated) {
    ns = (double)cdiv(tiles, kCus) * (kk * (f32 ? 32 : 6.2) + 2500);
  } else {
    ns = (double)cdiv(tiles, 2 * kCus) * (kk * (tiles <= kCus ? (f32 ? 20 : 4.7) : (f32 ? 34 : 7.2)) + 2500);
  }
  if (splits > 1) ns += 4000 + 2.0 * splits * m * n * prods * (f.gated ? 2 : 1) * 4 / 5000;
  return ns;
}

// EAS_HIP_OPS_GEMM picks the kernel ("tile64", "tile128", "tile256" or "auto") and, after a colon, the ranges that k is
// split into, where they can run the product; for measurements and tests.
bool forced(const GemmForm& f, int64_t k, int terms, GemmPlan* out) {
  const char* v = getenv("EAS_HIP_OPS_GEMM");
  if (!v || !*v) return false;
  GemmKernel kernel;
  if (!strncmp(v, "tile64", 6)) kernel = kGemmTile64;
  else if (!strncmp(v, "tile128", 7)) kernel = kGemmTile128;
  else if (!strncmp(v, "tile256", 7) && f.dtype != EAS_HIP_F32) kernel = kGemmTile256;
  else return false;
  const char* colon = strchr(v, ':');
  const int splits = colon ? atoi(colon + 1) : 1;
  const int64_t stages = cdiv(k > 0 ? k : 1, tile_of(kernel, f).bk) * terms;
  *out = {kernel, splits < 1 ? 1 : splits < stages ? splits : (int)stages, 0.0};
  return true;
}

// Where no kernel reaches the operands, one that `fit` refuses.
GemmPlan plan(const GemmForm& f, int64_t m, int64_t n, int64_t k, int terms, int prods) {
  GemmPlan pick;
  if (forced(f, k, terms, &pick)) return pick;
  if (!f.a_outer && m <= kFewRows && prods == 1 && reaches(few_kernel(m), f, m, n, k)) {
    const GemmKernel kernel = few_kernel(m);
    const GemmTile t = tile_of(kernel, f);
    const int64_t groups = cdiv(n, t.bn), stages = cdiv(k > 0 ? k : 1, t.bk) * terms;
    const int64_t want = kCus;
    int64_t splits = want / groups;
    if (splits > stages / 16) splits = stages / 16;
    if (splits < 1) splits = 1;
    return {kernel, (int)splits, 0.0};
  }
  GemmPlan best{kGemmTile64, 1, 1e300};
  for (int kernel = kGemmTile64; kernel <= kGemmTile256; ++kernel) {
    if ((kernel == kGemmTile256 && f.dtype == EAS_HIP_F32) || !reaches((GemmKernel)kernel, f, m, n, k)) continue;
    for (int s = 1; s <= 16; s *= 2) {
      if (s > 1 && (k * terms / s < 512)) break;
      const double ns = estimate((GemmKernel)kernel, f, m, n, k > 0 ? k : 1, terms, prods, s);
      if (ns < best.ns) best = {(GemmKernel)kernel, s, ns};
    }
  }
  return best;
}

// A few tiles beyond a whole number of rounds cost a round of their own.  The columns to leave to a launch of their own
// then, whose plan fits them: 4096 x 4096 x 4100 in 256 x 256 tiles is 16 of 272 tiles too many for one round (184 us;
// 4096 columns and 4 apart 131).  0: none, one launch is the faster.
int64_t columns_apart(const GemmForm& f, const GemmPlan& whole, int64_t m, int64_t n, int64_t k, int terms, int prods) {
  if (whole.ns == 0.0) return 0;  // few rows, or forced
  int64_t apart = 0;
  double least = whole.ns;
  for (int kernel = kGemmTile64; kernel <= kGemmTile256; ++kernel) {
    if ((kernel == kGemmTile256 && f.dtype == EAS_HIP_F32) || !reaches((GemmKernel)kernel, f, m, n, k)) continue;
    const GemmTile t = tile_of((GemmKernel)kernel, f);
    const int64_t high = cdiv(m, t.bm) * prods, side = kernel == kGemmTile64 && !f.gated ? 2 * kCus : kCus;
    const int64_t rounds = cdiv(high * cdiv(n, t.bn), side);
    if (rounds < 2) continue;
    const int64_t first = (rounds - 1) * side / high * t.bn;
    if (first < 1 || first >= n) continue;
    const double ns = estimate((GemmKernel)kernel, f, m, first, k > 0 ? k : 1, terms, prods, 1) + 3000 +
                      plan(f, m, n - first, k, terms, prods).ns;
    if (ns < 0.97 * least) least = ns, apart = n - first;
  }
  return apart;
}

// The plan's sizes into `p`, and its scratch
int fit(const GemmForm& form, const GemmPlan& g, GemmParams& p, Arena& ws) {
  OPS_CHECK(reaches(g.kernel, form, p.m, p.n, p.k), "an operand's rows are too long: 32-bit offsets do not reach a tile's rows");
  const GemmTile t = tile_of(g.kernel, form);
  p.kt = (int)cdiv(p.k > 0 ? p.k : 1, t.bk);
  p.tiles_m = (int)cdiv(p.m, t.bm);
  p.tiles_n = (int)cdiv(p.n, t.bn);
  p.width = t.bn;
  if (g.kernel <= kGemmSkinny4 && !form.b_outer) {
    // Columns in even shares, so that the last round has work for every CU too: 1 x 4096 x 14336 bf16 20.9 -> 19.9 us,
    // 64 x 4096 x 11008 25.9 -> 23.9, 16 x 5488 x 11119 f32 64.3 -> 59.5.  Not where a row of B crosses the columns: its
    // runs would start inside lines that two workgroups then fetch (1 x 4096 x 11008 20.6 -> 30.3 us).
    const int64_t rounds = cdiv((int64_t)p.tiles_n * g.splits, kCus), groups = rounds * kCus / g.splits;
    const int64_t width = up(cdiv(p.n, groups), 8);
    if (width < t.bn) p.width = (int)width, p.tiles_n = (int)cdiv(p.n, width);
  }
  // ranges of whole stages, none of them empty
  const int64_t total = (int64_t)p.kt * p.segs, per = cdiv(total, g.splits);
  p.splits = (int)cdiv(total, per);
  p.part = nullptr;
  if (p.splits > 1)
    p.part = (float*)ws.take((uint64_t)p.splits * p.prods * p.m * p.n * (form.gated ? 2 : 1) * sizeof(float));
  const int64_t threads = (int64_t)p.tiles_m * p.tiles_n * (g.kernel <= kGemmSkinny4 ? 256 : 512);
  OPS_CHECK(threads < (1ll << 32) && (int64_t)p.prods * p.splits < 65536, "the product has too many tiles");  // for a grid
  return EAS_HIP_OK;
}

int join(const GemmForm& form, const GemmParams& p, hipStream_t stream) {
  if (p.splits < 2) return EAS_HIP_OK;
  if (form.dtype == EAS_HIP_F16) OPS_HIP(gemm_join_typed<f16>(form.gated, p, stream));
  else if (form.dtype == EAS_HIP_BF16) OPS_HIP(gemm_join_typed<bf16>(form.gated, p, stream));
  else OPS_HIP(gemm_join_typed<float>(form.gated, p, stream));
  return EAS_HIP_OK;
}

int run_planned(const GemmForm& form, const GemmPlan& g, GemmParams p, Arena& ws, bool launch, hipStream_t stream) {
  OPS_TRY(fit(form, g, p, ws));
  if (!launch) return EAS_HIP_OK;
  if (form.dtype == EAS_HIP_F16) OPS_HIP(gemm_launch_typed<f16>(g.kernel, form, p, stream));
  else if (form.dtype == EAS_HIP_BF16) OPS_HIP(gemm_launch_typed<bf16>(g.kernel, form, p, stream));
  else OPS_HIP(gemm_launch_typed<float>(g.kernel, form, p, stream));
  return join(form, p, stream);
}

// Whether dx and dW are faster as one launch of 64 x 64 tiles, and then the ranges of dx's k: by the same times per k and
// fixed parts, every CU with two tiles at a time until they are used up.  0: no.
int pair_splits(const GemmForm& fx, const GemmParams& x, const GemmForm& fw, const GemmParams& w) {
  const GemmPlan gx = plan(fx, x.m, x.n, x.k, x.segs, x.prods), gw = plan(fw, w.m, w.n, w.k, w.segs, w.prods);
  if (fx.any || gx.ns == 0.0 || gw.ns == 0.0 || x.k == 0 || w.k == 0) return 0;  // few rows, forced, or nothing to sum
  if (!reaches(kGemmTile64, fx, x.m, x.n, x.k) || !reaches(kGemmTile64, fw, w.m, w.n, w.k)) return 0;
  if (columns_apart(fx, gx, x.m, x.n, x.k, x.segs, x.prods) || columns_apart(fw, gw, w.m, w.n, w.k, w.segs, w.prods)) return 0;
  const double alone = fx.dtype == EAS_HIP_F32 ? 20 : 4.7, two = fx.dtype == EAS_HIP_F32 ? 34 : 7.2;
  // a tile's prologue and epilogue beside another tile's k: 512 x 2048 x 1024 bf16 23.5 us by 2500 and 20.9 by 1200, f32 400 x
  // 400 x 3000 41 and 48
  const double fixed = fx.dtype == EAS_HIP_F32 ? 2500 : 1200;
  const GemmTile t = tile_of(kGemmTile64, fx);
  const int64_t wide = cdiv(x.m, t.bm) * cdiv(x.n, t.bn), rest = cdiv(w.m, t.bm) * cdiv(w.n, t.bn) * w.prods;
  const int64_t stages = cdiv(x.k, t.bk) * x.segs;
  const double kw = (double)cdiv(w.k, t.bk) * t.bk;
  if (wide * 16 + rest > (1 << 20)) return 0;
  double best = 0.95 * (gx.ns + gw.ns);
  int pick = 0;
  for (int s = 1; s <= 16 && s <= stages; ++s) {
    if (s > 1 && x.k * x.segs / s < 256) break;
    const double kx = (double)cdiv(stages, s) * t.bk, least = kx < kw ? kx : kw, most = kx < kw ? kw : kx;
    double ns = most * alone + 2500;
    if (wide * s + rest > kCus) {
      ns = (wide * s * (kx * two + fixed) + rest * (kw * two + fixed)) / (2 * kCus) + least * two / 2;
      if (ns < most * two + 2500) ns = most * two + 2500;
    }
    if (s > 1) ns += 4000 + 2.0 * s * x.m * x.n * 4 / 5000;
    if (ns < best) best = ns, pick = s;
  }
  return pick;
}

int run_pair(const GemmForm& fx, GemmParams x, int splits, const GemmForm& fw, GemmParams w, Arena& ws, bool launch, hipStream_t stream) {
  OPS_TRY(fit(fx, {kGemmTile64, splits, 0.0}, x, ws));
  OPS_TRY(fit(fw, {kGemmTile64, 1, 0.0}, w, ws));
  if (!launch) return EAS_HIP_OK;
  if (fx.dtype == EAS_HIP_F16) OPS_HIP(gemm_pair_typed<f16>(fx.b_outer, x, w, stream));
  else if (fx.dtype == EAS_HIP_BF16) OPS_HIP(gemm_pair_typed<bf16>(fx.b_outer, x, w, stream));
  else OPS_HIP(gemm_pair_typed<float>(fx.b_outer, x, w, stream));
  return join(fx, x, stream);
}

// Plans `p` (m, n, k, segs, prods and the operands are set), takes its scratch, and launches it.
int run_gemm(const GemmForm& form, const GemmParams& p, Arena& ws, bool launch, hipStream_t stream) {
  if (p.m == 0 || p.n == 0) return EAS_HIP_OK;
  const GemmPlan g = plan(form, p.m, p.n, p.k, p.segs, p.prods);
  const int64_t apart = columns_apart(form, g, p.m, p.n, p.k, p.segs, p.prods);
  if (!apart) return run_planned(form, g, p, ws, launch, stream);
  GemmParams first = p, rest = p;
  const int64_t n = p.n - apart, e = elem(form.dtype), ce = p.wide ? 4 : e;
  first.n = (int)n;
  rest.n = (int)apart;
  auto on = [](const void* q, int64_t bytes) { return q ? (char*)q + bytes : nullptr; };
  for (int i = 0; i < 2; ++i) {
    rest.b[i] = on(p.b[i], n * (form.b_outer ? 1 : p.ldb[i]) * e);
    rest.c[i] = on(p.c[i], n * ce);
    rest.pre[i] = on(p.pre[i], n * ce);
    rest.bias[i] = on(p.bias[i], n * e);
  }
  rest.res = on(p.res, n * ce);
  OPS_TRY(run_planned(form, plan(form, first.m, first.n, first.k, first.segs, first.prods), first, ws, launch, stream));
  return run_planned(form, plan(form, rest.m, rest.n, rest.k, rest.segs, rest.prods), rest, ws, launch, stream);
}

template <typename Args> int read_args(const Args* args, size_t size, Args* out) {
  OPS_CHECK(args != nullptr, "args must not be NULL");
  OPS_CHECK(size == sizeof(Args), "args_size is not this operator's");
  memcpy(out, args, sizeof(Args));
  return EAS_HIP_OK;
}

int check_workspace(const void* ws, uint64_t bytes, uint64_t need) {
  OPS_CHECK(need == 0 || (ws != nullptr && (uint64_t)ws % 16 == 0), "the workspace must be 16-byte aligned device memory");
  OPS_CHECK(bytes >= need, "the workspace is too small");
  return EAS_HIP_OK;
}

// ---- linear -------------------------------------------------------------------------

int check_linear(const eas_hip_linear_args& a) {
  OPS_CHECK(is_dtype(a.dtype) && (a.ydtype == a.dtype || a.ydtype == EAS_HIP_F32), "unsupported dtype");
  OPS_CHECK(is_act(a.activation), "unknown activation");
  OPS_CHECK(a.w_trans == 0 || a.w_trans == 1, "w_trans must be 0 or 1");
  OPS_CHECK(size_ok(a.m) && size_ok(a.k) && size_ok(a.n), "sizes must be in [0, 2^31 - 256]");
  OPS_CHECK(a.x_ld >= a.k && a.w_ld >= (a.w_trans ? a.k : a.n) && a.y_ld >= a.n && (!a.residual || a.residual_ld >= a.n) &&
                (!a.pre || a.pre_ld >= a.n),
            "a row stride is shorter than the row");
  const bool out = a.m && a.n;
  OPS_CHECK(!out || a.y, "y must not be NULL");
  OPS_CHECK(!out || !a.k || (a.x && a.w), "x and w must not be NULL");
  const int e = elem(a.dtype), ye = elem(a.ydtype);
  const Area outs[] = {{a.y, a.y_ld, a.m, a.n, ye}, {a.pre, a.pre_ld, a.m, a.n, ye}};
  const Area ins[] = {{a.x, a.x_ld, a.m, a.k, e}, {a.w, a.w_ld, a.w_trans ? a.n : a.k, a.w_trans ? a.k : a.n, e}, {a.bias, a.n, 1, a.n, e}};
  const Area in_place[] = {{a.residual, a.residual_ld, a.m, a.n, ye}};
  return check_apart(outs, 2, ins, 3, in_place, 1);
}

int linear(const eas_hip_linear_args& a, Arena& ws, bool launch, hipStream_t stream) {
  if (!a.m || !a.n) return EAS_HIP_OK;
  GemmForm form{a.dtype, false, !a.w_trans, false, false};
  Operand x{a.x, a.x_ld, a.m, a.k, true};
  Operand w{a.w, a.w_ld, a.w_trans ? a.n : a.k, a.w_trans ? a.k : a.n, a.w_trans != 0};
  form.a_row = row_bytes(&x, 1, a.dtype);
  form.b_row = row_bytes(&w, 1, a.dtype);
  form.any = few_rows(a.m, a.dtype) && !(direct(x, a.dtype) && direct(w, a.dtype) && reaches(few_kernel(a.m), form, a.m, a.n, a.k));
  PrepareParams before{};
  before.dtype = a.dtype;
  if (!form.any) {
    realign(before, x, a.dtype, ws);
    realign(before, w, a.dtype, ws);
    form.a_row = row_bytes(&x, 1, a.dtype);
    form.b_row = row_bytes(&w, 1, a.dtype);
  }
  if (launch) OPS_HIP(prepare_launch(before, stream));
  GemmParams p{};
  p.a[0] = x.p;
  p.lda[0] = x.ld;
  p.b[0] = w.p;
  p.ldb[0] = w.ld;
  p.c[0] = a.y;
  p.ldc[0] = a.y_ld;
  p.pre[0] = a.pre;
  p.ldpre[0] = a.pre_ld;
  p.bias[0] = a.bias;
  p.res = a.residual;
  p.ldres = a.residual_ld;
  p.m = (int)a.m;
  p.n = (int)a.n;
  p.k = (int)a.k;
  p.segs = p.prods = 1;
  p.act = a.activation;
  p.wide = a.ydtype == EAS_HIP_F32;
  return run_gemm(form, p, ws, launch, stream);
}

// ---- gated linear ---------------------------------------------------------------------

int check_gated(const eas_hip_gated_linear_args& a) {
  OPS_CHECK(is_dtype(a.dtype) && (a.ydtype == a.dtype || a.ydtype == EAS_HIP_F32), "unsupported dtype");
  OPS_CHECK(is_act(a.activation), "unknown activation");
  OPS_CHECK(a.w_trans == 0 || a.w_trans == 1, "w_trans must be 0 or 1");
  OPS_CHECK(size_ok(a.m) && size_ok(a.k) && size_ok(a.n), "sizes must be in [0, 2^31 - 256]");
  const int64_t wl = a.w_trans ? a.k : a.n;
  OPS_CHECK(a.x_ld >= a.k && a.w_gate_ld >= wl && a.w_up_ld >= wl && a.y_ld >= a.n &&
                (!a.gate || (a.gate_ld >= a.n && a.up_ld >= a.n)),
            "a row stride is shorter than the row");
  OPS_CHECK(!a.gate == !a.up, "gate and up go together");
  const bool out = a.m && a.n;
  OPS_CHECK(!out || a.y, "y must not be NULL");
  OPS_CHECK(!out || !a.k || (a.x && a.w_gate && a.w_up), "x, w_gate and w_up must not be NULL");
  const int e = elem(a.dtype), ye = elem(a.ydtype);
  const int64_t wr = a.w_trans ? a.n : a.k;
  const Area outs[] = {{a.y, a.y_ld, a.m, a.n, ye}, {a.gate, a.gate_ld, a.m, a.n, ye}, {a.up, a.up_ld, a.m, a.n, ye}};
  const Area ins[] = {{a.x, a.x_ld, a.m, a.k, e}, {a.w_gate, a.w_gate_ld, wr, wl, e}, {a.w_up, a.w_up_ld, wr, wl, e},
                      {a.bias_gate, a.n, 1, a.n, e}, {a.bias_up, a.n, 1, a.n, e}};
  return check_apart(outs, 3, ins, 5, nullptr, 0);
}

int gated(const eas_hip_gated_linear_args& a, Arena& ws, bool launch, hipStream_t stream) {
  if (!a.m || !a.n) return EAS_HIP_OK;
  GemmForm form{a.dtype, false, !a.w_trans, true, false};
  const int64_t rows = a.w_trans ? a.n : a.k, cols = a.w_trans ? a.k : a.n;
  Operand x{a.x, a.x_ld, a.m, a.k, true};
  Operand w[] = {{a.w_gate, a.w_gate_ld, rows, cols, a.w_trans != 0}, {a.w_up, a.w_up_ld, rows, cols, a.w_trans != 0}};
  form.a_row = row_bytes(&x, 1, a.dtype);
  form.b_row = row_bytes(w, 2, a.dtype);
  form.any = few_rows(a.m, a.dtype) && !(direct(x, a.dtype) && direct(w[0], a.dtype) && direct(w[1], a.dtype) &&
                                         reaches(few_kernel(a.m), form, a.m, a.n, a.k));
  PrepareParams before{};
  before.dtype = a.dtype;
  if (!form.any) {
    realign(before, x, a.dtype, ws);
    realign(before, w[0], a.dtype, ws);
    realign(before, w[1], a.dtype, ws);
    form.a_row = row_bytes(&x, 1, a.dtype);
    form.b_row = row_bytes(w, 2, a.dtype);
  }
  if (launch) OPS_HIP(prepare_launch(before, stream));
  GemmParams p{};
  p.a[0] = x.p;
  p.lda[0] = x.ld;
  p.b[0] = w[0].p;
  p.b[1] = w[1].p;
  p.ldb[0] = w[0].ld;
  p.ldb[1] = w[1].ld;
  p.c[0] = a.y;
  p.ldc[0] = a.y_ld;
  p.pre[0] = a.gate;
  p.pre[1] = a.up;
  p.ldpre[0] = a.gate_ld;
  p.ldpre[1] = a.up_ld;
  p.bias[0] = a.bias_gate;
  p.bias[1] = a.bias_up;
  p.m = (int)a.m;
  p.n = (int)a.n;
  p.k = (int)a.k;
  p.segs = p.prods = 1;
  p.act = a.activation;
  p.wide = a.ydtype == EAS_HIP_F32;
  return run_gemm(form, p, ws, launch, stream);
}

// ---- gradients ------------------------------------------------------------------------

// What linear's and gated_linear's gradients have in common: `terms` pairs of weights and of dz.
struct Backward {
  const void *dy, *x, *w[2], *pre[2];
  void *dx, *dw[2], *dbias[2];
  int64_t m, k, n, dy_ld, x_ld, w_ld[2], pre_ld[2], dx_ld, dw_ld[2];
  int dtype, wdtype, act;
  bool w_trans, gated;
};

int check_backward(const Backward& b) {
  const int terms = b.gated ? 2 : 1;
  OPS_CHECK(is_dtype(b.dtype) && (b.wdtype == b.dtype || b.wdtype == EAS_HIP_F32), "unsupported dtype");
  OPS_CHECK(is_act(b.act), "unknown activation");
  OPS_CHECK(size_ok(b.m) && size_ok(b.k) && size_ok(b.n), "sizes must be in [0, 2^31 - 256]");
  const int64_t wl = b.w_trans ? b.k : b.n;
  const bool pre = b.gated || b.act != EAS_HIP_ACT_NONE;
  OPS_CHECK(b.dy_ld >= b.n && (!b.dw[0] || b.x_ld >= b.k) && (!b.dx || b.dx_ld >= b.k), "a row stride is shorter than the row");
  for (int i = 0; i < terms; ++i)
    OPS_CHECK((!b.dx || b.w_ld[i] >= wl) && (!b.dw[0] || b.dw_ld[i] >= wl) && (!pre || b.pre_ld[i] >= b.n),
              "a row stride is shorter than the row");
  OPS_CHECK(!b.gated || (!b.dw[0] == !b.dw[1] && !b.dbias[0] == !b.dbias[1]), "the gradients of gate and up go together");
  if (b.m && b.n) {
    OPS_CHECK(b.dy, "dy must not be NULL");
    OPS_CHECK(!pre || (b.pre[0] && (!b.gated || b.pre[1])), "the activation's input must not be NULL");
    OPS_CHECK(!b.dw[0] || !b.k || b.x, "x must not be NULL");
    OPS_CHECK(!b.dx || !b.k || (b.w[0] && (!b.gated || b.w[1])), "w must not be NULL");
  }
  const int e = elem(b.dtype), we = elem(b.wdtype);
  const int64_t wr = b.w_trans ? b.n : b.k;
  const Area outs[] = {{b.dx, b.dx_ld, b.m, b.k, e}, {b.dw[0], b.dw_ld[0], wr, wl, we}, {b.dw[1], b.dw_ld[1], wr, wl, we},
                       {b.dbias[0], b.n, 1, b.n, we}, {b.dbias[1], b.n, 1, b.n, we}};
  const Area ins[] = {{b.dy, b.dy_ld, b.m, b.n, e}, {b.x, b.x_ld, b.m, b.k, e}, {b.w[0], b.w_ld[0], wr, wl, e}, {b.w[1], b.w_ld[1], wr, wl, e},
                      {pre ? b.pre[0] : nullptr, b.pre_ld[0], b.m, b.n, e}, {b.pre[1], b.pre_ld[1], b.m, b.n, e}};
  return check_apart(outs, 5, ins, 6, nullptr, 0);
}

int backward(const Backward& b, Arena& ws, bool launch, hipStream_t stream) {
  const int terms = b.gated ? 2 : 1;
  const bool products = b.k && (b.dx || b.dw[0]);
  const bool pre = b.gated || b.act != EAS_HIP_ACT_NONE;
  if (!products && !(b.dbias[0] && b.n)) return EAS_HIP_OK;
  PrepareParams d{};
  d.dy = b.dy;
  d.dy_ld = b.dy_ld;
  d.m = (int)b.m;
  d.n = (int)b.n;
  d.act = b.act;
  d.dtype = b.dtype;
  d.gated = b.gated;
  d.sum_wide = b.wdtype == EAS_HIP_F32;
  // what dz is taken from goes past the caches where it and dz would fill half of the memory-side one (256 MB): gated
  // 2048x14336 bf16 62 -> 53 us, 4096x8192 43 -> 41; not for less: 4096x4096 22.4 either way, 512x4096 gated 10.3 -> 11.8
  d.stream = b.m * b.n * elem(b.dtype) * (b.gated ? 5 : 3) > (128 << 20);
  // dz, as rows along n: for dx its rows run along the reduction, for dw across it
  Operand dz[2];
  for (int i = 0; i < terms; ++i) {
    dz[i] = {b.dy, b.dy_ld, b.m, b.n, true};
    d.pre[i] = pre ? b.pre[i] : nullptr;
    d.pre_ld[i] = b.pre_ld[i];
  }
  const bool write_dz = pre && products && b.m && b.n, sums = b.dbias[0] && b.n;
  if (write_dz) {
    d.dz_ld = up(b.n, 8);
    for (int i = 0; i < terms; ++i) {
      d.dz[i] = ws.take((uint64_t)(b.m * d.dz_ld * elem(b.dtype)));
      dz[i].p = d.dz[i];
      dz[i].ld = d.dz_ld;
    }
  } else if (products) {
    realign(d, dz[0], b.dtype, ws);
  }
  if (sums || write_dz) {
    const int64_t vecs = cdiv(b.n, 8), rows = b.m > 0 ? b.m : 1;
    int64_t chunks;
    if (sums && rows * b.n <= kOneChunk) {
      // few elements: all rows in one chunk, whose sums are the result, on narrow strips of columns
      d.tx = 64;
      while (d.tx > 1 && cdiv(vecs, d.tx) < kCus) d.tx /= 2;
      chunks = 1;
    } else {
      d.tx = 64;
      while (d.tx > 8 && d.tx / 2 >= vecs) d.tx /= 2;
      // about 1024 workgroups of at least 8 rows
      chunks = cdiv(1024, cdiv(vecs, d.tx));
      if (chunks > cdiv(rows, 8)) chunks = cdiv(rows, 8);
    }
    d.across = (int)cdiv(vecs, d.tx);
    if (chunks == 1) d.across = (int)up(d.across, 8);  // one run of strips for each XCD
    d.rows_per_chunk = (int)cdiv(rows, chunks);
    d.chunks = (int)cdiv(rows, d.rows_per_chunk);
    if (sums && d.chunks > 1) d.part = (float*)ws.take((uint64_t)d.chunks * terms * b.n * sizeof(float));
    if (sums && d.chunks == 1)
      for (int i = 0; i < terms; ++i) d.sum[i] = b.dbias[i];
  }
  Operand x{b.x, b.x_ld, b.m, b.k, false}, w[2];
  if (b.dw[0] && b.k && b.n) realign(d, x, b.dtype, ws);
  // dx [m, k] = sum of dz [m, n] w^T [n, k], and dw [k, n] = x^T [k, m] dz [m, n] or its transpose
  GemmForm fx{b.dtype, false, b.w_trans, false, false}, fw{b.dtype, true, true, false, false};
  if (b.dx && b.k) {
    bool as_they_are = true;  // dz's rows are aligned, but may end within 16 bytes of k
    for (int i = 0; i < terms; ++i) {
      w[i] = {b.w[i], b.w_ld[i], b.w_trans ? b.n : b.k, b.w_trans ? b.k : b.n, !b.w_trans};
      as_they_are = as_they_are && direct(w[i], b.dtype);
    }
    fx.a_row = row_bytes(dz, terms, b.dtype);
    fx.b_row = row_bytes(w, terms, b.dtype);
    fx.any = few_rows(b.m, b.dtype) && !(as_they_are && reaches(few_kernel(b.m), fx, b.m, b.k, b.n));
    for (int i = 0; i < terms && !fx.any; ++i) realign(d, w[i], b.dtype, ws);
    fx.b_row = row_bytes(w, terms, b.dtype);
  }
  fw.a_row = b.w_trans ? row_bytes(dz, terms, b.dtype) : row_bytes(&x, 1, b.dtype);
  fw.b_row = b.w_trans ? row_bytes(&x, 1, b.dtype) : row_bytes(dz, terms, b.dtype);
  if (launch) {
    OPS_HIP(prepare_launch(d, stream));
    if (d.part) {
      ColumnSumParams c{};
      c.part = d.part;
      for (int i = 0; i < terms; ++i) c.out[i] = b.dbias[i];
      c.n = (int)b.n;
      c.outs = terms;
      c.chunks = d.chunks;
      c.dtype = b.wdtype;
      OPS_HIP(column_sum_launch(c, stream));
    }
  }
  if (!b.k) return EAS_HIP_OK;
  const bool dx = b.dx && b.m, dw = b.dw[0] && b.n;
  GemmParams px{}, pw{};
  for (int i = 0; i < terms && dx; ++i) {
    px.a[i] = dz[i].p;
    px.lda[i] = dz[i].ld;
    px.b[i] = w[i].p;
    px.ldb[i] = w[i].ld;
  }
  px.c[0] = b.dx;
  px.ldc[0] = b.dx_ld;
  px.m = (int)b.m;
  px.n = (int)b.k;
  px.k = (int)b.n;
  px.segs = terms;
  px.prods = 1;
  for (int i = 0; i < terms; ++i) {
    const Operand &a = b.w_trans ? dz[i] : x, &c = b.w_trans ? x : dz[i];
    pw.a[i] = a.p;
    pw.lda[i] = a.ld;
    pw.b[i] = c.p;
    pw.ldb[i] = c.ld;
    pw.c[i] = b.dw[i];
    pw.ldc[i] = b.dw_ld[i];
  }
  pw.m = (int)(b.w_trans ? b.n : b.k);
  pw.n = (int)(b.w_trans ? b.k : b.n);
  pw.k = (int)b.m;
  pw.segs = 1;
  pw.prods = terms;
  pw.wide = b.wdtype == EAS_HIP_F32;
  const int pair = dx && dw ? pair_splits(fx, px, fw, pw) : 0;
  if (pair) return run_pair(fx, px, pair, fw, pw, ws, launch, stream);
  if (dx) OPS_TRY(run_gemm(fx, px, ws, launch, stream));
  if (dw) OPS_TRY(run_gemm(fw, pw, ws, launch, stream));
  return EAS_HIP_OK;
}

Backward of(const eas_hip_linear_backward_args& a) {
  Backward b{};
  b.dy = a.dy;
  b.x = a.x;
  b.w[0] = a.w;
  b.pre[0] = a.pre;
  b.dx = a.dx;
  b.dw[0] = a.dw;
  b.dbias[0] = a.dbias;
  b.m = a.m;
  b.k = a.k;
  b.n = a.n;
  b.dy_ld = a.dy_ld;
  b.x_ld = a.x_ld;
  b.w_ld[0] = a.w_ld;
  b.pre_ld[0] = a.pre_ld;
  b.dx_ld = a.dx_ld;
  b.dw_ld[0] = a.dw_ld;
  b.dtype = a.dtype;
  b.wdtype = a.wdtype;
  b.act = a.activation;
  b.w_trans = a.w_trans != 0;
  return b;
}

Backward of(const eas_hip_gated_linear_backward_args& a) {
  Backward b{};
  b.dy = a.dy;
  b.x = a.x;
  b.w[0] = a.w_gate;
  b.w[1] = a.w_up;
  b.pre[0] = a.gate;
  b.pre[1] = a.up;
  b.dx = a.dx;
  b.dw[0] = a.dw_gate;
  b.dw[1] = a.dw_up;
  b.dbias[0] = a.dbias_gate;
  b.dbias[1] = a.dbias_up;
  b.m = a.m;
  b.k = a.k;
  b.n = a.n;
  b.dy_ld = a.dy_ld;
  b.x_ld = a.x_ld;
  b.w_ld[0] = a.w_gate_ld;
  b.w_ld[1] = a.w_up_ld;
  b.pre_ld[0] = a.gate_ld;
  b.pre_ld[1] = a.up_ld;
  b.dx_ld = a.dx_ld;
  b.dw_ld[0] = a.dw_gate_ld;
  b.dw_ld[1] = a.dw_up_ld;
  b.dtype = a.dtype;
  b.wdtype = a.wdtype;
  b.act = a.activation;
  b.w_trans = a.w_trans != 0;
  b.gated = true;
  return b;
}

int check(const eas_hip_linear_args& a) { return check_linear(a); }
int check(const eas_hip_gated_linear_args& a) { return check_gated(a); }
int check(const eas_hip_linear_backward_args& a) { return check_backward(of(a)); }
int check(const eas_hip_gated_linear_backward_args& a) { return check_backward(of(a)); }
int work(const eas_hip_linear_args& a, Arena& ws, bool launch, hipStream_t s) { return linear(a, ws, launch, s); }
int work(const eas_hip_gated_linear_args& a, Arena& ws, bool launch, hipStream_t s) { return gated(a, ws, launch, s); }
int work(const eas_hip_linear_backward_args& a, Arena& ws, bool launch, hipStream_t s) { return backward(of(a), ws, launch, s); }
int work(const eas_hip_gated_linear_backward_args& a, Arena& ws, bool launch, hipStream_t s) { return backward(of(a), ws, launch, s); }

template <typename Args> int workspace_of(const Args* args, size_t size, uint64_t* bytes) {
  Args a;
  OPS_TRY(read_args(args, size, &a));
  OPS_CHECK(bytes != nullptr, "bytes must not be NULL");
  OPS_TRY(check(a));
  Arena ws{nullptr};
  OPS_TRY(work(a, ws, false, nullptr));
  *bytes = ws.used;
  return EAS_HIP_OK;
}

template <typename Args> int run(const Args* args, size_t size, void* stream) {
  Args a;
  OPS_TRY(read_args(args, size, &a));
  OPS_TRY(check(a));
  Arena count{nullptr};
  OPS_TRY(work(a, count, false, nullptr));
  OPS_TRY(check_workspace(a.workspace, a.workspace_bytes, count.used));
  Arena ws{(char*)a.workspace};
  return work(a, ws, true, (hipStream_t)stream);
}

// ---- layer norm -----------------------------------------------------------------------

int check_norm_backward(const eas_hip_layer_norm_backward_args& a) {
  OPS_CHECK(is_dtype(a.dtype) && (a.wdtype == a.dtype || a.wdtype == EAS_HIP_F32), "unsupported dtype");
  OPS_CHECK(size_ok(a.m) && a.n > 0 && a.n <= kMost, "rows must hold at least one element, and sizes be at most 2^31 - 256");
  OPS_CHECK(a.dy_ld >= a.n && a.x_ld >= a.n && (!a.dx || a.dx_ld >= a.n), "a row stride is shorter than the row");
  OPS_CHECK(!a.m || (a.dy && a.x && a.mean && a.rstd), "dy, x, mean and rstd must not be NULL");
  const int e = elem(a.dtype), we = elem(a.wdtype);
  const Area outs[] = {{a.dx, a.dx_ld, a.m, a.n, e}, {a.dweight, a.n, 1, a.n, we}, {a.dbias, a.n, 1, a.n, we}};
  const Area ins[] = {{a.weight, a.n, 1, a.n, we}, {a.mean, a.m, 1, a.m, 4}, {a.rstd, a.m, 1, a.m, 4}};
  const Area in_place[] = {{a.dy, a.dy_ld, a.m, a.n, e}, {a.x, a.x_ld, a.m, a.n, e}};
  return check_apart(outs, 3, ins, 3, in_place, 2);
}
uint64_t norm_backward_bytes(const eas_hip_layer_norm_backward_args& a, int* chunks) {
  *chunks = layer_norm_backward_chunks(a);
  return a.dweight || a.dbias ? (uint64_t)*chunks * 2 * (uint64_t)a.n * sizeof(float) : 0;
}

}  // namespace
}  // namespace eas

using namespace eas;

extern "C" {

int eas_hip_layer_norm(const eas_hip_layer_norm_args* args, size_t args_size, void* stream) {
  eas_hip_layer_norm_args a;
  OPS_TRY(read_args(args, args_size, &a));
  OPS_CHECK(is_dtype(a.dtype) && (a.wdtype == a.dtype || a.wdtype == EAS_HIP_F32), "unsupported dtype");
  OPS_CHECK(size_ok(a.m) && a.n > 0 && a.n <= kMost, "rows must hold at least one element, and sizes be at most 2^31 - 256");
  OPS_CHECK(a.x_ld >= a.n && a.y_ld >= a.n, "a row stride is shorter than the row");
  OPS_CHECK(a.eps >= 0.0f, "eps must be >= 0");
  if (!a.m) return EAS_HIP_OK;
  OPS_CHECK(a.x && a.y, "x and y must not be NULL");
  const int e = elem(a.dtype), we = elem(a.wdtype);
  const Area outs[] = {{a.y, a.y_ld, a.m, a.n, e}, {a.mean, a.m, 1, a.m, 4}, {a.rstd, a.m, 1, a.m, 4}};
  const Area ins[] = {{a.weight, a.n, 1, a.n, we}, {a.bias, a.n, 1, a.n, we}};
  const Area in_place[] = {{a.x, a.x_ld, a.m, a.n, e}};
  OPS_TRY(check_apart(outs, 3, ins, 2, in_place, 1));
  OPS_HIP(layer_norm_launch(a, (hipStream_t)stream));
  return EAS_HIP_OK;
}

int eas_hip_layer_norm_backward_workspace(const eas_hip_layer_norm_backward_args* args, size_t args_size, uint64_t* bytes) {
  eas_hip_layer_norm_backward_args a;
  OPS_TRY(read_args(args, args_size, &a));
  OPS_CHECK(bytes != nullptr, "bytes must not be NULL");
  OPS_TRY(check_norm_backward(a));
  int chunks;
  *bytes = norm_backward_bytes(a, &chunks);
  return EAS_HIP_OK;
}

int eas_hip_layer_norm_backward(const eas_hip_layer_norm_backward_args* args, size_t args_size, void* stream) {
  eas_hip_layer_norm_backward_args a;
  OPS_TRY(read_args(args, args_size, &a));
  OPS_TRY(check_norm_backward(a));
  int chunks;
  const uint64_t need = norm_backward_bytes(a, &chunks);
  OPS_TRY(check_workspace(a.workspace, a.workspace_bytes, need));
  float* part = a.dweight || a.dbias ? (float*)a.workspace : nullptr;  // null with no rows: no chunk is read
  if (a.m && (a.dx || part)) OPS_HIP(layer_norm_backward_launch(a, part, chunks, (hipStream_t)stream));
  if (a.dweight || a.dbias) {
    ColumnSumParams c{};
    c.part = part;
    c.out[0] = a.dweight;
    c.out[1] = a.dbias;
    c.n = (int)a.n;
    c.outs = 2;
    c.chunks = chunks;
    c.dtype = a.wdtype;
    OPS_HIP(column_sum_launch(c, (hipStream_t)stream));
  }
  return EAS_HIP_OK;
}

#define EAS_OP(name)                                                                                                 \
  int eas_hip_##name##_workspace(const eas_hip_##name##_args* args, size_t args_size, uint64_t* bytes) {             \
    return workspace_of(args, args_size, bytes);                                                                     \
  }                                                                                                                  \
  int eas_hip_##name(const eas_hip_##name##_args* args, size_t args_size, void* stream) { return run(args, args_size, stream); }
EAS_OP(linear)
EAS_OP(linear_backward)
EAS_OP(gated_linear)
EAS_OP(gated_linear_backward)

}  // extern "C"
