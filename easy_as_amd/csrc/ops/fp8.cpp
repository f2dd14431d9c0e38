// fp8.cpp — the entry points around 8-bit operands: the root-mean-square norm, the conversion and the product.
#include <cstdlib>

#include "host.h"

namespace eas {
namespace {

constexpr int kBlock = 128;
constexpr int64_t kFar = 1ll << 40;  // longest stride of a scale: offsets in 64 bits

// The area of a matrix of scales at any two strides of at least 0; beyond 2^58 elements, more than any memory, that many
Area scale_area(const void* p, int64_t rows, int64_t row, int64_t cols, int64_t col) {
  constexpr int64_t most = 1ll << 58;
  const __int128 all = rows && cols ? (__int128)(rows - 1) * row + (__int128)(cols - 1) * col + 1 : 0;
  const int64_t n = all < most ? (int64_t)all : most;
  return {p, n, 1, n, 4};
}
// Whether they are written each to a place of its own: along one stride of 1, lines apart by the other
bool scale_lines(int64_t rows, int64_t row, int64_t cols, int64_t col) {
  if (row < 0 || col < 0 || row > kFar || col > kFar) return false;
  return ((col == 1 || cols <= 1) && (row >= cols || rows <= 1)) || ((row == 1 || rows <= 1) && (col >= rows || cols <= 1));
}
// No output shares memory with another area, but the first two (or one) with those that are read in their place.
int check_places(const Area* outs, int n_outs, int n_over, const Area* ins, int n_ins, const Area* in_place, int n_in_place) {
  OPS_TRY(check_apart(outs, n_outs, ins, n_ins, nullptr, 0));
  for (int i = 0; i < n_outs; ++i)
    for (int j = 0; j < n_in_place; ++j)
      OPS_CHECK(!shares(outs[i], in_place[j]) || (i < n_over && same(outs[i], in_place[j])), "an output shares memory with an input");
  return EAS_HIP_OK;
}

// ---- root-mean-square norm ----------------------------------------------------------------

int check_rms(const eas_hip_rms_norm_args& a) {
  OPS_CHECK(is_dtype(a.dtype) && (a.wdtype == a.dtype || a.wdtype == EAS_HIP_F32) && (a.hdtype == a.dtype || a.hdtype == EAS_HIP_F32),
            "unsupported dtype");
  OPS_CHECK(size_ok(a.m) && a.n > 0 && a.n <= kMost, "rows must hold at least one element, and sizes be at most 2^31 - 256");
  OPS_CHECK(a.x_ld >= a.n && (!a.y || a.y_ld >= a.n) && (!a.residual || a.residual_ld >= a.n) && (!a.total || a.total_ld >= a.n) &&
                (!a.q || a.q_ld >= a.n),
            "a row stride is shorter than the row");
  OPS_CHECK(a.eps >= 0.0f, "eps must be >= 0");
  OPS_CHECK(!a.q == !a.q_scale, "q and q_scale go together");
  const int64_t blocks = cdiv(a.n, kBlock);
  OPS_CHECK(!a.q || scale_lines(a.m, a.q_scale_row, blocks, a.q_scale_block), "the scales must lie in lines that do not overlap");
  OPS_CHECK(!a.m || (a.x && (a.y || a.q)), "x, and y or q, must not be NULL");
  const int e = elem(a.dtype), we = elem(a.wdtype), he = elem(a.hdtype);
  const Area outs[] = {{a.y, a.y_ld, a.m, a.n, e}, {a.total, a.total_ld, a.m, a.n, he}, {a.rstd, a.m, 1, a.m, 4},
                       {a.q, a.q_ld, a.m, a.n, 1}, scale_area(a.q_scale, a.m, a.q_scale_row, blocks, a.q_scale_block)};
  const Area ins[] = {{a.weight, a.n, 1, a.n, we}};
  const Area in_place[] = {{a.x, a.x_ld, a.m, a.n, e}, {a.residual, a.residual_ld, a.m, a.n, he}};
  return check_places(outs, 5, 2, ins, 1, in_place, 2);
}

int check_rms_backward(const eas_hip_rms_norm_backward_args& a) {
  OPS_CHECK(is_dtype(a.dtype) && (a.wdtype == a.dtype || a.wdtype == EAS_HIP_F32) && (a.hdtype == a.dtype || a.hdtype == EAS_HIP_F32),
            "unsupported dtype");
  OPS_CHECK(size_ok(a.m) && a.n > 0 && a.n <= kMost, "rows must hold at least one element, and sizes be at most 2^31 - 256");
  OPS_CHECK(a.dy_ld >= a.n && a.h_ld >= a.n && (!a.dx || a.dx_ld >= a.n) && (!a.dtotal || a.dtotal_ld >= a.n),
            "a row stride is shorter than the row");
  OPS_CHECK(!a.m || (a.dy && a.h && a.rstd), "dy, h and rstd must not be NULL");
  const int e = elem(a.dtype), we = elem(a.wdtype), he = elem(a.hdtype);
  const Area outs[] = {{a.dx, a.dx_ld, a.m, a.n, he}, {a.dweight, a.n, 1, a.n, we}};
  const Area ins[] = {{a.weight, a.n, 1, a.n, we}, {a.rstd, a.m, 1, a.m, 4}};
  const Area in_place[] = {{a.dy, a.dy_ld, a.m, a.n, e}, {a.h, a.h_ld, a.m, a.n, he}, {a.dtotal, a.dtotal_ld, a.m, a.n, he}};
  return check_places(outs, 2, 1, ins, 2, in_place, 3);
}
uint64_t rms_backward_bytes(const eas_hip_rms_norm_backward_args& a, int* chunks) {
  *chunks = rms_norm_backward_chunks(a);
  return a.dweight && !rms_norm_backward_few(a) ? (uint64_t)*chunks * (uint64_t)a.n * sizeof(float) : 0;
}

// ---- conversion ---------------------------------------------------------------------------

int check_quantize(const eas_hip_quantize_args& a) {
  OPS_CHECK(is_dtype(a.dtype), "unsupported dtype");
  OPS_CHECK(is_act(a.activation), "unknown activation");
  OPS_CHECK((a.block_m == 1 || a.block_m == kBlock) && (a.block_n == 1 || a.block_n == kBlock) && a.block_m * a.block_n > 1,
            "blocks must be 1 x 128, 128 x 1 or 128 x 128");
  OPS_CHECK(size_ok(a.m) && size_ok(a.n), "sizes must be in [0, 2^31 - 256]");
  OPS_CHECK(a.x_ld >= a.n && a.q_ld >= a.n && (!a.gate || a.gate_ld >= a.n), "a row stride is shorter than the row");
  const int64_t rows = cdiv(a.m, a.block_m), cols = cdiv(a.n, a.block_n);
  OPS_CHECK(scale_lines(rows, a.scale_row, cols, a.scale_col), "the scales must lie in lines that do not overlap");
  OPS_CHECK(!a.m || !a.n || (a.x && a.q && a.scale), "x, q and scale must not be NULL");
  const int e = elem(a.dtype);
  const Area outs[] = {{a.q, a.q_ld, a.m, a.n, 1}, scale_area(a.scale, rows, a.scale_row, cols, a.scale_col)};
  const Area ins[] = {{a.x, a.x_ld, a.m, a.n, e}, {a.gate, a.gate_ld, a.m, a.n, e}};
  return check_apart(outs, 2, ins, 2, nullptr, 0);
}

// ---- product --------------------------------------------------------------------------------

// A matrix of bytes as it lies in memory
struct Operand8 {
  const void* p;
  int64_t ld, rows, cols;
  bool along_k;
};

// What the DMA takes: rows at any 4 bytes, and for rows along k whole 16-byte chunks of k (of others, what a chunk reads past
// a row's end goes to columns that are not stored).  Others are copied to rows that are.
bool direct(const Operand8& o) {
  return (uint64_t)o.p % 4 == 0 && o.ld % 4 == 0 && (o.ld <= (4 << 20) || o.ld <= up(o.cols, 16)) && (!o.along_k || o.cols % 16 == 0);
}
void realign(CopyBytesParams& c, Operand8& o, Arena& ws) {
  if (direct(o) || !o.rows || !o.cols) return;
  const int i = c.copies++;
  c.src[i] = (const uint8_t*)o.p;
  c.src_ld[i] = o.ld;
  c.rows[i] = (int)o.rows;
  c.cols[i] = (int)o.cols;
  c.dst_ld[i] = o.ld = up(o.cols, 16);
  o.p = c.dst[i] = (uint8_t*)ws.take((uint64_t)(o.rows * o.ld));
}

int check_fp8(const eas_hip_linear_fp8_args& a) {
  OPS_CHECK(is_dtype(a.ydtype), "unsupported dtype");
  OPS_CHECK(is_act(a.activation), "unknown activation");
  OPS_CHECK((a.x_trans | a.w_trans | a.w_blocks | 1) == 1, "x_trans, w_trans and w_blocks must be 0 or 1");
  OPS_CHECK(size_ok(a.m) && size_ok(a.k) && size_ok(a.n), "sizes must be in [0, 2^31 - 256]");
  OPS_CHECK(a.x_ld >= (a.x_trans ? a.m : a.k) && a.w_ld >= (a.w_trans ? a.k : a.n) && a.y_ld >= a.n &&
                (!a.residual || a.residual_ld >= a.n) && (!a.pre || a.pre_ld >= a.n),
            "a row stride is shorter than the row");
  OPS_CHECK(a.x_scale_row >= 0 && a.x_scale_block >= 0 && a.w_scale_block >= 0 && a.w_scale_col >= 0, "a scale's stride is negative");
  OPS_CHECK(a.x_scale_row <= kFar && a.x_scale_block <= kFar && a.w_scale_block <= kFar && a.w_scale_col <= kFar, "the scales lie too far apart");
  const bool out = a.m && a.n;
  OPS_CHECK(!out || a.y, "y must not be NULL");
  OPS_CHECK(!out || !a.k || (a.x && a.w && a.x_scale && a.w_scale), "x, w and their scales must not be NULL");
  const int ye = elem(a.ydtype);
  const int64_t kb = cdiv(a.k, kBlock), nb = a.w_blocks ? cdiv(a.n, kBlock) : a.n;
  // a tile's scales are read at 32-bit offsets from its first one
  constexpr int64_t kReach = (1ll << 31) - 8;
  OPS_CHECK(a.x_scale_row * 4 <= kReach / 255 && a.w_scale_col * 4 <= kReach / 255, "the scales lie too far apart");
  const Area outs[] = {{a.y, a.y_ld, a.m, a.n, ye}, {a.pre, a.pre_ld, a.m, a.n, ye}};
  const Area ins[] = {{a.x, a.x_ld, a.x_trans ? a.k : a.m, a.x_trans ? a.m : a.k, 1},
                      {a.w, a.w_ld, a.w_trans ? a.n : a.k, a.w_trans ? a.k : a.n, 1},
                      scale_area(a.x_scale, a.m, a.x_scale_row, kb, a.x_scale_block),
                      scale_area(a.w_scale, kb, a.w_scale_block, nb, a.w_scale_col),
                      {a.bias, a.n, 1, a.n, ye}};
  const Area in_place[] = {{a.residual, a.residual_ld, a.m, a.n, ye}};
  return check_apart(outs, 2, ins, 5, in_place, 1);
}

constexpr int64_t kFewRows = 64;

struct Fp8Plan {
  Fp8Kernel kernel;
  int bm, bn, splits;
  double ns;  // what it is expected to take
};

// Few rows: every workgroup reads its columns of w and all of x, at 31 bytes a ns and CU (what a ring holds in flight over
// a load's time, and less than the memory gives), so wide workgroups read x less often,
// and narrow ones need no split k, whose join costs a launch.  Columns in even shares of a round, by eights.  Measured, us
// (16 columns / 64 in four ranges of k): 1 x 14336 x 4096 12.9 / 15.0, 16 rows 16.9 / 15.9, 64 rows 32.7 / 23.1.
Fp8Plan plan_few(bool any, int64_t m, int64_t k, int64_t n) {
  const Fp8Kernel kernel = m <= 16 ? kFp8Skinny1 : m <= 32 ? kFp8Skinny2 : kFp8Skinny4;
  Fp8Plan best{kernel, 64, any && cdiv(n, 32) >= kCus ? 32 : 16, 1, 1e300};
  for (int cw = 16; cw <= (any ? best.bn : 64); cw *= 2) {
    if (any && cw < best.bn) continue;
    for (int s = 1; s <= 16 && (s == 1 || cdiv(k, kBlock) >= 8 * s); s *= 2) {
      const int64_t rounds = cdiv(cdiv(n, cw) * s, kCus), width = any ? cw : up(cdiv(n, rounds * kCus / s), 8);
      double ns = 3000 + (double)rounds * (double)(width + m) * k / s / 31;
      if (s > 1) ns += 4500 + 2.0 * s * m * n * 4 / 5000;
      if (ns < best.ns) best.ns = ns, best.bn = (int)width, best.splits = s;
    }
  }
  return best;
}

int side_of(Fp8Kernel tile) { return tile == kFp8Tile256 ? 256 : tile == kFp8Tile128 ? 128 : 64; }

// EAS_HIP_OPS_GEMM picks the tile ("tile64", "tile128" or "tile256") and, after a colon, the ranges that k is split into, where they can
// run the product; for measurements and tests.
bool forced(int64_t k, bool wide, Fp8Plan* out) {
  const char* v = getenv("EAS_HIP_OPS_GEMM");
  if (!v || !*v) return false;
  Fp8Kernel kernel;
  if (!strncmp(v, "tile128", 7)) kernel = kFp8Tile128;
  else if (!strncmp(v, "tile64", 6) && wide) kernel = kFp8Tile64;
  else if (!strncmp(v, "tile256", 7) && !wide) kernel = kFp8Tile256;
  else return false;
  const char* colon = strchr(v, ':');
  const int64_t splits = colon ? atoi(colon + 1) : 1, stages = cdiv(k > 0 ? k : 1, kBlock);
  *out = {kernel, side_of(kernel), side_of(kernel), (int)(splits < 1 ? 1 : splits < stages ? splits : stages), 0};
  return true;
}

// Nanoseconds of a launch by a model of its rounds: workgroups side by side on the card's CUs, a time per block of k of one round
// and a fixed part, and for a split k the parts' way through memory and the launch that joins them.  The times are those of
// launches of one round over 4 to 112 blocks: 256 x 256 tiles 1.5 us a block, 1.9 on all CUs; 128 x 128 0.54 and 0.62; for
// f32 y 1.4 alone on a CU and 2.3 for two, 64 x 64 0.62 alone, 1 for two and 1.48 for four.
double estimate(Fp8Kernel kernel, bool wide, int64_t m, int64_t n, int64_t blocks, int splits) {
  const int64_t t = side_of(kernel), tiles = cdiv(m, t) * cdiv(n, t) * splits;
  const double each = (double)cdiv(blocks, splits);
  // whole rounds of `slots` workgroups, and one of the rest, whose block takes `rest` ns
  auto rounds = [&](int64_t slots, double whole, double fixed, auto rest) {
    const int64_t left = tiles % slots;
    return (double)(tiles / slots) * (each * whole + fixed) + (left ? each * rest(left) + fixed : 0.0);
  };
  double ns;
  if (kernel == kFp8Tile256) ns = rounds(kCus, 1900, 6000, [](int64_t n) { return n > kCus * 3 / 4 ? 1900.0 : 1500.0; });
  else if (kernel == kFp8Tile64) ns = rounds(4 * kCus, 1480, 2800, [](int64_t n) { return n > 2 * kCus ? 1480.0 : n > kCus ? 1000.0 : 620.0; });
  else if (!wide) ns = rounds(kCus, 620, 3000, [](int64_t n) { return n > kCus * 3 / 4 ? 620.0 : 540.0; });
  else ns = rounds(2 * kCus, 2300, 3000, [](int64_t n) { return n > kCus ? 2300.0 : 1400.0; });
  if (splits > 1) ns += 4000 + 2.0 * splits * m * n * 4 / 5000;
  return ns;
}

Fp8Plan plan_fp8(bool few, bool any, int64_t m, int64_t k, int64_t n, bool wide) {
  Fp8Plan best{kFp8Tile128, 0, 0, 0, 1e300};
  if (forced(k, wide, &best)) return best;
  if (few) return plan_few(any, m, k, n);
  const int64_t blocks = cdiv(k > 0 ? k : 1, kBlock);
  for (int s = 1; s <= 16 && (s == 1 || blocks >= 4 * s); s *= 2)
    for (const Fp8Kernel kernel : {kFp8Tile128, wide ? kFp8Tile64 : kFp8Tile256}) {
      const double ns = estimate(kernel, wide, m, n, blocks, s);
      if (ns < best.ns) best = {kernel, side_of(kernel), side_of(kernel), s, ns};
    }
  return best;
}

// A product in one launch, or in two: whole rounds of large tiles, and then the rows or the columns behind those as they are
// best by themselves.  Measured, us, in one launch / in two: 4099 x 4096 x 4096 112.7 / 78.3, 2600 x 14336 x 6400 355 / 242,
// f32 2900 x 4096 x 3300 118 / 112.  A second launch of much the same tiles gains nothing (3000 x 4096 x 9000 129.8 / 135.6),
// and neither do rounds of 128 x 128 tiles for 16-bit y (500 x 8192 x 9000 71.1 / 74.6).
struct Fp8Parts {
  int count;
  int64_t m[2], n[2];  // the second one begins behind the first, along the axis in which that is smaller than the whole
  Fp8Plan plan[2];
};
Fp8Parts parts_fp8(bool along_k, bool few, bool any, int64_t m, int64_t k, int64_t n, bool wide) {
  Fp8Parts best{1, {m}, {n}, {plan_fp8(few, any, m, k, n, wide)}};
  Fp8Plan tile;
  if (few || forced(k, wide, &tile)) return best;
  const Fp8Kernel kernel = wide ? kFp8Tile128 : kFp8Tile256;
  const int64_t side = side_of(kernel), tm = cdiv(m, side), tn = cdiv(n, side), slots = wide ? 2 * kCus : kCus;
  const int64_t whole = tm * tn / slots * slots;  // tiles in whole rounds
  if (!whole || whole == tm * tn) return best;
  double least = best.plan[0].ns;
  for (int axis = 0; axis < 2; ++axis) {
    const int64_t first = whole / (axis ? tm : tn) * side, all = axis ? n : m;
    if (!first || first >= all) continue;
    const int64_t m1 = axis ? m : first, n1 = axis ? first : n, m2 = axis ? m : m - first, n2 = axis ? n - first : n;
    const Fp8Plan rest = plan_fp8(along_k && m2 <= kFewRows, false, m2, k, n2, wide);
    const double ns = estimate(kernel, wide, m1, n1, cdiv(k > 0 ? k : 1, kBlock), 1), both = ns + 2000 + rest.ns;  // from launch to launch
    if (both < least) {
      least = both;
      best = {2, {m1, m2}, {n1, n2}, {{kernel, (int)side, (int)side, 1, ns}, rest}};
    }
  }
  return best;
}

// The plan's sizes into `g`, and its scratch
int fit_fp8(const Fp8Plan& plan, GemmParams& g, Arena& ws) {
  g.kt = (int)cdiv(g.k > 0 ? g.k : 1, kBlock);
  g.tiles_m = (int)cdiv(g.m, plan.bm);
  g.tiles_n = (int)cdiv(g.n, plan.bn);
  g.width = plan.bn;
  const int64_t per = cdiv(g.kt, plan.splits);  // ranges of whole blocks, none of them empty
  g.splits = (int)cdiv(g.kt, per);
  if (g.splits > 1) g.part = (float*)ws.take((uint64_t)g.splits * g.m * g.n * sizeof(float));
  const int64_t threads = (int64_t)g.tiles_m * g.tiles_n * 512;
  OPS_CHECK(threads < (1ll << 32) && g.splits < 65536, "the product has too many tiles");  // for a grid
  return EAS_HIP_OK;
}

int fp8_work(const eas_hip_linear_fp8_args& a, Arena& ws, bool launch, hipStream_t stream) {
  if (!a.m || !a.n) return EAS_HIP_OK;
  Operand8 x{a.x, a.x_ld, a.x_trans ? a.k : a.m, a.x_trans ? a.m : a.k, !a.x_trans};
  Operand8 w{a.w, a.w_ld, a.w_trans ? a.n : a.k, a.w_trans ? a.k : a.n, a.w_trans != 0};
  // a tile's rows within 32-bit offsets of its first one
  constexpr int64_t kReach = ((1ll << 31) - 4) / 256;
  Fp8Plan tile;  // forced
  const bool few = a.m <= kFewRows && x.along_k && w.along_k && !forced(a.k, a.ydtype == EAS_HIP_F32, &tile);
  // up to 16 rows go through registers where they are not direct; for more a copy is faster, although it moves w, all the work, three
  // times (64 x 4095 x 14336: 80 us through registers)
  const Fp8Form form{!x.along_k, !w.along_k, !a.w_blocks,
                     few && a.m <= 16 && !(direct(x) && direct(w) && x.ld <= kReach && w.ld <= kReach)};
  CopyBytesParams copy{};
  if (!form.any) {
    realign(copy, x, ws);
    realign(copy, w, ws);
    OPS_CHECK(x.ld <= kReach && w.ld <= kReach, "an operand's rows are too long: 32-bit offsets do not reach a tile's rows");
  }
  Fp8Params p{};
  p.xs = a.x_scale;
  p.ws = a.w_scale;
  p.xs_row = a.x_scale_row;
  p.xs_block = a.x_scale_block;
  p.ws_block = a.w_scale_block;
  p.ws_col = a.w_scale_col;
  p.ytype = a.ydtype;
  GemmParams& g = p.g;
  g.a[0] = x.p;
  g.lda[0] = x.ld;
  g.b[0] = w.p;
  g.ldb[0] = w.ld;
  g.c[0] = a.y;
  g.ldc[0] = a.y_ld;
  g.pre[0] = a.pre;
  g.ldpre[0] = a.pre_ld;
  g.bias[0] = a.bias;
  g.res = a.residual;
  g.ldres = a.residual_ld;
  g.m = (int)a.m;
  g.n = (int)a.n;
  g.k = (int)a.k;
  g.segs = g.prods = 1;
  g.act = a.activation;
  const int ye = elem(a.ydtype);
  const Fp8Parts parts = parts_fp8(x.along_k && w.along_k, few, form.any, a.m, a.k, a.n, a.ydtype == EAS_HIP_F32);
  if (launch) OPS_HIP(copy_bytes_launch(copy, stream));
  int64_t m0 = 0, n0 = 0;
  for (int i = 0; i < parts.count; ++i) {
    Fp8Params q = p;
    GemmParams& g = q.g;
    auto at = [&](const void* base, int64_t ld) { return base ? (char*)base + (m0 * ld + n0) * ye : nullptr; };
    q.xs += m0 * q.xs_row;
    q.ws += (a.w_blocks ? n0 / kBlock : n0) * q.ws_col;
    g.a[0] = (const char*)g.a[0] + m0 * (x.along_k ? x.ld : 1);
    g.b[0] = (const char*)g.b[0] + n0 * (w.along_k ? w.ld : 1);
    g.c[0] = at(g.c[0], g.ldc[0]);
    g.pre[0] = at(g.pre[0], g.ldpre[0]);
    g.res = at(g.res, g.ldres);
    if (g.bias[0]) g.bias[0] = (const char*)g.bias[0] + n0 * ye;
    g.m = (int)parts.m[i];
    g.n = (int)parts.n[i];
    OPS_TRY(fit_fp8(parts.plan[i], g, ws));
    if (launch) {
      OPS_HIP(fp8_launch(parts.plan[i].kernel, form, q, stream));
      if (g.splits > 1) {
        if (a.ydtype == EAS_HIP_F16) OPS_HIP(gemm_join_typed<f16>(false, g, stream));
        else if (a.ydtype == EAS_HIP_BF16) OPS_HIP(gemm_join_typed<bf16>(false, g, stream));
        else OPS_HIP(gemm_join_typed<float>(false, g, stream));
      }
    }
    if (parts.m[i] < a.m) m0 = parts.m[i];
    else n0 = parts.n[i];
  }
  return EAS_HIP_OK;
}

}  // namespace
}  // namespace eas

using namespace eas;

extern "C" {

int eas_hip_rms_norm(const eas_hip_rms_norm_args* args, size_t args_size, void* stream) {
  eas_hip_rms_norm_args a;
  OPS_TRY(read_args(args, args_size, &a));
  OPS_TRY(check_rms(a));
  if (a.m) OPS_HIP(rms_norm_launch(a, (hipStream_t)stream));
  return EAS_HIP_OK;
}

int eas_hip_rms_norm_backward_workspace(const eas_hip_rms_norm_backward_args* args, size_t args_size, uint64_t* bytes) {
  eas_hip_rms_norm_backward_args a;
  OPS_TRY(read_args(args, args_size, &a));
  OPS_CHECK(bytes != nullptr, "bytes must not be NULL");
  OPS_TRY(check_rms_backward(a));
  int chunks;
  *bytes = rms_backward_bytes(a, &chunks);
  return EAS_HIP_OK;
}

int eas_hip_rms_norm_backward(const eas_hip_rms_norm_backward_args* args, size_t args_size, void* stream) {
  eas_hip_rms_norm_backward_args a;
  OPS_TRY(read_args(args, args_size, &a));
  OPS_TRY(check_rms_backward(a));
  int chunks;
  const uint64_t need = rms_backward_bytes(a, &chunks);
  OPS_TRY(check_workspace(a.workspace, a.workspace_bytes, need));
  if (rms_norm_backward_few(a)) {
    OPS_HIP(rms_norm_backward_launch(a, nullptr, chunks, (hipStream_t)stream));
    return EAS_HIP_OK;
  }
  float* part = a.dweight ? (float*)a.workspace : nullptr;  // null with no rows: no chunk is read
  if (a.m && (a.dx || part)) OPS_HIP(rms_norm_backward_launch(a, part, chunks, (hipStream_t)stream));
  if (a.dweight) {
    ColumnSumParams c{};
    c.part = part;
    c.out[0] = a.dweight;
    c.n = (int)a.n;
    c.outs = 1;
    c.chunks = chunks;
    c.dtype = a.wdtype;
    OPS_HIP(column_sum_launch(c, (hipStream_t)stream));
  }
  return EAS_HIP_OK;
}

int eas_hip_quantize(const eas_hip_quantize_args* args, size_t args_size, void* stream) {
  eas_hip_quantize_args a;
  OPS_TRY(read_args(args, args_size, &a));
  OPS_TRY(check_quantize(a));
  if (a.m && a.n) OPS_HIP(quantize_launch(a, (hipStream_t)stream));
  return EAS_HIP_OK;
}

int eas_hip_linear_fp8_workspace(const eas_hip_linear_fp8_args* args, size_t args_size, uint64_t* bytes) {
  eas_hip_linear_fp8_args a;
  OPS_TRY(read_args(args, args_size, &a));
  OPS_CHECK(bytes != nullptr, "bytes must not be NULL");
  OPS_TRY(check_fp8(a));
  Arena ws{nullptr};
  OPS_TRY(fp8_work(a, ws, false, nullptr));
  *bytes = ws.used;
  return EAS_HIP_OK;
}

int eas_hip_linear_fp8(const eas_hip_linear_fp8_args* args, size_t args_size, void* stream) {
  eas_hip_linear_fp8_args a;
  OPS_TRY(read_args(args, args_size, &a));
  OPS_TRY(check_fp8(a));
  Arena count{nullptr};
  OPS_TRY(fp8_work(a, count, false, nullptr));
  OPS_TRY(check_workspace(a.workspace, a.workspace_bytes, count.used));
  Arena ws{(char*)a.workspace};
  return fp8_work(a, ws, true, (hipStream_t)stream);
}

}  // extern "C"
