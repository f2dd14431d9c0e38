// gemm.h — the matrix product under linear, gated_linear and their gradients (gfx950 MFMA).
//
// Every kernel moves its operands HBM -> LDS with 16-byte DMA chunks and multiplies with 16-row MFMAs, which take
// 64 bytes of k per row at a time: 32 elements of 16 bits in one v_mfma_f32_16x16x32, 16 of fp32 in four
// v_mfma_f32_16x16x4.  An operand whose memory rows run along k keeps them in LDS, and a lane reads its 16 bytes
// with one ds_read_b128; one whose rows run along m or n is transposed by the LDS read (ds_read_b64_tr_b16; fp32
// one ds_read_b32 per k).  The MFMA's first operand is B, so a lane holds 4 consecutive columns of one row of C.
//
// The DMA's range check gives zeros past the last row of an operand, and lanes past the end of k point outside.
// Its offsets are 32-bit: each stage moves the 64-bit base instead, so an operand may have any size, but a tile's rows
// have to lie within 2^31 bytes of its first one.  The host gives the kernels operands for which they do, with rows at any
// 4 bytes, and of whole 16-byte chunks of k where they run along k.
//
// The tiles are bound by the matrix cores, the small ones by LDS reads (for as many MFMAs a 64 x 64 tile
// reads twice what a 128 x 128 one does), few rows by the weights' way from HBM.
#ifndef EAS_OPS_GEMM_H
#define EAS_OPS_GEMM_H

#include "device.h"

namespace eas {

typedef int rsrc_t __attribute__((ext_vector_type(4)));
#define EAS_LDS __attribute__((address_space(3)))
// s_waitcnt with only vmcnt limited, and with only lgkmcnt(0)
#define EAS_WAITVM(n) (((n) & 15) | (((n) >> 4) << 14) | (0x7 << 4) | (0xF << 8))
#define EAS_WAITLGKM0 (15 | (3 << 14) | (0x7 << 4))

// raw buffer resource: base, range in bytes (reads at or past it return 0)
static __device__ __forceinline__ rsrc_t make_rsrc(const char* base, int64_t bytes) {
  const uint64_t a = (uint64_t)base;
  // clamped to [0, 2^31 - 4] by 32-bit comparisons, which stay on the scalar unit
  const int high = (int)(bytes >> 32);
  const uint32_t low = (uint32_t)bytes;
  const uint32_t n = high < 0 ? 0u : high > 0 || low > 0x7ffffffcu ? 0x7ffffffcu : low;
  rsrc_t r;
  r[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)a);
  r[1] = __builtin_amdgcn_readfirstlane((int)((uint32_t)(a >> 32) & 0xffffu));
  r[2] = __builtin_amdgcn_readfirstlane((int)n);
  r[3] = 0x00020000;
  return r;
}
// 16 bytes per lane, HBM -> LDS; lane i writes [lds + 16 i, lds + 16 i + 16).  As asm, so that the compiler does not
// wait for it before every LDS read; the loops count their own loads.
static __device__ __forceinline__ void dma16(rsrc_t r, uint32_t voff, uint32_t lds) {
  asm volatile("buffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff), "s"(r), "{m0}"(lds) : "memory");
}
// the same for lines that nothing reads again: past the caches
static __device__ __forceinline__ void dma16_stream(rsrc_t r, uint32_t voff, uint32_t lds) {
  asm volatile("buffer_load_dwordx4 %0, %1, 0 offen nt lds" ::"v"(voff), "s"(r), "{m0}"(lds) : "memory");
}
constexpr uint32_t kOutside = 0x80000000u;  // past every range

template <int V> struct int_c { static constexpr int value = V; };

// ---- operand types: a fragment is 16 bytes a lane, 64 bytes of k for 16 rows --------

template <typename T> struct Mma;
template <> struct Mma<f16> {
  typedef f16 frag __attribute__((ext_vector_type(8)));
  typedef __fp16 tr __attribute__((__vector_size__(4 * sizeof(__fp16))));
  static __device__ __forceinline__ tr read_tr(const char* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4f16((EAS_LDS tr*)p);
  }
  static __device__ __forceinline__ f32x4 mma(frag n, frag m, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(n, m, c, 0, 0, 0);
  }
};
template <> struct Mma<bf16> {
  typedef bf16 frag __attribute__((ext_vector_type(8)));
  typedef bf16 tr __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ tr read_tr(const char* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((EAS_LDS tr*)p);
  }
  static __device__ __forceinline__ f32x4 mma(frag n, frag m, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(n, m, c, 0, 0, 0);
  }
};
template <> struct Mma<float> {
  typedef f32x4 frag;
  static __device__ __forceinline__ f32x4 mma(frag n, frag m, f32x4 c) {
    const float n0 = n[0], n1 = n[1], n2 = n[2], n3 = n[3], m0 = m[0], m1 = m[1], m2 = m[2], m3 = m[3];
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(n0, m0, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(n1, m1, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(n2, m2, c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x4f32(n3, m3, c, 0, 0, 0);
  }
};

// ---- an operand's tile: R rows of the outer index by KB bytes of k, in LDS ------------
//
// k-rows: R rows of KB bytes (64, 128 or 256), 16-byte chunk c of row r at c ^ swz(r).  A ds_read_b128 takes its lanes 16 at a
// time: 0-3 and 12-15 with 20-27, 4-11 with 16-19 and 28-31, and the same from lane 32 on.  With swz = -(r/4) mod 4 (64-byte
// rows, four a bank cycle), (r/2) mod 8 (128-byte rows, two) and r mod 16 (256-byte rows) each such set meets every bank once; (r/4) mod 4 meets
// half of them twice (4096 x 8192 x 4096 with both operands so: 5.2e7 LDS cycles, 2.6e7 of them conflicts).
// outer-rows: KB / sizeof(T) rows (k) of R elements, chunk c of row r at c ^ swz(r).  16 bits: the four rows of a
// transposing read 64 bytes apart, and rows 8 apart on other banks too; rows r and r + 4 share the mask.  fp32: the
// rows 4 g + t that the four lane groups read at once 64 bytes apart.
template <typename T, bool OUTER, int R, int KB> struct Tile {
  static constexpr int E = sizeof(T), CE = 16 / E, BK = KB / E;
  static constexpr int ROW = OUTER ? R * E : KB;        // bytes of an LDS row
  static constexpr int BYTES = R * KB, LOADS = BYTES / 1024;
  static constexpr int CH = ROW / 16;                   // chunks per row
  typedef typename Mma<T>::frag frag;

  static __device__ __forceinline__ int swz(int r) {
    if constexpr (!OUTER) return KB == 64 ? -(r >> 2) & 3 : KB == 128 ? (r >> 1) & 7 : r & 15;
    else if constexpr (E == 4) return 4 * ((r >> 2) & 3);
    else if constexpr (ROW == 128) return 2 * ((r >> 1) & 1) + 4 * ((r >> 3) & 1);
    else return (4 * (r & 3)) ^ (2 * ((r >> 3) & 1));
  }
  // DMA load q (1 KB): this lane's offset from the stage's base, kOutside where its row or chunk lies past the
  // operand's outer extent (`left` elements from the tile's origin), and its first k in the stage (k-rows)
  static __device__ __forceinline__ uint32_t lane_offset(int q, int lane, int64_t ld, int64_t left, int* k) {
    const int r = (64 / CH) * q + lane / CH, c = (lane % CH) ^ swz(r);
    *k = c * CE;
    const bool in = OUTER ? (int64_t)c * CE < left : r < left;
    return in ? (uint32_t)r * (uint32_t)(ld * E) + (uint32_t)(c * 16) : kOutside;
  }
  // the chunk that lane_offset's lane holds: its row, and its first element in the row
  static __device__ __forceinline__ void chunk(int q, int lane, int* row, int* col) {
    *row = (64 / CH) * q + lane / CH;
    *col = ((lane % CH) ^ swz(*row)) * CE;
  }
  // the stage's resource; origin: the tile's first element at k = 0
  static __device__ __forceinline__ rsrc_t resource(const char* origin, int64_t ld, int64_t left, int k, int k0) {
    if constexpr (OUTER)  // a dword that holds the last element whole
      return make_rsrc(origin + (int64_t)k0 * ld * E, ((((int64_t)(k - 1 - k0) * ld + left) * E) + 3) & ~(int64_t)3);
    else
      return make_rsrc(origin + (int64_t)k0 * E, (((left - 1) * ld + (k - k0)) * E + 15) & ~(int64_t)15);
  }
  static __device__ __forceinline__ const char* origin(const void* p, int64_t ld, int64_t outer0) {
    return (const char*)p + (OUTER ? outer0 : outer0 * ld) * E;
  }
  // The same, stage by stage: kept on the scalar unit, so that the waves that multiply spend nothing on it
  struct Source {
    const char* p;   // the tile's first element of the stage
    int64_t bytes;   // from there to the operand's end
    int64_t step;
    __device__ __forceinline__ void set(const void* op, int64_t ld, int64_t outer0, int64_t left, int k, int k0) {
      step = OUTER ? (int64_t)BK * ld * E : KB;
      p = origin(op, ld, outer0) + (OUTER ? (int64_t)k0 * ld * E : (int64_t)k0 * E);
      bytes = OUTER ? ((((int64_t)(k - 1 - k0) * ld + left) * E) + 3) & ~(int64_t)3
                    : (((left - 1) * ld + (k - k0)) * E + 15) & ~(int64_t)15;
    }
    __device__ __forceinline__ void next() {
      p += step;
      bytes -= step;
    }
    __device__ __forceinline__ rsrc_t resource(bool any) const { return make_rsrc(p, any ? bytes : 0); }
  };
  // offset of the fragment of 16 outer rows from `o`, the stage's first 64 bytes of k; later ones: at()
  static __device__ __forceinline__ int frag_offset(int lane, int o) {
    const int g = lane >> 4, i = lane & 15;
    if constexpr (!OUTER) {
      const int r = o + i;
      return r * ROW + ((g ^ swz(r)) * 16);
    } else if constexpr (E == 4) {
      const int r = 4 * g, col = o + i;
      return r * ROW + (((col >> 2) ^ swz(r)) * 16) + (col & 3) * 4;
    } else {
      // ds_read_b64_tr_b16: source lane i of a 16-lane group addresses row i/4, columns 4 (i%4)..+3; result lane i
      // receives column i of the four rows
      const int r = 8 * g + (i >> 2), col = o + 4 * (i & 3);
      return r * ROW + (((col >> 3) ^ swz(r)) * 16) + (col & 7) * 2;
    }
  }
  // the fragment at `off` (frag_offset), 64-byte step h of the stage
  static __device__ __forceinline__ frag read(const char* tile, int off, int h) {
    if constexpr (!OUTER) {
      return *(const frag*)(tile + (off ^ (64 * h)));  // chunks 4 on, within the row's swizzle
    } else if constexpr (E == 4) {
      const char* p = tile + off + h * 16 * ROW;
      return (frag){*(const float*)p, *(const float*)(p + ROW), *(const float*)(p + 2 * ROW), *(const float*)(p + 3 * ROW)};
    } else {
      const char* p = tile + off + h * 32 * ROW;
      const auto lo = Mma<T>::read_tr(p), hi = Mma<T>::read_tr(p + 4 * ROW);
      typedef T half __attribute__((ext_vector_type(4)));
      const half l = __builtin_bit_cast(half, lo), u = __builtin_bit_cast(half, hi);
      return (frag){l[0], l[1], l[2], l[3], u[0], u[1], u[2], u[3]};
    }
  }
  static constexpr int READS = OUTER ? (E == 4 ? 4 : 2) : 1;
};

// ---- epilogue ----------------------------------------------------------------------

// the biases of 8 columns; absent ones are 0
template <typename T, bool GATED>
static __device__ __forceinline__ void load_bias(const GemmParams& p, int64_t col, float (&bz)[8], float (&bu)[8]) {
  const int left = col < p.n ? (int)(p.n - col < 8 ? p.n - col : 8) : 0;
  load_upto8((const T*)p.bias[0] + col, p.bias[0] ? left : 0, bz);
  if constexpr (GATED) load_upto8((const T*)p.bias[1] + col, p.bias[1] ? left : 0, bu);
}

// 8 columns of one row from (row, col) on: z (gated: z and u) through bias, activation and residual to memory
template <typename T, bool GATED>
static __device__ __forceinline__ void finish8(const GemmParams& p, int prod, int64_t row, int64_t col, float (&z)[8], float (&u)[8],
                                               const float (&bz)[8], const float (&bu)[8]) {
  const int left = (int)(p.n - col < 8 ? p.n - col : 8);
  float t[8];
  if (p.res) load_upto8<T>(p.res, p.wide, row * p.ldres + col, left, t);
#pragma unroll
  for (int e = 0; e < 8; ++e) z[e] += bz[e];
  if constexpr (GATED) {
#pragma unroll
    for (int e = 0; e < 8; ++e) u[e] += bu[e];
    if (p.pre[1]) store_upto8<T>(p.pre[1], p.wide, row * p.ldpre[1] + col, left, u);
  }
  if (p.pre[0]) store_upto8<T>(p.pre[0], p.wide, row * p.ldpre[0] + col, left, z);
  activate8<sizeof(T) == 2>(p.act, z);
  if constexpr (GATED) {
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] *= u[e];
  }
  if (p.res) {
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] += t[e];
  }
  void* c = prod ? p.c[1] : p.c[0];
  const int64_t ldc = prod ? p.ldc[1] : p.ldc[0];
  store_upto8<T>(c, p.wide, row * ldc + col, left, z);
}

// the sums of one range of k, for gemm_join
template <bool GATED>
static __device__ __forceinline__ void store_part(const GemmParams& p, int prod, int split, int64_t row, int64_t col,
                                                  const float (&z)[8], const float (&u)[8]) {
  const int left = (int)(p.n - col < 8 ? p.n - col : 8);
  float* part = p.part + (((int64_t)split * p.prods + prod) * p.m + row) * p.n * (GATED ? 2 : 1) + col;
  store_upto8(part, left, z);
  if constexpr (GATED) store_upto8(part + p.n, left, u);
}

// Rows of f32 sums in LDS to memory: `rows` rows of LD floats, columns [0, W) (gated: gate [0, W), up [W, 2 W)).
// row_of(r) is the row of C behind LDS row r.
template <typename T, bool GATED, int W, int LD, int NTHREADS, typename RowOf>
static __device__ __forceinline__ void finish_rows(const GemmParams& p, const float* sums, int rows, int prod, int split,
                                                   int n0, int tid, RowOf row_of) {
  constexpr int PER = W / 8;
  static_assert(NTHREADS % PER == 0, "a thread stays in its columns");
  const int c = (tid % PER) * 8;
  if (n0 + c >= p.n) return;
  float bz[8], bu[8];
  if (p.splits == 1) load_bias<T, GATED>(p, n0 + c, bz, bu);
#pragma unroll 1
  for (int r = tid / PER; r < rows; r += NTHREADS / PER) {
    const int64_t row = row_of(r);
    if (row >= p.m) continue;
    float z[8], u[8];
    const f32x4 z0 = *(const f32x4*)(sums + r * LD + c), z1 = *(const f32x4*)(sums + r * LD + c + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) z[e] = z0[e], z[e + 4] = z1[e];
    if constexpr (GATED) {
      const f32x4 u0 = *(const f32x4*)(sums + r * LD + W + c), u1 = *(const f32x4*)(sums + r * LD + W + c + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) u[e] = u0[e], u[e + 4] = u1[e];
    }
    if (p.splits > 1) store_part<GATED>(p, prod, split, row, n0 + c, z, u);
    else finish8<T, GATED>(p, prod, row, n0 + c, z, u, bz, bu);
  }
}

// ---- the workgroup's tile ----------------------------------------------------------

// Workgroup w runs on XCD w % 8: each XCD takes a contiguous range of tiles, GROUP tile rows high, column by column,
// so that the tiles in flight on it share rows of A and columns of B in its L2.
template <int GROUP>
static __device__ __forceinline__ void tile_of(const GemmParams& p, int id, int& tm, int& tn) {
  const int total = p.tiles_m * p.tiles_n;
  const int xcd = id & 7, q = total >> 3, r = total & 7;
  const int t = xcd * q + (xcd < r ? xcd : r) + (id >> 3);
  const int span = GROUP * p.tiles_n, group = t / span, first = group * GROUP;
  const int high = p.tiles_m - first < GROUP ? p.tiles_m - first : GROUP;
  const int in = t - group * span;
  tm = first + in % high;
  tn = in / high;
}

// The range of stages of this split, over both segments
static __device__ __forceinline__ void stages_of(const GemmParams& p, int split, int& lo, int& hi) {
  const int total = p.kt * p.segs, per = (total + p.splits - 1) / p.splits;
  lo = split * per;
  hi = lo + per < total ? lo + per : total;
}

// ---- tiles of BM x BN on producers and consumers --------------------------------------
//
// 8 waves.  Waves 4-7 move the stages (128 bytes of k, a ring of NSTAGE) and run no arithmetic, waves 0-3 hold
// BM/2 x BN/2 of the tile each and read the fragments of one 64-byte half between the MFMAs of the half before.
// GATED: the B tile is two tiles of BN/2 columns, gate's and up's, and a wave holds the same columns of both.
//
// For fp32, and where 256 x 256 tiles are too few.  Measured: 4.7 ns a k for a 64 x 64 tile alone on a CU and 7.2 for two,
// 8.3 for 128 x 128 (1024^3 bf16 8.0 us; 2048 x 4096 x 1024 in two ranges of k 23 us, 740 TFLOP/s); fp32 20, 34 and 61 ns.
constexpr int kTileStages = 4;
template <typename T, bool AOUT, bool BOUT, bool GATED, int BM, int BN> constexpr int tile_bytes() {
  return kTileStages * (Tile<T, AOUT, BM, 128>::BYTES + (GATED ? 2 : 1) * Tile<T, BOUT, BN / (GATED ? 2 : 1), 128>::BYTES);
}
// tile `id` of a product and range of k `slice`
template <typename T, bool AOUT, bool BOUT, bool GATED, int BM, int BN>
static __device__ __forceinline__ void tile_product(const GemmParams& p, char* smem, int id, int slice) {
  constexpr int NSUB = GATED ? 2 : 1, SUBN = BN / NSUB, KB = 128;
  typedef Tile<T, AOUT, BM, KB> TA;
  typedef Tile<T, BOUT, SUBN, KB> TB;
  typedef Mma<T> M;
  constexpr int BK = TA::BK, NSTAGE = kTileStages, STAGE = TA::BYTES + NSUB * TB::BYTES;
  constexpr int NA = BM / 32, NB = BN / 32;              // fragments of a wave
  constexpr int NAI = TA::LOADS / 4, NBI = NSUB * TB::LOADS / 4;  // loads per producer and stage
  constexpr int LD = BN + 4;
  static_assert(BM * LD * 4 <= NSTAGE * STAGE && NSTAGE * STAGE <= 160 * 1024, "the epilogue's rows fit the ring");
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int tm, tn, lo, hi;
  tile_of<8>(p, id, tm, tn);
  const int prod = slice % p.prods, split = slice / p.prods;
  stages_of(p, split, lo, hi);
  const int m0 = tm * BM, n0 = tn * SUBN, nst = hi - lo;

  if (wave >= 4) {
    const int pw = wave - 4, sub = GATED ? pw >> 1 : 0;
    const int64_t mleft = p.m - m0, nleft = p.n - n0;
    const uint32_t lds = (uint32_t)(size_t)(EAS_LDS char*)smem;
    const uint32_t lds_a = lds + pw * NAI * 1024, lds_b = lds + TA::BYTES + pw * NBI * 1024;
    auto pick = [&](int s, const char*& oa, const char*& ob, int64_t& la, int64_t& lb) {
      const int ia = p.prods > 1 ? prod : s, ib = GATED ? sub : ia;
      la = ia ? p.lda[1] : p.lda[0];
      lb = ib ? p.ldb[1] : p.ldb[0];
      oa = TA::origin(ia ? p.a[1] : p.a[0], la, m0);
      ob = TB::origin(ib ? p.b[1] : p.b[0], lb, n0);
    };
    const char *oa, *ob;
    int64_t la, lb;
    uint32_t va[NAI], vb[NBI];
    int ka[NAI], kb[NBI];
    auto lanes = [&]() {
#pragma unroll
      for (int i = 0; i < NAI; ++i) va[i] = TA::lane_offset(pw * NAI + i, lane, la, mleft, &ka[i]);
#pragma unroll
      for (int i = 0; i < NBI; ++i) vb[i] = TB::lane_offset((GATED ? (pw & 1) : pw) * NBI + i, lane, lb, nleft, &kb[i]);
    };
    int seg = lo >= p.kt ? 1 : 0;
    pick(seg, oa, ob, la, lb);
    lanes();
    auto dma = [&](int s) __attribute__((always_inline)) {  // stage s of this split
      const uint32_t at = (uint32_t)((s % NSTAGE) * STAGE);
      if (s >= nst) {  // past the end: zeros into a slot that nobody reads, to keep the count of loads
        const rsrc_t none = make_rsrc((const char*)p.a[0], 0);
#pragma unroll
        for (int i = 0; i < NAI; ++i) dma16(none, kOutside, lds_a + at + i * 1024);
#pragma unroll
        for (int i = 0; i < NBI; ++i) dma16(none, kOutside, lds_b + at + i * 1024);
        return;
      }
      int kt = lo + s;
      if (kt >= p.kt) {
        if (seg == 0) {
          seg = 1;
          pick(1, oa, ob, la, lb);
          lanes();
        }
        kt -= p.kt;
      }
      const int k0 = kt * BK;
      const rsrc_t ra = TA::resource(oa, la, mleft, p.k, k0), rb = TB::resource(ob, lb, nleft, p.k, k0);
      if (k0 + BK <= p.k) {
#pragma unroll
        for (int i = 0; i < NAI; ++i) dma16(ra, va[i], lds_a + at + i * 1024);
#pragma unroll
        for (int i = 0; i < NBI; ++i) dma16(rb, vb[i], lds_b + at + i * 1024);
      } else {
#pragma unroll
        for (int i = 0; i < NAI; ++i) dma16(ra, !AOUT && k0 + ka[i] >= p.k ? kOutside : va[i], lds_a + at + i * 1024);
#pragma unroll
        for (int i = 0; i < NBI; ++i) dma16(rb, !BOUT && k0 + kb[i] >= p.k ? kOutside : vb[i], lds_b + at + i * 1024);
      }
    };
    // one barrier per stage, as many as the consumers
    constexpr int PER = NAI + NBI;
#pragma unroll
    for (int s = 0; s < NSTAGE; ++s) dma(s);
    __builtin_amdgcn_s_waitcnt(EAS_WAITVM((NSTAGE - 1) * PER));  // stage 0 landed
    __syncthreads();
    for (int s = 0; s + 1 < nst; ++s) {
      __builtin_amdgcn_s_waitcnt(EAS_WAITVM((NSTAGE - 2) * PER));  // stage s + 1 landed
      __syncthreads();
      dma(s + NSTAGE);  // the slot of stage s, whose fragments every consumer has read
    }
    __builtin_amdgcn_s_waitcnt(EAS_WAITVM(0));
    __syncthreads();  // the ring is free
    __syncthreads();  // the sums are in it
  } else {
    const int wm = wave >> 1, wn = wave & 1;
    int oa[NA], ob[NB];
#pragma unroll
    for (int i = 0; i < NA; ++i) oa[i] = TA::frag_offset(lane, wm * (BM / 2) + i * 16);
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int c = wn * (SUBN / 2) + (j % (NB / NSUB)) * 16;
      ob[j] = TB::frag_offset(lane, c);
    }
    f32x4 acc[NA][NB];
#pragma unroll
    for (int i = 0; i < NA; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j) acc[i][j] = (f32x4){};
    typedef typename M::frag afrag_t[NA];
    typedef typename M::frag bfrag_t[NB];
    auto read_half = [&](int h, afrag_t& fa, bfrag_t& fb) __attribute__((always_inline)) {
      const char* st = smem + (h / 2 % NSTAGE) * STAGE;
#pragma unroll
      for (int i = 0; i < NA; ++i) fa[i] = TA::read(st, oa[i], h & 1);
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        fb[j] = TB::read(st + TA::BYTES + (j / (NB / NSUB)) * TB::BYTES, ob[j], h & 1);
      }
    };
    auto mmas = [&](const afrag_t& fa, const bfrag_t& fb) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < NA; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = M::mma(fb[j], fa[i], acc[i][j]);
    };
    // Half h: its MFMAs, and between them the reads of half h + 1.  Before the second half of a stage: the barrier at
    // which the next stage has landed, and after which the producers refill this stage's slot, both of whose halves
    // every consumer has read by then.
    auto step = [&](int h, const afrag_t& fa, const bfrag_t& fb, afrag_t& na, bfrag_t& nb) __attribute__((always_inline)) {
      constexpr int NMFMA = NA * NB * (TA::E == 4 ? 4 : 1), NREAD = NA * TA::READS + NB * TB::READS;
      if (h & 1) __syncthreads();
      __builtin_amdgcn_sched_barrier(0);
      read_half(h + 1, na, nb);
      mmas(fa, fb);
#pragma unroll
      for (int s = 0; s < NREAD / 2; ++s) {  // the LDS reads two by two after the first MFMAs
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, NMFMA - NREAD / 2, 0);
      __builtin_amdgcn_sched_barrier(0);
    };
    __syncthreads();  // stage 0 landed
    afrag_t a0, a1;
    bfrag_t b0, b1;
    read_half(0, a0, b0);
    for (int s = 0; s + 1 < nst; ++s) {
      step(2 * s, a0, b0, a1, b1);
      step(2 * s + 1, a1, b1, a0, b0);
    }
    step(2 * nst - 2, a0, b0, a1, b1);
    mmas(a1, b1);
    __syncthreads();  // the ring is free
    float* sums = (float*)smem;
    // lane l of a 16 x 16 tile holds columns 4 (l/16)..+3 of row l%16
#pragma unroll
    for (int i = 0; i < NA; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const int sub = j / (NB / NSUB), c = sub * SUBN + wn * (SUBN / 2) + (j % (NB / NSUB)) * 16;
        *(f32x4*)(sums + (wm * (BM / 2) + i * 16 + (lane & 15)) * LD + c + 4 * (lane >> 4)) = acc[i][j];
      }
    __syncthreads();  // the sums are in it
  }
  finish_rows<T, GATED, SUBN, LD, 512>(p, (const float*)smem, BM, prod, split, n0, tid, [&](int r) { return (int64_t)m0 + r; });
}

template <typename T, bool AOUT, bool BOUT, bool GATED, int BM, int BN>
static __global__ __launch_bounds__(512) void gemm_tile(const GemmParams p) {
  __shared__ __attribute__((aligned(1024))) char smem[tile_bytes<T, AOUT, BOUT, GATED, BM, BN>()];
  tile_product<T, AOUT, BOUT, GATED, BM, BN>(p, smem, blockIdx.x, blockIdx.y);
}

// A gradient's two products in one launch, `dx`'s tiles and then `dw`'s, where neither fills the card: each alone takes as
// long as one tile's k, with CUs that wait for it.  300 x 512 x 1031 f32 gated, all of the gradient: 45.2 -> 33.4 us; 1024^3
// bf16 26.7 -> 22.2; 517 x 1023 x 2047 f16 32.9 -> 27.9.
template <typename T, bool BOUT>
static __global__ __launch_bounds__(512) void gemm_pair(const GemmParams dx, const GemmParams dw) {
  constexpr int A = tile_bytes<T, false, BOUT, false, 64, 64>(), B = tile_bytes<T, true, true, false, 64, 64>();
  __shared__ __attribute__((aligned(1024))) char smem[A > B ? A : B];
  const int tiles = dx.tiles_m * dx.tiles_n, first = tiles * dx.splits, id = blockIdx.x;
  if (id < first) {
    tile_product<T, false, BOUT, false, 64, 64>(dx, smem, id % tiles, id / tiles);
  } else {
    const int rest = dw.tiles_m * dw.tiles_n;
    tile_product<T, true, true, false, 64, 64>(dw, smem, (id - first) % rest, (id - first) / rest);
  }
}

// ---- tiles of 256 x 256 -----------------------------------------------------------------
//
// 16-bit operands.  8 waves, two per SIMD, that both load and multiply: wave (g, w) holds rows [128 g, 128 g + 128) of
// columns [64 w, 64 w + 64) (gated: 32 of gate's and the same 32 of up's), 128 sums a lane.  Four stages of 32 k in a
// ring; one barrier a stage.  A stage's 32 MFMAs a wave take 512 cycles of its SIMD, its fragments 12 KB a wave, so the
// matrix cores bound it, at the clock that they leave: 4096^3 bf16 110 us (1250 TFLOP/s, matrix cores busy 61 % of the
// cycles) once the clock has settled, with bias, gelu and the product kept 122.  Two groups of waves that load and multiply
// in turns took 139 in the form tried here; the lifted GEMMs' body of that kind (codegen/gemm_kernels.py) takes 103 for the
// same product with f32 stores.
template <typename T, bool AOUT, bool BOUT, bool GATED>
static __global__ __launch_bounds__(512) void gemm_tile256(const GemmParams p) {
  constexpr int BM = 256, BN = 256, KB = 64, NSUB = GATED ? 2 : 1, SUBN = BN / NSUB, NSTAGE = 4;
  typedef Tile<T, AOUT, BM, KB> TA;
  typedef Tile<T, BOUT, SUBN, KB> TB;
  typedef Mma<T> M;
  constexpr int BK = TA::BK, STAGE = TA::BYTES + NSUB * TB::BYTES;  // 32 KB
  constexpr int LD = BN + 4, ROWS = 128;                            // rows of an epilogue pass
  constexpr int BYTES = NSTAGE * STAGE > ROWS * LD * 4 ? NSTAGE * STAGE : ROWS * LD * 4;
  static_assert(sizeof(T) == 2 && BYTES <= 160 * 1024, "16-bit operands; LDS");
  __shared__ __attribute__((aligned(1024))) char smem[BYTES];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = wave >> 2, w = wave & 3;
  int tm, tn, lo, hi;
  tile_of<4>(p, blockIdx.x, tm, tn);
  const int prod = blockIdx.y % p.prods, split = blockIdx.y / p.prods;
  stages_of(p, split, lo, hi);
  const int m0 = tm * BM, n0 = tn * SUBN, nst = hi - lo;
  const int64_t mleft = p.m - m0, nleft = p.n - n0;

  // Each wave moves 2 KB of A and 2 KB of B per stage (gated: waves 0-3 gate's columns, 4-7 up's), in four loads.
  const int sub = GATED ? g : 0, qb = (GATED ? w : wave) * 2;
  const uint32_t lds = (uint32_t)(size_t)(EAS_LDS char*)smem;
  const uint32_t lds_a = lds + wave * 2048, lds_b = lds + TA::BYTES + wave * 2048;
  typename TA::Source sa;
  typename TB::Source sb;
  uint32_t va[2], vb[2];
  // The source of stage t on, where it changes: at a segment's first stage, and at its last one where that is not
  // whole (rows along k end within it).  `change`: the next such stage.
  int seg = 0, change = 0;
  auto set_source = [&](int t) __attribute__((always_inline)) {
    const int at = lo + t;
    seg = at >= p.kt ? 1 : 0;
    const int kt = at - (seg ? p.kt : 0), k0 = kt * BK;
    const int ia = p.prods > 1 ? prod : seg, ib = GATED ? sub : ia;
    const int64_t la = ia ? p.lda[1] : p.lda[0], lb = ib ? p.ldb[1] : p.ldb[0];
    sa.set(ia ? p.a[1] : p.a[0], la, m0, mleft, p.k, k0);
    sb.set(ib ? p.b[1] : p.b[0], lb, n0, nleft, p.k, k0);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      int k;
      va[i] = TA::lane_offset(wave * 2 + i, lane, la, mleft, &k);
      if (!AOUT && k0 + k >= p.k) va[i] = kOutside;
      vb[i] = TB::lane_offset(qb + i, lane, lb, nleft, &k);
      if (!BOUT && k0 + k >= p.k) vb[i] = kOutside;
    }
    const int whole = p.k / BK;  // stages
    change = kt < whole && whole < p.kt ? t + whole - kt : t + p.kt - kt;
  };
  // load d of a stage; past the last stage it moves zeros, into a slot whose fragments are not used
  auto dma_one = [&](int t, int slot, int d) __attribute__((always_inline)) {  // d: 0, 1 A; 2, 3 B
    if (d < 2) dma16(sa.resource(t < nst), va[d], lds_a + (uint32_t)(slot + d * 1024));
    else dma16(sb.resource(t < nst), vb[d - 2], lds_b + (uint32_t)(slot + (d - 2) * 1024));
  };
  auto advance = [&](int t) __attribute__((always_inline)) {  // from stage t - 1 to stage t
    if (t == change) {
      if (t < nst) set_source(t);
    } else {
      sa.next();
      sb.next();
    }
  };
  int fo_a[8], fo_b[4];
#pragma unroll
  for (int i = 0; i < 8; ++i) fo_a[i] = TA::frag_offset(lane, g * 128 + i * 16);
#pragma unroll
  for (int j = 0; j < 4; ++j) fo_b[j] = TB::frag_offset(lane, GATED ? w * 32 + (j & 1) * 16 : w * 64 + j * 16);
  f32x4 acc[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = (f32x4){};
  typename M::frag fa[8], b0[4], b1[4];
  typedef typename M::frag bfrag_t[4];
  // slot: a stage's place in the ring, in bytes
  auto read_a = [&](int slot, int i) __attribute__((always_inline)) { fa[i] = TA::read(smem + slot, fo_a[i], 0); };
  auto read_b = [&](int slot, bfrag_t& b, int j) __attribute__((always_inline)) {
    b[j] = TB::read(smem + slot + TA::BYTES + (GATED ? j / 2 : 0) * TB::BYTES, fo_b[j], 0);
  };
  auto after = [&](int slot) __attribute__((always_inline)) { return slot + STAGE == NSTAGE * STAGE ? 0 : slot + STAGE; };
  // Stage s: its MFMAs, two rows of 16 at a time, and among them the fragments of stage s + 1: B's beside B's, each A
  // fragment in place once its MFMAs are issued, so that its read has most of a stage to land.  The DMA of stage s +
  // NSTAGE - 1 refills the slot of stage s - 1, whose last fragments every wave had multiplied before the barrier.
  int next = STAGE, fill = (NSTAGE - 1) * STAGE;
  auto step = [&](int s, const bfrag_t& b, bfrag_t& xb) __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(EAS_WAITVM(4 * (NSTAGE - 3)));  // this wave's loads of stage s + 1 landed
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    const int t = s + NSTAGE - 1;
    advance(t);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      __builtin_amdgcn_sched_barrier(0);
      dma_one(t, fill, c);
#pragma unroll
      for (int i = 2 * c; i < 2 * c + 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = M::mma(b[j], fa[i], acc[i][j]);
      read_b(next, xb, c);
      read_a(next, 2 * c);
      read_a(next, 2 * c + 1);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, TB::READS, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 3, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, TA::READS, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, TA::READS, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    next = after(next);
    fill = after(fill);
  };
#pragma unroll 1
  for (int t = 0; t < NSTAGE - 1; ++t) {
    advance(t);
#pragma unroll
    for (int d = 0; d < 4; ++d) dma_one(t, t * STAGE, d);
  }
  __builtin_amdgcn_s_waitcnt(EAS_WAITVM(4 * (NSTAGE - 2)));  // stage 0 landed
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 4; ++j) read_b(0, b0, j);
#pragma unroll
  for (int i = 0; i < 8; ++i) read_a(0, i);
  // stages two by two, as B's fragments alternate; an odd last one has a stage of zeros beside it
#pragma unroll 1
  for (int s = 0; s < nst; s += 2) {
    step(s, b0, b1);
    step(s + 1, b1, b0);
  }
  __builtin_amdgcn_s_waitcnt(EAS_WAITVM(0));  // the zeros past the last stage
  // The sums through LDS, 128 rows a pass: 64 of each group.  A lane of a 16 x 16 tile holds columns 4 (l/16)..+3 of
  // row l%16.
  float* sums = (float*)smem;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    __syncthreads();  // the ring, or the rows of the pass before, are read
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = GATED ? (j >> 1) * SUBN + w * 32 + (j & 1) * 16 : w * 64 + j * 16;
        *(f32x4*)(sums + (g * 64 + i * 16 + (lane & 15)) * LD + c + 4 * (lane >> 4)) = acc[4 * h + i][j];
      }
    __syncthreads();
    finish_rows<T, GATED, SUBN, LD, 512>(p, sums, ROWS, prod, split, n0, tid,
                                         [&](int r) { return (int64_t)m0 + (r >> 6) * 128 + h * 64 + (r & 63); });
  }
}

// ---- few rows: A of at most 16 MT rows -------------------------------------------------
//
// Bound by the bytes of B.  A workgroup takes CW columns (gated: of both weights) and a range of k, its four waves a
// quarter of that range each: a wave streams its stages (KB bytes of k) into a ring of its own, with no barrier in the
// loop, multiplies, and the waves add their sums through LDS at the end.  Few columns leave CUs idle: k is then split
// over workgroups too (p.splits) and the parts joined.  The weights go past the caches, in runs of 256 bytes of their
// rows (128: 15 % slower), or of 128 where they run along k.  1 x 14336 x 4096 f16 20 us and the join 4 (4.8 TB/s of
// weights); 16 x 4096 x 14336 gated 42 and 4.6 (5.0 TB/s; weights along k 36.6, 6.4 TB/s): what a CU takes, 31 bytes a ns,
// and CUs without columns keep it from HBM's 6.8.
//
// ANY: the stages go through registers, two of them ahead of the one that is multiplied, so operands may have any
// alignment and length.
template <typename T, bool BOUT, bool GATED, int MT, bool ANY>
static __global__ __launch_bounds__(256) void gemm_skinny(const GemmParams p) {
  constexpr int NSUB = GATED ? 2 : 1, CW = skinny_columns(BOUT), KB = skinny_bytes(BOUT);
  typedef Tile<T, false, 16 * MT, KB> TA;
  typedef Tile<T, BOUT, CW, KB> TB;
  typedef Mma<T> M;
  // GATED: a stage's two weights take two places of the ring, each beside the same rows of A
  constexpr int BK = TA::BK, PLACE = TA::BYTES + TB::BYTES, LOADS = TA::LOADS + TB::LOADS;
  constexpr int NST = ANY ? 1 : 16 * PLACE <= 160 * 1024 ? 4 : 12 * PLACE <= 160 * 1024 ? 3 : 2;
  constexpr int RING = NST * PLACE, W = 64, LD = NSUB * W + 4, NC = CW / 16, STEPS = KB / 64;
  constexpr int SUMS = 4 * 16 * MT * LD * 4, BYTES = 4 * RING > SUMS ? 4 * RING : SUMS;
  static_assert(BYTES <= 160 * 1024 && (NST - 1) * LOADS < 64, "LDS, and the loads that a wave can count");
  __shared__ __attribute__((aligned(1024))) char smem[BYTES];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int split = blockIdx.y, n0 = blockIdx.x * p.width, nend = p.n - n0 < p.width ? p.n : n0 + p.width;
  int lo, hi;
  stages_of(p, split, lo, hi);
  const int per = (hi - lo + 3) / 4;
  lo += wave * per;
  const int left = hi - lo < per ? hi - lo : per;
  const int places = left > 0 ? left * NSUB : 0;
  const int64_t mleft = p.m, nleft = nend - n0;
  char* ring = smem + wave * RING;
  int fa[MT], fb[NC];
#pragma unroll
  for (int i = 0; i < MT; ++i) fa[i] = TA::frag_offset(lane, 16 * i);
#pragma unroll
  for (int j = 0; j < NC; ++j) fb[j] = TB::frag_offset(lane, 16 * j);
  typedef f32x4 acc_t[MT][NSUB][NC];
  auto multiply = [&](const char* st, acc_t& acc, int u) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < STEPS; ++h) {
      typename M::frag a[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) a[i] = TA::read(st, fa[i], h);
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        const typename M::frag b = TB::read(st + TA::BYTES, fb[j], h);
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[i][u][j] = M::mma(b, a[i], acc[i][u][j]);
      }
    }
  };
  acc_t acc;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int u = 0; u < NSUB; ++u)
#pragma unroll
      for (int j = 0; j < NC; ++j) acc[i][u][j] = (f32x4){};
  if constexpr (ANY) {
    typedef typename Vec8<T>::type unit_t;  // a 16-byte chunk
    unit_t units[2][LOADS];
    // chunk `lane` of 1 KB piece q of a tile, wherever it lies in memory: its row, its first element in the row, and how
    // many of the row's elements are left from there
    auto fetch = [&](unit_t (&r)[LOADS], int s) __attribute__((always_inline)) {
      const int u = s % NSUB, at = lo + s / NSUB, seg = at >= p.kt ? 1 : 0, k0 = (at - (seg ? p.kt : 0)) * BK;
      const int64_t la = seg ? p.lda[1] : p.lda[0];
      const T* a = (const T*)(seg ? p.a[1] : p.a[0]);
#pragma unroll
      for (int i = 0; i < TA::LOADS; ++i) {
        int row, col;
        TA::chunk(i, lane, &row, &col);
        r[i] = raw8(a + (row < p.m ? row : 0) * la + k0 + col, row < p.m && k0 + col < p.k ? (p.k - k0 - col < 8 ? p.k - k0 - col : 8) : 0);
      }
      const int ib = GATED ? u : seg;
      const int64_t lb = ib ? p.ldb[1] : p.ldb[0];
      const T* b = (const T*)(ib ? p.b[1] : p.b[0]);
#pragma unroll
      for (int i = 0; i < TB::LOADS; ++i) {
        int row, col;
        TB::chunk(i, lane, &row, &col);
        const int64_t first = BOUT ? n0 + col : k0 + col, end = BOUT ? nend : p.k, outer = BOUT ? k0 + row : n0 + row;
        const bool in = outer < (BOUT ? p.k : nend) && first < end;
        r[TA::LOADS + i] = raw8(b + (in ? outer * lb + first : 0), in ? (int)(end - first < 8 ? end - first : 8) : 0);
      }
    };
    // The wave's LDS accesses run in order; the fences keep the compiler from moving one lane's read before another's
    // write.
    auto order = [&]() __attribute__((always_inline)) {
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    };
    auto place = [&](unit_t (&r)[LOADS], int s, int u) __attribute__((always_inline)) {
      order();
#pragma unroll
      for (int i = 0; i < LOADS; ++i) *(typename M::frag*)(ring + i * 1024 + lane * 16) = (typename M::frag)r[i];
      if (s + 2 < places) fetch(r, s + 2);
      order();
      multiply(ring, acc, u);
    };
    if (0 < places) fetch(units[0], 0);
    if (1 < places) fetch(units[1], 1);
#pragma unroll 1
    for (int s = 0; s < places; s += 2) {
      place(units[0], s, 0);
      if (s + 1 < places) place(units[1], s + 1, NSUB - 1);
    }
  } else {
  typename TA::Source sa;
  typename TB::Source sb[NSUB];
  uint32_t va[TA::LOADS], vb[NSUB][TB::LOADS];
  // The source of stage t on, where it changes: at a segment's first stage, and at its last one where that is not
  // whole.  `change`: the next such stage.
  int change = 0;
  auto set_source = [&](int t) __attribute__((always_inline)) {
    const int at = lo + t, seg = at >= p.kt ? 1 : 0, kt = at - (seg ? p.kt : 0), k0 = kt * BK;
    const int64_t la = seg ? p.lda[1] : p.lda[0];
    sa.set(seg ? p.a[1] : p.a[0], la, 0, mleft, p.k, k0);
#pragma unroll
    for (int i = 0; i < TA::LOADS; ++i) {
      int k;
      va[i] = TA::lane_offset(i, lane, la, mleft, &k);
      if (k0 + k >= p.k) va[i] = kOutside;
    }
#pragma unroll
    for (int u = 0; u < NSUB; ++u) {
      const int ib = GATED ? u : seg;
      const int64_t lb = ib ? p.ldb[1] : p.ldb[0];
      sb[u].set(ib ? p.b[1] : p.b[0], lb, n0, nleft, p.k, k0);
#pragma unroll
      for (int i = 0; i < TB::LOADS; ++i) {
        int k;
        vb[u][i] = TB::lane_offset(i, lane, lb, nleft, &k);
        if (!BOUT && k0 + k >= p.k) vb[u][i] = kOutside;
      }
    }
    const int whole = p.k / BK;
    change = kt < whole && whole < p.kt ? t + whole - kt : t + p.kt - kt;
  };
  const uint32_t lds = (uint32_t)(size_t)(EAS_LDS char*)ring;
  // place s of this wave: stage s / NSUB, weight u = s % NSUB
  auto dma = [&](int s, int u) __attribute__((always_inline)) {
    const uint32_t at = lds + (uint32_t)((s % NST) * PLACE);
    if (u == 0) {
      if (s / NSUB == change) {
        set_source(s / NSUB);
      } else {
        sa.next();
#pragma unroll
        for (int v = 0; v < NSUB; ++v) sb[v].next();
      }
    }
    const rsrc_t rb = sb[u].resource(true);
#pragma unroll
    for (int i = 0; i < TB::LOADS; ++i) dma16_stream(rb, vb[u][i], at + TA::BYTES + i * 1024);
    const rsrc_t ra = sa.resource(true);
#pragma unroll
    for (int i = 0; i < TA::LOADS; ++i) dma16(ra, va[i], at + i * 1024);
  };
  static_assert(NST - 1 <= 3, "places issued before the loop");
  if (0 < places) dma(0, 0);
  if (NST > 2 && 1 < places) dma(1, 1 % NSUB);
  if (NST > 3 && 2 < places) dma(2, 0);
#pragma unroll 1
  for (int s0 = 0; s0 < places; s0 += NSUB) {
#pragma unroll
    for (int u = 0; u < NSUB; ++u) {
      const int s = s0 + u;
      // this wave's place s landed; up to NST - 2 newer ones stay in flight
      const int later = places - 1 - s < NST - 2 ? places - 1 - s : NST - 2;
      if (later >= 2) __builtin_amdgcn_s_waitcnt(EAS_WAITVM(2 * LOADS));
      else if (later == 1) __builtin_amdgcn_s_waitcnt(EAS_WAITVM(LOADS));
      else __builtin_amdgcn_s_waitcnt(EAS_WAITVM(0));
      if (s + NST - 1 < places) dma(s + NST - 1, (u + NST - 1) % NSUB);  // refills the place read at step s - 1
      __builtin_amdgcn_sched_barrier(0);
      multiply(ring + (s % NST) * PLACE, acc, u);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  }
  float* sums = (float*)smem;  // [wave][16 MT][LD], 64 columns a pass
#pragma unroll
  for (int c0 = 0; c0 < CW; c0 += W) {
    __syncthreads();  // every wave is past its loop, or past the columns before
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int u = 0; u < NSUB; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *(f32x4*)(sums + (wave * 16 * MT + i * 16 + (lane & 15)) * LD + u * W + j * 16 + 4 * (lane >> 4)) = acc[i][u][c0 / 16 + j];
    __syncthreads();
    constexpr int PER = W / 8;
#pragma unroll 1
    for (int it = tid; it < 16 * MT * PER; it += 256) {
      const int r = it / PER, c = (it % PER) * 8;
      if (r >= p.m || n0 + c0 + c >= nend) continue;
      float z[8], u[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float* q = sums + r * LD + c + e;
        constexpr int S = 16 * MT * LD;
        z[e] = (q[0] + q[S]) + (q[2 * S] + q[3 * S]);
        u[e] = GATED ? (q[W] + q[W + S]) + (q[W + 2 * S] + q[W + 3 * S]) : 0.0f;
      }
      if (p.splits > 1) {
        store_part<GATED>(p, 0, split, r, n0 + c0 + c, z, u);
      } else {
        float bz[8], bu[8];
        load_bias<T, GATED>(p, n0 + c0 + c, bz, bu);
        finish8<T, GATED>(p, 0, r, n0 + c0 + c, z, u, bz, bu);
      }
    }
  }
}

// ---- the parts of a split k -----------------------------------------------------------
//
// One thread for 8 columns of a row, the parts added in the order of k.  Bound by a launch and a way to memory and back
// for few rows (3 to 5 us), by the parts' bytes else (2 x 2048 x 4096: 14.8 us, 5.4 TB/s).
template <typename T, bool GATED>
static __global__ __launch_bounds__(64) void gemm_join(const GemmParams p) {
  const int64_t per = (p.n + 7) / 8, total = per * p.m * p.prods;
  for (int64_t it = (int64_t)blockIdx.x * 64 + threadIdx.x; it < total; it += (int64_t)gridDim.x * 64) {
    const int prod = (int)(it / (per * p.m));
    const int64_t in = it - prod * per * p.m, row = in / per, col = (in % per) * 8;
    const int left = (int)(p.n - col < 8 ? p.n - col : 8);
    const int64_t rows = (int64_t)p.m * p.prods, ld = (int64_t)p.n * (GATED ? 2 : 1);
    const float* q = p.part + ((int64_t)prod * p.m + row) * ld + col;
    float z[8] = {}, u[8] = {};
    // four parts' loads at a time, added in the order of k
    for (int s = 0; s < p.splits; s += 4) {
      float t[4][8], v[4][8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int n = s + i < p.splits ? left : 0;
        load_upto8(q + (s + i) * rows * ld, n, t[i]);
        if constexpr (GATED) load_upto8(q + (s + i) * rows * ld + p.n, n, v[i]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          z[e] += t[i][e];
          if constexpr (GATED) u[e] += v[i][e];
        }
    }
    float bz[8], bu[8];
    load_bias<T, GATED>(p, col, bz, bu);
    finish8<T, GATED>(p, prod, row, col, z, u, bz, bu);
  }
}

// ---- launchers ------------------------------------------------------------------------

template <typename T, bool AOUT, bool BOUT, bool GATED>
static hipError_t launch_form(GemmKernel kernel, bool any, const GemmParams& p, hipStream_t stream) {
  const dim3 tiles(p.tiles_m * p.tiles_n, p.prods * p.splits);
  switch (kernel) {
    case kGemmTile64:
      if constexpr (GATED) gemm_tile<T, AOUT, BOUT, true, 64, 128><<<tiles, 512, 0, stream>>>(p);
      else gemm_tile<T, AOUT, BOUT, false, 64, 64><<<tiles, 512, 0, stream>>>(p);
      break;
    case kGemmTile128:
      gemm_tile<T, AOUT, BOUT, GATED, 128, 128><<<tiles, 512, 0, stream>>>(p);
      break;
    case kGemmTile256:
      if constexpr (sizeof(T) == 2) gemm_tile256<T, AOUT, BOUT, GATED><<<tiles, 512, 0, stream>>>(p);
      else return hipErrorInvalidValue;
      break;
    default:
      if constexpr (!AOUT) {
        const dim3 grid(p.tiles_n, p.splits);
        if constexpr (sizeof(T) == 2) {
          if (any) {
            if (kernel == kGemmSkinny1) gemm_skinny<T, BOUT, GATED, 1, true><<<grid, 256, 0, stream>>>(p);
            else if (kernel == kGemmSkinny2) gemm_skinny<T, BOUT, GATED, 2, true><<<grid, 256, 0, stream>>>(p);
            else gemm_skinny<T, BOUT, GATED, 4, true><<<grid, 256, 0, stream>>>(p);
            break;
          }
        }
        if (kernel == kGemmSkinny1) gemm_skinny<T, BOUT, GATED, 1, false><<<grid, 256, 0, stream>>>(p);
        else if (kernel == kGemmSkinny2) gemm_skinny<T, BOUT, GATED, 2, false><<<grid, 256, 0, stream>>>(p);
        else gemm_skinny<T, BOUT, GATED, 4, false><<<grid, 256, 0, stream>>>(p);
        break;
      }
      return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

template <typename T>
hipError_t gemm_launch_typed(GemmKernel kernel, const GemmForm& f, const GemmParams& p, hipStream_t stream) {
  if (f.gated) {
    if (f.a_outer) return hipErrorInvalidValue;
    return f.b_outer ? launch_form<T, false, true, true>(kernel, f.any, p, stream) : launch_form<T, false, false, true>(kernel, f.any, p, stream);
  }
  if (f.a_outer) return f.b_outer ? launch_form<T, true, true, false>(kernel, f.any, p, stream) : hipErrorInvalidValue;
  return f.b_outer ? launch_form<T, false, true, false>(kernel, f.any, p, stream) : launch_form<T, false, false, false>(kernel, f.any, p, stream);
}

template <typename T>
hipError_t gemm_pair_typed(bool b_outer, const GemmParams& dx, const GemmParams& dw, hipStream_t stream) {
  const unsigned grid = (unsigned)(dx.tiles_m * dx.tiles_n * dx.splits + dw.tiles_m * dw.tiles_n * dw.prods * dw.splits);
  if (b_outer) gemm_pair<T, true><<<grid, 512, 0, stream>>>(dx, dw);
  else gemm_pair<T, false><<<grid, 512, 0, stream>>>(dx, dw);
  return hipGetLastError();
}

template <typename T> hipError_t gemm_join_typed(bool gated, const GemmParams& p, hipStream_t stream) {
  const int64_t items = (int64_t)p.m * p.prods * ((p.n + 7) / 8);
  const unsigned blocks = (unsigned)((items + 63) / 64 < 16384 ? (items + 63) / 64 : 16384);
  if (gated) gemm_join<T, true><<<blocks, 64, 0, stream>>>(p);
  else gemm_join<T, false><<<blocks, 64, 0, stream>>>(p);
  return hipGetLastError();
}

}  // namespace eas

#endif  // EAS_OPS_GEMM_H
