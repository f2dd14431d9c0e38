// elementwise.hip — the pass before the matrix products (the epilogues' gradients with their sums over rows, operands
// moved to aligned rows) and the sums' second stage.
#include "device.h"

namespace eas {

// ---- before the products: gradients of the epilogues, and aligned copies ---------------
//
// One launch for both, which are independent: the first p.dz_groups workgroups take dz, the others copy.
//
// dz.  linear: dz = dy act'(z); gated: dg = dy u act'(g), du = dy act(g).  tx threads along a row, 8 columns each, and ty
// = 256 / tx rows at a time; a workgroup takes one chunk of rows, and its sums over them meet across lanes, then waves.
// dz's rows are 16-byte aligned, and zero from n to the next multiple of 8, as the products read them.  16-bit operands
// round dz to their type, which the matrix cores multiply; the sums over rows take it unrounded.  Against 64 bits the
// gradients are then off by 2.3e-3 (bf16) and 2.9e-4 (f16) in the 2-norm, the rounding of dz as much as that of the
// result, 1.7e-3 and 2.1e-4 alone; the low half of dz as a second segment would halve the products' rate (4096^3
// linear_backward: 229 us of 255 are products).  An f16 dz is
// infinite beyond 65504 and loses digits below 6e-5.  Bound by memory: gated 2048x14336 bf16 52.6 us (5.6 TB/s), 4096x4096 bf16 gelu 21.5 us (4.7 TB/s).  Two rows ahead; one took 23.9 us for
// the latter, four 21.9.  Even rows as buffers, with no branch around their loads: 23.1 -> 21.5.  Few rows are bound by a
// load's way there and back, and take all rows in one chunk, on strips of as little as 8 columns; neighbouring strips go
// to one XCD, whose L2 then holds the lines that they share (517x2048 f16 with sums 11.6 -> 8.8 us).
//
// Copies.  One thread per 8 elements of a destination row; reads at any alignment, writes at 16 bytes.  Four vectors a
// thread, all loads first, were slower (500x4097x4097 bf16 53.1 -> 54.6 us with its product).
//
// FORM: kAny rows, or even ones, a wave's whole 512 columns of each, read through the caches (kEven) or past them (kStream)
enum { kAny, kEven, kStream };
template <typename T, bool GATED, int FORM>
static __device__ __forceinline__ void dz_part(const PrepareParams& p, float* sums) {
  const int tx = p.tx, ty = 256 / tx, x = threadIdx.x % tx, y = threadIdx.x / tx;
  int across = blockIdx.x % p.across;
  const int chunk = blockIdx.x / p.across;
  if (p.chunks == 1) across = across % 8 * (p.across / 8) + across / 8;  // across is a multiple of 8 then
  const int64_t col = ((int64_t)across * tx + x) * 8;
  const int left = col < p.n ? (p.n - col < 8 ? (int)(p.n - col) : 8) : 0;
  float sg[8] = {}, su[8] = {};
  const int64_t r0 = (int64_t)chunk * p.rows_per_chunk, r1 = r0 + p.rows_per_chunk < p.m ? r0 + p.rows_per_chunk : p.m;
  constexpr int AHEAD = 2;
  typedef typename Vec8<T>::type raw_t;
  // one row's gradients, from what was read of it
  auto row = [&](const raw_t& dy, const raw_t& z, const raw_t& w, float (&g)[8], float (&u)[8]) __attribute__((always_inline)) {
    float d[8], f[8], a[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      d[e] = (float)dy[e];
      if (GATED || p.pre[0]) g[e] = (float)z[e];
      if (GATED) u[e] = (float)w[e];
    }
    if (GATED || p.pre[0]) activate_grad8<sizeof(T) == 2>(p.act, g, f, a);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (GATED) {
        g[e] = d[e] * u[e] * a[e];
        u[e] = d[e] * f[e];
        su[e] += u[e];
      } else {
        g[e] = p.pre[0] ? d[e] * a[e] : d[e];
      }
      sg[e] += g[e];
    }
  };
  if constexpr (FORM != kAny) {
    // the next two rows' loads are always under way
    const int64_t first = r0 + __builtin_amdgcn_readfirstlane(threadIdx.x / 64), wide = (p.n + 7) / 8 * 8;
    raw_t dy[AHEAD], z[AHEAD], w[AHEAD];
    auto fetch = [&](int i, int64_t r) __attribute__((always_inline)) {
      dy[i] = row_load<T, true, FORM == kStream>((const T*)p.dy + r * p.dy_ld, p.n, r < r1, (int)col, left);
      z[i] = row_load<T, true, FORM == kStream>((const T*)p.pre[0] + r * p.pre_ld[0], p.n, r < r1 && (GATED || p.pre[0]), (int)col, left);
      if (GATED) w[i] = row_load<T, true, FORM == kStream>((const T*)p.pre[1] + r * p.pre_ld[1], p.n, r < r1, (int)col, left);
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      fetch(i, first + i * 4);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll 1
    for (int64_t r = first; r < r1; r += 4 * AHEAD)
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int64_t at = r + 4 * i;
        float g[8], u[8];
        row(dy[i], z[i], w[i], g, u);
        fetch(i, at + 4 * AHEAD);
        row_store<T, true>((T*)p.dz[0] + at * p.dz_ld, wide, at < r1 && p.dz[0], (int)col, 8, false, g);
        if (GATED) row_store<T, true>((T*)p.dz[1] + at * p.dz_ld, wide, at < r1 && p.dz[0], (int)col, 8, false, u);
      }
  } else if (left > 0) {
    // both rows' loads are under way before the first is used
    for (int64_t r = r0 + y; r < r1; r += AHEAD * ty) {
      raw_t dy[AHEAD], z[AHEAD], w[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int64_t at = r + i * ty;
        const int n = at < r1 ? left : 0;
        dy[i] = raw8((const T*)p.dy + at * p.dy_ld + col, n);
        if (GATED || p.pre[0]) z[i] = raw8((const T*)p.pre[0] + at * p.pre_ld[0] + col, n);
        if (GATED) w[i] = raw8((const T*)p.pre[1] + at * p.pre_ld[1] + col, n);
      }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int64_t at = r + i * ty;
        if (at >= r1) break;
        float g[8], u[8];
        row(dy[i], z[i], w[i], g, u);
        if (p.dz[0]) {  // columns past n are zero: dy's zeros times finite factors
          store8((T*)p.dz[0] + at * p.dz_ld + col, g);
          if (GATED) store8((T*)p.dz[1] + at * p.dz_ld + col, u);
        }
      }
    }
  }
  if (!p.part && !p.sum[0]) return;
  // the lanes of a wave that hold the same columns, then the four waves; the same order on every run
  constexpr int SUMS = GATED ? 2 : 1;
  for (int o = tx; o < 64; o *= 2)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      sg[e] += __shfl_xor(sg[e], o);
      if (GATED) su[e] += __shfl_xor(su[e], o);
    }
  const int columns = 8 * tx, wave = threadIdx.x / 64;
  if ((int)(threadIdx.x % 64) < tx)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      sums[wave * columns + x * 8 + e] = sg[e];
      if (GATED) sums[(4 + wave) * columns + x * 8 + e] = su[e];
    }
  __syncthreads();
  for (int i = threadIdx.x; i < columns * SUMS; i += 256) {
    const int w = i >= columns, j = i - w * columns;
    const float* from = sums + 4 * w * columns + j;
    const float s = (from[0] + from[columns]) + (from[2 * columns] + from[3 * columns]);
    const int64_t c = (int64_t)across * columns + j;
    if (c < p.n) {
      if (p.part) p.part[((int64_t)chunk * SUMS + w) * p.n + c] = s;
      else if (p.sum_wide) ((float*)p.sum[w])[c] = s;
      else ((T*)p.sum[w])[c] = (T)s;
    }
  }
}

template <typename T, bool GATED, int FORM>
static __global__ __launch_bounds__(256) void prepare(const PrepareParams p) {
  __shared__ float sums[(GATED ? 8 : 4) * 64 * 8];
  if ((int)blockIdx.x < p.dz_groups) {
    dz_part<T, GATED, FORM>(p, sums);
    return;
  }
  typedef T aligned_t __attribute__((ext_vector_type(8)));
  const int64_t step = (int64_t)(gridDim.x - p.dz_groups) * 256;
  int64_t it = (int64_t)(blockIdx.x - p.dz_groups) * 256 + threadIdx.x;
#pragma unroll
  for (int w = 0; w < 3; ++w) {
    if (w >= p.copies) break;
    const int64_t per = p.dst_ld[w] / 8, total = per * p.rows[w];
    for (; it < total; it += step) {
      const int64_t r = total >> 32 ? it / per : (uint32_t)it / (uint32_t)per, c = (it - r * per) * 8;
      *(aligned_t*)((T*)p.dst[w] + r * p.dst_ld[w] + c) =
          raw8((const T*)p.src[w] + r * p.src_ld[w] + c, c < p.cols[w] ? (int)(p.cols[w] - c < 8 ? p.cols[w] - c : 8) : 0);
    }
    it -= total;  // the next matrix's items follow on
  }
}

template <typename T> static void prepare_typed(int form, unsigned grid, const PrepareParams& p, hipStream_t stream) {
  if (p.gated) {
    if (form == kAny) prepare<T, true, kAny><<<grid, 256, 0, stream>>>(p);
    else if (form == kEven) prepare<T, true, kEven><<<grid, 256, 0, stream>>>(p);
    else prepare<T, true, kStream><<<grid, 256, 0, stream>>>(p);
  } else {
    if (form == kAny) prepare<T, false, kAny><<<grid, 256, 0, stream>>>(p);
    else if (form == kEven) prepare<T, false, kEven><<<grid, 256, 0, stream>>>(p);
    else prepare<T, false, kStream><<<grid, 256, 0, stream>>>(p);
  }
}

hipError_t prepare_launch(PrepareParams p, hipStream_t stream) {
  int64_t items = 0;
  for (int i = 0; i < p.copies; ++i) items += p.dst_ld[i] / 8 * p.rows[i];
  const int64_t copiers = (items + 255) / 256 < 8192 ? (items + 255) / 256 : 8192;
  p.dz_groups = p.chunks * p.across;
  const unsigned grid = (unsigned)(p.dz_groups + copiers);
  if (!grid) return hipSuccess;
  const int form = p.tx != 64 || p.n > (1 << 28) || !even_rows(p.dy, p.dy_ld, p.n) || !even_rows(p.pre[0], p.pre_ld[0], p.n) ||
                           !even_rows(p.pre[1], p.pre_ld[1], p.n)
                       ? (int)kAny
                       : p.stream ? (int)kStream : (int)kEven;
  if (p.dtype == EAS_HIP_F16) prepare_typed<f16>(form, grid, p, stream);
  else if (p.dtype == EAS_HIP_BF16) prepare_typed<bf16>(form, grid, p, stream);
  else prepare_typed<float>(form, grid, p, stream);
  return hipGetLastError();
}

// ---- sums over chunks ---------------------------------------------------------------
//
// A workgroup sums 32 columns: 32 threads of each take every 32nd chunk, four loads ahead, then meet in LDS; always in
// the same order.
template <typename T>
static __global__ __launch_bounds__(1024) void column_sum(const ColumnSumParams p) {
  __shared__ float sums[32][33];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int64_t total = (int64_t)p.n * p.outs;
  for (int64_t first = (int64_t)blockIdx.x * 32; first < total; first += (int64_t)gridDim.x * 32) {
    const int64_t c = first + x;
    float s[4] = {};
    if (c < total) {
      int k = y;
      for (; k + 96 < p.chunks; k += 128)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] += p.part[(k + 32 * i) * total + c];
      for (; k < p.chunks; k += 32) s[0] += p.part[k * total + c];
    }
    sums[y][x] = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    if (y == 0 && c < total) {
      float v = 0.0f;
#pragma unroll
      for (int k = 0; k < 32; ++k) v += sums[k][x];
      T* out = (T*)(c < p.n ? p.out[0] : p.out[1]);
      if (out) out[c < p.n ? c : c - p.n] = (T)v;
    }
    __syncthreads();  // the sums are read
  }
}

hipError_t column_sum_launch(const ColumnSumParams& p, hipStream_t stream) {
  const int64_t groups = ((int64_t)p.n * p.outs + 31) / 32;
  const unsigned blocks = (unsigned)(groups < (1 << 20) ? groups : 1 << 20);  // a grid holds fewer than 2^32 threads
  if (p.dtype == EAS_HIP_F16) column_sum<f16><<<blocks, 1024, 0, stream>>>(p);
  else if (p.dtype == EAS_HIP_BF16) column_sum<bf16><<<blocks, 1024, 0, stream>>>(p);
  else column_sum<float><<<blocks, 1024, 0, stream>>>(p);
  return hipGetLastError();
}

}  // namespace eas
