// elementwise.hip — the pass before the matrix products (the epilogues' gradients with their sums over rows, operands
// moved to aligned rows) and the sums' second stage.
#include "device.h"

namespace eas {

// ---- before the products: gradients of the epilogues, and aligned copies ---------------
//
// One launch for both, which are independent: the first p.dz_groups workgroups take dz, the others copy.
//
// dz.  linear: dz = dy act'(z); gated: dg = dy u act'(g), du = dy act(g).  tx threads along a row, 8 columns each, and ty
// = 256 / tx rows at a time; a workgroup takes one chunk of rows, and its sums over them meet in LDS.  dz's rows are
// 16-byte aligned, and zero from n to the next multiple of 8, as the products read them.
//
// Copies.  One thread per 8 elements of a destination row; reads at any alignment, writes at 16 bytes.
template <typename T, bool GATED>
static __device__ __forceinline__ void dz_part(const PrepareParams& p, float* sums, float* half) {
  const int tx = p.tx, ty = 256 / tx, x = threadIdx.x % tx, y = threadIdx.x / tx;
  const int across = blockIdx.x % p.across, chunk = blockIdx.x / p.across;
  const int64_t col = ((int64_t)across * tx + x) * 8;
  const int left = col < p.n ? (p.n - col < 8 ? (int)(p.n - col) : 8) : 0;
  float sg[8] = {}, su[8] = {};
  if (left > 0) {
    const int64_t r0 = (int64_t)chunk * p.rows_per_chunk, r1 = r0 + p.rows_per_chunk < p.m ? r0 + p.rows_per_chunk : p.m;
#pragma unroll 2
    for (int64_t r = r0 + y; r < r1; r += ty) {
      float d[8], g[8], f[8], a[8];
      load_upto8((const T*)p.dy + r * p.dy_ld + col, left, d);
      if (GATED || p.pre[0]) {
        load_upto8((const T*)p.pre[0] + r * p.pre_ld[0] + col, left, g);
        activate_grad8<sizeof(T) == 2>(p.act, g, f, a);
      }
      if constexpr (GATED) {
        float u[8];
        load_upto8((const T*)p.pre[1] + r * p.pre_ld[1] + col, left, u);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          g[e] = d[e] * u[e] * a[e];
          u[e] = d[e] * f[e];
          sg[e] += g[e];
          su[e] += u[e];
        }
        if (p.dz[0]) {  // columns past n are zero: dy's zeros times finite factors
          store8((T*)p.dz[0] + r * p.dz_ld + col, g);
          store8((T*)p.dz[1] + r * p.dz_ld + col, u);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          g[e] = p.pre[0] ? d[e] * a[e] : d[e];
          sg[e] += g[e];
        }
        if (p.dz[0]) store8((T*)p.dz[0] + r * p.dz_ld + col, g);
      }
    }
  }
  if (!p.part && !p.sum[0]) return;
  // `each` threads add a column's ty sums, then one adds theirs; the same order on every run
  const int columns = 8 * tx, each = columns < 256 ? 256 / columns : 1;
#pragma unroll
  for (int w = 0; w < (GATED ? 2 : 1); ++w) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[y * columns + e * tx + x] = w ? su[e] : sg[e];
    __syncthreads();
    for (int i = threadIdx.x; i < columns * each; i += 256) {
      float s = 0.0f;
      for (int k = i / columns; k < ty; k += each) s += sums[k * columns + i % columns];
      if (each > 1) half[i] = s;
      else sums[i] = s;  // its own column's first place, which no other thread reads
    }
    __syncthreads();
    for (int i = threadIdx.x; i < columns; i += 256) {
      float s = each > 1 ? 0.0f : sums[i];
      if (each > 1)
        for (int k = 0; k < each; ++k) s += half[k * columns + i];
      const int64_t c = ((int64_t)across * tx + i % tx) * 8 + i / tx;
      if (c < p.n) {
        if (p.part) {
          p.part[((int64_t)chunk * (GATED ? 2 : 1) + w) * p.n + c] = s;
        } else if (p.sum_wide) {
          ((float*)p.sum[w])[c] = s;
        } else {
          ((T*)p.sum[w])[c] = (T)s;
        }
      }
    }
  }
}

template <typename T, bool GATED>
static __global__ __launch_bounds__(256) void prepare(const PrepareParams p) {
  __shared__ float sums[256 * 8], half[256];
  if ((int)blockIdx.x < p.dz_groups) {
    dz_part<T, GATED>(p, sums, half);
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
      const int64_t r = it / per, c = (it % per) * 8;
      *(aligned_t*)((T*)p.dst[w] + r * p.dst_ld[w] + c) =
          raw8((const T*)p.src[w] + r * p.src_ld[w] + c, c < p.cols[w] ? (int)(p.cols[w] - c < 8 ? p.cols[w] - c : 8) : 0);
    }
    it -= total;  // the next matrix's items follow on
  }
}

hipError_t prepare_launch(PrepareParams p, hipStream_t stream) {
  int64_t items = 0;
  for (int i = 0; i < p.copies; ++i) items += p.dst_ld[i] / 8 * p.rows[i];
  const int64_t copiers = (items + 255) / 256 < 8192 ? (items + 255) / 256 : 8192;
  p.dz_groups = p.chunks * p.across;
  const unsigned grid = (unsigned)(p.dz_groups + copiers);
  if (!grid) return hipSuccess;
  if (p.dtype == EAS_HIP_F16) {
    if (p.gated) prepare<f16, true><<<grid, 256, 0, stream>>>(p);
    else prepare<f16, false><<<grid, 256, 0, stream>>>(p);
  } else if (p.dtype == EAS_HIP_BF16) {
    if (p.gated) prepare<bf16, true><<<grid, 256, 0, stream>>>(p);
    else prepare<bf16, false><<<grid, 256, 0, stream>>>(p);
  } else {
    if (p.gated) prepare<float, true><<<grid, 256, 0, stream>>>(p);
    else prepare<float, false><<<grid, 256, 0, stream>>>(p);
  }
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
  const int64_t total = (int64_t)p.n * p.outs, c = (int64_t)blockIdx.x * 32 + x;
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
}

hipError_t column_sum_launch(const ColumnSumParams& p, hipStream_t stream) {
  const unsigned blocks = (unsigned)(((int64_t)p.n * p.outs + 31) / 32);
  if (p.dtype == EAS_HIP_F16) column_sum<f16><<<blocks, 1024, 0, stream>>>(p);
  else if (p.dtype == EAS_HIP_BF16) column_sum<bf16><<<blocks, 1024, 0, stream>>>(p);
  else column_sum<float><<<blocks, 1024, 0, stream>>>(p);
  return hipGetLastError();
}

}  // namespace eas
