// elementwise.hip — the passes around the matrix products: operands moved to aligned rows, the epilogues' gradients
// with their sums over rows, and the sums' second stage.
#include "device.h"

namespace eas {

// ---- aligned copies ---------------------------------------------------------------
//
// One thread per 8 elements of a destination row; reads at any alignment, writes at 16 bytes.
template <typename T>
static __global__ __launch_bounds__(256) void realign(const RealignParams p) {
  const int w = blockIdx.y;
  const T* src = (const T*)(w == 0 ? p.src[0] : w == 1 ? p.src[1] : p.src[2]);
  T* dst = (T*)(w == 0 ? p.dst[0] : w == 1 ? p.dst[1] : p.dst[2]);
  const int64_t src_ld = w == 0 ? p.src_ld[0] : w == 1 ? p.src_ld[1] : p.src_ld[2];
  const int64_t dst_ld = w == 0 ? p.dst_ld[0] : w == 1 ? p.dst_ld[1] : p.dst_ld[2];
  const int rows = w == 0 ? p.rows[0] : w == 1 ? p.rows[1] : p.rows[2];
  const int cols = w == 0 ? p.cols[0] : w == 1 ? p.cols[1] : p.cols[2];
  const int64_t per = dst_ld / 8, total = per * rows;
  for (int64_t it = (int64_t)blockIdx.x * 256 + threadIdx.x; it < total; it += (int64_t)gridDim.x * 256) {
    const int64_t r = it / per, c = (it % per) * 8;
    typename Vec8<T>::type v = {};
    const T* s = src + r * src_ld + c;
    if (c + 8 <= cols) {
      v = *(const typename Vec8<T>::type*)s;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c + e < cols) v[e] = s[e];
    }
    typedef T aligned_t __attribute__((ext_vector_type(8)));
    *(aligned_t*)(dst + r * dst_ld + c) = v;
  }
}

hipError_t realign_launch(const RealignParams& p, int dtype, hipStream_t stream) {
  int64_t most = 0;
  for (int i = 0; i < p.count; ++i) {
    const int64_t items = p.dst_ld[i] / 8 * p.rows[i];
    most = items > most ? items : most;
  }
  if (!most) return hipSuccess;
  const int64_t blocks = (most + 255) / 256;
  const dim3 grid((unsigned)(blocks < 8192 ? blocks : 8192), p.count);
  if (dtype == EAS_HIP_F32) realign<float><<<grid, 256, 0, stream>>>(p);
  else realign<f16><<<grid, 256, 0, stream>>>(p);  // the bits of either 16-bit type
  return hipGetLastError();
}

// ---- gradients of the epilogues ------------------------------------------------------
//
// linear: dz = dy act'(z).  gated: dg = dy u act'(g), du = dy act(g).  TX threads along a row, 8 columns each, and
// 256 / TX rows at a time; a workgroup takes one chunk of rows, and its sums over them meet in LDS.  dz's rows are
// 16-byte aligned, and zero from n to the next multiple of 8, as the products read them.
template <typename T, bool GATED>
static __global__ __launch_bounds__(256) void dz_kernel(const DzParams p, int tx) {
  __shared__ float sums[256 * 8];
  const int x = threadIdx.x % tx, y = threadIdx.x / tx, ty = 256 / tx;
  const int64_t col = ((int64_t)blockIdx.x * tx + x) * 8;
  const int left = col < p.n ? (p.n - col < 8 ? (int)(p.n - col) : 8) : 0;
  float sg[8] = {}, su[8] = {};
  if (left > 0) {
    const int64_t r0 = (int64_t)blockIdx.y * p.rows_per_chunk, r1 = r0 + p.rows_per_chunk < p.m ? r0 + p.rows_per_chunk : p.m;
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
  if (!p.part) return;
#pragma unroll
  for (int w = 0; w < (GATED ? 2 : 1); ++w) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[(y * 8 + e) * tx + x] = w ? su[e] : sg[e];
    __syncthreads();
    // column e of thread x: entries [row group][e][x]
    for (int i = threadIdx.x; i < 8 * tx; i += 256) {
      const int e = i / tx, xx = i % tx;
      float s = 0.0f;
      for (int k = 0; k < ty; ++k) s += sums[(k * 8 + e) * tx + xx];
      const int64_t c = ((int64_t)blockIdx.x * tx + xx) * 8 + e;
      if (c < p.n) p.part[((int64_t)blockIdx.y * (GATED ? 2 : 1) + w) * p.n + c] = s;
    }
  }
}

template <typename T> static void dz_typed(const DzParams& p, dim3 grid, int tx, hipStream_t stream) {
  if (p.gated) dz_kernel<T, true><<<grid, 256, 0, stream>>>(p, tx);
  else dz_kernel<T, false><<<grid, 256, 0, stream>>>(p, tx);
}

hipError_t dz_launch(const DzParams& p, hipStream_t stream) {
  const int vecs = (p.n + 7) / 8;
  int tx = 64;
  while (tx > 8 && tx / 2 >= vecs) tx /= 2;
  const dim3 grid((vecs + tx - 1) / tx, p.chunks);
  if (p.dtype == EAS_HIP_F16) dz_typed<f16>(p, grid, tx, stream);
  else if (p.dtype == EAS_HIP_BF16) dz_typed<bf16>(p, grid, tx, stream);
  else dz_typed<float>(p, grid, tx, stream);
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
