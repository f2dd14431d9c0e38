// quantize.hip — matrices to 8 bits with a scale for each block: of a row, of a column, or 128 x 128.
//
// v = act(x), or act(gate) x, in 32 bits, held in registers between the search for a block's largest magnitude and its
// conversion: one read, one write.  A workgroup takes 128 columns of up to 128 rows, 16 threads of 8 columns by 16 rows
// at a time; a row's block is 16 neighbouring lanes, a column's meets through LDS.  Bound by memory.
#include "e4m3.h"

namespace eas {

enum QuantizeBlocks { kBlockRows, kBlockColumns, kBlockSquares };

// TURNS: rows of a thread, 16 apart
template <typename T, QuantizeBlocks BLOCKS, int TURNS>
static __device__ __forceinline__ void quantize_one(const eas_hip_quantize_args& p, int64_t by, int64_t bx) {
  const int x = threadIdx.x & 15, y = threadIdx.x >> 4, wave = threadIdx.x >> 6;
  const int64_t r0 = by * 16 * TURNS, c = bx * kBlock + x * 8;
  const int left = c < p.n ? (p.n - c < 8 ? (int)(p.n - c) : 8) : 0;
  float v[TURNS][8];
  {
    typename Vec8<T>::type a[TURNS], g[TURNS];
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
      const int64_t r = r0 + 16 * i + y;
      a[i] = raw8((const T*)p.x + r * p.x_ld + c, r < p.m ? left : 0);
      g[i] = raw8((const T*)p.gate + r * p.gate_ld + c, r < p.m && p.gate ? left : 0);
    }
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
      float z[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[i][e] = (float)a[i][e];
        z[e] = p.gate ? (float)g[i][e] : v[i][e];
      }
      activate8<sizeof(T) == 2>(p.activation, z);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = p.gate ? z[e] * v[i][e] : z[e];
    }
  }
  if constexpr (BLOCKS == kBlockRows) {
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
      const int64_t r = r0 + 16 * i + y;
      const float scale = scale_of(max16(amax8(v[i], 0.0f)));
      const u32x2 q = to_e4m3(v[i], scale, 1.0f / scale);
      if (r < p.m) {
        store_bytes((uint8_t*)p.q + r * p.q_ld + c, left, q);
        if (x == 0) p.scale[r * p.scale_row + bx * p.scale_col] = scale;
      }
    }
  } else if constexpr (BLOCKS == kBlockSquares) {
    __shared__ float most[4];
    float a = 0.0f;
#pragma unroll
    for (int i = 0; i < TURNS; ++i) a = amax8(v[i], a);
    a = max16(a);
    a = fmaxf(a, __shfl_xor(a, 16));
    a = fmaxf(a, __shfl_xor(a, 32));
    if ((threadIdx.x & 63) == 0) most[wave] = a;
    __syncthreads();
    const float scale = scale_of(fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]))), inverse = 1.0f / scale;
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
      const int64_t r = r0 + 16 * i + y;
      const u32x2 q = to_e4m3(v[i], scale, inverse);
      if (r < p.m) store_bytes((uint8_t*)p.q + r * p.q_ld + c, left, q);
    }
    if (threadIdx.x == 0) p.scale[by * p.scale_row + bx * p.scale_col] = scale;
  } else {
    __shared__ float most[4][kBlock];
    float a[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      a[e] = 0.0f;
#pragma unroll
      for (int i = 0; i < TURNS; ++i) a[e] = fmaxf(a[e], is_finite(v[i][e]) ? fabsf(v[i][e]) : 0.0f);
      a[e] = fmaxf(a[e], __shfl_xor(a[e], 16));
      a[e] = fmaxf(a[e], __shfl_xor(a[e], 32));
    }
    if ((threadIdx.x & 63) < 16) {
#pragma unroll
      for (int e = 0; e < 8; ++e) most[wave][x * 8 + e] = a[e];
    }
    __syncthreads();
    float scale[8], inverse[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int k = x * 8 + e;
      scale[e] = scale_of(fmaxf(fmaxf(most[0][k], most[1][k]), fmaxf(most[2][k], most[3][k])));
      inverse[e] = 1.0f / scale[e];
    }
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
      const int64_t r = r0 + 16 * i + y;
      const u32x2 q = to_e4m3(v[i], scale, inverse);
      if (r < p.m) store_bytes((uint8_t*)p.q + r * p.q_ld + c, left, q);
    }
    if (y == 0)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < left) p.scale[by * p.scale_row + (c + e) * p.scale_col] = scale[e];
  }
}

template <typename T, QuantizeBlocks BLOCKS, int TURNS>
static __global__ __launch_bounds__(256) void quantize_tiles(const eas_hip_quantize_args p) {
  const int64_t across = (p.n + kBlock - 1) / kBlock, total = across * ((p.m + 16 * TURNS - 1) / (16 * TURNS));
  for (int64_t it = blockIdx.x; it < total; it += gridDim.x) {
    if (BLOCKS != kBlockRows && it != blockIdx.x) __syncthreads();  // the tile before is done with LDS
    const int64_t by = it / across;
    quantize_one<T, BLOCKS, TURNS>(p, by, it - by * across);
  }
}

template <typename T> static void quantize_typed(const eas_hip_quantize_args& a, hipStream_t stream) {
  const int64_t tiles = ((a.n + kBlock - 1) / kBlock) * ((a.m + kBlock - 1) / kBlock);
  const unsigned grid = (unsigned)(tiles < (1 << 20) ? tiles : 1 << 20);
  if (a.block_m == 1) quantize_tiles<T, kBlockRows, 8><<<grid, 256, 0, stream>>>(a);
  else if (a.block_n == 1) quantize_tiles<T, kBlockColumns, 8><<<grid, 256, 0, stream>>>(a);
  else quantize_tiles<T, kBlockSquares, 8><<<grid, 256, 0, stream>>>(a);
}

hipError_t quantize_launch(const eas_hip_quantize_args& a, hipStream_t stream) {
  if (a.dtype == EAS_HIP_F16) quantize_typed<f16>(a, stream);
  else if (a.dtype == EAS_HIP_BF16) quantize_typed<bf16>(a, stream);
  else quantize_typed<float>(a, stream);
  return hipGetLastError();
}

}  // namespace eas
