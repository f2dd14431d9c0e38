// quantize.hip — matrices to 8 bits with a scale for each block: of a row, of a column, or 128 x 128.
//
// v = act(x), or act(gate) x, in 32 bits, held in registers between the search for a block's largest magnitude and its
// conversion: one read, one write.  A workgroup takes a strip of columns, XT threads of 8 across and NT / XT rows at a time,
// TURNS times: a row's block is 16 neighbouring lanes, a column's or a square's meets through LDS.  Bound by memory: 2048 x
// 14336 bf16 silu(gate) * x by rows 30.0 us (4.9 TB/s), 4099 x 4096 bf16 by columns 13.6 (3.7).
#include "e4m3.h"

namespace eas {

enum QuantizeBlocks { kBlockRows, kBlockColumns, kBlockSquares };

template <typename T, QuantizeBlocks BLOCKS, int NT, int XT, int TURNS>
static __device__ __forceinline__ void quantize_one(const eas_hip_quantize_args& p, int64_t by, int64_t bx) {
  constexpr int STEP = NT / XT, WAVES = NT / 64;
  static_assert(BLOCKS == kBlockRows || STEP * TURNS == kBlock, "a block's rows are one workgroup's");
  static_assert(BLOCKS == kBlockColumns || XT * 8 == kBlock, "a block's columns are one workgroup's");
  const int x = threadIdx.x % XT, y = threadIdx.x / XT, wave = threadIdx.x >> 6;
  const int64_t r0 = by * STEP * TURNS, c = (bx * XT + x) * 8;
  const int left = c < p.n ? (p.n - c < 8 ? (int)(p.n - c) : 8) : 0;
  float v[TURNS][8];
  {
    typename Vec8<T>::type a[TURNS], g[TURNS];
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
      const int64_t r = r0 + STEP * i + y;
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
      const int64_t r = r0 + STEP * i + y;
      const float scale = scale_of(block_max(v[i]));
      const u32x2 q = to_e4m3(v[i], scale, 1.0f / scale);
      if (r < p.m) {
        store_bytes((uint8_t*)p.q + r * p.q_ld + c, left, q);
        if (x == 0) p.scale[r * p.scale_row + bx * p.scale_col] = scale;
      }
    }
  } else if constexpr (BLOCKS == kBlockSquares) {
    __shared__ float most[WAVES];
    float a = 0.0f;
#pragma unroll
    for (int i = 0; i < TURNS; ++i) a = amax8(v[i], a);
    a = max16(a);
    a = fmaxf(a, __shfl_xor(a, 16));
    a = fmaxf(a, __shfl_xor(a, 32));
    if ((threadIdx.x & 63) == 0) most[wave] = a;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) a = fmaxf(a, most[w]);
    const float scale = scale_of(a), inverse = 1.0f / scale;
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
      const int64_t r = r0 + STEP * i + y;
      const u32x2 q = to_e4m3(v[i], scale, inverse);
      if (r < p.m) store_bytes((uint8_t*)p.q + r * p.q_ld + c, left, q);
    }
    if (threadIdx.x == 0) p.scale[by * p.scale_row + bx * p.scale_col] = scale;
  } else {
    // each row of 16 lanes holds two rows' columns; then a thread for each column, which has the one division
    static_assert(XT == 8, "a row of 16 lanes holds the columns twice");
    constexpr int CW = XT * 8;
    __shared__ __attribute__((aligned(16))) float most[4 * WAVES][CW], scales[2][CW];
    float scale[8], inverse[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float a = 0.0f;
#pragma unroll
      for (int i = 0; i < TURNS; ++i) a = fmaxf(a, is_finite(v[i][e]) ? fabsf(v[i][e]) : 0.0f);
      scale[e] = max_dpp<0x128>(a);  // row_ror:8
    }
    if ((threadIdx.x & 15) < XT) {
      f32x4* to = (f32x4*)(most[threadIdx.x >> 4] + x * 8);
      to[0] = (f32x4){scale[0], scale[1], scale[2], scale[3]};
      to[1] = (f32x4){scale[4], scale[5], scale[6], scale[7]};
    }
    __syncthreads();
    if (threadIdx.x < CW) {
      const int k = threadIdx.x;
      float a = most[0][k];
#pragma unroll
      for (int w = 1; w < 4 * WAVES; ++w) a = fmaxf(a, most[w][k]);
      a = scale_of(a);
      scales[0][k] = a;
      scales[1][k] = 1.0f / a;
      if (bx * CW + k < p.n) p.scale[by * p.scale_row + (bx * CW + k) * p.scale_col] = a;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      const f32x4 a = *(const f32x4*)(scales[0] + x * 8 + e), b = *(const f32x4*)(scales[1] + x * 8 + e);
#pragma unroll
      for (int i = 0; i < 4; ++i) scale[e + i] = a[i], inverse[e + i] = b[i];
    }
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
      const int64_t r = r0 + STEP * i + y;
      const u32x2 q = to_e4m3(v[i], scale, inverse);
      if (r < p.m) store_bytes((uint8_t*)p.q + r * p.q_ld + c, left, q);
    }
  }
}

template <typename T, QuantizeBlocks BLOCKS, int NT, int XT, int TURNS>
static __global__ __launch_bounds__(NT) void quantize_tiles(const eas_hip_quantize_args p) {
  const int64_t across = (p.n + XT * 8 - 1) / (XT * 8), total = across * ((p.m + NT / XT * TURNS - 1) / (NT / XT * TURNS));
  for (int64_t it = blockIdx.x; it < total; it += gridDim.x) {
    if (BLOCKS != kBlockRows && it != blockIdx.x) __syncthreads();  // the tile before is done with LDS
    const int64_t by = it / across;
    quantize_one<T, BLOCKS, NT, XT, TURNS>(p, by, it - by * across);
  }
}

template <typename T, QuantizeBlocks BLOCKS, int NT, int XT, int TURNS> static void quantize_blocks(const eas_hip_quantize_args& a, hipStream_t stream) {
  const int64_t tiles = ((a.n + XT * 8 - 1) / (XT * 8)) * ((a.m + NT / XT * TURNS - 1) / (NT / XT * TURNS));
  quantize_tiles<T, BLOCKS, NT, XT, TURNS><<<(unsigned)(tiles < (1 << 20) ? tiles : 1 << 20), NT, 0, stream>>>(a);
}

// Rows two to a thread, 32 to a workgroup (2048 x 14336 bf16 gated 29.9 us; four 32.5, one of 512 threads 33.2).  Columns in strips of 64 by
// 256 threads (4099 x 4096 bf16 13.6 us; by 128 threads 17.9, by 1024 16.9).  Squares by 512 threads (4096 x 4096 bf16 13.2; by
// 256 15.8).
template <typename T> static void quantize_typed(const eas_hip_quantize_args& a, hipStream_t stream) {
  if (a.block_m == 1) quantize_blocks<T, kBlockRows, 256, 16, 2>(a, stream);
  else if (a.block_n == 1) quantize_blocks<T, kBlockColumns, 256, 8, 4>(a, stream);
  else quantize_blocks<T, kBlockSquares, 512, 16, 4>(a, stream);
}

hipError_t quantize_launch(const eas_hip_quantize_args& a, hipStream_t stream) {
  if (a.dtype == EAS_HIP_F16) quantize_typed<f16>(a, stream);
  else if (a.dtype == EAS_HIP_BF16) quantize_typed<bf16>(a, stream);
  else quantize_typed<float>(a, stream);
  return hipGetLastError();
}

}  // namespace eas
