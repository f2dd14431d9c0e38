// quantize.hip — matrices to 8 bits with a scale for each block: of a row, of a column, or 128 x 128.
//
// v = act(x), or act(gate) x, in 32 bits, held in registers between the search for a block's largest magnitude and its
// conversion: one read, one write.  A workgroup takes a strip of columns, XT threads of 8 across and NT / XT rows at a time,
// TURNS times: a row's block is 16 neighbouring lanes, a column's or a square's meets through LDS.  Bound by memory: 8192 x 4096
// bf16 by rows 23.3 us (4.4 TB/s), 4099 x 4096 by columns 12.9 (3.9); 2048 x 14336 bf16 by rows relu(gate) * x 30.3 (4.9),
// silu(gate) * x 32.4 and gelu(gate) * x 42, whose arithmetic is no longer hidden.
#include <type_traits>

#include "e4m3.h"

namespace eas {

// ---- activations in 32 bits ---------------------------------------------------------
//
// A scale is v's own 32 bits, and a quotient next to a tie rounds by its last ones, so act(z) is within 2^-20 of itself at every
// z: 13 units of 2^-24 at the most, the steps' roundings added up.  The activations of 16-bit products (device.h) are up to
// 1.3e-5 off in the tails, and 0 below silu's -88; with them silu(gate) * x took 30.2 us for 32.4.  What those lose is the
// exponent's rounding, here kept as a second summand of it, and a unit of the hardware's reciprocal, here corrected.  SiLU is
// z / (1 + exp(-z)), the tanh form the same of z (c0 + c1 z^2), and gelu z Phi(z), Phi(-|z|) = exp(-z^2 / 2) t P(t), t = 1 / (1 +
// 5/16 |z|), P a minimax fit of the relative error (1.1e-8) up to |z| = 15.  FAR: for z whose exponentials may leave the range,
// which are of negative exponents only and held 2^64 times as large.  All go by the roundings of each step, so that no
// product may join an addition.
struct Power {
  float f, scale;  // f scale = exp(-(a + low))
};
template <bool FAR> static __device__ __forceinline__ Power power(float a, float low) {
#pragma clang fp contract(off)
  const float t = a * -0x1.715476p+0f;
  const bool far = FAR && t < -120.0f;
  const float f = __builtin_amdgcn_exp2f(far ? t + 64.0f : t);
  const float r = __builtin_fmaf(t, 0x1.05c61p-29f, __builtin_fmaf(t, -0x1.62e43p-1f, -a)) - low;
  return {__builtin_fmaf(f, r, f), far ? 0x1p-64f : 1.0f};
}
static __device__ __forceinline__ float reciprocal(float d) {
  const float r = __builtin_amdgcn_rcpf(d);
  return __builtin_fmaf(__builtin_fmaf(-d, r, 1.0f), r, r);
}
// z / (1 + exp(-(a + low))); FAR: a and low are |z|'s
template <bool FAR> static __device__ __forceinline__ float times_sigmoid(float z, float a, float low) {
  const Power p = power<FAR>(a, low);
  const float r = reciprocal(__builtin_fmaf(p.f, p.scale, 1.0f));
  return FAR && z < 0.0f ? z * (p.f * r) * p.scale : z * r;
}
template <bool FAR> static __device__ __forceinline__ float silu32(float z) {
  return times_sigmoid<FAR>(z, FAR ? fminf(fabsf(z), 400.0f) : z, 0.0f);
}
template <bool FAR> static __device__ __forceinline__ float gelu_tanh32(float z) {
#pragma clang fp contract(off)
  constexpr float c0 = 0x1.988454p+0f, c0_low = -0x1.857936p-25f;  // sqrt(8 / pi)
  constexpr float c1 = 0x1.2444f2p-4f, c1_low = 0x1.49b16ap-29f;  // 0.044715 of that
  const float a = FAR ? fminf(fabsf(z), 30.0f) : z, aa = a * a, q = aa * c1, p = q + c0;
  const float more = fmaxf(q, c0), less = fminf(q, c0);
  const float p_low = (less - (p - more)) +
                      (__builtin_fmaf(aa, c1, -q) + __builtin_fmaf(__builtin_fmaf(a, a, -aa), c1, __builtin_fmaf(aa, c1_low, c0_low)));
  const float b = a * p;
  return times_sigmoid<FAR>(z, b, __builtin_fmaf(a, p_low, __builtin_fmaf(a, p, -b)));
}
template <bool FAR> static __device__ __forceinline__ float gelu32(float z) {
#pragma clang fp contract(off)
  const float a = FAR ? fminf(fabsf(z), 40.0f) : fabsf(z), half = 0.5f * a, b = a * half;
  const Power p = power<FAR>(b, __builtin_fmaf(a, half, -b));
  const float s = reciprocal(__builtin_fmaf(0.3125f, a, 1.0f));
  float g = __builtin_fmaf(-0.0192170553f, s, 0.0924713537f);
  g = __builtin_fmaf(g, s, -0.153514698f);
  g = __builtin_fmaf(g, s, 0.0774997398f);
  g = __builtin_fmaf(g, s, -0.00518122735f);
  g = __builtin_fmaf(g, s, 0.0569405369f);
  g = __builtin_fmaf(g, s, 0.0896129459f);
  g = __builtin_fmaf(g, s, 0.111983962f);
  g = __builtin_fmaf(g, s, 0.124738492f);
  g = __builtin_fmaf(g, s, 0.124665953f);
  g *= s;
  return z < 0.0f ? z * (p.f * g) * p.scale : z * __builtin_fmaf(-p.f * p.scale, g, 1.0f);
}
// act(z) of 8 values
template <int ACT> static __device__ __forceinline__ void activate32(float (&z)[8]) {
  constexpr float reach = ACT == EAS_HIP_ACT_SILU ? 80.0f : ACT == EAS_HIP_ACT_GELU ? 12.5f : 9.5f;
  auto all = [&](auto far) __attribute__((always_inline)) {
    constexpr bool FAR = decltype(far)::value;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      z[e] = ACT == EAS_HIP_ACT_SILU ? silu32<FAR>(z[e]) : ACT == EAS_HIP_ACT_GELU ? gelu32<FAR>(z[e]) : gelu_tanh32<FAR>(z[e]);
      if (FAR) __builtin_amdgcn_sched_barrier(0);  // one at a time, in few registers
    }
  };
  bool near = true;
#pragma unroll
  for (int e = 0; e < 8; ++e) near &= fabsf(z[e]) <= reach;  // not NaN
  if (near) all(std::false_type());
  else all(std::true_type());
}

enum QuantizeBlocks { kBlockRows, kBlockColumns, kBlockSquares };

template <typename T, int ACT, QuantizeBlocks BLOCKS, int NT, int XT, int TURNS>
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
      if constexpr (ACT) activate32<ACT>(z);
      else if (p.activation == EAS_HIP_ACT_RELU) activate8<false>(EAS_HIP_ACT_RELU, z);
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

template <typename T, int ACT, QuantizeBlocks BLOCKS, int NT, int XT, int TURNS>
static __global__ __launch_bounds__(NT) void quantize_tiles(const eas_hip_quantize_args p) {
  const int64_t across = (p.n + XT * 8 - 1) / (XT * 8), total = across * ((p.m + NT / XT * TURNS - 1) / (NT / XT * TURNS));
  for (int64_t it = blockIdx.x; it < total; it += gridDim.x) {
    if (BLOCKS != kBlockRows && it != blockIdx.x) __syncthreads();  // the tile before is done with LDS
    const int64_t by = it / across;
    quantize_one<T, ACT, BLOCKS, NT, XT, TURNS>(p, by, it - by * across);
  }
}

template <typename T, int ACT, QuantizeBlocks BLOCKS, int NT, int XT, int TURNS>
static void quantize_blocks(const eas_hip_quantize_args& a, hipStream_t stream) {
  const int64_t tiles = ((a.n + XT * 8 - 1) / (XT * 8)) * ((a.m + NT / XT * TURNS - 1) / (NT / XT * TURNS));
  quantize_tiles<T, ACT, BLOCKS, NT, XT, TURNS><<<(unsigned)(tiles < (1 << 20) ? tiles : 1 << 20), NT, 0, stream>>>(a);
}

// Rows two to a thread, 32 to a workgroup (8192 x 4096 bf16 23.3 us; four 24.6, one of 512 threads 26.0).  Columns in strips of
// 64 by 256 threads (4099 x 4096 bf16 12.9 us; by 128 threads 16.6, by 1024 17.0).  Squares by 512 threads (4096 x 4096 bf16
// 12.8; by 256 14.8).
template <typename T, int ACT> static void quantize_sized(const eas_hip_quantize_args& a, hipStream_t stream) {
  if (a.block_m == 1) quantize_blocks<T, ACT, kBlockRows, 256, 16, 2>(a, stream);
  else if (a.block_n == 1) quantize_blocks<T, ACT, kBlockColumns, 256, 8, 4>(a, stream);
  else quantize_blocks<T, ACT, kBlockSquares, 512, 16, 4>(a, stream);
}

// A kernel for each activation: by rows 57 registers, eight waves a SIMD (all in one 73; silu(gate) * x 36.9 us
// for 33.7 in the same run, and 8192 x 4096 without any 25.4 for 23.3).
template <typename T> static void quantize_typed(const eas_hip_quantize_args& a, hipStream_t stream) {
  if (a.activation == EAS_HIP_ACT_SILU) quantize_sized<T, EAS_HIP_ACT_SILU>(a, stream);
  else if (a.activation == EAS_HIP_ACT_GELU) quantize_sized<T, EAS_HIP_ACT_GELU>(a, stream);
  else if (a.activation == EAS_HIP_ACT_GELU_TANH) quantize_sized<T, EAS_HIP_ACT_GELU_TANH>(a, stream);
  else quantize_sized<T, EAS_HIP_ACT_NONE>(a, stream);
}

hipError_t quantize_launch(const eas_hip_quantize_args& a, hipStream_t stream) {
  if (a.dtype == EAS_HIP_F16) quantize_typed<f16>(a, stream);
  else if (a.dtype == EAS_HIP_BF16) quantize_typed<bf16>(a, stream);
  else quantize_typed<float>(a, stream);
  return hipGetLastError();
}

}  // namespace eas
