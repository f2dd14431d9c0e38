// e4m3.h — 8-bit values and their blocks' scales (gfx950).
//
// A scale is the block's largest finite magnitude over 448, at least 2^-126, so that it and its reciprocal are normal
// numbers.  An element is v / scale to 32 bits, as a division would round it: v times the reciprocal, and one
// correction by what is left over (a product by the reciprocal alone rounds a quotient next to a tie between two 8-bit
// values to the other side now and then).  The correction makes NaN of infinities, and no finite quotient is beyond 448 by more
// than a rounding, so the conversion, to nearest with ties to even, needs no clamp.
#ifndef EAS_OPS_E4M3_H
#define EAS_OPS_E4M3_H

#include "device.h"

namespace eas {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
constexpr float kLargest = 448.0f;
constexpr float kLeastScale = 0x1p-126f;
constexpr int kBlock = 128;

static __device__ __forceinline__ bool is_finite(float v) { return __builtin_isfpclass(v, 0x1f8); }

// the larger of `most` and the finite ones of v
static __device__ __forceinline__ float amax8(const float (&v)[8], float most) {
#pragma unroll
  for (int e = 0; e < 8; ++e) most = fmaxf(most, is_finite(v[e]) ? fabsf(v[e]) : 0.0f);
  return most;
}
template <int CTRL> static __device__ __forceinline__ float max_dpp(float v) {
  const int i = __builtin_bit_cast(int, v);
  return fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, CTRL, 0xf, 0xf, false)));
}
// the largest of each row of 16 lanes, in all of them
static __device__ __forceinline__ float max16(float v) {
  v = max_dpp<0x121>(v);  // row_ror:1
  v = max_dpp<0x122>(v);
  v = max_dpp<0x124>(v);
  return max_dpp<0x128>(v);
}
template <int CTRL> static __device__ __forceinline__ uint32_t umax_dpp(uint32_t v) {
  const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, false);
  return o > v ? o : v;
}
// The largest finite magnitude of 16 lanes' 8 values.  As integers magnitudes are in order, infinities and NaN last: only
// where one is found the others are looked through by themselves.
static __device__ __forceinline__ float block_max(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v[e]) & 0x7fffffffu;
    m = b > m ? b : m;
  }
  m = umax_dpp<0x121>(m);
  m = umax_dpp<0x122>(m);
  m = umax_dpp<0x124>(m);
  m = umax_dpp<0x128>(m);
  if (m >= 0x7f800000u) return max16(amax8(v, 0.0f));  // the same in all 16
  return __builtin_bit_cast(float, m);
}
static __device__ __forceinline__ float scale_of(float most) { return fmaxf(most / kLargest, kLeastScale); }

// 8 values over their scales; inverse: 1 / scale
static __device__ __forceinline__ u32x2 to_e4m3(const float (&v)[8], const float (&scale)[8], const float (&inverse)[8]) {
  float t[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float a = v[e] * inverse[e];
    t[e] = __builtin_fmaf(__builtin_fmaf(-a, scale[e], v[e]), inverse[e], a);
  }
  u32x2 q;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(t[4 * i], t[4 * i + 1], 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(t[4 * i + 2], t[4 * i + 3], w, true);
    q[i] = (uint32_t)w;
  }
  return q;
}
static __device__ __forceinline__ u32x2 to_e4m3(const float (&v)[8], float scale, float inverse) {
  const float s[8] = {scale, scale, scale, scale, scale, scale, scale, scale};
  const float i[8] = {inverse, inverse, inverse, inverse, inverse, inverse, inverse, inverse};
  return to_e4m3(v, s, i);
}
// the first `n` of 8 bytes (n >= 8: all) to any address
static __device__ __forceinline__ void store_bytes(uint8_t* p, int n, u32x2 q) {
  if (n >= 8) {
    typedef uint32_t any_t __attribute__((ext_vector_type(2), aligned(1)));
    *(any_t*)p = q;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) p[e] = (uint8_t)(q[e / 4] >> (8 * (e % 4)));
  }
}

}  // namespace eas

#endif  // EAS_OPS_E4M3_H
