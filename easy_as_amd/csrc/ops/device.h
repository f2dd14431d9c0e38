// device.h — device helpers shared by the operators' kernels (gfx950).
#ifndef EAS_OPS_DEVICE_H
#define EAS_OPS_DEVICE_H

#include <hip/hip_runtime.h>

#include <cstdint>

#include "ops.h"

namespace eas {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename T> struct DtypeOf;
template <> struct DtypeOf<f16> { static constexpr int value = EAS_HIP_F16; };
template <> struct DtypeOf<bf16> { static constexpr int value = EAS_HIP_BF16; };
template <> struct DtypeOf<float> { static constexpr int value = EAS_HIP_F32; };

// Rows of N elements whose first one lies at any element boundary: vectors of 8 with the alignment of one
// element.  Global loads and stores of 16 bytes accept every alignment on this target.
template <typename T> struct Vec8 {
  typedef T type __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};

template <typename T> static __device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  typename Vec8<T>::type x;
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = (T)v[e];
  *(typename Vec8<T>::type*)p = x;
}
// store8 past the caches
template <typename T> static __device__ __forceinline__ void stream8(T* p, const float (&v)[8]) {
  typename Vec8<T>::type x;
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = (T)v[e];
  __builtin_nontemporal_store(x, (typename Vec8<T>::type*)p);
}
// 8 elements as they lie in memory; those from `n` on are 0
template <bool STREAM = false, typename T> static __device__ __forceinline__ typename Vec8<T>::type raw8(const T* p, int n) {
  typename Vec8<T>::type v = {};
  if (n >= 8) {
    if constexpr (STREAM) v = __builtin_nontemporal_load((const typename Vec8<T>::type*)p);
    else v = *(const typename Vec8<T>::type*)p;
  } else if (n > 0) {
    // all loads at once, those past the end of the last element; one after the other under its own condition each
    // would wait for the one before
    T t[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = p[e < n ? e : n - 1];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < n ? t[e] : (T)0.0f;
  }
  return v;
}
// the first `n` of 8 (n >= 8: all); the others read as 0 and are not written
template <typename T> static __device__ __forceinline__ void load_upto8(const T* p, int n, float (&v)[8]) {
  const typename Vec8<T>::type x = raw8(p, n);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (float)x[e];
}
template <typename T> static __device__ __forceinline__ void store_upto8(T* p, int n, const float (&v)[8]) {
  if (n >= 8) {
    store8(p, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) p[e] = (T)v[e];
  }
}
// the same for memory of one of two types, chosen per launch: T, or f32 where `wide`
template <typename T>
static __device__ __forceinline__ void load_upto8(const void* p, bool wide, int64_t at, int n, float (&v)[8]) {
  if (sizeof(T) == 4 || wide) load_upto8((const float*)p + at, n, v);
  else load_upto8((const T*)p + at, n, v);
}
template <typename T>
static __device__ __forceinline__ void store_upto8(void* p, bool wide, int64_t at, int n, const float (&v)[8]) {
  if (sizeof(T) == 4 || wide) store_upto8((float*)p + at, n, v);
  else store_upto8((T*)p + at, n, v);
}

// ---- rows as buffers -------------------------------------------------------------
//
// A thread's 8 columns of a row.  EVEN: rows of whole 4 bytes at multiples of 4, as a buffer of the row's length, or of
// none where it is not `live`: what lies past the end reads as zero and is not written, with no branch around the
// access.  Behind a branch that may skip a load, the compiler cannot count the accesses under way, and waits for the
// loads ahead (and the stores) at every row: forward 2048 x 8192 bf16 16.8 us with branches and 13.4 without, backward
// 8192 x 4096 45.0 and 42.7.  Else, 16-bit elements at odd addresses or in rows of an odd length, the branches are there.
template <typename T> static __device__ __forceinline__ __amdgpu_buffer_rsrc_t row_buffer(const T* row, int64_t n, bool live) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)row, 0, live ? (int)(n * (int64_t)sizeof(T)) : 0, 0x00020000);
}
template <typename T, bool EVEN, bool STREAM = false>
static __device__ __forceinline__ typename Vec8<T>::type row_load(const T* row, int64_t n, bool live, int c, int left) {
  if constexpr (!EVEN) {
    return raw8<STREAM>(row + c, live ? left : 0);
  } else {
    const __amdgpu_buffer_rsrc_t b = row_buffer(row, n, live);
    u32x4 v[sizeof(T) / 2];
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i)
      v[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(b, c * (int)sizeof(T) + 16 * i, 0, STREAM ? 2 : 0));
    return __builtin_bit_cast(typename Vec8<T>::type, v);
  }
}
template <typename T, bool EVEN>
static __device__ __forceinline__ void row_store(T* row, int64_t n, bool live, int c, int left, bool stream, const float (&x)[8]) {
  if constexpr (!EVEN) {
    if (!live) return;
    if (stream && left == 8) stream8(row + c, x);
    else store_upto8(row + c, left, x);
  } else {
    struct vec { u32x4 v[sizeof(T) / 2]; };
    typename Vec8<T>::type y;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = (T)x[e];
    const vec out = __builtin_bit_cast(vec, y);
    const __amdgpu_buffer_rsrc_t b = row_buffer(row, n, live);
    if (stream) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) __builtin_amdgcn_raw_buffer_store_b128(out.v[i], b, c * (int)sizeof(T) + 16 * i, 0, 2);  // nt
    } else {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) __builtin_amdgcn_raw_buffer_store_b128(out.v[i], b, c * (int)sizeof(T) + 16 * i, 0, 0);
    }
  }
}
// rows of whole 4 bytes at multiples of 4; 32-bit ones are
static inline bool even_rows(const void* p, int64_t ld, int64_t n) { return !p || ((uint64_t)p % 4 == 0 && ld % 2 == 0 && n % 2 == 0); }

// ---- activations --------------------------------------------------------------
//
// In 32 bits, from z in 32 bits.  FAST (16-bit operands): the hardware's exp2 and reciprocal, each within about
// one unit in the last place of 32 bits, and the normal integral by a formula within 6e-8, and within 1.1e-5 of itself where
// it is small: with what the exponents' roundings add (z^2 2^-23), far below a 16-bit result's rounding (4.9e-4 and 3.9e-3
// relative) at every z.  Else the library's functions.
template <bool FAST> static __device__ __forceinline__ float exp_(float x) {
  if constexpr (FAST) return __builtin_amdgcn_exp2f(x * 1.44269504088896340736f);
  else return expf(x);
}
template <bool FAST> static __device__ __forceinline__ float rcp_(float x) {
  if constexpr (FAST) return __builtin_amdgcn_rcpf(x);
  else return 1.0f / x;
}
template <bool FAST> static __device__ __forceinline__ float sigmoid_(float x) { return rcp_<FAST>(1.0f + exp_<FAST>(-x)); }

// z sigmoid(a) = (z m) (m r): m = exp(a / 2) for a < 0, else 1, and r = 1 / (1 + exp(-|a|)).  As z / (1 + exp(-a)) it
// would be 0 once exp(-a) leaves the range, where the tanh form's a is -88 and z only -10.
template <bool FAST> static __device__ __forceinline__ void half_sigmoid_(float a, float& m, float& r) {
  const float h = exp_<FAST>(-0.5f * fabsf(a));
  r = rcp_<FAST>(__builtin_fmaf(h, h, 1.0f));
  m = a < 0.0f ? h : 1.0f;
}

// Phi(z), the normal distribution's integral, and exp(-z^2/2).  The tail Phi(-|z|) is computed for itself, so that negative
// z keep its digits (0.5 (1 + erf) has none left below -6), and taken from 1 for positive ones.  FAST: Phi(-|z|) =
// exp(-z^2/2) t P(t), t = 1 / (1 + c |z|), the polynomial P a minimax fit over all z of the error over the larger of 1e-7
// and 2e-5 Phi.
template <bool FAST> static __device__ __forceinline__ float phi_(float z, float& e) {
  if constexpr (FAST) {
    const float t = rcp_<true>(__builtin_fmaf(0.3570646048f, fabsf(z), 1.0f));
    e = __builtin_amdgcn_exp2f(z * z * -0.721347520444f);
    float p = __builtin_fmaf(0.0435247980f, t, -0.1702376604f);
    p = __builtin_fmaf(p, t, 0.1727778912f);
    p = __builtin_fmaf(p, t, 0.0346730500f);
    p = __builtin_fmaf(p, t, 0.1354271173f);
    p = __builtin_fmaf(p, t, 0.1413480937f);
    p = __builtin_fmaf(p, t, 0.1424867660f);
    const float q = p * t * e;  // Phi(-|z|)
    return z < 0.0f ? q : 1.0f - q;
  } else {
    e = expf(-0.5f * z * z);
    return 0.5f * erfcf(z * -0.70710678118654752440f);
  }
}

// act(z) of 8 values; `act` is the same for the whole launch
template <bool FAST> static __device__ __forceinline__ void activate8(int act, float (&z)[8]) {
  switch (act) {
    case EAS_HIP_ACT_RELU:
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] = z[i] > 0.0f || z[i] != z[i] ? z[i] : 0.0f;
      break;
    case EAS_HIP_ACT_SILU:
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] *= sigmoid_<FAST>(z[i]);
      break;
    case EAS_HIP_ACT_GELU:
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float e;
        z[i] *= phi_<FAST>(z[i], e);
      }
      break;
    case EAS_HIP_ACT_GELU_TANH:  // 0.5 (1 + tanh u) = sigmoid(2 u)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float m, r;
        half_sigmoid_<FAST>(z[i] * __builtin_fmaf(0.07135481627f, z[i] * z[i], 1.59576912161f), m, r);
        z[i] = z[i] * m * (m * r);
      }
      break;
    default:
      break;
  }
}

// f = act(z) and d = act'(z) of 8 values
template <bool FAST>
static __device__ __forceinline__ void activate_grad8(int act, const float (&z)[8], float (&f)[8], float (&d)[8]) {
  switch (act) {
    case EAS_HIP_ACT_RELU:
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        f[i] = z[i] > 0.0f || z[i] != z[i] ? z[i] : 0.0f;
        d[i] = z[i] > 0.0f ? 1.0f : 0.0f;
      }
      break;
    case EAS_HIP_ACT_SILU:
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float s = sigmoid_<FAST>(z[i]);
        f[i] = z[i] * s;
        d[i] = __builtin_fmaf(f[i], 1.0f - s, s);
      }
      break;
    case EAS_HIP_ACT_GELU:
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float e;
        const float p = phi_<FAST>(z[i], e);
        f[i] = z[i] * p;
        d[i] = __builtin_fmaf(z[i] * 0.39894228040143267794f, e, p);
      }
      break;
    case EAS_HIP_ACT_GELU_TANH:
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float zz = z[i] * z[i];
        float m, r;
        half_sigmoid_<FAST>(z[i] * __builtin_fmaf(0.07135481627f, zz, 1.59576912161f), m, r);
        const float s = m * (m * r);
        f[i] = z[i] * m * (m * r);
        d[i] = __builtin_fmaf(f[i] * (1.0f - s), __builtin_fmaf(0.21406444882f, zz, 1.59576912161f), s);
      }
      break;
    default:
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        f[i] = z[i];
        d[i] = 1.0f;
      }
      break;
  }
}

// ---- sums over a wave and a workgroup -------------------------------------------

// lane l of each operand: v plus v of the lane that DPP control CTRL gives, in the rows of 16 lanes of ROWS
template <int CTRL, int ROWS> static __device__ __forceinline__ float add_dpp(float v) {
  const int other = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false);
  return v + __builtin_bit_cast(float, other);
}
// The sum over the wave, in every lane: within rows of 16 lanes by shifts, across them by broadcasts of their last
// lanes, with no trip through LDS.
static __device__ __forceinline__ float wave_sum(float v) {
  v = add_dpp<0x111, 0xf>(v);  // row_shr:1
  v = add_dpp<0x112, 0xf>(v);
  v = add_dpp<0x114, 0xf>(v);
  v = add_dpp<0x118, 0xf>(v);
  v = add_dpp<0x142, 0xa>(v);  // row_bcast:15 into rows 1 and 3
  v = add_dpp<0x143, 0xc>(v);  // row_bcast:31 into rows 2 and 3
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

}  // namespace eas

#endif  // EAS_OPS_DEVICE_H
