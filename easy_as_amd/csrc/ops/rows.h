// rows.h — what the kernels of the two norms share: sums over a row, its parameters, and how rows are shared out.
#ifndef EAS_OPS_ROWS_H
#define EAS_OPS_ROWS_H

#include "device.h"

namespace eas {

// Sums over the TPR threads of a row (whole waves).  `slots`: two sets of N floats per wave of the workgroup, used in
// turns (`turn`), so that one barrier separates a set's writers from its readers, and the next but one writers from them.
template <int TPR, int WG, int N>
static __device__ __forceinline__ void row_sums(float (&v)[N], float* slots, int& turn) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
  if constexpr (TPR > 64) {
    float* set = slots + (turn & 1) * (WG / 64) * N;
    ++turn;
    const int wave = threadIdx.x >> 6, first = (threadIdx.x / TPR) * (TPR / 64);
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) set[wave * N + i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = 0.0f;
#pragma unroll
      for (int k = 0; k < TPR / 64; ++k) v[i] += set[(first + k) * N + i];
    }
  }
}

// one f32 of a row's
static __device__ __forceinline__ float uniform(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)));
}
template <bool EVEN> static __device__ __forceinline__ float stat_load(const float* p, bool live) {
  if constexpr (EVEN) return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(row_buffer(p, 1, live), 0, 0, 0));
  else return live ? *p : 0.0f;
}
template <bool EVEN> static __device__ __forceinline__ void stat_store(float* p, bool live, bool mine, float v) {
  if constexpr (EVEN) {
    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, v), row_buffer(p, 1, live), mine ? 0 : 4, 0, 0);
  } else {
    if (live && mine) *p = v;
  }
}

// weight or bias from column c on; absent ones are `none` everywhere
template <typename T>
static __device__ __forceinline__ void load_param(const void* p, bool wide, float none, int64_t c, int left, float (&v)[8]) {
  if (p) {
    load_upto8<T>(p, wide, c, left, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = none;
  }
}

// the same with EVEN rows' access, in two steps: all of a thread's loads are under way before the first is used
struct RawParam { u32x4 v[2]; };
template <typename T, bool EVEN>
static __device__ __forceinline__ void fetch_param(const void* p, bool wide, int64_t n, int c, RawParam& raw) {
  if constexpr (EVEN) {
    const int size = wide ? 4 : (int)sizeof(T);
    const __amdgpu_buffer_rsrc_t b = row_buffer((const char*)p, n * size, p);
    raw.v[0] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(b, c * size, 0, 0));
    if (size == 4) raw.v[1] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(b, c * size + 16, 0, 0));
  }
}
template <typename T, bool EVEN>
static __device__ __forceinline__ void take_param(const void* p, bool wide, float none, int c, int left, const RawParam& raw, float (&v)[8]) {
  if constexpr (!EVEN) {
    load_param<T>(p, wide, none, c, left, v);
  } else if (!p) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = none;
  } else if (sizeof(T) == 4 || wide) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const f32x4 x = __builtin_bit_cast(f32x4, raw.v[i]);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * i + e] = x[e];
    }
  } else if constexpr (sizeof(T) == 2) {
    const typename Vec8<T>::type x = __builtin_bit_cast(typename Vec8<T>::type, raw.v[0]);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)x[e];
  }
}

// Workgroups that each take the same number of turns but the last: at most `most`
static inline int64_t even_groups(int64_t turns, int64_t most) {
  const int64_t each = (turns + most - 1) / most;
  return (turns + each - 1) / each;
}

}  // namespace eas

#endif  // EAS_OPS_ROWS_H
