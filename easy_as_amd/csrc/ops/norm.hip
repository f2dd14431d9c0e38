// norm.hip — layer norm over rows, and its gradients.
//
// Forward: mean = sum(x)/n, rstd = (sum((x - mean)^2)/n + eps)^-1/2, y = (x - mean) rstd weight + bias.  A row stays
// in registers from its one read to its one write: TPR threads of VPT vectors of 8, two sums over them, the second
// about the mean (no cancellation between large squares).  Rows beyond 16384 elements are read three times instead.
//
// Backward, with g = dy weight and xh = (x - mean) rstd: dx = rstd (g - mean(g) - xh mean(g xh)), dweight =
// sum(dy xh) and dbias = sum(dy) over rows.  A thread owns its columns: it adds their dweight and dbias over all the
// rows that its workgroup takes, each workgroup writes one row of partial sums, and column_sum adds those.
//
// Both are bound by memory.  Forward 8192 x 4096 bf16: 22.8 us (5.9 TB/s of x and y; a copy of as much reaches 6.6).
// Backward of the same: 42.2 us with the sums' second launch (4.7 TB/s of x, dy and dx; the sums on the way, two barriers
// a row and one workgroup a CU keep it from more).
#include "rows.h"

namespace eas {

// Mean and sum of squared differences from it over a row, squares(c) being the thread's sum of squares about c: each wave's own first, then the waves' joined by M2 = sum of
// M2_i + c_i (mean_i - mean)^2, every term of which is positive.  `count`: the wave's columns.
template <int TPR, int WG, typename Squares>
static __device__ __forceinline__ void row_moments(float sum, float count, float n, Squares squares, float* slots, int& turn,
                                                   float& mean, float& m2) {
  if constexpr (TPR == 64) {
    mean = wave_sum(sum) / n;
    m2 = wave_sum(squares(mean));
  } else {
    const float s = wave_sum(sum), own = count > 0.0f ? s / count : 0.0f;
    const float q = wave_sum(squares(own));
    float* set = slots + (turn & 1) * (WG / 64) * 4;
    ++turn;
    const int wave = threadIdx.x >> 6, first = (threadIdx.x / TPR) * (TPR / 64);
    if ((threadIdx.x & 63) == 0) {
      set[wave * 4] = s;
      set[wave * 4 + 1] = q;
      set[wave * 4 + 2] = own;
      set[wave * 4 + 3] = count;
    }
    __syncthreads();
    mean = 0.0f;
#pragma unroll
    for (int k = 0; k < TPR / 64; ++k) mean += set[(first + k) * 4];
    mean /= n;
    m2 = 0.0f;
#pragma unroll
    for (int k = 0; k < TPR / 64; ++k) {
      const float* w = set + (first + k) * 4;
      const float d = w[2] - mean;
      m2 += w[1] + w[3] * d * d;
    }
  }
}

// ---- forward ----------------------------------------------------------------------

// A workgroup takes RPW rows at a time, those of the grid side by side in memory, and loads its next ones before it
// reduces these: the loads are in flight while the sums meet.
template <typename T, bool EVEN, int VPT, int TPR>
static __global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void norm_rows(const eas_hip_layer_norm_args p, bool stream_y) {
  constexpr int WG = TPR < 256 ? 256 : TPR, RPW = WG / TPR;
  __shared__ float slots[2 * (WG / 64) * 4];
  typedef typename Vec8<T>::type raw_t;
  const int t = threadIdx.x % TPR, lane = threadIdx.x & 63;
  const int64_t n = p.n;
  const bool wide = p.wdtype == EAS_HIP_F32;
  float w[VPT][8], b[VPT][8];
  int left[VPT];
  float count = 0.0f;  // columns of this wave
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    const int64_t c = ((int64_t)v * TPR + t) * 8, c0 = c - lane * 8;
    left[v] = c >= n ? 0 : n - c < 8 ? (int)(n - c) : 8;
    count += c0 >= n ? 0.0f : (float)(n - c0 < 512 ? n - c0 : 512);
  }
  int turn = 0;
  const bool whole = n == 8 * VPT * TPR;
  const int64_t first = (int64_t)blockIdx.x * RPW, stride = (int64_t)gridDim.x * RPW, end = p.m;
  raw_t ahead[VPT];
  auto fetch = [&](int64_t r) {
#pragma unroll
    for (int v = 0; v < VPT; ++v) ahead[v] = row_load<T, EVEN>((const T*)p.x + r * p.x_ld, n, r < end, (v * TPR + t) * 8, left[v]);
  };
  const int group = __builtin_amdgcn_readfirstlane(threadIdx.x / TPR);
  fetch(first + group);
  {
    RawParam raw[2][VPT];
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      fetch_param<T, EVEN>(p.weight, wide, n, (v * TPR + t) * 8, raw[0][v]);
      fetch_param<T, EVEN>(p.bias, wide, n, (v * TPR + t) * 8, raw[1][v]);
    }
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      take_param<T, EVEN>(p.weight, wide, 1.0f, (v * TPR + t) * 8, left[v], raw[0][v], w[v]);
      take_param<T, EVEN>(p.bias, wide, 0.0f, (v * TPR + t) * 8, left[v], raw[1][v], b[v]);
    }
  }
  // every thread of the workgroup runs every turn: the sums' barriers are the workgroup's
  for (int64_t r0 = first; r0 < end; r0 += stride) {
    const int64_t r = r0 + group;
    float x[VPT][8];
    float s = 0.0f;
#pragma unroll
    for (int v = 0; v < VPT; ++v)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[v][e] = (float)ahead[v][e];
        s += x[v][e];
      }
    fetch(r + stride);
    float mean, m2;
    row_moments<TPR, WG>(s, count, (float)n, [&](float about) {
      float q = 0.0f;
      if (whole) {  // the same for the whole launch
#pragma unroll
        for (int v = 0; v < VPT; ++v)
#pragma unroll
          for (int e = 0; e < 8; ++e) q = __builtin_fmaf(x[v][e] - about, x[v][e] - about, q);
      } else {
#pragma unroll
        for (int v = 0; v < VPT; ++v)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float d = e < left[v] ? x[v][e] - about : 0.0f;
            q = __builtin_fmaf(d, d, q);
          }
      }
      return q;
    }, slots, turn, mean, m2);
    const float rstd = 1.0f / sqrtf(m2 / (float)n + p.eps);
    const bool live = r < end;
    stat_store<EVEN>(p.mean + r, live && p.mean, t == 0, mean);
    stat_store<EVEN>(p.rstd + r, live && p.rstd, t == 0, rstd);
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[v][e] = __builtin_fmaf((x[v][e] - mean) * rstd, w[v][e], b[v][e]);
      row_store<T, EVEN>((T*)p.y + r * p.y_ld, n, live, (v * TPR + t) * 8, left[v], stream_y, x[v]);
    }
  }
}

// rows of any length, one workgroup each
template <typename T> static __global__ __launch_bounds__(1024) void norm_long(const eas_hip_layer_norm_args p) {
  __shared__ float slots[2 * 16];
  const bool wide = p.wdtype == EAS_HIP_F32;
  const int64_t n = p.n;
  int turn = 0;
  for (int64_t r = blockIdx.x; r < p.m; r += gridDim.x) {
    const T* x = (const T*)p.x + r * p.x_ld;
    float s[1] = {}, v[8], w[8], b[8];
    for (int64_t c = threadIdx.x * 8; c < n; c += 8192) {
      load_upto8(x + c, n - c < 8 ? (int)(n - c) : 8, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[0] += v[e];
    }
    row_sums<1024, 1024, 1>(s, slots, turn);
    const float mean = s[0] / (float)n;
    s[0] = 0.0f;
    for (int64_t c = threadIdx.x * 8; c < n; c += 8192) {
      const int left = n - c < 8 ? (int)(n - c) : 8;
      load_upto8(x + c, left, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[0] += e < left ? (v[e] - mean) * (v[e] - mean) : 0.0f;
    }
    row_sums<1024, 1024, 1>(s, slots, turn);
    const float rstd = 1.0f / sqrtf(s[0] / (float)n + p.eps);
    if (threadIdx.x == 0) {
      if (p.mean) p.mean[r] = mean;
      if (p.rstd) p.rstd[r] = rstd;
    }
    for (int64_t c = threadIdx.x * 8; c < n; c += 8192) {
      const int left = n - c < 8 ? (int)(n - c) : 8;
      load_upto8(x + c, left, v);
      load_param<T>(p.weight, wide, 1.0f, c, left, w);
      load_param<T>(p.bias, wide, 0.0f, c, left, b);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = __builtin_fmaf((v[e] - mean) * rstd, w[e], b[e]);
      store_upto8((T*)p.y + r * p.y_ld + c, left, v);
    }
  }
}

template <typename T, bool EVEN, int VPT, int TPR> static void norm_rows_launch(const eas_hip_layer_norm_args& a, hipStream_t stream) {
  constexpr int WG = TPR < 256 ? 256 : TPR, RPW = WG / TPR;
  // y past the memory-side cache (256 MB) where x and y would share it: 8192 x 4096 bf16 28.7 -> 22.8 us; not where they
  // are beyond it anyway: fp32 51.0 -> 54.2
  const bool stream_y = a.m * a.n * (int64_t)sizeof(T) * 2 <= (256 << 20);
  norm_rows<T, EVEN, VPT, TPR><<<(unsigned)even_groups((a.m + RPW - 1) / RPW, 256 * (1024 / WG)), WG, 0, stream>>>(a, stream_y);
}

template <typename T, bool EVEN> static void norm_typed(const eas_hip_layer_norm_args& a, hipStream_t stream) {
  if (a.n <= 512) norm_rows_launch<T, EVEN, 1, 64>(a, stream);
  else if (a.n <= 1024) norm_rows_launch<T, EVEN, 2, 64>(a, stream);
  else if (a.n <= 2048) norm_rows_launch<T, EVEN, 1, 256>(a, stream);
  else if (a.n <= 4096) norm_rows_launch<T, EVEN, 2, 256>(a, stream);
  else if (a.n <= 6144) norm_rows_launch<T, EVEN, 3, 256>(a, stream);
  else if (a.n <= 8192) norm_rows_launch<T, EVEN, 4, 256>(a, stream);
  else if (a.n <= 12288) norm_rows_launch<T, EVEN, 3, 512>(a, stream);
  else if (a.n <= 16384) norm_rows_launch<T, EVEN, 4, 512>(a, stream);
  else norm_long<T><<<(unsigned)(a.m < 512 ? a.m : 512), 1024, 0, stream>>>(a);
}

hipError_t layer_norm_launch(const eas_hip_layer_norm_args& a, hipStream_t stream) {
  const bool even = even_rows(a.x, a.x_ld, a.n) && even_rows(a.y, a.y_ld, a.n) && even_rows(a.weight, 0, a.n) && even_rows(a.bias, 0, a.n);
  if (a.dtype == EAS_HIP_F16) even ? norm_typed<f16, true>(a, stream) : norm_typed<f16, false>(a, stream);
  else if (a.dtype == EAS_HIP_BF16) even ? norm_typed<bf16, true>(a, stream) : norm_typed<bf16, false>(a, stream);
  else norm_typed<float, true>(a, stream);
  return hipGetLastError();
}

// ---- backward ---------------------------------------------------------------------

template <typename T, bool EVEN, int VPT, int TPR>
static __global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void norm_backward_rows(const eas_hip_layer_norm_backward_args p, float* part) {
  constexpr int WG = TPR < 256 ? 256 : TPR, RPW = WG / TPR;
  __shared__ float slots[2 * (WG / 64) * 2];
  __shared__ float meet[RPW > 1 ? RPW * VPT * TPR * 8 : 1];
  constexpr int AHEAD = TPR * VPT > 1024 ? 1 : 2;  // 512 threads leave 256 registers each
  typedef typename Vec8<T>::type raw_t;
  const int t = threadIdx.x % TPR, group = __builtin_amdgcn_readfirstlane(threadIdx.x / TPR);
  const int64_t n = p.n;
  const bool wide = p.wdtype == EAS_HIP_F32;
  float w[VPT][8], dw[VPT][8] = {}, db[VPT][8] = {};
  int left[VPT];
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    const int64_t c = ((int64_t)v * TPR + t) * 8;
    left[v] = c >= n ? 0 : n - c < 8 ? (int)(n - c) : 8;
  }
  const float inv = 1.0f / (float)n;
  int turn = 0;
  const int64_t first = (int64_t)blockIdx.x * RPW, stride = (int64_t)gridDim.x * RPW, end = p.m;
  // the next rows of this thread, in flight while this one is reduced
  struct Row {
    raw_t x[VPT], d[VPT];
    float mean, rstd;
  };
  auto fetch = [&](Row& q, int64_t r) __attribute__((always_inline)) {
    const bool live = r < end;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      q.x[v] = row_load<T, EVEN>((const T*)p.x + r * p.x_ld, n, live, (v * TPR + t) * 8, left[v]);
      q.d[v] = row_load<T, EVEN>((const T*)p.dy + r * p.dy_ld, n, live, (v * TPR + t) * 8, left[v]);
    }
    q.mean = stat_load<EVEN>(p.mean + r, live);
    q.rstd = stat_load<EVEN>(p.rstd + r, live);
  };
  auto one = [&](Row& q, int64_t r0) __attribute__((always_inline)) {
    const int64_t r = r0 + group;
    const float mean = uniform(q.mean), rstd = uniform(q.rstd);  // the wave's row
    // c = x - mean and xh = c rstd: dweight adds (dy rstd) c, and dx = c (-rstd^2 mean(g xh)) + (g rstd - rstd mean(g)),
    // 11 operations an element.  Past the row's end, and for a row past the last, dy is 0 and c finite.
    float c[VPT][8], g[VPT][8];
    float sums[2] = {};
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        c[v][e] = (float)q.x[v][e] - mean;
        g[v][e] = (float)q.d[v][e];
        dw[v][e] = __builtin_fmaf(g[v][e] * rstd, c[v][e], dw[v][e]);
        db[v][e] += g[v][e];
        g[v][e] *= w[v][e];
        sums[0] += g[v][e];
        sums[1] = __builtin_fmaf(g[v][e], c[v][e], sums[1]);
      }
    }
    fetch(q, r + AHEAD * stride);
    row_sums<TPR, WG, 2>(sums, slots, turn);
    const float a = -rstd * (sums[0] * inv), b = -rstd * rstd * (sums[1] * rstd * inv);
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
#pragma unroll
      for (int e = 0; e < 8; ++e) c[v][e] = __builtin_fmaf(c[v][e], b, __builtin_fmaf(g[v][e], rstd, a));
      row_store<T, EVEN>((T*)p.dx + r * p.dx_ld, n, r < end && p.dx, (v * TPR + t) * 8, left[v], false, c[v]);
    }
  };
  Row rows[AHEAD];
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) {
    fetch(rows[k], first + k * stride + group);
    __builtin_amdgcn_sched_barrier(0);  // in the order of their use, which the counts of loads under way go by
  }
  {
    RawParam raw[VPT];
#pragma unroll
    for (int v = 0; v < VPT; ++v) fetch_param<T, EVEN>(p.weight, wide, n, (v * TPR + t) * 8, raw[v]);
#pragma unroll
    for (int v = 0; v < VPT; ++v) take_param<T, EVEN>(p.weight, wide, 1.0f, (v * TPR + t) * 8, left[v], raw[v], w[v]);
  }
#pragma unroll 1
  for (int64_t r0 = first; r0 < end; r0 += AHEAD * stride)
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) one(rows[k], r0 + k * stride);
  if (!part) return;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float* out = part + ((int64_t)blockIdx.x * 2 + k) * n;
    if constexpr (RPW > 1) {  // the row groups' sums first
      __syncthreads();
#pragma unroll
      for (int v = 0; v < VPT; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e) meet[(group * VPT * 8 + v * 8 + e) * TPR + t] = k ? db[v][e] : dw[v][e];
      __syncthreads();
      for (int i = threadIdx.x; i < VPT * 8 * TPR; i += WG) {
        const int64_t c = ((int64_t)(i / (8 * TPR)) * TPR + i % TPR) * 8 + (i / TPR) % 8;
        float s = 0.0f;
#pragma unroll
        for (int q = 0; q < RPW; ++q) s += meet[q * VPT * 8 * TPR + i];
        if (c < n) out[c] = s;
      }
    } else {
#pragma unroll
      for (int v = 0; v < VPT; ++v) store_upto8(out + ((int64_t)v * TPR + t) * 8, left[v], k ? db[v] : dw[v]);
    }
  }
}

// rows beyond what the registers hold: dx one row per workgroup, read twice
template <typename T>
static __global__ __launch_bounds__(1024) void norm_backward_long(const eas_hip_layer_norm_backward_args p) {
  __shared__ float slots[2 * 32];
  const bool wide = p.wdtype == EAS_HIP_F32;
  const int64_t n = p.n;
  int turn = 0;
  for (int64_t r = blockIdx.x; r < p.m; r += gridDim.x) {
    const T *x = (const T*)p.x + r * p.x_ld, *dy = (const T*)p.dy + r * p.dy_ld;
    const float mean = p.mean[r], rstd = p.rstd[r];
    float sums[2] = {}, v[8], d[8], w[8];
    auto load = [&](int64_t c) {
      const int left = n - c < 8 ? (int)(n - c) : 8;
      load_upto8(x + c, left, v);
      load_upto8(dy + c, left, d);
      load_param<T>(p.weight, wide, 1.0f, c, left, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = e < left ? (v[e] - mean) * rstd : 0.0f;
        d[e] *= w[e];
      }
      return left;
    };
    for (int64_t c = threadIdx.x * 8; c < n; c += 8192) {
      load(c);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sums[0] += d[e];
        sums[1] = __builtin_fmaf(d[e], v[e], sums[1]);
      }
    }
    row_sums<1024, 1024, 2>(sums, slots, turn);
    const float a = sums[0] / (float)n, b = sums[1] / (float)n;
    for (int64_t c = threadIdx.x * 8; c < n; c += 8192) {
      const int left = load(c);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = rstd * (d[e] - a - v[e] * b);
      store_upto8((T*)p.dx + r * p.dx_ld + c, left, v);
    }
  }
}
// and the sums over rows by columns: 64 threads of 8 columns, 4 rows at a time
template <typename T>
static __global__ __launch_bounds__(256) void norm_backward_columns(const eas_hip_layer_norm_backward_args p, float* part) {
  __shared__ float sums[2][4][8][64];
  const int x = threadIdx.x & 63, y = threadIdx.x >> 6;
  const int64_t n = p.n, c = ((int64_t)blockIdx.x * 64 + x) * 8;
  const int left = c >= n ? 0 : n - c < 8 ? (int)(n - c) : 8;
  float dw[8] = {}, db[8] = {}, v[8], d[8];
  for (int64_t r = (int64_t)blockIdx.y * 4 + y; r < p.m; r += (int64_t)gridDim.y * 4) {
    const float mean = p.mean[r], rstd = p.rstd[r];
    load_upto8((const T*)p.x + r * p.x_ld + c, left, v);
    load_upto8((const T*)p.dy + r * p.dy_ld + c, left, d);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      dw[e] = __builtin_fmaf(d[e], (v[e] - mean) * rstd, dw[e]);
      db[e] += d[e];
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) sums[0][y][e][x] = dw[e], sums[1][y][e][x] = db[e];
  __syncthreads();
  for (int i = threadIdx.x; i < 1024; i += 256) {
    const int k = i >> 9, e = (i >> 6) & 7, xx = i & 63;
    const int64_t col = ((int64_t)blockIdx.x * 64 + xx) * 8 + e;
    if (col < n)
      part[((int64_t)blockIdx.y * 2 + k) * n + col] = (sums[k][0][e][xx] + sums[k][1][e][xx]) + (sums[k][2][e][xx] + sums[k][3][e][xx]);
  }
}

constexpr int64_t kBackwardRegisters = 16384;  // longest row of the register kernels

static int backward_threads(int64_t n) { return n <= 1024 ? 64 : n <= 2048 ? 128 : n <= 4096 ? 256 : 512; }

// Workgroups, each of which writes one row of partial sums: one a CU, with two rows of each in flight.  Twice as many
// read and write twice the partial sums for the same time (8192 x 4096 bf16 42.7 us and 45.4, 4096 x 4096 fp32 43.2 and
// 45.7, both with the launch that adds the partial sums).
int layer_norm_backward_chunks(const eas_hip_layer_norm_backward_args& a) {
  if (!a.m) return 0;
  if (a.n > kBackwardRegisters) {
    const int64_t rows = (a.m + 3) / 4;
    return (int)(rows < 32 ? rows : 32);
  }
  const int tpr = backward_threads(a.n), wg = tpr < 256 ? 256 : tpr, rpw = wg / tpr;
  return (int)even_groups((a.m + rpw - 1) / rpw, 256);
}

template <typename T, bool EVEN, int VPT, int TPR>
static void backward_rows_launch(const eas_hip_layer_norm_backward_args& a, float* part, int chunks, hipStream_t stream) {
  norm_backward_rows<T, EVEN, VPT, TPR><<<chunks, TPR < 256 ? 256 : TPR, 0, stream>>>(a, part);
}

template <typename T, bool EVEN>
static void backward_typed(const eas_hip_layer_norm_backward_args& a, float* part, int chunks, hipStream_t stream) {
  if (a.n <= 512) backward_rows_launch<T, EVEN, 1, 64>(a, part, chunks, stream);
  else if (a.n <= 1024) backward_rows_launch<T, EVEN, 2, 64>(a, part, chunks, stream);
  else if (a.n <= 2048) backward_rows_launch<T, EVEN, 2, 128>(a, part, chunks, stream);
  else if (a.n <= 4096) backward_rows_launch<T, EVEN, 2, 256>(a, part, chunks, stream);
  else if (a.n <= 8192) backward_rows_launch<T, EVEN, 2, 512>(a, part, chunks, stream);
  else if (a.n <= 12288) backward_rows_launch<T, EVEN, 3, 512>(a, part, chunks, stream);
  else if (a.n <= kBackwardRegisters) backward_rows_launch<T, EVEN, 4, 512>(a, part, chunks, stream);
  else {
    if (part)  // before dx, which may take dy's place
      norm_backward_columns<T><<<dim3((unsigned)((a.n + 511) / 512), chunks), 256, 0, stream>>>(a, part);
    if (a.dx) norm_backward_long<T><<<(unsigned)(a.m < 512 ? a.m : 512), 1024, 0, stream>>>(a);
  }
}

hipError_t layer_norm_backward_launch(const eas_hip_layer_norm_backward_args& a, float* part, int chunks, hipStream_t stream) {
  const bool even = even_rows(a.x, a.x_ld, a.n) && even_rows(a.dy, a.dy_ld, a.n) && even_rows(a.dx, a.dx_ld, a.n) &&
                    even_rows(a.weight, 0, a.n);
  if (a.dtype == EAS_HIP_F16) even ? backward_typed<f16, true>(a, part, chunks, stream) : backward_typed<f16, false>(a, part, chunks, stream);
  else if (a.dtype == EAS_HIP_BF16) even ? backward_typed<bf16, true>(a, part, chunks, stream) : backward_typed<bf16, false>(a, part, chunks, stream);
  else backward_typed<float, true>(a, part, chunks, stream);
  return hipGetLastError();
}

}  // namespace eas
