// rms.hip — the root-mean-square norm with the residual's addition and an 8-bit output, and its gradients.
//
// Forward: h = x + residual in 32 bits, rstd = (sum(h^2)/n + eps)^-1/2, y = h rstd weight, and y in 8 bits by blocks of
// 128 columns.  A row stays in registers from its one read to its last write: TPR threads of VPT vectors of 8, one sum
// over them; 16 neighbouring lanes hold a block, whose largest magnitude they find by rotating their values among them.
// Rows beyond 16384 elements are read twice instead.
//
// Backward, with g = dy weight: dx = rstd (g - h rstd^2 mean(g h)) + dtotal, dweight = sum(dy h rstd) over rows.  A
// thread owns its columns: it adds their dweight over all the rows that its workgroup takes, each workgroup writes one
// row of partial sums, and column_sum adds those.
//
// Both are bound by memory.  Forward 8192 x 4096 bf16 with residual, total and q: 39.3 us (6.0 TB/s).  Backward of the same
// with dtotal: 46.6 us with the sums' second launch (5.8 TB/s), 4.8 of it that.
#include "e4m3.h"
#include "rows.h"

namespace eas {

// ---- forward ----------------------------------------------------------------------

// y in 8 bits from column c on (t: its thread's place in the row), and its block's scale.  EVEN rows: the stores as a
// buffer's, with no branch around them.
template <bool EVEN>
static __device__ __forceinline__ void store_q(const eas_hip_rms_norm_args& p, int64_t r, bool live, int64_t c, int left, const float (&y)[8]) {
  const float scale = scale_of(block_max(y));
  const u32x2 q = to_e4m3(y, scale, 1.0f / scale);
  const bool mine = (threadIdx.x & 15) == 0 && left > 0;
  const int64_t b = c / kBlock;
  if constexpr (EVEN) {
    __builtin_amdgcn_raw_buffer_store_b64(q, row_buffer((const char*)p.q + r * p.q_ld, p.n, live), (int)c, 0, 0);
    const int64_t blocks = (p.n - 1) / kBlock;
    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, scale),
                                          row_buffer(p.q_scale + r * p.q_scale_row, blocks * p.q_scale_block + 1, live),
                                          mine ? (int)(b * p.q_scale_block * 4) : 0x7ffffff0, 0, 0);
  } else {
    if (!live) return;
    store_bytes((uint8_t*)p.q + r * p.q_ld + c, left, q);
    if (mine) p.q_scale[r * p.q_scale_row + b * p.q_scale_block] = scale;
  }
}

// H: residual's and total's type.  A workgroup takes RPW rows at a time, those of the grid side by side in memory, and
// loads its next ones before it reduces these: the loads are in flight while the sums meet.
template <typename T, typename H, bool EVEN, bool STREAM, int VPT, int TPR>
static __global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void rms_rows(const eas_hip_rms_norm_args p, bool stream_total) {
  constexpr int WG = TPR < 256 ? 256 : TPR, RPW = WG / TPR;
  __shared__ float slots[2 * (WG / 64)];
  const int t = threadIdx.x % TPR;
  const int64_t n = p.n;
  const bool wide = p.wdtype == EAS_HIP_F32;
  float w[VPT][8];
  int left[VPT];
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    const int64_t c = ((int64_t)v * TPR + t) * 8;
    left[v] = c >= n ? 0 : n - c < 8 ? (int)(n - c) : 8;
  }
  int turn = 0;
  const int64_t first = (int64_t)blockIdx.x * RPW, stride = (int64_t)gridDim.x * RPW, end = p.m;
  typename Vec8<T>::type ahead[VPT];
  typename Vec8<H>::type res[VPT];
  auto fetch = [&](int64_t r) __attribute__((always_inline)) {
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      ahead[v] = row_load<T, EVEN, STREAM>((const T*)p.x + r * p.x_ld, n, r < end, (v * TPR + t) * 8, left[v]);
      res[v] = row_load<H, EVEN, STREAM>((const H*)p.residual + r * p.residual_ld, n, r < end && p.residual, (v * TPR + t) * 8, left[v]);
    }
  };
  const int group = __builtin_amdgcn_readfirstlane(threadIdx.x / TPR);
  fetch(first + group);
  {
    RawParam raw[VPT];
#pragma unroll
    for (int v = 0; v < VPT; ++v) fetch_param<T, EVEN>(p.weight, wide, n, (v * TPR + t) * 8, raw[v]);
#pragma unroll
    for (int v = 0; v < VPT; ++v) take_param<T, EVEN>(p.weight, wide, 1.0f, (v * TPR + t) * 8, left[v], raw[v], w[v]);
  }
  // every thread of the workgroup runs every turn: the sums' barriers are the workgroup's
  for (int64_t r0 = first; r0 < end; r0 += stride) {
    const int64_t r = r0 + group;
    const bool live = r < end;
    float h[VPT][8];
    float s[1] = {};
#pragma unroll
    for (int v = 0; v < VPT; ++v)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        h[v][e] = (float)ahead[v][e] + (float)res[v][e];  // past the row's end 0
        s[0] = __builtin_fmaf(h[v][e], h[v][e], s[0]);
      }
    fetch(r + stride);
#pragma unroll
    for (int v = 0; v < VPT; ++v)
      row_store<H, EVEN>((H*)p.total + r * p.total_ld, n, live && p.total, (v * TPR + t) * 8, left[v], stream_total, h[v]);
    row_sums<TPR, WG, 1>(s, slots, turn);
    const float rstd = 1.0f / sqrtf(s[0] / (float)n + p.eps);
    stat_store<EVEN>(p.rstd + r, live && p.rstd, t == 0, rstd);
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
#pragma unroll
      for (int e = 0; e < 8; ++e) h[v][e] = h[v][e] * rstd * w[v][e];
      row_store<T, EVEN>((T*)p.y + r * p.y_ld, n, live && p.y, (v * TPR + t) * 8, left[v], false, h[v]);
      if (p.q) store_q<EVEN>(p, r, live, (v * TPR + t) * 8, left[v], h[v]);
    }
  }
}

// rows of any length, one workgroup each
template <typename T, typename H> static __global__ __launch_bounds__(1024) void rms_long(const eas_hip_rms_norm_args p) {
  __shared__ float slots[2 * 16];
  const bool wide = p.wdtype == EAS_HIP_F32;
  const int64_t n = p.n, wave = threadIdx.x & ~63;
  int turn = 0;
  for (int64_t r = blockIdx.x; r < p.m; r += gridDim.x) {
    float s[1] = {}, h[8], t[8], w[8];
    auto load = [&](int64_t c) {
      const int left = n - c < 8 ? (c < n ? (int)(n - c) : 0) : 8;
      load_upto8((const T*)p.x + r * p.x_ld + c, left, h);
      load_upto8((const H*)p.residual + r * p.residual_ld + c, p.residual ? left : 0, t);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] += t[e];
      return left;
    };
    for (int64_t c = threadIdx.x * 8; c < n; c += 8192) {
      load(c);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[0] = __builtin_fmaf(h[e], h[e], s[0]);
    }
    row_sums<1024, 1024, 1>(s, slots, turn);
    const float rstd = 1.0f / sqrtf(s[0] / (float)n + p.eps);
    if (threadIdx.x == 0 && p.rstd) p.rstd[r] = rstd;
    // whole waves: a block's lanes find its largest magnitude together
    for (int64_t c0 = wave * 8; c0 < n; c0 += 8192) {
      const int64_t c = c0 + (threadIdx.x & 63) * 8;
      const int left = load(c);
      if (p.total) store_upto8((H*)p.total + r * p.total_ld + c, left, h);
      load_param<T>(p.weight, wide, 1.0f, c, left, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] = h[e] * rstd * w[e];
      if (p.y) store_upto8((T*)p.y + r * p.y_ld + c, left, h);
      if (p.q) store_q<false>(p, r, true, c, left, h);
    }
  }
}

// Whether rows of `ld` elements start where a 128-byte line does: past the caches, a line that two rows share is read twice
// (1031 x 4099 f32 14.8 -> 22.1 us).
static bool whole_lines(const void* p, int64_t ld, int size) { return !p || ((uint64_t)p % 128 == 0 && ld * size % 128 == 0); }

template <typename T, typename H, bool EVEN, int VPT, int TPR> static void rms_rows_launch(const eas_hip_rms_norm_args& a, hipStream_t stream) {
  constexpr int WG = TPR < 256 ? 256 : TPR, RPW = WG / TPR;
  const unsigned grid = (unsigned)even_groups((a.m + RPW - 1) / RPW, 256 * (1024 / WG));
  // Past the memory-side cache (256 MB): what is read, where all that is moved would fill most of it (8192 x 4096 bf16 45.6 ->
  // 39.6 us with total so; 2048 x 8192 20.3 -> 23.1), and total from a quarter on (2048 x 8192 25.9 -> 20.3).
  const int64_t moved = a.m * a.n * ((int64_t)sizeof(T) * (a.y ? 2 : 1) + (int64_t)sizeof(H) * ((a.residual ? 1 : 0) + (a.total ? 1 : 0)) + (a.q ? 1 : 0));
  const bool stream_total = moved > (64 << 20);
  if constexpr (EVEN && VPT * TPR >= 512) {
    if (moved > (192 << 20) && whole_lines(a.x, a.x_ld, sizeof(T)) && whole_lines(a.residual, a.residual_ld, sizeof(H))) {
      rms_rows<T, H, EVEN, true, VPT, TPR><<<grid, WG, 0, stream>>>(a, stream_total);
      return;
    }
  }
  rms_rows<T, H, EVEN, false, VPT, TPR><<<grid, WG, 0, stream>>>(a, stream_total);
}

template <typename T, typename H, bool EVEN> static void rms_sized(const eas_hip_rms_norm_args& a, hipStream_t stream) {
  if (a.n <= 512) rms_rows_launch<T, H, EVEN, 1, 64>(a, stream);
  else if (a.n <= 1024) rms_rows_launch<T, H, EVEN, 2, 64>(a, stream);
  else if (a.n <= 2048) rms_rows_launch<T, H, EVEN, 1, 256>(a, stream);
  else if (a.n <= 4096) rms_rows_launch<T, H, EVEN, 2, 256>(a, stream);
  else if (a.n <= 6144) rms_rows_launch<T, H, EVEN, 3, 256>(a, stream);
  else if (a.n <= 8192) rms_rows_launch<T, H, EVEN, 4, 256>(a, stream);
  else if (a.n <= 12288) rms_rows_launch<T, H, EVEN, 3, 512>(a, stream);
  else if (a.n <= 16384) rms_rows_launch<T, H, EVEN, 4, 512>(a, stream);
  else rms_long<T, H><<<(unsigned)(a.m < 512 ? a.m : 512), 1024, 0, stream>>>(a);
}

template <typename T> static void rms_typed(bool even, const eas_hip_rms_norm_args& a, hipStream_t stream) {
  if (a.hdtype == EAS_HIP_F32 && sizeof(T) == 2) even ? rms_sized<T, float, true>(a, stream) : rms_sized<T, float, false>(a, stream);
  else even ? rms_sized<T, T, true>(a, stream) : rms_sized<T, T, false>(a, stream);
}

hipError_t rms_norm_launch(const eas_hip_rms_norm_args& a, hipStream_t stream) {
  bool even = true;
  if (a.dtype != EAS_HIP_F32)
    even = even_rows(a.x, a.x_ld, a.n) && even_rows(a.y, a.y_ld, a.n) && even_rows(a.residual, a.residual_ld, a.n) &&
           even_rows(a.total, a.total_ld, a.n) && even_rows(a.weight, 0, a.n);
  // 8-bit rows of whole 4 bytes at multiples of 4, and scales within a buffer's reach
  if (a.q) even = even && (uint64_t)a.q % 4 == 0 && a.q_ld % 4 == 0 && a.n % 4 == 0 && (a.n / kBlock + 1) * a.q_scale_block < (1 << 28);
  if (a.dtype == EAS_HIP_F16) rms_typed<f16>(even, a, stream);
  else if (a.dtype == EAS_HIP_BF16) rms_typed<bf16>(even, a, stream);
  else rms_typed<float>(even, a, stream);
  return hipGetLastError();
}

// ---- backward ---------------------------------------------------------------------

template <typename T, typename H, bool EVEN, bool STREAM, int VPT, int TPR>
static __device__ __forceinline__ void backward_part(const eas_hip_rms_norm_backward_args& p, float* part, int group_id, int groups) {
  constexpr int WG = TPR < 256 ? 256 : TPR, RPW = WG / TPR;
  __shared__ float slots[2 * (WG / 64)];
  __shared__ float meet[RPW > 1 ? RPW * VPT * TPR * 8 : 1];
  constexpr int AHEAD = TPR * VPT > 1024 ? 1 : 2;  // 512 threads leave 256 registers each; four vectors of f32 pass them all the same, by 78 to 91
  const int t = threadIdx.x % TPR, group = __builtin_amdgcn_readfirstlane(threadIdx.x / TPR);
  const int64_t n = p.n;
  const bool wide = p.wdtype == EAS_HIP_F32;
  float w[VPT][8], dw[VPT][8] = {};
  int left[VPT];
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    const int64_t c = ((int64_t)v * TPR + t) * 8;
    left[v] = c >= n ? 0 : n - c < 8 ? (int)(n - c) : 8;
  }
  const float inv = 1.0f / (float)n;
  int turn = 0;
  const int64_t first = (int64_t)group_id * RPW, stride = (int64_t)groups * RPW, end = p.m;
  // the next rows of this thread, in flight while this one is reduced
  struct Row {
    typename Vec8<H>::type h[VPT], d[VPT];
    typename Vec8<T>::type g[VPT];
    float rstd;
  };
  auto fetch = [&](Row& q, int64_t r) __attribute__((always_inline)) {
    const bool live = r < end;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int c = (v * TPR + t) * 8;
      q.h[v] = row_load<H, EVEN, STREAM>((const H*)p.h + r * p.h_ld, n, live, c, left[v]);
      q.g[v] = row_load<T, EVEN, STREAM>((const T*)p.dy + r * p.dy_ld, n, live, c, left[v]);
      q.d[v] = row_load<H, EVEN, STREAM>((const H*)p.dtotal + r * p.dtotal_ld, n, live && p.dtotal, c, left[v]);
    }
    q.rstd = stat_load<EVEN>(p.rstd + r, live);
  };
  auto one = [&](Row& q, int64_t r0) __attribute__((always_inline)) {
    const int64_t r = r0 + group;
    const float rstd = uniform(q.rstd);  // the wave's row
    // Past the row's end, and for a row past the last, dy, h and dtotal are 0
    float h[VPT][8], g[VPT][8], d[VPT][8];
    float sums[1] = {};
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        h[v][e] = (float)q.h[v][e];
        g[v][e] = (float)q.g[v][e] * rstd;
        d[v][e] = (float)q.d[v][e];
        dw[v][e] = __builtin_fmaf(g[v][e], h[v][e], dw[v][e]);
        g[v][e] *= w[v][e];
        sums[0] = __builtin_fmaf(g[v][e], h[v][e], sums[0]);
      }
    }
    fetch(q, r + AHEAD * stride);
    row_sums<TPR, WG, 1>(sums, slots, turn);
    const float b = -rstd * rstd * (sums[0] * inv);
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
#pragma unroll
      for (int e = 0; e < 8; ++e) h[v][e] = __builtin_fmaf(h[v][e], b, g[v][e]) + d[v][e];
      row_store<H, EVEN>((H*)p.dx + r * p.dx_ld, n, r < end && p.dx, (v * TPR + t) * 8, left[v], false, h[v]);
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
  float* out = part + (int64_t)group_id * n;
  if constexpr (RPW > 1) {  // the row groups' sums first
    __syncthreads();
#pragma unroll
    for (int v = 0; v < VPT; ++v)
#pragma unroll
      for (int e = 0; e < 8; ++e) meet[(group * VPT * 8 + v * 8 + e) * TPR + t] = dw[v][e];
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
    for (int v = 0; v < VPT; ++v) store_upto8(out + ((int64_t)v * TPR + t) * 8, left[v], dw[v]);
  }
}

template <typename T, typename H, bool EVEN, bool STREAM, int VPT, int TPR>
static __global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void rms_backward_rows(const eas_hip_rms_norm_backward_args p, float* part) {
  backward_part<T, H, EVEN, STREAM, VPT, TPR>(p, part, blockIdx.x, gridDim.x);
}

// Few elements: dx by the first `groups` workgroups, and dweight itself, whose sums a workgroup makes for each 8 columns, in
// one launch.  A second one for partial sums costs as much as the first (517 x 1023 f16 10.7 -> 6.4 us).  The columns'
// workgroups read h and dy again, from L2: neighbouring strips go to one XCD, whose lines they share.
template <typename T, typename H, bool EVEN, int VPT, int TPR>
static __global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void rms_backward_few(const eas_hip_rms_norm_backward_args p, int groups, int strips) {
  constexpr int WG = TPR < 256 ? 256 : TPR;
  const int id = blockIdx.x - groups;
  if (id < 0) {
    backward_part<T, H, EVEN, false, VPT, TPR>(p, nullptr, blockIdx.x, groups);
    return;
  }
  __shared__ float sums[WG / 64][8];
  const int strip = id % 8 * (strips / 8) + id / 8;  // strips is a multiple of 8
  const int64_t n = p.n, c = (int64_t)strip * 8;
  const int left = c >= n ? 0 : n - c < 8 ? (int)(n - c) : 8;
  float dw[8] = {};
  for (int64_t r = threadIdx.x; r < p.m; r += WG) {
    float h[8], d[8];
    const float rstd = p.rstd[r];
    load_upto8((const H*)p.h + r * p.h_ld + c, left, h);
    load_upto8((const T*)p.dy + r * p.dy_ld + c, left, d);
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[e] = __builtin_fmaf(d[e] * rstd, h[e], dw[e]);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) dw[e] = wave_sum(dw[e]);
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[threadIdx.x >> 6][e] = dw[e];
  __syncthreads();
  if ((int)threadIdx.x < left) {
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < WG / 64; ++w) s += sums[w][threadIdx.x];
    if (p.wdtype == EAS_HIP_F32) ((float*)p.dweight)[c + threadIdx.x] = s;
    else ((T*)p.dweight)[c + threadIdx.x] = (T)s;
  }
}

// rows beyond what the registers hold: dx one row per workgroup, read twice
template <typename T, typename H>
static __global__ __launch_bounds__(1024) void rms_backward_long(const eas_hip_rms_norm_backward_args p) {
  __shared__ float slots[2 * 16];
  const bool wide = p.wdtype == EAS_HIP_F32;
  const int64_t n = p.n;
  int turn = 0;
  for (int64_t r = blockIdx.x; r < p.m; r += gridDim.x) {
    const float rstd = p.rstd[r];
    float sums[1] = {}, h[8], g[8], w[8];
    auto load = [&](int64_t c) {
      const int left = n - c < 8 ? (int)(n - c) : 8;
      load_upto8((const H*)p.h + r * p.h_ld + c, left, h);
      load_upto8((const T*)p.dy + r * p.dy_ld + c, left, g);
      load_param<T>(p.weight, wide, 1.0f, c, left, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) g[e] = g[e] * rstd * w[e];
      return left;
    };
    for (int64_t c = threadIdx.x * 8; c < n; c += 8192) {
      load(c);
#pragma unroll
      for (int e = 0; e < 8; ++e) sums[0] = __builtin_fmaf(g[e], h[e], sums[0]);
    }
    row_sums<1024, 1024, 1>(sums, slots, turn);
    const float b = -rstd * rstd * (sums[0] / (float)n);
    for (int64_t c = threadIdx.x * 8; c < n; c += 8192) {
      const int left = load(c);
      load_upto8((const H*)p.dtotal + r * p.dtotal_ld + c, p.dtotal ? left : 0, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] = __builtin_fmaf(h[e], b, g[e]) + w[e];
      store_upto8((H*)p.dx + r * p.dx_ld + c, left, h);
    }
  }
}
// and the sums over rows by columns: 64 threads of 8 columns, 4 rows at a time
template <typename T, typename H>
static __global__ __launch_bounds__(256) void rms_backward_columns(const eas_hip_rms_norm_backward_args p, float* part) {
  __shared__ float sums[4][8][64];
  const int x = threadIdx.x & 63, y = threadIdx.x >> 6;
  const int64_t n = p.n, c = ((int64_t)blockIdx.x * 64 + x) * 8;
  const int left = c >= n ? 0 : n - c < 8 ? (int)(n - c) : 8;
  float dw[8] = {}, h[8], d[8];
  for (int64_t r = (int64_t)blockIdx.y * 4 + y; r < p.m; r += (int64_t)gridDim.y * 4) {
    const float rstd = p.rstd[r];
    load_upto8((const H*)p.h + r * p.h_ld + c, left, h);
    load_upto8((const T*)p.dy + r * p.dy_ld + c, left, d);
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[e] = __builtin_fmaf(d[e] * rstd, h[e], dw[e]);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) sums[y][e][x] = dw[e];
  __syncthreads();
  for (int i = threadIdx.x; i < 512; i += 256) {
    const int e = i >> 6, xx = i & 63;
    const int64_t col = ((int64_t)blockIdx.x * 64 + xx) * 8 + e;
    if (col < n) part[(int64_t)blockIdx.y * n + col] = (sums[0][e][xx] + sums[1][e][xx]) + (sums[2][e][xx] + sums[3][e][xx]);
  }
}

constexpr int64_t kBackwardRegisters = 16384;  // longest row of the register kernels

static int backward_threads(int64_t n) { return n <= 1024 ? 64 : n <= 2048 ? 128 : n <= 4096 ? 256 : 512; }

// Few elements, whose dweight is summed by strips of 8 columns, without scratch.  Measured, bf16, us, in one launch / in two: 256 x
// 4096 5.5 / 9.3, 1024 x 1024 5.5 / 10.1, 2048 x 512 6.0 / 10.0, 4096 x 128 9.4 / 10.3; the rule takes it also at 4096 x 256, 12.4 /
// 10.1, and 64 x 16384, 13.0 / 10.6, and leaves 512 x 4096, 7.0 / 9.9, and 1024 x 4096, 10.6 / 12.1.  More rows: 8192 x 128 22.4 / 9.9.
bool rms_norm_backward_few(const eas_hip_rms_norm_backward_args& a) {
  return a.m && a.dx && a.dweight && a.n <= kBackwardRegisters && a.m * a.n <= (1 << 20) && a.m <= 4096;
}

// Workgroups, each of which writes one row of partial sums.  Of long rows 32 chunks, us (8 / 32 / 128): 2048 x 20000 bf16 106 / 92 / 93,
// 256 x 20000 18.6 / 18.9 / 21.3, 64 x 60000 25.4 / 27.8 / 27.8.
int rms_norm_backward_chunks(const eas_hip_rms_norm_backward_args& a) {
  if (!a.m) return 0;
  if (a.n > kBackwardRegisters) {
    const int64_t rows = (a.m + 3) / 4;
    return (int)(rows < 32 ? rows : 32);
  }
  const int tpr = backward_threads(a.n), wg = tpr < 256 ? 256 : tpr, rpw = wg / tpr;
  return (int)even_groups((a.m + rpw - 1) / rpw, 256);
}

template <typename T, typename H, bool EVEN, int VPT, int TPR>
static void backward_rows_launch(const eas_hip_rms_norm_backward_args& a, float* part, int chunks, hipStream_t stream) {
  constexpr int WG = TPR < 256 ? 256 : TPR;
  if (rms_norm_backward_few(a)) {
    const int strips = (int)((a.n + 63) / 64 * 8);
    if (a.dx == a.dy || a.dx == a.h) {  // the strips first, which read what dx takes the place of
      rms_backward_few<T, H, EVEN, VPT, TPR><<<strips, WG, 0, stream>>>(a, 0, strips);
      rms_backward_few<T, H, EVEN, VPT, TPR><<<chunks, WG, 0, stream>>>(a, chunks, 0);
    } else {
      rms_backward_few<T, H, EVEN, VPT, TPR><<<chunks + strips, WG, 0, stream>>>(a, chunks, strips);
    }
    return;
  }
  if constexpr (EVEN && VPT * TPR >= 512) {
    // what is read past the memory-side cache, where it would fill much of it: 8192 x 4096 bf16 53.0 -> 47.4 us, 2048 x 8192 30.2 -> 28.3;
    // not 1024 x 4096, 13.4 -> 13.9
    const int64_t moved = a.m * a.n * ((int64_t)sizeof(T) + (int64_t)sizeof(H) * (a.dtotal ? 3 : 2));
    if (moved > (128 << 20) && whole_lines(a.h, a.h_ld, sizeof(H)) && whole_lines(a.dy, a.dy_ld, sizeof(T)) &&
        whole_lines(a.dtotal, a.dtotal_ld, sizeof(H))) {
      rms_backward_rows<T, H, EVEN, true, VPT, TPR><<<chunks, WG, 0, stream>>>(a, part);
      return;
    }
  }
  rms_backward_rows<T, H, EVEN, false, VPT, TPR><<<chunks, WG, 0, stream>>>(a, part);
}

template <typename T, typename H, bool EVEN>
static void backward_sized(const eas_hip_rms_norm_backward_args& a, float* part, int chunks, hipStream_t stream) {
  if (a.n <= 512) backward_rows_launch<T, H, EVEN, 1, 64>(a, part, chunks, stream);
  else if (a.n <= 1024) backward_rows_launch<T, H, EVEN, 2, 64>(a, part, chunks, stream);
  else if (a.n <= 2048) backward_rows_launch<T, H, EVEN, 2, 128>(a, part, chunks, stream);
  else if (a.n <= 4096) backward_rows_launch<T, H, EVEN, 2, 256>(a, part, chunks, stream);
  else if (a.n <= 8192) backward_rows_launch<T, H, EVEN, 2, 512>(a, part, chunks, stream);
  else if (a.n <= 12288) backward_rows_launch<T, H, EVEN, 3, 512>(a, part, chunks, stream);
  else if (a.n <= kBackwardRegisters) backward_rows_launch<T, H, EVEN, 4, 512>(a, part, chunks, stream);
  else {
    if (part)  // before dx, which may take dy's or h's place
      rms_backward_columns<T, H><<<dim3((unsigned)((a.n + 511) / 512), chunks), 256, 0, stream>>>(a, part);
    if (a.dx) rms_backward_long<T, H><<<(unsigned)(a.m < 512 ? a.m : 512), 1024, 0, stream>>>(a);
  }
}

template <typename T>
static void backward_typed(bool even, const eas_hip_rms_norm_backward_args& a, float* part, int chunks, hipStream_t stream) {
  if constexpr (sizeof(T) == 4) backward_sized<T, T, true>(a, part, chunks, stream);
  else if (a.hdtype == EAS_HIP_F32)
    even ? backward_sized<T, float, true>(a, part, chunks, stream) : backward_sized<T, float, false>(a, part, chunks, stream);
  else even ? backward_sized<T, T, true>(a, part, chunks, stream) : backward_sized<T, T, false>(a, part, chunks, stream);
}

hipError_t rms_norm_backward_launch(const eas_hip_rms_norm_backward_args& a, float* part, int chunks, hipStream_t stream) {
  const bool even = even_rows(a.h, a.h_ld, a.n) && even_rows(a.dy, a.dy_ld, a.n) && even_rows(a.dx, a.dx_ld, a.n) &&
                    even_rows(a.dtotal, a.dtotal_ld, a.n) && even_rows(a.weight, 0, a.n);
  if (a.dtype == EAS_HIP_F16) backward_typed<f16>(even, a, part, chunks, stream);
  else if (a.dtype == EAS_HIP_BF16) backward_typed<bf16>(even, a, part, chunks, stream);
  else backward_typed<float>(even, a, part, chunks, stream);
  return hipGetLastError();
}

}  // namespace eas
