// ops.h — what the operators' translation units share: kernel parameters and launchers.
#ifndef EAS_OPS_OPS_H
#define EAS_OPS_OPS_H

#include <hip/hip_runtime_api.h>

#include <cstddef>
#include <cstdint>

#include "eas_hip.h"

namespace eas {

typedef _Float16 f16;
typedef __bf16 bf16;

// One matrix product, or two of the same shape.  C[m, n] = sum over k of A[m, k] B[k, n], and what the epilogue
// makes of it.  An operand is `k-rows` when its memory rows run along k (A as [m][k], B as [n][k]) and
// `outer-rows` when they run along m or n (A as [k][m], B as [k][n]).
struct GemmParams {
  const void* a[2];      // [1]: of the second segment or product
  const void* b[2];      // [1]: of the second segment or product, or the gated product's up weights
  void* c[2];            // [1]: of the second product
  void* pre[2];          // optional: the product before the activation; gated: gate and up
  const void* bias[2];   // optional; gated: gate's and up's
  const void* res;       // optional
  float* part;           // with splits > 1: [split][product][m][n (gated: gate | up)]
  int64_t lda[2], ldb[2], ldc[2], ldpre[2], ldres;
  int m, n, k;           // k: of each segment
  int segs;              // 2: C = A0 B0 + A1 B1
  int prods;             // 2: C0 = A0 B0 and C1 = A1 B1
  int splits;            // ranges of k, joined by gemm_join
  int act;
  int wide;              // c, pre and res are f32, whatever the operands are
  int kt;                // stages of a segment in the chosen kernel
  int tiles_m, tiles_n;
  int width;             // few rows: columns of a workgroup, a multiple of 8 up to skinny_columns
};

enum GemmKernel { kGemmSkinny1, kGemmSkinny2, kGemmSkinny4, kGemmTile64, kGemmTile128, kGemmTile256 };

struct GemmForm {        // what a kernel is compiled for
  int dtype;
  bool a_outer, b_outer; // outer-rows operands
  bool gated;
  bool any;              // few rows of 16-bit operands: rows of any alignment and length, through registers
  int64_t a_row = 0, b_row = 0;  // bytes from row to row of the operands, the larger of two; for the plan
};

// The few-row kernels' columns per workgroup (gated: of each weight) and bytes of k per stage, by the layout of B: runs
// of 256 bytes of its rows, or of 128 where they run along k.
constexpr int skinny_columns(bool b_outer) { return b_outer ? 128 : 64; }
constexpr int skinny_bytes(bool b_outer) { return b_outer ? 64 : 128; }
// Launches `p`, whose kt, tiles_m and tiles_n are the kernel's.
template <typename T> hipError_t gemm_launch_typed(GemmKernel kernel, const GemmForm& form, const GemmParams& p, hipStream_t stream);
// A gradient's dx (b_outer: its weights are outer rows) and dW (dw.prods of them), whose kt and tiles are kGemmTile64's
template <typename T> hipError_t gemm_pair_typed(bool b_outer, const GemmParams& dx, const GemmParams& dw, hipStream_t stream);
// Sums the parts of a launch with splits > 1 in the order of k and runs its epilogue.
template <typename T> hipError_t gemm_join_typed(bool gated, const GemmParams& p, hipStream_t stream);

// What comes before the products, in one launch: the gradients of an epilogue, elementwise, with their sums over rows,
// and up to three matrices copied to rows at a multiple of 16 bytes, the elements from `cols` to `dst_ld` zero.
struct PrepareParams {
  const void* dy;
  const void* pre[2];    // linear: z (null: dz is dy); gated: gate and up
  void* dz[2];           // of the operands' type (null: the sums alone); gated: dg and du
  float* part;           // [chunk][sum][n] sums over a chunk's rows
  void* sum[2];          // without part, of one chunk: the sums themselves, of the operands' type or f32
  int64_t dy_ld, pre_ld[2], dz_ld;
  int m, n, rows_per_chunk, chunks, across, tx;  // chunks 0: no dz and no sums
  int act, dtype, sum_wide;
  bool gated, stream;    // stream: dy and pre past the caches
  const void* src[3];
  void* dst[3];
  int64_t src_ld[3], dst_ld[3];
  int rows[3], cols[3];
  int copies;
  int dz_groups;         // filled in by the launch
};
hipError_t prepare_launch(PrepareParams p, hipStream_t stream);

// out[i] = sum over chunks of part[chunk][i], for `outs` outputs of n each, of type dtype
struct ColumnSumParams {
  const float* part;
  void* out[2];
  int n, outs, chunks, dtype;
};
hipError_t column_sum_launch(const ColumnSumParams& p, hipStream_t stream);

hipError_t layer_norm_launch(const eas_hip_layer_norm_args& a, hipStream_t stream);
int layer_norm_backward_chunks(const eas_hip_layer_norm_backward_args& a);
hipError_t layer_norm_backward_launch(const eas_hip_layer_norm_backward_args& a, float* part, int chunks, hipStream_t stream);

// eas_hip.cpp's error slot
int fail_status(int code, const char* message);

}  // namespace eas

#endif  // EAS_OPS_OPS_H
