// host.h — what the operators' entry points share: refusals, scratch and the areas that arguments cover.
#ifndef EAS_OPS_HOST_H
#define EAS_OPS_HOST_H

#include <cstring>

#include "ops.h"

namespace eas {

#define OPS_CHECK(cond, message) \
  do {                           \
    if (!(cond)) return fail_status(EAS_HIP_ERR_INVALID, message); \
  } while (0)
#define OPS_HIP(call)                                                                               \
  do {                                                                                              \
    const hipError_t e_ = (call);                                                                   \
    if (e_ != hipSuccess) return fail_status(EAS_HIP_ERR_RUNTIME, hipGetErrorString(e_));           \
  } while (0)

#define OPS_TRY(call)      \
  do {                     \
    const int rc_ = (call); \
    if (rc_) return rc_;   \
  } while (0)

constexpr int kCus = 256;
constexpr int64_t kOneChunk = 1 << 21;  // most elements whose sums over rows are made in one stage
constexpr int64_t kMost = 0x7fffff00;  // rows and columns are 32-bit in the kernels

inline int elem(int dtype) { return dtype == EAS_HIP_F32 ? 4 : 2; }
inline bool is_dtype(int d) { return d == EAS_HIP_F16 || d == EAS_HIP_BF16 || d == EAS_HIP_F32; }
inline bool is_act(int a) { return a >= EAS_HIP_ACT_NONE && a <= EAS_HIP_ACT_SILU; }
inline bool size_ok(int64_t n) { return n >= 0 && n <= kMost; }
inline int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }
inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Scratch, laid out the same way when its size is asked for and when it is used.
struct Arena {
  char* base;      // null: only the size is wanted
  uint64_t used = 0;
  void* take(uint64_t bytes) {
    void* p = base ? base + used : nullptr;
    used += (uint64_t)up((int64_t)bytes, 256);
    return p;
  }
};

// Whether two matrices share an element, by their address ranges; matrices of one row stride side by side in the same
// rows (halves of a wider one) do not.
struct Area {
  const void* p;
  int64_t ld, rows, cols;
  int elem;
};
inline bool shares(const Area& a, const Area& b) {
  if (!a.p || !b.p || !a.rows || !b.rows || !a.cols || !b.cols) return false;
  const char *pa = (const char*)a.p, *pb = (const char*)b.p;
  const int64_t la = ((a.rows - 1) * a.ld + a.cols) * a.elem, lb = ((b.rows - 1) * b.ld + b.cols) * b.elem;
  if (pa + la <= pb || pb + lb <= pa) return false;
  if (a.ld * a.elem != b.ld * b.elem) return true;
  const int64_t row = a.ld * a.elem;
  int64_t d = (pb - pa) % row;
  if (d < 0) d += row;
  return d < a.cols * a.elem || row - d < b.cols * b.elem;
}
inline bool same(const Area& a, const Area& b) { return a.p == b.p && a.elem == b.elem && (a.ld == b.ld || a.rows <= 1); }
// No output shares memory with another area, but those named as its input in place.
inline int check_apart(const Area* outs, int n_outs, const Area* ins, int n_ins, const Area* in_place, int n_in_place) {
  for (int i = 0; i < n_outs; ++i) {
    for (int j = i + 1; j < n_outs; ++j) OPS_CHECK(!shares(outs[i], outs[j]), "two outputs share memory");
    for (int j = 0; j < n_ins; ++j) OPS_CHECK(!shares(outs[i], ins[j]), "an output shares memory with an input");
    for (int j = 0; j < n_in_place; ++j)
      OPS_CHECK(!shares(outs[i], in_place[j]) || (i == 0 && same(outs[0], in_place[j])), "an output shares memory with an input");
  }
  return EAS_HIP_OK;
}

template <typename Args> int read_args(const Args* args, size_t size, Args* out) {
  OPS_CHECK(args != nullptr, "args must not be NULL");
  OPS_CHECK(size == sizeof(Args), "args_size is not this operator's");
  memcpy(out, args, sizeof(Args));
  return EAS_HIP_OK;
}

inline int check_workspace(const void* ws, uint64_t bytes, uint64_t need) {
  OPS_CHECK(need == 0 || (ws != nullptr && (uint64_t)ws % 16 == 0), "the workspace must be 16-byte aligned device memory");
  OPS_CHECK(bytes >= need, "the workspace is too small");
  return EAS_HIP_OK;
}

}  // namespace eas

#endif  // EAS_OPS_HOST_H
