// Arguments of the products with an operand held in few bits (w4.cu, act8.cu).
#pragma once
#include <stdint.h>

#include "../../include/subcuber_b200.h"
#include "sw_host.h"

namespace sb200 {
namespace lowbit {

// Weights in format W4 (lowbit_format.cuh); zeros == nullptr: symmetric.
struct W4 {
  DType dtype;  // of the scales and of the activations: kF16 or kBF16
  int n, k, group;
  const void* codes;
  const void* scales;
  const void* zeros;
};

// Activations in format ACT8; rows of codes start every `pitch` bytes, rows of exponents every `exp_pitch`.
struct Act8 {
  DType dtype;  // of the activations and of dY: kF16 or kBF16
  int m, k;
  const void* codes;
  long long pitch;
  const void* exps;
  long long exp_pitch;
};

inline bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
// Rows of a 16-bit matrix that TMA can read as they are.
inline bool tma_rows(const void* p, long long ld) { return aligned(p, 16) && ld % 8 == 0; }

// Extents are held in 32 bits, rounded up to whole tiles too.
constexpr int kMaxExtent = 0x7fffff00;

// The device-side waits of a product: how long one lasts at most, and the test aid that makes them run out (left tiles are not
// announced to the matrix instructions).
struct Waits {
  unsigned long long ns;
  int drop;
};
// From a call's options (null: 2 s); only those that concern waits are supported.
inline int waits_of(const sb200_gemm_options* o, Waits* w) {
  *w = Waits{2000000000ull, 0};
  if (!o) return kOk;
  if (o->sm_limit != 0 || o->no_split != 0) return kErrNotSupported;
  if (o->wait_limit_us > 0) w->ns = 1000ull * static_cast<unsigned long long>(o->wait_limit_us);
  w->drop = o->drop_split_flags != 0;
  return kOk;
}

// Bytes of a copy of a 16-bit matrix with rows that start on 16 bytes.
inline size_t copy_bytes(long long rows, int cols) {
  const size_t row = (static_cast<size_t>(cols) + 7) / 8 * 16;
  return (static_cast<size_t>(rows) * row + 255) / 256 * 256;
}

// dst (rows x cols_d, packed, cols_d the next multiple of 8) = src (rows x cols, leading dimension ld) of 16-bit elements,
// zeros behind (act8.cu).
int copy_rows_16bit(void* dst, int cols_d, const void* src, int rows, int cols, long long ld, cudaStream_t stream);
// Expansion to 16 bits (w4.cu, act8.cu).
int dequantize_w4(const W4& w, void* out, long long ldo, cudaStream_t stream);
int restore_act8(const Act8& a, void* x, long long ldx, cudaStream_t stream);

// The products on the tensor cores (expand_product.cu).  Workspace: a status word, a copy of the 16-bit operand where its
// rows are not aligned, the operand in 16 bits where it is expanded first, and the parts of a divided reduction at its end.  The bytes asked for grow with m, so that a
// workspace serves every smaller m.
constexpr size_t kStatusBytes = 256;
constexpr int kDecodeMaxRows = 64;
size_t expand_w4_workspace(int m, int n, int k, bool x_aligned);
int decode_w4(const W4& w, const void* x, long long ldx, void* y, long long ldy, int m, void* status, const Waits& waits,
              cudaStream_t stream);
int expand_w4(const W4& w, const void* x, long long ldx, void* y, long long ldy, int m, void* workspace, size_t workspace_bytes,
              const Waits& waits, cudaStream_t stream);
size_t expand_act8_workspace(int m, int n, int k, bool dy_aligned);
int expand_act8(const Act8& a, const void* dy, long long lddy, bool out_f32, const void* base, long long ldbase, void* dw,
                long long lddw, int n, void* workspace, const Waits& waits, cudaStream_t stream);

}  // namespace lowbit
}  // namespace sb200
