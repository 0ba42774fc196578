// Activations saved in 8 bits (format ACT8 of lowbit_format.cuh): saving, restoring, and the weight gradient
// dW = base + X^T dY of a linear layer from them.
#include <stdint.h>

#include "../../include/subcuber_b200.h"
#include "lowbit_format.cuh"
#include "lowbit_host.h"

namespace sb200 {
namespace lowbit {
namespace {

constexpr int kThreads = 256;

// A thread handles 16 channels of a token, half a block.  A power of two of threads stand along a row, the others of
// the 256 on further rows.
struct Cut {
  int pieces;         // 16-channel pieces of a row
  int cols_log2;      // threads along a row, as a power of two
  long long parts;    // thread blocks along a row
  long long blocks;   // thread blocks in all
};

Cut cut_of(int m, int pieces) {
  Cut c;
  c.pieces = pieces;
  c.cols_log2 = 1;
  while (c.cols_log2 < 8 && (1 << c.cols_log2) < c.pieces) ++c.cols_log2;
  c.parts = ceil_div(c.pieces, 1 << c.cols_log2);
  c.blocks = c.parts * ceil_div(m, kThreads >> c.cols_log2);
  return c;
}

// 16 neighbouring values of a row, zeros behind `k`.  A row that does not start on 16 bytes is read in the aligned 8-byte
// words that hold its values, which are shifted together.
template <typename T>
__device__ __forceinline__ void load16(const T* row, int k0, int k, bool wide, T (&v)[16]) {
  if (wide && k0 + 16 <= k) {
    reinterpret_cast<uint4*>(v)[0] = __ldg(reinterpret_cast<const uint4*>(row + k0));
    reinterpret_cast<uint4*>(v)[1] = __ldg(reinterpret_cast<const uint4*>(row + k0) + 1);
    return;
  }
  const uintptr_t at = reinterpret_cast<uintptr_t>(row + k0), end = reinterpret_cast<uintptr_t>(row + k);
  const uint32_t off = at & 7;
  const unsigned long long* word = reinterpret_cast<const unsigned long long*>(at - off);
  unsigned long long w[5];
#pragma unroll
  for (int i = 0; i < 5; ++i) w[i] = k0 < k && at - off + 8 * i < end ? __ldg(word + i) : 0ull;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    unsigned long long x = off ? (w[i] >> (8 * off)) | (w[i + 1] << (64 - 8 * off)) : w[i];
    const int left = k - k0 - 4 * i;
    if (left < 4) x = left <= 0 ? 0ull : x & (~0ull >> (64 - 16 * left));
    reinterpret_cast<unsigned long long*>(v)[i] = x;
  }
}

// The step of a block is 2^(floor(log2 amax) - 6): magnitudes reach 64..127 and the largest error is half a step, but
// for magnitudes above 127.5 steps, which are held at 127 (off by less than one step, 0.8 %).  The exponent is read
// from the bits of the largest magnitude; scaling by a power of two is exact, so rint() is the only rounding.
template <typename T>
__global__ void __launch_bounds__(kThreads) act8_save_kernel(const T* __restrict__ x, long long ldx, int m, int k,
                                                             uint8_t* __restrict__ codes, long long pitch,
                                                             uint8_t* __restrict__ exps, long long exp_pitch, Cut cut, bool wide) {
  const long long rb = blockIdx.x / cut.parts;
  const int part = static_cast<int>(blockIdx.x % cut.parts);
  const long long row = (rb << (8 - cut.cols_log2)) + (threadIdx.x >> cut.cols_log2);
  const int piece = (part << cut.cols_log2) + (threadIdx.x & ((1 << cut.cols_log2) - 1));
  const bool live = row < m && piece < cut.pieces;
  const int k0 = piece * 16;
  __align__(16) T v[16];
  load16<T>(x + (live ? row : 0) * ldx, k0, live ? k : 0, wide, v);
  typedef typename Half<T>::two T2;
  const T2* pair = reinterpret_cast<const T2*>(v);
  T2 most = __habs2(pair[0]);  // NaN stays NaN
#pragma unroll
  for (int i = 1; i < 8; ++i) most = __hmax2_nan(most, __habs2(pair[i]));
  // magnitudes compare as their bits, NaN above infinity
  uint32_t top = max(__float_as_uint(to_f32(low_of(most))), __float_as_uint(to_f32(high_of(most)))) & 0x7fffffffu;
  const uint32_t other = __shfl_xor_sync(0xffffffffu, top, 1);
  top = other > top ? other : top;
  int e = static_cast<int>(top >> 23) - 127 - 6;
  const bool bad = top >= 0x7f800000u || e > ActRange<T>::hi;
  if (e < ActRange<T>::lo) e = ActRange<T>::lo;
  const float inv = __uint_as_float(static_cast<uint32_t>(127 - (bad ? 0 : e)) << 23);
  const uint32_t keep = bad ? 0u : 0x7f7f7f7fu;
  const uint32_t* words = reinterpret_cast<const uint32_t*>(v);
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)  // adding 2^23 rounds to a whole number (nearest, ties to even) in the last bits
      q[i] = __float_as_uint(fminf(__fmaf_rn(fabsf(to_f32(v[4 * j + i])), inv, 8388608.f), 8388735.f));
    const uint32_t mags = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
    const uint32_t signs = __byte_perm(words[2 * j], words[2 * j + 1], 0x7531);  // the upper bytes of four values
    w[j] = (mags & keep) | (signs & 0x80808080u);
  }
  if (!live) return;
  // the second half of a row's last block may lie behind the row, which ends at k rounded up to 16
  if (k0 < k) *reinterpret_cast<uint4*>(codes + row * pitch + k0) = make_uint4(w[0], w[1], w[2], w[3]);
  if (!(piece & 1)) exps[row * exp_pitch + (piece >> 1)] = static_cast<uint8_t>(bad ? kActNaN : e + 127);
}

// Rows of 16-bit values to rows on 16 bytes, zeros behind their ends.
__global__ void __launch_bounds__(kThreads) copy_rows_kernel(uint16_t* __restrict__ dst, int cols_d, const uint16_t* __restrict__ src,
                                                             int rows, int cols, long long ld, Cut cut) {
  const long long row = ((blockIdx.x / cut.parts) << (8 - cut.cols_log2)) + (threadIdx.x >> cut.cols_log2);
  const int piece = (static_cast<int>(blockIdx.x % cut.parts) << cut.cols_log2) + (threadIdx.x & ((1 << cut.cols_log2) - 1));
  const int k0 = piece * 16;
  if (row >= rows || k0 >= cols_d) return;
  __align__(16) uint16_t v[16];
  load16<uint16_t>(src + row * ld, k0, cols, false, v);
  uint4* to = reinterpret_cast<uint4*>(dst + row * cols_d + k0);
  to[0] = reinterpret_cast<const uint4*>(v)[0];
  if (k0 + 8 < cols_d) to[1] = reinterpret_cast<const uint4*>(v)[1];
}

template <typename T>
__global__ void __launch_bounds__(kThreads) act8_restore_kernel(const uint8_t* __restrict__ codes, long long pitch,
                                                                const uint8_t* __restrict__ exps, long long exp_pitch, int m,
                                                                int k, T* __restrict__ x, long long ldx, Cut cut, bool wide) {
  const long long rb = blockIdx.x / cut.parts;
  const int part = static_cast<int>(blockIdx.x % cut.parts);
  const long long row = (rb << (8 - cut.cols_log2)) + (threadIdx.x >> cut.cols_log2);
  const int piece = (part << cut.cols_log2) + (threadIdx.x & ((1 << cut.cols_log2) - 1));
  const int k0 = piece * 16;
  // rows that do not start on 16 bytes leave through shared memory where a warp lies within one row
  const bool staged = !wide && cut.cols_log2 >= 5;
  __shared__ __align__(16) T stage[kThreads * 16];
  if (row >= m || (k0 >= k && !staged)) return;
  __align__(16) T v[16] = {};
  if (k0 < k) {
    const uint4 raw = __ldg(reinterpret_cast<const uint4*>(codes + row * pitch + k0));
    const Act8Step<T> step(exps[row * exp_pitch + (piece >> 1)]);
    reinterpret_cast<uint4*>(v)[0] = expand_act8<T>(raw.x, raw.y, step);
    reinterpret_cast<uint4*>(v)[1] = expand_act8<T>(raw.z, raw.w, step);
  }
  if (staged) {
    const int lane = threadIdx.x & 31, first = k0 - lane * 16;
    T* mine = stage + (threadIdx.x - lane) * 16;
    reinterpret_cast<uint4*>(mine + lane * 16)[0] = reinterpret_cast<const uint4*>(v)[0];
    reinterpret_cast<uint4*>(mine + lane * 16)[1] = reinterpret_cast<const uint4*>(v)[1];
    __syncwarp();
    if (first < k) store_row<T>(x + row * ldx + first, mine, min(512, k - first), lane);
    return;
  }
  T* to = x + row * ldx + k0;
  if (wide && k0 + 16 <= k) {
    reinterpret_cast<uint4*>(to)[0] = reinterpret_cast<const uint4*>(v)[0];
    reinterpret_cast<uint4*>(to)[1] = reinterpret_cast<const uint4*>(v)[1];
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (k0 + i < k) to[i] = v[i];
  }
}

int check(const Act8& a) {
  if (a.dtype != kF16 && a.dtype != kBF16) return kErrNotSupported;
  if (a.m < 0 || a.k <= 0 || a.pitch < a.k || a.exp_pitch < ceil_div(a.k, kActBlock)) return kErrInvalidProblem;
  if (a.m > 0 && (!a.codes || !a.exps)) return kErrInvalidProblem;
  if (a.m > kMaxExtent || a.k > kMaxExtent || a.exp_pitch > 0x7fffffffll) return kErrNotSupported;
  if (!aligned(a.codes, 16) || a.pitch % 16 || !aligned(a.exps, 4) || a.exp_pitch % 4) return kErrMisalignedOperand;
  return kOk;
}

template <typename T>
int save(const void* x, long long ldx, const Act8& a, cudaStream_t stream) {
  const Cut cut = cut_of(a.m, 2 * ceil_div(a.k, kActBlock));  // whole blocks of 32: both halves take part in the maximum
  if (cut.blocks > 0x7fffffffll) return kErrNotSupported;
  act8_save_kernel<T><<<static_cast<unsigned>(cut.blocks), kThreads, 0, stream>>>(
      static_cast<const T*>(x), ldx, a.m, a.k, static_cast<uint8_t*>(const_cast<void*>(a.codes)), a.pitch,
      static_cast<uint8_t*>(const_cast<void*>(a.exps)), a.exp_pitch, cut, aligned(x, 16) && ldx % 8 == 0);
  return static_cast<int>(cudaGetLastError());
}

template <typename T>
int restore(const Act8& a, void* x, long long ldx, cudaStream_t stream) {
  const Cut cut = cut_of(a.m, ceil_div(a.k, 16));
  if (cut.blocks > 0x7fffffffll) return kErrNotSupported;
  act8_restore_kernel<T><<<static_cast<unsigned>(cut.blocks), kThreads, 0, stream>>>(
      static_cast<const uint8_t*>(a.codes), a.pitch, static_cast<const uint8_t*>(a.exps), a.exp_pitch, a.m, a.k,
      static_cast<T*>(x), ldx, cut, aligned(x, 16) && ldx % 8 == 0);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace

int copy_rows_16bit(void* dst, int cols_d, const void* src, int rows, int cols, long long ld, cudaStream_t stream) {
  const Cut cut = cut_of(rows, ceil_div(cols_d, 16));
  if (cut.blocks > 0x7fffffffll) return kErrNotSupported;
  copy_rows_kernel<<<static_cast<unsigned>(cut.blocks), kThreads, 0, stream>>>(static_cast<uint16_t*>(dst), cols_d,
                                                                               static_cast<const uint16_t*>(src), rows, cols, ld, cut);
  return static_cast<int>(cudaGetLastError());
}

int restore_act8(const Act8& a, void* x, long long ldx, cudaStream_t stream) {
  return a.dtype == kF16 ? restore<__half>(a, x, ldx, stream) : restore<__nv_bfloat16>(a, x, ldx, stream);
}

}  // namespace lowbit
}  // namespace sb200

using sb200::lowbit::Act8;

extern "C" int sb200_act8_save(int dtype, const void* x, long long ldx, int m, int k, void* codes, long long pitch,
                               void* exponents, long long exp_pitch, sb200_stream_t stream) {
  const Act8 a{static_cast<sb200::DType>(dtype), m, k, codes, pitch, exponents, exp_pitch};
  if (int rc = sb200::lowbit::check(a)) return rc;
  if (ldx < k) return SB200_ERR_INVALID_PROBLEM;
  if (m == 0) return SB200_OK;
  if (!x) return SB200_ERR_INVALID_PROBLEM;
  if (!sb200::lowbit::aligned(x, 2)) return SB200_ERR_MISALIGNED_OPERAND;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return dtype == sb200::kF16 ? sb200::lowbit::save<__half>(x, ldx, a, s) : sb200::lowbit::save<__nv_bfloat16>(x, ldx, a, s);
}

extern "C" int sb200_act8_restore(int dtype, const void* codes, long long pitch, const void* exponents, long long exp_pitch,
                                  int m, int k, void* x, long long ldx, sb200_stream_t stream) {
  const Act8 a{static_cast<sb200::DType>(dtype), m, k, codes, pitch, exponents, exp_pitch};
  if (int rc = sb200::lowbit::check(a)) return rc;
  if (ldx < k) return SB200_ERR_INVALID_PROBLEM;
  if (m == 0) return SB200_OK;
  if (!x) return SB200_ERR_INVALID_PROBLEM;
  if (!sb200::lowbit::aligned(x, 2)) return SB200_ERR_MISALIGNED_OPERAND;
  return sb200::lowbit::restore_act8(a, x, ldx, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" size_t sb200_act8_wgrad_workspace_bytes(int dtype, int out_dtype, int m, int n, int k, int dy_aligned) {
  (void)dtype;
  (void)out_dtype;
  if (m < 0 || n <= 0 || k <= 0) return 256;
  return sb200::lowbit::expand_act8_workspace(m, n, k, dy_aligned != 0);
}

extern "C" int sb200_act8_wgrad_opt(int dtype, const void* codes, long long pitch, const void* exponents, long long exp_pitch,
                                    const void* dy, long long lddy, int out_dtype, const void* base, long long ldbase, void* dw,
                                    long long lddw, int m, int n, int k, void* workspace, size_t workspace_bytes,
                                    sb200_stream_t stream, const sb200_gemm_options* options) {
  const Act8 a{static_cast<sb200::DType>(dtype), m, k, codes, pitch, exponents, exp_pitch};
  sb200::lowbit::Waits waits;
  if (int rc = sb200::lowbit::check(a)) return rc;
  if (int rc = sb200::lowbit::waits_of(options, &waits)) return rc;
  if ((out_dtype != sb200::kF32 && out_dtype != dtype) || n > sb200::lowbit::kMaxExtent) return SB200_ERR_NOT_SUPPORTED;
  if (n <= 0 || !dw || lddw < n || lddy < n || (m > 0 && !dy) || (base && ldbase < n)) return SB200_ERR_INVALID_PROBLEM;
  const uintptr_t width = out_dtype == sb200::kF32 ? 4 : 2;
  if (!sb200::lowbit::aligned(dy, 2) || !sb200::lowbit::aligned(dw, width) || !sb200::lowbit::aligned(base, width))
    return SB200_ERR_MISALIGNED_OPERAND;
  if (!workspace || workspace_bytes < sb200_act8_wgrad_workspace_bytes(dtype, out_dtype, m, n, k, sb200::lowbit::tma_rows(dy, lddy)) ||
      !sb200::lowbit::aligned(workspace, 256))
    return SB200_ERR_WORKSPACE_NULL;
  return sb200::lowbit::expand_act8(a, dy, lddy, out_dtype == sb200::kF32, base, ldbase, dw, lddw, n, workspace, waits,
                                    reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int sb200_act8_wgrad(int dtype, const void* codes, long long pitch, const void* exponents, long long exp_pitch,
                                const void* dy, long long lddy, int out_dtype, const void* base, long long ldbase, void* dw,
                                long long lddw, int m, int n, int k, void* workspace, size_t workspace_bytes,
                                sb200_stream_t stream) {
  return sb200_act8_wgrad_opt(dtype, codes, pitch, exponents, exp_pitch, dy, lddy, out_dtype, base, ldbase, dw, lddw, m, n, k,
                              workspace, workspace_bytes, stream, nullptr);
}
