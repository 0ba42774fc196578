// Weights in 4 bits (format W4 of lowbit_format.cuh): packing, quantisation, expansion, and the product y = x W^T.
#include <stdint.h>

#include "../../include/subcuber_b200.h"
#include "lowbit_format.cuh"
#include "lowbit_host.h"
#include "per_device.h"
#include "w4_rows.cuh"

namespace sb200 {
namespace lowbit {
namespace {

// A block of threads handles one row tile (16 rows) and kSpanBlocks tiles of 128 inputs.  To quantise, half a warp takes a row and
// a lane sixteen neighbouring inputs of each 256, two words of the format: what is done once for a group is then done by half
// as many lanes as with one word (4096 x 4096, bf16, groups of 128 with zeros: 11.1 us, 13.0 with one).  The codes are put
// together in shared memory and leave as whole tiles.
constexpr int kSpanBlocks = 4, kSpan = kSpanBlocks * kW4Block;
constexpr int kThreads = 256;
constexpr int kLaneInputs = 16, kTurn = 16 * kLaneInputs, kTurns = kSpan / kTurn;

// The lane's 16-bit values of a row for every turn, zeros behind `k`; the lanes of half a warp take neighbours.  A row that does
// not start on 16 bytes is read in the aligned 8-byte words that hold it: a lane takes four words, the rest from the lane
// behind (the last lane reads one more), and shifts them together.  Words without a value of the row are not read.  All loads
// are issued before the first value is used (tile after tile, one word for a lane: 17.1 us in place of 13.0).
template <typename T>
__device__ __forceinline__ void load_words(const T* row, int first, int k, bool wide, T (&v)[kTurns][kLaneInputs], int lane) {
  if (wide && first - (lane & 15) * kLaneInputs <= k - kSpan) {  // the same for the lanes of a row
#pragma unroll
    for (int b = 0; b < kTurns; ++b)
#pragma unroll
      for (int i = 0; i < 2; ++i) reinterpret_cast<uint4*>(v[b])[i] = __ldg(reinterpret_cast<const uint4*>(row + first + b * kTurn) + i);
    return;
  }
  const uintptr_t end = reinterpret_cast<uintptr_t>(row + k);
  const uint32_t off = reinterpret_cast<uintptr_t>(row + first) & 7;  // the same for the lanes of a row, and every turn
  unsigned long long w[kTurns][5];
#pragma unroll
  for (int b = 0; b < kTurns; ++b) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(row + first + b * kTurn) - off;
    const unsigned long long* word = reinterpret_cast<const unsigned long long*>(at);
#pragma unroll
    for (int i = 0; i < 5; ++i)
      w[b][i] = k > 0 && at + 8 * i < end && (i < 4 || (off && (lane & 15) == 15)) ? __ldg(word + i) : 0ull;
  }
#pragma unroll
  for (int b = 0; b < kTurns; ++b) {
    const unsigned long long behind = __shfl_down_sync(0xffffu << (lane & 16), w[b][0], 1, 16);
    if ((lane & 15) != 15) w[b][4] = behind;
    unsigned long long* to = reinterpret_cast<unsigned long long*>(v[b]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      to[i] = off ? (w[b][i] >> (8 * off)) | (w[b][i + 1] << (64 - 8 * off)) : w[b][i];
      const int left = k - (first + b * kTurn) - 4 * i;
      if (left < 4) to[i] = left <= 0 ? 0ull : to[i] & (~0ull >> (64 - 16 * left));
    }
  }
}

// Bytes of a tile where the word of (row, eight inputs) goes: word = 4 j + t.
__device__ __forceinline__ int word_offset(int row, int word) {
  return (row >> 3) * 512 + ((row & 7) * 4 + (word & 3)) * 16 + (word >> 2) * 4;
}

// Scales that are normal numbers of their type and whose reciprocals are normal floats.
template <typename T> struct UsualScale;
template <> struct UsualScale<__half> { static constexpr float least = 0x1p-14f, most = 65504.f; };
template <> struct UsualScale<__nv_bfloat16> { static constexpr float least = 0x1p-100f, most = 0x1p100f; };

template <typename T2> __device__ __forceinline__ uint32_t bits_of(T2 v) { return *reinterpret_cast<const uint32_t*>(&v); }
template <typename T> __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {  // NaN stays NaN
  typedef typename Half<T>::two T2;
  return bits_of(__hmax2_nan(*reinterpret_cast<const T2*>(&a), *reinterpret_cast<const T2*>(&b)));
}

// Quantisation, one group at a time.  Symmetric: scale = amax / 7 and codes 8 + rint(w / scale).  Else the range
// [min(0, w), max(0, w)] is laid over 0..15, which keeps zero exact: scale = (hi - lo) / 15, zero = rint(-lo / scale).
// The scale is rounded to the 16-bit type FIRST and the codes are made for the rounded one.  Divisions are the
// correctly rounded ones, so that a code next to a border does not depend on how the quotient was formed.  A group with
// an infinity or a NaN gets a scale that is not finite and stands for NaN.
template <typename T, int G, bool SYM>
__global__ void __launch_bounds__(kThreads) w4_quantize_kernel(const T* __restrict__ w, long long ldw, int n, int k,
                                                               uint8_t* __restrict__ codes, T* __restrict__ scales,
                                                               uint8_t* __restrict__ zeros, bool wide) {
  __shared__ __align__(16) uint8_t tile[kSpanBlocks * kW4TileBytes];
  const int blocks = w4_blocks(k);
  const int spans = ceil_div(blocks, kSpanBlocks);
  const int rt = blockIdx.x / spans, span = blockIdx.x % spans;
  const int lane = threadIdx.x & 31, word = (lane & 7) * 2, r = threadIdx.x >> 4;
  const int row = rt * kW4Rows + r;
  const int first = span * kSpan + (lane & 15) * kLaneInputs;
  __align__(16) T v[kTurns][kLaneInputs];
  load_words<T>(w + (row < n ? row : 0) * ldw, first, row < n ? k : 0, wide, v, lane);
#pragma unroll
  for (int b = 0; b < kTurns; ++b) {
    // The largest value above zero and the largest magnitude below it (SYM: the largest magnitude), which travel as
    // one pair; NaN stays NaN.
    typedef typename Half<T>::two T2;
    const T2* pair = reinterpret_cast<const T2*>(v[b]);
    T2 top = SYM ? __habs2(pair[0]) : pair[0], low = pair[0];
#pragma unroll
    for (int i = 1; i < kLaneInputs / 2; ++i) {
      top = __hmax2_nan(top, SYM ? __habs2(pair[i]) : pair[i]);
      if (!SYM) low = __hmin2_nan(low, pair[i]);
    }
    uint32_t most = bits_of(top);
    if (SYM) {
      most = max2<T>(most, __byte_perm(most, 0, 0x1032));
    } else {
      const uint32_t below = bits_of(low) ^ 0x80008000u;
      most = max2<T>(max2<T>(__byte_perm(most, below, 0x5410), __byte_perm(most, below, 0x7632)), 0u);
    }
#pragma unroll
    for (int i = G / kLaneInputs / 2; i >= 1; i >>= 1) most = max2<T>(most, __shfl_xor_sync(0xffffffffu, most, i));
    most &= 0x7fff7fffu;  // no zero keeps a sign
    const T2 ends = *reinterpret_cast<const T2*>(&most);
    const float hi = to_f32(low_of(ends)), lo = to_f32(high_of(ends));
    // amax / 7 may be a product with 1 / 7: amax has 11 significant bits at most, so that the quotient is a fourteenth of a
    // 16-bit step or more away from where the rounding to 16 bits changes.  hi - lo has more bits.
    const float range = SYM ? hi : hi + lo;  // NaN and infinity stay
    const T s16 = from_f32<T>(SYM ? range * (1.f / 7.f) : __fdiv_rn(range, 15.f));
    const float s = to_f32(s16);
    int z = SYM ? 8 : 0;
    uint32_t packed[2] = {z * 0x11111111u, z * 0x11111111u};
    // rint(x / s) without a division.  x and s have 11 significant bits at most, so that a quotient up to 2^5 that is
    // not halfway between two whole numbers is at least 2^-13 away from that; the product with the reciprocal is off by
    // 2^-17 at most.  Adding it to 768 leaves multiples of 2^-14: a quotient that is halfway becomes exactly so, and no
    // other one crosses.  Adding 1.5 * 2^23 - 768 then rounds to nearest, ties to even, as rint(x / s) does, and leaves the
    // whole number in the last bits.
    constexpr int kWhole = 0x4b400000;
    auto whole = [](float a, float inv) { return __float_as_int(__fadd_rn(__fmaf_rn(a, inv, 768.f), 12582144.f)); };
    if (s >= UsualScale<T>::least && s <= UsualScale<T>::most) {
      // The scale was rounded by 2^-8 of itself at most, so that a symmetric quotient stays within -7..7 and the others
      // within z + 1 units of each end: the only code that can leave 0..15 is 16.  The codes of a word are summed at their
      // places with what `whole` puts on top of each, which comes off once for all (modulo 2^32).
      const float inv = __fdividef(1.f, s);
      if (!SYM) z = whole(lo, inv) - kWhole;
      const int least = kWhole - z;  // code 0
      packed[0] = packed[1] = 0u - static_cast<uint32_t>(least) * 0x11111111u;
#pragma unroll
      for (int i = 0; i < kLaneInputs; ++i) {
        int c = whole(to_f32(v[b][i]), inv);
        if (!SYM) c = min(c, least + 15);
        packed[i / 8] += static_cast<uint32_t>(c) << (4 * w4_nibble(i % 8));
      }
    } else if (s > 0.f && s < INFINITY) {
      // Scales that may have lost bits when they were rounded (subnormal ones), or whose reciprocal is not a normal number:
      // they are brought into range first, the values with them (a power of two: exact), and all codes are held in 0..15.
      const float shift = s < 0x1p-100f ? 0x1p64f : s > 0x1p100f ? 0x1p-64f : 1.f;
      const float inv = __fdividef(1.f, s * shift);
      if (!SYM) z = min(whole(lo * shift, inv) - kWhole, 15);
      packed[0] = packed[1] = 0;
#pragma unroll
      for (int i = 0; i < kLaneInputs; ++i)
        packed[i / 8] += static_cast<uint32_t>(min(max(whole(to_f32(v[b][i]) * shift, inv) - (kWhole - z), 0), 15)) << (4 * w4_nibble(i % 8));
    }
    const int of_span = b * (kTurn / kW4Block) + ((lane >> 3) & 1), block = span * kSpanBlocks + of_span;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      *reinterpret_cast<uint32_t*>(tile + of_span * kW4TileBytes + word_offset(r, word + i)) = packed[i];
    if (word % (G / 8) == 0 && block < blocks) {
      const long long at = ((static_cast<long long>(rt) * blocks + block) * kW4Rows + r) * (kW4Block / G) + word / (G / 8);
      scales[at] = s16;
      if (!SYM) zeros[at] = static_cast<uint8_t>(z);
    }
  }
  __syncthreads();
  if (span * kSpanBlocks + static_cast<int>(threadIdx.x) / (kW4TileBytes / 16) < blocks)
    reinterpret_cast<uint4*>(codes)[(static_cast<long long>(rt) * blocks + span * kSpanBlocks) * (kW4TileBytes / 16) +
                                    threadIdx.x] = reinterpret_cast<const uint4*>(tile)[threadIdx.x];
}

// Codes that are there already, one byte each, and their tables [groups][n] into the format's order.
__global__ void __launch_bounds__(kThreads) w4_pack_kernel(const uint8_t* __restrict__ q, long long ldq,
                                                           const uint16_t* __restrict__ s, long long lds,
                                                           const uint8_t* __restrict__ z, long long ldz, int n, int k, int G,
                                                           uint8_t* __restrict__ codes, uint16_t* __restrict__ scales,
                                                           uint8_t* __restrict__ zeros) {
  const int blocks = w4_blocks(k);
  const int rt = blockIdx.x / blocks, block = blockIdx.x % blocks;
  const int r = threadIdx.x >> 4, pair = threadIdx.x & 15;  // one word for each thread
  const int row = rt * kW4Rows + r;
  const int k0 = block * kW4Block + pair * 8;
  const long long group = k0 / G;
  const bool real = row < n && group * G < k;
  const uint32_t zero = z && real ? z[group * ldz + row] & 15u : 8u;
  uint32_t word = 0;
  for (int i = 0; i < 8; ++i) {
    const int kk = k0 + i;
    uint32_t c = zero;  // inputs behind k stand for 0: another code times a large scale would be infinite
    if (row < n && kk < k) c = q[row * ldq + kk] & 15u;
    word |= c << (4 * w4_nibble(i));
  }
  *reinterpret_cast<uint32_t*>(codes + (static_cast<long long>(rt) * blocks + block) * kW4TileBytes + word_offset(r, pair)) = word;
  if (k0 % G == 0) {
    const long long at = w4_table_at(row, k0 / G, blocks, G);
    scales[at] = real ? s[group * lds + row] : 0;
    if (z) zeros[at] = real ? zero : 0;
  }
}

// Expansion: a thread takes the 16 bytes of (row, t), four words of eight inputs, and leaves them in shared memory; a warp
// then stores two rows of up to 512 neighbours in aligned words.  Rows that do not start on 16 bytes are stored in 4-byte words (or
// 2-byte ones at their ends) of the values that fall into them.
template <typename T>
__global__ void __launch_bounds__(kThreads) w4_dequantize_kernel(const uint8_t* __restrict__ codes, const T* __restrict__ scales,
                                                                 const uint8_t* __restrict__ zeros, int n, int k, int G,
                                                                 T* __restrict__ out, long long ldo) {
  __shared__ __align__(16) T rows[kW4Rows][kSpan + 8];
  const int blocks = w4_blocks(k);
  const int spans = ceil_div(blocks, kSpanBlocks);
  const int rt = blockIdx.x / spans, span = blockIdx.x % spans;
  const int block = span * kSpanBlocks + (threadIdx.x >> 6);
  const int piece = threadIdx.x & 63;
  const int r = (piece >> 5) * 8 + ((piece & 31) >> 2), t = piece & 3;
  if (block < blocks) {
    const uint4 raw = __ldg(reinterpret_cast<const uint4*>(codes) +
                            (static_cast<long long>(rt) * blocks + block) * (kW4TileBytes / 16) + piece);
    const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
    const int per = kW4Block / G;
    const long long at = ((static_cast<long long>(rt) * blocks + block) * kW4Rows + r) * per;
    T* to = &rows[r][(threadIdx.x >> 6) * kW4Block + 8 * t];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t s = reinterpret_cast<const uint16_t*>(scales)[at + j * per / 4], z = zeros ? zeros[at + j * per / 4] : 8u;
      *reinterpret_cast<uint4*>(to + 32 * j) =
          expand_w4<T>(words[j], Half<T>::magic + __byte_perm(z, 0, 0x4040), __byte_perm(s, 0, 0x1010), 0x000f000fu, Half<T>::magic);
    }
  }
  __syncthreads();
  const int first = span * kSpan, count = min(kSpan, k - first);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int row = rt * kW4Rows + warp + 8 * h;
    if (row >= n) continue;
    store_row<T>(out + row * ldo + first, rows[warp + 8 * h], count, lane);
  }
}

template <typename T, int PER>
int rows_product(const void* x, long long ldx, const W4& w, void* y, long long ldy, int m, cudaStream_t stream) {
  const RowsParams p{x, ldx, static_cast<const uint8_t*>(w.codes), static_cast<const uint8_t*>(w.scales),
                     static_cast<const uint8_t*>(w.zeros), y, ldy, m, w.n, w.k, w4_blocks(w.k)};
  // one row tile to a warp while that is at most two blocks for each SM, else two, which read x half as often (one row, 2048 x
  // 2048: 2.5 us, 3.0 with two; 4096 x 8192: 7.5 and 7.6; 8192 x 8192: 11.9 us, 13.4 with one; between, 6144 x 8192: 11.7 us,
  // 10.7 with one, but 12.9 and 13.0 at eight rows of x, and 7104 x 2048 4.9 and 5.5; four row tiles were slower everywhere)
  if (w4_row_tiles(w.n) <= 2 * sm_count_of_current_device()) return launch_rows<T, PER, 1, 4>(p, stream);
  return launch_rows<T, PER, 2, 3>(p, stream);
}

template <typename T>
int rows_product_any(const void* x, long long ldx, const W4& w, void* y, long long ldy, int m, cudaStream_t stream) {
  if (w.group == 32) return rows_product<T, 4>(x, ldx, w, y, ldy, m, stream);
  if (w.group == 64) return rows_product<T, 2>(x, ldx, w, y, ldy, m, stream);
  return rows_product<T, 1>(x, ldx, w, y, ldy, m, stream);
}

// Up to here, the columns of one warp instruction, the codes are multiplied as they are (w4_rows.cuh); more rows go to
// tcgen05.mma (w4_decode.cuh).  In one run, this kernel and the other one: 8192 x 8192: 1 row 12.1 and 17.3 us, 8 rows 13.3 and 18.1,
// 9 rows 18.3 (the other); 2048 x 2048: 1 row 2.3 and 5.9, 8 rows 2.4 and 6.4, 9 rows 6.8; 16384 x 4096: 8 rows 14.1 and 17.8.
constexpr int kFewRows = 8;

int check(const W4& w) {
  if (w.dtype != kF16 && w.dtype != kBF16) return kErrNotSupported;
  if (w.n <= 0 || w.k <= 0 || !w.codes || !w.scales) return kErrInvalidProblem;
  if (w.n > kMaxExtent || w.k > kMaxExtent) return kErrNotSupported;
  if (w.group != 32 && w.group != 64 && w.group != 128) return kErrNotSupported;
  if (!aligned(w.codes, 16) || !aligned(w.scales, 16) || !aligned(w.zeros, 16)) return kErrMisalignedOperand;
  return kOk;
}

// Thread blocks of a launch over (row tiles) x (parts of a row); the grid's x axis holds 2^31 - 1 of them.
int grid_of(int n, int parts, unsigned* grid) {
  const long long g = static_cast<long long>(w4_row_tiles(n)) * parts;
  if (g > 0x7fffffffll) return kErrNotSupported;
  *grid = static_cast<unsigned>(g);
  return kOk;
}

template <typename T, int G>
int quantize(const void* w, long long ldw, const W4& q, cudaStream_t stream) {
  unsigned grid;
  if (int rc = grid_of(q.n, ceil_div(w4_blocks(q.k), kSpanBlocks), &grid)) return rc;
  const T* from = static_cast<const T*>(w);
  const bool wide = tma_rows(w, ldw);
  uint8_t* codes = static_cast<uint8_t*>(const_cast<void*>(q.codes));
  T* scales = static_cast<T*>(const_cast<void*>(q.scales));
  uint8_t* zeros = static_cast<uint8_t*>(const_cast<void*>(q.zeros));
  if (zeros) w4_quantize_kernel<T, G, false><<<grid, kThreads, 0, stream>>>(from, ldw, q.n, q.k, codes, scales, zeros, wide);
  else w4_quantize_kernel<T, G, true><<<grid, kThreads, 0, stream>>>(from, ldw, q.n, q.k, codes, scales, zeros, wide);
  return static_cast<int>(cudaGetLastError());
}

template <typename T>
int quantize_any(const void* w, long long ldw, const W4& q, cudaStream_t stream) {
  switch (q.group) {
    case 32: return quantize<T, 32>(w, ldw, q, stream);
    case 64: return quantize<T, 64>(w, ldw, q, stream);
    default: return quantize<T, 128>(w, ldw, q, stream);
  }
}

template <typename T>
int dequantize(const W4& w, void* out, long long ldo, cudaStream_t stream) {
  unsigned grid;
  if (int rc = grid_of(w.n, ceil_div(w4_blocks(w.k), kSpanBlocks), &grid)) return rc;
  w4_dequantize_kernel<T><<<grid, kThreads, 0, stream>>>(static_cast<const uint8_t*>(w.codes), static_cast<const T*>(w.scales),
                                                         static_cast<const uint8_t*>(w.zeros), w.n, w.k, w.group,
                                                         static_cast<T*>(out), ldo);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace

int dequantize_w4(const W4& w, void* out, long long ldo, cudaStream_t stream) {
  return w.dtype == kF16 ? dequantize<__half>(w, out, ldo, stream) : dequantize<__nv_bfloat16>(w, out, ldo, stream);
}

}  // namespace lowbit
}  // namespace sb200

using sb200::lowbit::W4;

extern "C" size_t sb200_w4_codes_bytes(int n, int k) {
  if (n <= 0 || k <= 0) return 0;
  return static_cast<size_t>(sb200::lowbit::w4_row_tiles(n)) * sb200::lowbit::w4_blocks(k) * sb200::lowbit::kW4TileBytes;
}

extern "C" size_t sb200_w4_table_entries(int n, int k, int group) {
  if (n <= 0 || k <= 0 || (group != 32 && group != 64 && group != 128)) return 0;
  return static_cast<size_t>(sb200::lowbit::w4_table_entries(n, k, group));
}

extern "C" int sb200_w4_quantize(int dtype, const void* w, long long ldw, int n, int k, int group, void* codes, void* scales,
                                 void* zeros, sb200_stream_t stream) {
  const W4 q{static_cast<sb200::DType>(dtype), n, k, group, codes, scales, zeros};
  if (int rc = sb200::lowbit::check(q)) return rc;
  if (!w || ldw < k) return SB200_ERR_INVALID_PROBLEM;
  if (!sb200::lowbit::aligned(w, 2)) return SB200_ERR_MISALIGNED_OPERAND;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return dtype == sb200::kF16 ? sb200::lowbit::quantize_any<__half>(w, ldw, q, s)
                              : sb200::lowbit::quantize_any<__nv_bfloat16>(w, ldw, q, s);
}

extern "C" int sb200_w4_pack(int dtype, const void* q, long long ldq, const void* q_scales, long long lds, const void* q_zeros,
                             long long ldz, int n, int k, int group, void* codes, void* scales, void* zeros,
                             sb200_stream_t stream) {
  const W4 w{static_cast<sb200::DType>(dtype), n, k, group, codes, scales, zeros};
  if (int rc = sb200::lowbit::check(w)) return rc;
  if (!q || !q_scales || ldq < k || lds < n || !q_zeros != !zeros || (q_zeros && ldz < n)) return SB200_ERR_INVALID_PROBLEM;
  if (!sb200::lowbit::aligned(q_scales, 2)) return SB200_ERR_MISALIGNED_OPERAND;
  unsigned grid;
  if (int rc = sb200::lowbit::grid_of(n, sb200::lowbit::w4_blocks(k), &grid)) return rc;
  sb200::lowbit::w4_pack_kernel<<<grid, sb200::lowbit::kThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      static_cast<const uint8_t*>(q), ldq, static_cast<const uint16_t*>(q_scales), lds, static_cast<const uint8_t*>(q_zeros), ldz,
      n, k, group, static_cast<uint8_t*>(codes), static_cast<uint16_t*>(scales), static_cast<uint8_t*>(zeros));
  return static_cast<int>(cudaGetLastError());
}

extern "C" int sb200_w4_dequantize(int dtype, const void* codes, const void* scales, const void* zeros, int n, int k,
                                   int group, void* out, long long ldo, sb200_stream_t stream) {
  const W4 w{static_cast<sb200::DType>(dtype), n, k, group, codes, scales, zeros};
  if (int rc = sb200::lowbit::check(w)) return rc;
  if (!out || ldo < k) return SB200_ERR_INVALID_PROBLEM;
  if (!sb200::lowbit::aligned(out, 2)) return SB200_ERR_MISALIGNED_OPERAND;
  return sb200::lowbit::dequantize_w4(w, out, ldo, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" size_t sb200_w4_gemm_workspace_bytes(int dtype, int m, int n, int k, int group, int x_aligned) {
  (void)dtype;
  (void)group;
  if (n <= 0 || k <= 0 || m <= 0) return 0;
  return sb200::lowbit::expand_w4_workspace(m, n, k, x_aligned != 0);
}

extern "C" int sb200_w4_gemm_opt(int dtype, const void* x, long long ldx, const void* codes, const void* scales,
                                 const void* zeros, void* y, long long ldy, int m, int n, int k, int group, void* workspace,
                                 size_t workspace_bytes, sb200_stream_t stream, const sb200_gemm_options* options) {
  using namespace sb200::lowbit;
  const W4 w{static_cast<sb200::DType>(dtype), n, k, group, codes, scales, zeros};
  Waits waits;
  if (int rc = check(w)) return rc;
  if (int rc = waits_of(options, &waits)) return rc;
  if (m < 0 || ldx < k || ldy < n) return SB200_ERR_INVALID_PROBLEM;
  if (m > kMaxExtent) return SB200_ERR_NOT_SUPPORTED;
  if (m == 0) return SB200_OK;
  if (!x || !y) return SB200_ERR_INVALID_PROBLEM;
  if (!aligned(x, 2) || !aligned(y, 2)) return SB200_ERR_MISALIGNED_OPERAND;
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < expand_w4_workspace(m, n, k, tma_rows(x, ldx)))
    return SB200_ERR_WORKSPACE_NULL;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  if (!tma_rows(x, ldx)) {  // every kernel wants rows of x that start on 16 bytes
    const int cols = (k + 7) / 8 * 8;
    if (int rc = copy_rows_16bit(ws + kStatusBytes, cols, x, m, k, ldx, s)) return rc;
    x = ws + kStatusBytes;
    ldx = cols;
  }
  if (m <= kFewRows)
    return dtype == sb200::kF16 ? rows_product_any<__half>(x, ldx, w, y, ldy, m, s)
                                : rows_product_any<__nv_bfloat16>(x, ldx, w, y, ldy, m, s);
  if (m <= kDecodeMaxRows) return decode_w4(w, x, ldx, y, ldy, m, workspace, waits, s);
  return expand_w4(w, x, ldx, y, ldy, m, workspace, workspace_bytes, waits, s);
}

extern "C" int sb200_w4_gemm(int dtype, const void* x, long long ldx, const void* codes, const void* scales,
                             const void* zeros, void* y, long long ldy, int m, int n, int k, int group, void* workspace,
                             size_t workspace_bytes, sb200_stream_t stream) {
  return sb200_w4_gemm_opt(dtype, x, ldx, codes, scales, zeros, y, ldy, m, n, k, group, workspace, workspace_bytes, stream,
                           nullptr);
}
