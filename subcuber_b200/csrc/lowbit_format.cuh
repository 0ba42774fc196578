// The two formats in which an operand of a product is held in few bits, and the element arithmetic on them.
//
//   W4     weights n x k in 4 bits:  W[n][k] = scale(n, k / G) * (code[n][k] - zero(n, k / G)),  code in 0..15, zero in 0..15
//          (8 where there is no table of zeros), G = 32, 64 or 128.  Rows are padded to 16, inputs to 128.  A tile of 16 rows
//          x 128 inputs is 1 KiB of consecutive bytes, tiles run along the inputs first.  Inside a tile the 16 bytes at
//          512 h + 16 (4 g + t) belong to row 8 h + g; their word j holds the inputs 32 j + 8 t + (0..7), input i at nibble
//          (i >> 1) + 4 (i & 1).  That is the fragment order of a 16 x 8 x 16 matrix instruction: lane 4 g + t loads its 16 bytes
//          at once, one word lies within one group whatever G is, and the four pairs of nibbles that `w >> 4 p` leaves 16 bits
//          apart are neighbouring inputs, so that an expanded word is 16 bytes in the order of the activations.
//          Scales have the 16-bit type of the activations, zeros are bytes; both tables run with the tiles:
//          [row tile][128 inputs][row of the tile][group of the 128 inputs], so that the groups of a row in a tile are one load.
//          What belongs to padding has scale 0.
//   ACT8   activations m x k in 8 bits:  X[m][k] = +-magnitude * 2^(E[m][k / 32] - 127), bit 7 of the byte is the sign, bits 0-6
//          the magnitude.  A magnitude has 7 bits and the step is a power of two, so every X is exact in bf16 and (with the
//          steps kept to 2^-24 .. 2^9) in f16: a product of X is a product of 16-bit operands without another rounding.
//          E = 255 marks a block that held an infinity or a NaN (bf16: or a magnitude of 2^127 and more); it reads as NaN.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace sb200 {
namespace lowbit {

constexpr int kW4Rows = 16;     // rows of a tile
constexpr int kW4Block = 128;   // inputs of a tile
constexpr int kW4TileBytes = kW4Rows * kW4Block / 2;
constexpr int kActBlock = 32;   // channels that share an exponent
constexpr int kActNaN = 255;    // the exponent of a block that reads as NaN

__host__ __device__ inline int ceil_div(int a, int b) { return a / b + (a % b != 0); }
__host__ __device__ inline int w4_blocks(int k) { return ceil_div(k, kW4Block); }
__host__ __device__ inline int w4_row_tiles(int n) { return ceil_div(n, kW4Rows); }
__host__ __device__ inline long long w4_padded_rows(int n) { return static_cast<long long>(w4_row_tiles(n)) * kW4Rows; }

// Entries of the tables, and where that of (row, group of the whole row) is.
__host__ __device__ inline long long w4_table_entries(int n, int k, int G) {
  return w4_padded_rows(n) * w4_blocks(k) * (kW4Block / G);
}
__host__ __device__ inline long long w4_table_at(int row, int group, int blocks, int G) {
  const int per = kW4Block / G;
  return ((static_cast<long long>(row / kW4Rows) * blocks + group / per) * kW4Rows + row % kW4Rows) * per + group % per;
}

// Nibble of input i (0..7) in its word.
__host__ __device__ constexpr int w4_nibble(int i) { return (i >> 1) + 4 * (i & 1); }

// Exponent range of the steps of ACT8: bf16 steps start at the smallest normal number (matrix units may flush smaller
// ones) and end where 2^(e + 7) is still finite; f16 steps cover the whole type, subnormals included.
template <typename T> struct ActRange;
template <> struct ActRange<__half> { static constexpr int lo = -24, hi = 9; };
template <> struct ActRange<__nv_bfloat16> { static constexpr int lo = -126, hi = 120; };

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
__device__ __forceinline__ __half low_of(__half2 v) { return __low2half(v); }
__device__ __forceinline__ __half high_of(__half2 v) { return __high2half(v); }
__device__ __forceinline__ __nv_bfloat16 low_of(__nv_bfloat162 v) { return __low2bfloat16(v); }
__device__ __forceinline__ __nv_bfloat16 high_of(__nv_bfloat162 v) { return __high2bfloat16(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }

// 2^(E - 127) of a stored exponent, NaN for kActNaN.  E is at least 1.
__device__ __forceinline__ float act8_step(int e) {
  return __uint_as_float(e == kActNaN ? 0x7fffffffu : static_cast<uint32_t>(e) << 23);
}
// ---- expansion to 16 bits, two values at a time

template <typename T> struct Half;
template <> struct Half<__half> {
  static constexpr uint32_t fmt = 0;              // of the instruction descriptor
  static constexpr uint32_t magic = 0x64006400u;  // 1024, last bit 1
  typedef __half2 two;
};
template <> struct Half<__nv_bfloat16> {
  static constexpr uint32_t fmt = 1;
  static constexpr uint32_t magic = 0x43004300u;  // 128, last bit 1
  typedef __nv_bfloat162 two;
};
template <typename T> __device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
  typedef typename Half<T>::two H;
  const H r = __hsub2(*reinterpret_cast<const H*>(&a), *reinterpret_cast<const H*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <typename T> __device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
  typedef typename Half<T>::two H;
  const H r = __hmul2(*reinterpret_cast<const H*>(&a), *reinterpret_cast<const H*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// (a & b) | c in one instruction.  The constants are kept in registers: with two of them written into the expression the
// compiler takes two instructions, each of which has room for one.
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
__device__ __forceinline__ uint32_t in_register(uint32_t constant) {
  uint32_t r;
  asm volatile("mov.b32 %0, %1;" : "=r"(r) : "r"(constant));
  return r;
}

// Eight codes of a word to eight weights, in the order of the inputs.  bias = magic + zero, scale twice.
// mask = 0x000f000f and magic, both in registers.
template <typename T>
__device__ __forceinline__ uint4 expand_w4(uint32_t w, uint32_t bias, uint32_t scale, uint32_t mask, uint32_t magic) {
  uint4 r;
  r.x = mul2<T>(sub2<T>(and_or(w, mask, magic), bias), scale);
  r.y = mul2<T>(sub2<T>(and_or(w >> 4, mask, magic), bias), scale);
  r.z = mul2<T>(sub2<T>(and_or(w >> 8, mask, magic), bias), scale);
  r.w = mul2<T>(sub2<T>(and_or(w >> 12, mask, magic), bias), scale);
  return r;
}

// Two bytes (sign, 7 bits of magnitude) to two values.
//   bf16  the magnitude is OR-ed under the exponent of 2^(e + 7), where its last bit is worth 2^e: the number is
//         +-(2^(e+7) + magnitude 2^e), and subtracting its own leading term leaves the value.  `e` holds that exponent's
//         bits twice; all ones (a block that reads as NaN) gives infinity - infinity or NaN.
//   f16   the magnitude under the exponent of 1024 in the same way, then a product with 2^e (`s`), which is exact.
template <typename T> struct Act8Step;
template <> struct Act8Step<__nv_bfloat16> {
  uint32_t e;
  __device__ __forceinline__ explicit Act8Step(uint32_t exponent) {
    const uint32_t field = exponent + 7u > 255u ? 255u : exponent + 7u;
    e = (field << 7) | (field << 23);
  }
  __device__ __forceinline__ uint32_t two(uint32_t bytes_twice) const {
    const uint32_t p = and_or(bytes_twice, 0x807f807fu, e);
    return sub2<__nv_bfloat16>(p, p & 0xff80ff80u);
  }
};
template <> struct Act8Step<__half> {
  uint32_t s, magic;
  __device__ __forceinline__ explicit Act8Step(uint32_t exponent) : magic(in_register(0x64006400u)) {
    const __half2 h = __float2half2_rn(act8_step(static_cast<int>(exponent)));
    s = *reinterpret_cast<const uint32_t*>(&h);
  }
  __device__ __forceinline__ uint32_t two(uint32_t bytes_twice) const {
    const uint32_t p = and_or(bytes_twice, 0x807f807fu, magic);
    return mul2<__half>(sub2<__half>(p, p & 0xfc00fc00u), s);
  }
};
template <typename T>
__device__ __forceinline__ uint4 expand_act8(uint32_t w0, uint32_t w1, const Act8Step<T>& st) {  // eight channels
  uint4 r;
  r.x = st.two(__byte_perm(w0, 0, 0x1100));
  r.y = st.two(__byte_perm(w0, 0, 0x3322));
  r.z = st.two(__byte_perm(w1, 0, 0x1100));
  r.w = st.two(__byte_perm(w1, 0, 0x3322));
  return r;
}

// Asynchronous copies of 4 and 16 bytes, zeros where `from` has none to give.
__device__ __forceinline__ void copy_async_16(uint32_t to, const void* from, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_async_4(uint32_t to, const void* from, bool real) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(real ? 4 : 0) : "memory");
}
__device__ __forceinline__ uint32_t lds_u16(uint32_t smem_addr) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(smem_addr));
  return v;
}
__device__ __forceinline__ uint32_t lds_u8(uint32_t smem_addr) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(smem_addr));
  return v;
}

// A warp stores `count` 16-bit values that lie in shared memory (on 16 bytes) to consecutive places of global memory.
template <typename T>
__device__ __forceinline__ void store_row(T* to, const T* from, int count, int lane) {
  const uint32_t off = reinterpret_cast<uintptr_t>(to) & 15;
  if (off == 0) {
    for (int i = lane * 8; i + 8 <= count; i += 256) *reinterpret_cast<uint4*>(to + i) = *reinterpret_cast<const uint4*>(from + i);
    const int done = count & ~7;
    if (lane < count - done) to[done + lane] = from[done + lane];
    return;
  }
  const int head = (off >> 1) & 1;  // a value before the first whole 4-byte word
  if (head && lane == 0) to[0] = from[0];
  const int pairs = (count - head) >> 1;
  for (int i = lane; i < pairs; i += 32) {
    const uint32_t a = *reinterpret_cast<const uint16_t*>(from + head + 2 * i), b = *reinterpret_cast<const uint16_t*>(from + head + 2 * i + 1);
    *reinterpret_cast<uint32_t*>(to + head + 2 * i) = a | (b << 16);
  }
  if (((count - head) & 1) && lane == 0) to[count - 1] = from[count - 1];
}

}  // namespace lowbit
}  // namespace sb200
