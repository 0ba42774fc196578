// y = x W^T for up to 8 rows of x, weights in format W4.
//
// Bound.  The bytes of the weights are the floor (8192 x 8192, groups of 128: 34.6 MB, 5.3 us at the measured copy rate); one row
// takes 11.8 us (2.9 TB/s), eight take 12.8.  What holds it there is the issue of instructions: a tile of 1 KiB costs a warp
// about 240, most of them logical operations and subtractions that turn codes into numbers; of the active cycles 60 %
// issue, the integer pipe is busy for 57 % and the tensor pipe for 21 %.  Two codes cost four
// operations (shift, and-or, subtract, and a quarter of the matrix instruction); in f16 two of the three shifts of a word could go, since
// the upper code of a byte, masked in place, is worth 16 units that a fused multiply-add takes off exactly.
//
// Mathematics.  Codes are small whole numbers and exact in 16 bits, so that the matrix instruction multiplies (code -
// zero) with x without any rounding; the sums of one group are scaled in fp32 afterwards:
//     y[m][n] = sum over groups g of scale(n, g) * (sum over k in g of (code - zero) x[m][k])
// A 4-bit code becomes a 16-bit number by bits alone: OR-ed into the last bits of 1024 (f16) or 128 (bf16) it adds exactly
// its value, and one packed subtraction of (1024 | 128) + zero leaves code - zero, for two codes at a time.
//
// Split.  A warp walks over tiles of 16 rows x 128 inputs: the weights are the left operand of mma.m16n8k16 (16 rows x 16
// inputs) and 8 rows of x the right one.  The order of inputs inside an instruction is free as long as both operands
// have the same, so a lane takes its word's eight inputs as they lie in memory.  The eight warps of a block take the tiles of its
// RT row tiles in turn; their sums meet in shared memory in the order of the warps, so that results do not change from call to
// call.
//
// Memory.  The kernel lives from bytes in flight (6.5 TB/s at about 1 us of latency under load are 44 KB for each SM), and
// registers do not hold them: every warp has a ring of AHEAD stages in shared memory that it fills with 16-byte asynchronous
// copies of its own, so that no barrier but the warp's own is needed.  The warps of a block work on different inputs; copies of x go
// through the first-level cache, where the blocks of an SM find what another one fetched.  With one row that is worth up to a sixth
// (in one run, 2048 x 2048: 2.3 us, past it 2.7; 4096 x 8192: 7.8, 8.4; 8192 x 8192: 11.7, 12.0), with eight it may cost a tenth
// (8192 x 8192: 13.1, 13.2; 4096 x 4096, groups of 32: 6.5, 5.8).
#pragma once
#include "lowbit_format.cuh"
#include "per_device.h"
#include "ptx.cuh"

namespace sb200 {
namespace lowbit {

constexpr int kRowWarps = 8;
constexpr int kRowThreads = kRowWarps * 32;

// Codes 2 q and 2 q + 1 (in the order of the inputs) of a word, minus the zero point.
template <typename T>
__device__ __forceinline__ uint32_t code_pair(uint32_t w, int q, uint32_t bias, uint32_t mask, uint32_t magic) {
  return sub2<T>(and_or(w >> (4 * q), mask, magic), bias);
}
template <typename T> __device__ __forceinline__ void mma_16x8x16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16x8x16<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16x8x16<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

struct RowsParams {
  const void* x;   // rows on 16 bytes
  long long ldx;
  const uint8_t* codes;
  const uint8_t* scales;
  const uint8_t* zeros;  // or null
  void* y;
  long long ldy;
  int m, n, k, blocks;
};

// The first `bytes` of 16, zeros behind; through the first-level cache.
__device__ __forceinline__ void copy_async_part(uint32_t to, const void* from, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}

// Bytes of a stage: codes, scales and zeros of RT row tiles, then 128 inputs of eight rows of x.
__host__ __device__ constexpr int rows_tile_bytes(int per) { return kW4TileBytes + kW4Rows * 3 * per; }
__host__ __device__ constexpr int rows_stage_bytes(int per, int rt) { return rt * rows_tile_bytes(per) + 8 * 256; }
__host__ __device__ constexpr int rows_smem(int per, int rt, int ahead) { return kRowWarps * ahead * rows_stage_bytes(per, rt); }

template <typename T, int PER, int RT, int AHEAD, bool ZEROS>
__global__ void __launch_bounds__(kRowThreads) w4_rows_kernel(const RowsParams p) {
  constexpr int kTile = rows_tile_bytes(PER), kStage = rows_stage_bytes(PER, RT);
  static_assert(kRowWarps * 8 * (RT * 16 + 1) * 4 <= rows_smem(PER, RT, AHEAD), "the sums reuse the rings");
  extern __shared__ __align__(128) uint8_t smem_rows[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int tile0 = static_cast<int>(blockIdx.x) * RT;  // first row tile of the block
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem_rows)) + warp * (AHEAD * kStage);

  // where this lane's copies come from; they move on by a tile of 128 inputs for each warp of the block
  const uint8_t *codes[RT], *table[RT];
  const bool copies_table = lane < 2 * PER || (ZEROS && lane < 3 * PER);  // 2 PER pieces of scales, PER of zeros
  const int table_step = kRowWarps * kW4Rows * PER * (lane < 2 * PER ? 2 : 1);
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    // row tiles behind the weights read the last one and are not stored
    const long long tile = static_cast<long long>(min(tile0 + r, w4_row_tiles(p.n) - 1)) * p.blocks + warp;
    codes[r] = p.codes + tile * kW4TileBytes + lane * 16;
    table[r] = lane < 2 * PER ? p.scales + tile * (kW4Rows * 2 * PER) + lane * 16
                              : p.zeros + tile * (kW4Rows * PER) + (lane - 2 * PER) * 16;
  }
  // Piece (row, c) of 16 of a row of x: eight inputs.  Odd rows keep their upper and lower eight pieces the other way
  // round, so that eight lanes read eight different 16-byte columns.  Rows from m on are not copied: what the ring holds
  // there reaches columns of the result that are not stored.
  const int xc = lane & 15, xrow = lane >> 4;
  const T* x = static_cast<const T*>(p.x) + xrow * p.ldx;
  int fetch_k = warp * kW4Block + xc * 8, fetch_b = warp, fill = 0;
  auto fetch = [&]() {
    if (fetch_b < p.blocks) {
      const uint32_t to = ring + fill * kStage;
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        copy_async_16(to + r * kTile + lane * 16, codes[r], true);
        copy_async_16(to + r * kTile + 512 + lane * 16, codes[r] + 512, true);
        if (copies_table) copy_async_16(to + r * kTile + kW4TileBytes + lane * 16, table[r], true);
        codes[r] += kRowWarps * kW4TileBytes;
        table[r] += table_step;
      }
      const int left = min(max(p.k - fetch_k, 0), 8) * 2;
      const T* from = x + (left ? fetch_k : 0);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (2 * i + xrow < p.m)
          copy_async_part(to + RT * kTile + (2 * i + xrow) * 256 + ((xc ^ (xrow << 2)) << 4), from + 2 * i * p.ldx, left);
    }
    fetch_b += kRowWarps;
    fetch_k += kRowWarps * kW4Block;
    fill = fill + 1 == AHEAD ? 0 : fill + 1;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  float total[RT][4] = {};
#pragma unroll
  for (int a = 0; a < AHEAD - 1; ++a) fetch();
  int stage = 0;
  const uint32_t mask = in_register(0x000f000fu), magic = in_register(Half<T>::magic);
  const uint32_t xat = g * 256 + ((t ^ ((g & 1) << 2)) << 4);  // of word 0; word j is 64 j further, exclusive-or
  for (int b = warp; b < p.blocks; b += kRowWarps) {
    asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD - 2) : "memory");
    __syncwarp();  // every lane's copies of this stage are there, and all have read the stage that is filled next
    fetch();
    const uint32_t at = ring + stage * kStage;
    stage = stage + 1 == AHEAD ? 0 : stage + 1;
    uint4 xv[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) xv[j] = ptx::lds_v4(at + RT * kTile + (xat ^ (j << 6)));
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const uint32_t tile = at + r * kTile;
      const uint4 lo4 = ptx::lds_v4(tile + lane * 16), hi4 = ptx::lds_v4(tile + 512 + lane * 16);
      const uint32_t lo[4] = {lo4.x, lo4.y, lo4.z, lo4.w}, hi[4] = {hi4.x, hi4.y, hi4.z, hi4.w};
#pragma unroll
      for (int gr = 0; gr < PER; ++gr) {
        uint32_t bias[2];
        float scale[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int entry = (8 * h + g) * PER + gr;
          const uint16_t s = static_cast<uint16_t>(lds_u16(tile + kW4TileBytes + 2 * entry));
          scale[h] = to_f32(*reinterpret_cast<const T*>(&s));
          bias[h] = Half<T>::magic +
                    (ZEROS ? __byte_perm(lds_u8(tile + kW4TileBytes + kW4Rows * 2 * PER + entry), 0, 0x4040) : 0x00080008u);
        }
        float acc[4] = {};
#pragma unroll
        for (int jj = 0; jj < 4 / PER; ++jj) {
          const int j = gr * (4 / PER) + jj;
          const uint32_t xw[4] = {xv[j].x, xv[j].y, xv[j].z, xv[j].w};
#pragma unroll
          for (int q = 0; q < 4; q += 2) {
            const uint32_t a4[4] = {code_pair<T>(lo[j], q, bias[0], mask, magic), code_pair<T>(hi[j], q, bias[1], mask, magic),
                                    code_pair<T>(lo[j], q + 1, bias[0], mask, magic), code_pair<T>(hi[j], q + 1, bias[1], mask, magic)};
            mma_16x8x16<T>(acc, a4, xw[q], xw[q + 1]);
          }
        }
        total[r][0] = fmaf(scale[0], acc[0], total[r][0]);
        total[r][1] = fmaf(scale[0], acc[1], total[r][1]);
        total[r][2] = fmaf(scale[1], acc[2], total[r][2]);
        total[r][3] = fmaf(scale[1], acc[3], total[r][3]);
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  float(*part)[8][RT * 16 + 1] = reinterpret_cast<float(*)[8][RT * 16 + 1]>(smem_rows);
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int i = 0; i < 4; ++i) part[warp][2 * t + (i & 1)][r * 16 + g + 8 * (i >> 1)] = total[r][i];
  __syncthreads();
  constexpr int kCols = RT * 16;
  for (int e = threadIdx.x; e < p.m * kCols; e += kRowThreads) {
    const int row = e / kCols, c = e % kCols, col = static_cast<int>(blockIdx.x) * kCols + c;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) s += part[w][row][c];
    if (col < p.n) static_cast<T*>(p.y)[row * p.ldy + col] = from_f32<T>(s);
  }
}

template <typename T, int PER, int RT, int AHEAD, bool ZEROS>
int launch_rows_kernel(const RowsParams& p, cudaStream_t stream) {
  constexpr int kSmem = rows_smem(PER, RT, AHEAD);
  if (kSmem > 48 * 1024) {
    static PerDeviceOnce attr;
    const int rc = attr.run_once([] {
      return static_cast<int>(cudaFuncSetAttribute(w4_rows_kernel<T, PER, RT, AHEAD, ZEROS>,
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    });
    if (rc) return rc;
  }
  w4_rows_kernel<T, PER, RT, AHEAD, ZEROS><<<ceil_div(w4_row_tiles(p.n), RT), kRowThreads, kSmem, stream>>>(p);
  return static_cast<int>(cudaGetLastError());
}
template <typename T, int PER, int RT, int AHEAD>
int launch_rows(const RowsParams& p, cudaStream_t stream) {
  return p.zeros ? launch_rows_kernel<T, PER, RT, AHEAD, true>(p, stream)
                 : launch_rows_kernel<T, PER, RT, AHEAD, false>(p, stream);
}

}  // namespace lowbit
}  // namespace sb200
