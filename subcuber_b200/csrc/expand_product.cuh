// Products whose left operand is held in few bits and is expanded to 16 bits on its way to the tensor cores:
//     W4    y^T = W x^T      left rows = outputs of the layer,  right columns = rows of x,   reduction = inputs
//     ACT8  dW  = X^T dY     left rows = channels,              right columns = columns of dY, reduction = tokens
//
// A pair of CTAs computes a tile of 256 left rows x `bn` columns with tcgen05.mma.cta_group::2.  Per step of 64 of the
// reduction each CTA's converter warps (two groups of four, in turn) expand the 128 x 64 values of its own left rows into the swizzled shared-memory
// tile that the tensor cores read; TMA brings the codes and the CTA's half of the right operand, so that no
// converter has a load of its own in flight when it hands a tile to the tensor cores.  The expansion costs no pass over
// memory: the operand travels in 4 or 8 bits and is never written out in 16.  (One rounding to 16 bits for each weight is what the
// tensor cores ask of an operand whose scale changes along the reduction.)
//   W4    the tile is K-major (a word of the format is the 16 bytes of eight neighbouring inputs); weights are rounded to 16
//         bits once, code - zero is exact before.
//   ACT8  the tile is MN-major (tokens are rows in memory, channels run along a row); every value is exact in 16 bits.
//
// A left tile is expanded once for every tile of columns.  With many of those it is cheaper to expand the operand once into 16
// bits in the workspace and to multiply that (DENSE: the left tiles come by TMA too, there are no converters): 1280 rows
// through 8192 x 4096 4-bit weights take 78 us, expanded on the way 86 us; a gradient of 4096 x 1280 from 4096 tokens
// 60 and 69 us (expand_product.cu has more sizes).
//
// Bound.  Dense, a large product: the tensor pipe is busy for 89 % of the cycles (2048 rows; a gradient of 2048 x 2304: 75 %), and
// under a long load the power limit lowers the clock (4096 rows through 8192 x 4096: 1.2 PFLOP/s in a long run, 1.5 in a short
// one; a gradient of 4096 x 8192 from 16384 tokens 1.1 and 1.5).  Expanded on the way: tensor pipe 51 % (4-bit) and 55 % (8-bit), the
// converters issue in 36 and 42 % of the cycles, and operands, codes and expanded tiles share the bandwidth of shared memory.  Small products: about 9 us for the launch, the
// setup, the first loads, the last sums and the end, and 0.37 us for every step of 64 that a narrow tile takes.
//
// Sums.  The tensor cores chop when they add to an accumulator (measured on B200, exact products of normal values:
// relative error 3.4e-5 after 2048 additions, 1.5e-6 after 128, growing with their number), which is too coarse for a gradient kept in
// fp32.  So an accumulator in tensor memory takes kSubSteps steps only; then eight epilogue warps add it to the tile's
// running sum in their registers, rounding to nearest, while the MMAs go on in the other accumulator.  With 128 sums a thread
// the epilogue warps need more registers than the others can spare at launch: the warps trade them (setmaxnreg).
#pragma once
#include <cuda.h>

#include "lowbit_format.cuh"
#include "lowbit_host.h"
#include "ptx.cuh"

namespace sb200 {
namespace lowbit {

enum ExpandKind { kExpandW4 = 0, kExpandAct8 = 1 };

struct ExpandParams {
  CUtensorMap left;         // codes: W4: 64-bit words (one for each input, so that coordinates fit), a row for each row tile;
                            // ACT8: bytes, a row for each token
                            // dense: the left operand in 16 bits, [row][input] (W4), [block of 64 channels][token][64] (ACT8)
  CUtensorMap right;        // x [tokens][inputs] (W4) or dY [tokens][columns] (ACT8)
  const void* scales;       // W4
  const uint8_t* zeros;     // W4, or null
  const uint8_t* exps;      // ACT8
  int exp_pitch;            // ACT8
  int right_blocked;        // ACT8: `right` is [block of 64 columns][token][64], one box for a CTA's whole half
  int rows, cols;           // of the result: left rows, right columns
  int depth;                // length of the reduction
  int bn;                   // columns of a tile, a multiple of 32 up to 256
  int tiles_r, tiles_c;
  int steps;                // steps of 64 of the reduction
  int slices;               // parts of the reduction; more than one: parts are written to `part` in fp32
  void* out;                // ACT8: [rows][ldo]; W4: [cols][ldo] (transposed)
  long long ldo;
  const void* base;         // ACT8, or null
  long long ldbase;
  int out_f32;
  float* part;              // [slices][the result's shape, packed]
  int* status;
  Waits waits;
};

constexpr int kPairRows = 256, kCtaRows = 128, kStep = 64, kMaxCols = 256;
constexpr int kSubSteps = 8;       // steps that one accumulator takes: 32 additions
constexpr int kExpandStages = 5;
constexpr int kRawStages = 4;      // tiles of codes: a step (ACT8: 64 tokens x 128 channels) or two (W4: 128 rows x 128 inputs)
constexpr int kRawBytes = 8192;
constexpr int kLeftBytes = kCtaRows * 128;           // 128 x 64 values of 16 bits
constexpr int kRightBytes = (kMaxCols / 2) * 128;    // at most 128 columns x 64
constexpr int kStageBytes = kLeftBytes + kRightBytes;
constexpr int kRightBlock = 64 * 128;                // 64 columns x 64 tokens (MN-major)
constexpr int kExpandThreads = 640;  // warpgroups: 0 = producers and MMA, 1-2 = epilogue, 3-4 = converters
constexpr int kEpilogueWarps = 8;
constexpr int kConvertWarps = 4;  // of a group; the two groups take the steps (W4: pairs of steps) in turn
constexpr int kPieces = kRawBytes / 16 / (32 * kConvertWarps);  // of 16 bytes of codes that a converter thread expands
constexpr int kProducers = 3;
constexpr int kTransposeBytes = 32 * 32 * 4;         // per epilogue warp
// scales and zeros of 128 rows (W4, PER groups each), or exponents of 64 tokens (ACT8, four blocks each)
__host__ __device__ constexpr int table_bytes(int kind, int per) { return kind == kExpandW4 ? kCtaRows * 3 * per : kStep * 4; }
__host__ __device__ constexpr int expand_smem(int kind, int per) {
  return 1024 + kExpandStages * kStageBytes + kRawStages * (kRawBytes + table_bytes(kind, per)) +
         (kind == kExpandAct8 ? kEpilogueWarps * kTransposeBytes : 0) + 1024;
}
// The dense form has no converters; its ring takes what they leave.
constexpr int kDenseStages = 6, kDenseThreads = 384;
constexpr int kDenseSmem = 1024 + kDenseStages * kStageBytes + kEpilogueWarps * kTransposeBytes + 1024;
// registers a thread: at launch (all threads), and after the trade; the sum of what the warpgroups take must not
// exceed what the block was launched with (the host checks the kernel's count before a launch)
constexpr int kRegsLaunch = 96, kRegsControl = 48, kRegsEpilogue = 152, kRegsConvert = 64;
static_assert(128 * kRegsControl + 256 * kRegsEpilogue + 64 * kConvertWarps * kRegsConvert <= kExpandThreads * kRegsLaunch, "register trade");
static_assert(expand_smem(kExpandW4, 4) <= 232448 && expand_smem(kExpandAct8, 1) <= 232448, "shared memory of a CTA");

template <int N> __device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

__device__ __forceinline__ void tmem_ld_32x8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}

// The calling thread arrives at `bar` once its asynchronous copies have landed.
__device__ __forceinline__ void copy_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(ptx::smem_u32(bar)) : "memory");
}

__device__ __forceinline__ uint2 lds_v2(uint32_t smem_addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(smem_addr));
  return v;
}

struct ExpandUnit {
  int row0, col0;  // of the pair's tile
  int k0, k1;      // steps
  int slice;
};

// Units in order: all tiles of a slice, tiles in bands of 16 tile rows, down the rows of a band first, so that the tiles that
// run together share both operands' panels in L2.
__device__ __forceinline__ ExpandUnit expand_unit(const ExpandParams& p, int u) {
  constexpr int kBand = 16;
  const int tiles = p.tiles_r * p.tiles_c;
  ExpandUnit r;
  r.slice = u / tiles;
  int t = u - r.slice * tiles;
  const int band = t / (kBand * p.tiles_c);
  t -= band * kBand * p.tiles_c;
  const int high = min(kBand, p.tiles_r - band * kBand);
  r.row0 = (band * kBand + t % high) * kPairRows;
  r.col0 = (t / high) * p.bn;
  // slices are cut at whole pairs of steps (a tile of the 4-bit format is two)
  const long long pairs = (p.steps + 1) / 2;
  r.k0 = static_cast<int>(2 * (pairs * r.slice / p.slices));
  r.k1 = min(p.steps, static_cast<int>(2 * (pairs * (r.slice + 1) / p.slices)));
  return r;
}

__device__ __forceinline__ void give_up(const ExpandParams& p, volatile int* abort_flag, int code) {
  *abort_flag = 1;
  atomicCAS(p.status, 0, code);
}

__device__ __forceinline__ float lds_f32(uint32_t a) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ void sts_f32(uint32_t a, float v) { asm volatile("st.shared.f32 [%0], %1;" ::"r"(a), "f"(v) : "memory"); }

// A warp's 32 rows x 128 columns of sums, a row to a lane, from and to a row-major matrix: 32 x 32 values at a time change
// places between lanes and registers in shared memory (`swap`, value (row, column) at word 32 row + (column ^ row)), so that
// memory sees whole rows.
template <typename E>
__device__ __forceinline__ void load_tile_rows(float (&sum)[128], const E* base, long long ld, int row0, int col0, int nrows,
                                               int ncols, uint32_t swap, int lane) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    if (c * 32 < ncols) {
      const bool in = c * 32 + lane < ncols;
      const E* from = base + row0 * ld + col0 + c * 32 + lane;
#pragma unroll 1
      for (int b = 0; b < 32; b += 8) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i, from += ld) v[i] = in && b + i < nrows ? to_f32(*from) : 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sts_f32(swap + (b + i) * 128 + ((lane ^ (b + i)) << 2), v[i]);
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 32; ++i) sum[c * 32 + i] = lds_f32(swap + lane * 128 + ((i ^ lane) << 2));
      __syncwarp();
    }
  }
}
template <typename E>
__device__ __forceinline__ void store_tile_rows(const float (&sum)[128], E* out, long long ld, int row0, int col0, int nrows,
                                                int ncols, uint32_t swap, int lane) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    if (c * 32 < ncols) {
#pragma unroll
      for (int i = 0; i < 32; ++i) sts_f32(swap + lane * 128 + ((i ^ lane) << 2), sum[c * 32 + i]);
      __syncwarp();
      const bool in = c * 32 + lane < ncols;
      E* to = out + row0 * ld + col0 + c * 32 + lane;
#pragma unroll 8
      for (int i = 0; i < 32; ++i, to += ld) {
        const float v = lds_f32(swap + i * 128 + ((lane ^ i) << 2));
        if (in && i < nrows) *to = from_f32<E>(v);
      }
      __syncwarp();
    }
  }
}
// The same to the transposed matrix: a column of the tile is a row there, 32 lanes store 32 neighbours.
template <typename E>
__device__ __forceinline__ void store_tile_cols(const float (&sum)[128], E* out, long long ld, int row0, int col0, int nrows,
                                                int ncols, int lane) {
  E* to = out + col0 * ld + row0 + lane;
#pragma unroll
  for (int c = 0; c < 128; ++c, to += ld)
    if (c < ncols && lane < nrows) *to = from_f32<E>(sum[c]);
}

template <typename T, int KIND, int PER, bool DENSE>
__global__ void __launch_bounds__(DENSE ? kDenseThreads : kExpandThreads, 1)
expand_product_kernel(const __grid_constant__ ExpandParams p) {
  constexpr int kStages = DENSE ? kDenseStages : kExpandStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr int kTable = table_bytes(KIND, PER);
  uint8_t* raw = smem + kStages * kStageBytes;
  float* transpose = reinterpret_cast<float*>(raw + (DENSE ? 0 : kRawStages * kRawBytes));
  uint8_t* tables = reinterpret_cast<uint8_t*>(transpose) + (KIND == kExpandAct8 || DENSE ? kEpilogueWarps * kTransposeBytes : 0);
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(tables + (DENSE ? 0 : kRawStages * kTable));
  uint64_t* empty_bar = full_bar + kStages;
  uint64_t* slot_full = empty_bar + kStages;
  uint64_t* slot_free = slot_full + 2;
  uint64_t* left_bar = slot_free + 2;  // this CTA's left tile of a stage is written
  uint64_t* raw_full = left_bar + kStages;
  uint64_t* raw_empty = raw_full + kRawStages;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(raw_empty + kRawStages);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = ptx::cluster_ctarank();  // 0 = leader
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int units = p.tiles_r * p.tiles_c * p.slices;

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    // all blocks of the grid are resident, so this store comes long before any bounded wait can run out
    if (blockIdx.x == 0) *p.status = 0;
    for (int s = 0; s < kStages; ++s) {
      ptx::mbar_init(&full_bar[s], DENSE ? 1 : 2);  // the leader's producer, the peer's left tile
      ptx::mbar_init(&left_bar[s], kConvertWarps);
      ptx::mbar_init(&empty_bar[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      ptx::mbar_init(&slot_full[s], 1);
      ptx::mbar_init(&slot_free[s], 2 * kEpilogueWarps);
    }
    for (int s = 0; s < kRawStages; ++s) {
      ptx::mbar_init(&raw_full[s], 1 + 32);  // the codes, and a producer's lanes' parts of the tables
      ptx::mbar_init(&raw_empty[s], kConvertWarps);
    }
    ptx::fence_mbar_init();
  }
  if (warp == 1) {
    ptx::tmem_alloc_pair(tmem_holder, 512);
    ptx::tmem_relinquish_pair();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::cluster_sync_all();
  ptx::tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_holder;
  const int half = p.bn / 2;  // columns of the right operand that a CTA brings

  if (warp < 4) {
    if (!DENSE) regs_dec<kRegsControl>();
    if (warp != 1) {
      // ---- producers: codes, tables and the CTA's half of the right operand.  The loads of one warp complete one after the
      // other (about 240 ns each, whatever they hold), so three warps take the steps (W4: pairs of steps) in turn.
      const int boxes = KIND == kExpandW4 ? 1 : (half + 63) / 64;
      const uint32_t bytes = 2u * ((KIND == kExpandW4 ? half * 128 : boxes * kRightBlock) + (DENSE ? kLeftBytes : 0));  // both CTAs'
      constexpr int kEach = KIND == kExpandW4 && !DENSE ? 2 : 1;  // steps of a tile of codes
      if (warp == 0 && lane == 0) {
        ptx::prefetch_tmap(&p.right);
        ptx::prefetch_tmap(&p.left);
      }
      uint32_t stage = 0, phase = 0, rstage = 0, rphase = 0;
      int turn = warp == 0 ? 0 : warp - 1;
      bool ok = true;
      for (int u = pair; ok && u < units; u += pairs) {
        const ExpandUnit w = expand_unit(p, u);
        const int row0 = w.row0 + static_cast<int>(rank) * kCtaRows;
        const int col0 = w.col0 + static_cast<int>(rank) * half;
        // where this lane's pieces of the tables come from; W4: of 24 PER pieces of 16 bytes (2 PER of scales for each of the
        // eight row tiles, then PER of zeros), three at most; ACT8: the exponents of two tokens, 32 apart
        constexpr int kCopies = DENSE ? 1 : KIND == kExpandW4 ? (24 * PER + 31) / 32 : 2;
        const uint8_t* from[kCopies];
        bool real[kCopies];
#pragma unroll
        for (int c = 0; c < kCopies; ++c) {
          if (DENSE) break;
          if (KIND == kExpandW4) {
            const int i = c * 32 + lane;
            const bool zero = i >= 16 * PER;
            const int j = zero ? i - 16 * PER : i, each = zero ? PER : 2 * PER;
            const int tile = row0 / kW4Rows + j / each;
            real[c] = i < 24 * PER && tile < w4_row_tiles(p.rows) && (!zero || p.zeros);
            from[c] = static_cast<const uint8_t*>(p.scales);
            if (real[c]) from[c] = (zero ? p.zeros : from[c]) + (static_cast<long long>(tile) * w4_blocks(p.depth) * each + j % each) * 16;
          } else {
            real[c] = row0 < p.rows;
            from[c] = p.exps + (real[c] ? row0 / kActBlock : 0);
          }
        }
        for (int kk = w.k0; ok && kk < w.k1; kk += kEach) {
          const bool mine = turn == 0;
          turn = mine ? kProducers - 1 : turn - 1;
          if (mine && !DENSE) {
            if (!ptx::mbar_wait_warp<false>(&raw_empty[rstage], rphase ^ 1u, abort_flag, p.waits.ns)) {
              if (lane == 0) give_up(p, abort_flag, 101);
              ok = false;
              break;
            }
            if (ptx::elect_one()) {
              ptx::mbar_arrive_expect_tx(&raw_full[rstage], kRawBytes);
              if (KIND == kExpandW4) ptx::tma_load_2d(raw + rstage * kRawBytes, &p.left, &raw_full[rstage], kk * kStep, row0 / kW4Rows);
              else ptx::tma_load_2d(raw + rstage * kRawBytes, &p.left, &raw_full[rstage], row0, kk * kStep);
            }
            __syncwarp();
            const uint32_t table = ptx::smem_u32(tables + rstage * kTable);
#pragma unroll
            for (int c = 0; c < kCopies; ++c) {
              const int i = c * 32 + lane;
              if (KIND == kExpandW4) {
                if (i < 24 * PER) copy_async_16(table + i * 16, from[c] + (real[c] ? kk * (i >= 16 * PER ? 8 * PER : 16 * PER) : 0), real[c]);
              } else {
                const int token = kk * kStep + i;
                const bool in = real[c] && token < p.depth;
                copy_async_4(table + i * 4, from[c] + (in ? static_cast<long long>(token) * p.exp_pitch : 0), in);
              }
            }
            copy_async_arrive(&raw_full[rstage]);
          }
          if (++rstage == kRawStages) { rstage = 0; rphase ^= 1u; }
#pragma unroll
          for (int h = 0; h < kEach; ++h) {
            if (mine) {
              if (!ptx::mbar_wait_warp<false>(&empty_bar[stage], phase ^ 1u, abort_flag, p.waits.ns)) {
                if (lane == 0) give_up(p, abort_flag, 101);
                ok = false;
                break;
              }
              if (!(DENSE && p.waits.drop) && ptx::elect_one()) {
                if (rank == 0) ptx::mbar_arrive_expect_tx(&full_bar[stage], bytes);
                uint8_t* to = smem + stage * kStageBytes + kLeftBytes;
                if (DENSE) {
                  if (KIND == kExpandW4) ptx::tma_load_2d_pair(to - kLeftBytes, &p.left, &full_bar[stage], kk * kStep, row0);
                  else ptx::tma_load_3d_pair(to - kLeftBytes, &p.left, &full_bar[stage], 0, kk * kStep, row0 / 64);
                }
                if (KIND == kExpandW4) {
                  ptx::tma_load_2d_pair(to, &p.right, &full_bar[stage], (kk + h) * kStep, col0);
                } else if (p.right_blocked) {
                  ptx::tma_load_3d_pair(to, &p.right, &full_bar[stage], 0, kk * kStep, col0 / 64);
                } else {
                  for (int b = 0; b < boxes; ++b)
                    ptx::tma_load_2d_pair(to + b * kRightBlock, &p.right, &full_bar[stage], col0 + b * 64, kk * kStep);
                }
              }
              __syncwarp();
            }
            if (++stage == kStages) { stage = 0; phase ^= 1u; }
          }
        }
      }
    } else if (warp == 1 && rank == 0) {
      // ---- MMA issuer (leader)
      const uint32_t idesc = (1u << 4) | (Half<T>::fmt << 7) | (Half<T>::fmt << 10) |
                             (KIND == kExpandAct8 ? (1u << 15) | (1u << 16) : 0u) |
                             (static_cast<uint32_t>(p.bn >> 3) << 17) | (static_cast<uint32_t>(kPairRows >> 4) << 24);
      const uint32_t lbo = KIND == kExpandW4 ? 16 : kRightBlock;
      const uint32_t advance = (KIND == kExpandW4 ? 32 : 16 * 128) >> 4;  // 16 of the reduction
      const uint64_t a0 = ptx::umma_desc_sw128(ptx::smem_u32(smem), lbo, 1024);
      const uint64_t b0 = ptx::umma_desc_sw128(ptx::smem_u32(smem) + kLeftBytes, lbo, 1024);
      uint32_t stage = 0, phase = 0, slot = 0, free_bits = 0;
      bool ok = true;
      for (int u = pair; ok && u < units; u += pairs) {
        const ExpandUnit w = expand_unit(p, u);
        int sub = 0;
        for (int kk = w.k0; kk < w.k1; ++kk) {
          if (sub == 0) {
            if (!ptx::mbar_wait_warp<false>(&slot_free[slot], ((free_bits >> slot) & 1u) ^ 1u, abort_flag, p.waits.ns)) {
              if (lane == 0) give_up(p, abort_flag, 102);
              ok = false;
              break;
            }
            free_bits ^= 1u << slot;
            ptx::tc_fence_after_sync();
          }
          if (!ptx::mbar_wait_warp<false>(&full_bar[stage], phase, abort_flag, p.waits.ns)) {
            if (lane == 0) give_up(p, abort_flag, 102);
            ok = false;
            break;
          }
          if (!DENSE && !ptx::mbar_wait_warp<false>(&left_bar[stage], phase, abort_flag, p.waits.ns)) {
            if (lane == 0) give_up(p, abort_flag, 102);
            ok = false;
            break;
          }
          const uint64_t as = a0 + ((stage * kStageBytes) >> 4), bs = b0 + ((stage * kStageBytes) >> 4);
          const bool last = sub == kSubSteps - 1 || kk == w.k1 - 1;
          if (ptx::elect_one()) {
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
              ptx::umma_f16_pair(tmem_base + slot * kMaxCols, as + ks * advance, bs + ks * advance, idesc, (sub | ks) ? 1u : 0u);
            ptx::umma_commit_pair(&empty_bar[stage], 3);
            if (last) ptx::umma_commit_pair(&slot_full[slot], 3);
          }
          __syncwarp();
          if (++stage == kStages) { stage = 0; phase ^= 1u; }
          ++sub;
          if (last) { sub = 0; slot ^= 1u; }
        }
      }
    }
    else if (!DENSE) {
      // ---- passes on to the leader that the peer's left tile is written.  One thread's arrival crosses to the other CTA
      // for each step instead of one from each converter warp.
      uint32_t stage = 0, phase = 0;
      bool ok = true;
      for (int u = pair; ok && u < units; u += pairs) {
        const ExpandUnit w = expand_unit(p, u);
        for (int kk = w.k0; kk < w.k1; ++kk) {
          if (!ptx::mbar_wait_warp<false>(&left_bar[stage], phase, abort_flag, p.waits.ns)) {
            if (lane == 0) give_up(p, abort_flag, 104);
            ok = false;
            break;
          }
          if (lane == 0) ptx::mbar_arrive_remote(&full_bar[stage], 0);
          __syncwarp();
          if (++stage == kStages) { stage = 0; phase ^= 1u; }
        }
      }
    }
  } else if (warp < 12) {
    // ---- epilogue: warp = 32 rows (of its lane quarter) x half of the tile's columns
    if (!DENSE) regs_inc<kRegsEpilogue>();
    const int quarter = warp & 3, side = (warp - 4) >> 2;
    const uint32_t swap = ptx::smem_u32(transpose) + (warp - 4) * kTransposeBytes;
    const uint32_t tmem = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + side * half;
    uint32_t slot = 0, full_bits = 0;
    bool ok = true;
    for (int u = pair; ok && u < units; u += pairs) {
      const ExpandUnit w = expand_unit(p, u);
      const int row0 = w.row0 + static_cast<int>(rank) * kCtaRows + quarter * 32;
      const int col0 = w.col0 + side * half;
      const int ncols = min(half, p.cols - col0), nrows = min(32, p.rows - row0);  // at most 0: outside
      float sum[128];
#pragma unroll
      for (int i = 0; i < 128; ++i) sum[i] = 0.f;
      if (KIND == kExpandAct8 && p.base && p.slices == 1) {
        // the sums start from the base, which is read while the tile's first MMAs run
        if (p.out_f32) load_tile_rows(sum, static_cast<const float*>(p.base), p.ldbase, row0, col0, nrows, ncols, swap, lane);
        else load_tile_rows(sum, static_cast<const T*>(p.base), p.ldbase, row0, col0, nrows, ncols, swap, lane);
      }
      for (int kk = w.k0; kk < w.k1; kk += kSubSteps) {
        if (!ptx::mbar_wait_warp<false>(&slot_full[slot], (full_bits >> slot) & 1u, abort_flag, p.waits.ns)) {
          if (lane == 0) give_up(p, abort_flag, 103);
          ok = false;
          break;
        }
        full_bits ^= 1u << slot;
        ptx::tc_fence_after_sync();
        const uint32_t from = tmem + slot * kMaxCols;
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          if (c * 8 < half) {
            uint32_t r[8];
            tmem_ld_32x8(from + c * 8, r);
            ptx::tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[c * 8 + i] += __uint_as_float(r[i]);
          }
        }
        ptx::tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive_remote(&slot_free[slot], 0);
        slot ^= 1u;
      }
      if (!ok) break;
      if (KIND == kExpandW4) {
        if (p.slices > 1) store_tile_cols(sum, p.part + static_cast<long long>(w.slice) * p.rows * p.cols, p.rows, row0, col0, nrows, ncols, lane);
        else store_tile_cols(sum, static_cast<T*>(p.out), p.ldo, row0, col0, nrows, ncols, lane);
      } else {
        if (p.slices > 1) store_tile_rows(sum, p.part + static_cast<long long>(w.slice) * p.rows * p.cols, p.cols, row0, col0, nrows, ncols, swap, lane);
        else if (p.out_f32) store_tile_rows(sum, static_cast<float*>(p.out), p.ldo, row0, col0, nrows, ncols, swap, lane);
        else store_tile_rows(sum, static_cast<T*>(p.out), p.ldo, row0, col0, nrows, ncols, swap, lane);
      }
    }
  } else if (!DENSE) {
    // ---- converters
    if (!DENSE) regs_dec<kRegsConvert>();
    const int group = (warp - 12) / kConvertWarps, tid = threadIdx.x % (kConvertWarps * 32);
    const uint32_t left = ptx::smem_u32(smem), codes = ptx::smem_u32(raw);
    uint32_t stage = 0, phase = 0, rstage = 0, rphase = 0, turn = group;
    bool ok = true;
    auto next_stage = [&]() { if (++stage == kStages) { stage = 0; phase ^= 1u; } };
    auto next_raw = [&]() { if (++rstage == kRawStages) { rstage = 0; rphase ^= 1u; } };
    auto acquire = [&]() -> bool {  // the stage's previous contents have been read
      if (ptx::mbar_wait_warp<false>(&empty_bar[stage], phase ^ 1u, abort_flag, p.waits.ns)) return true;
      if (lane == 0) give_up(p, abort_flag, 104);
      return false;
    };
    auto publish = [&]() {
      ptx::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0 && !p.waits.drop) ptx::mbar_arrive(&left_bar[stage]);
      next_stage();
    };
    auto raw_ready = [&]() -> bool {
      if (ptx::mbar_wait_warp<false>(&raw_full[rstage], rphase, abort_flag, p.waits.ns)) return true;
      if (lane == 0) give_up(p, abort_flag, 104);
      return false;
    };
    auto raw_done = [&]() {  // every lane has read the codes and tables
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&raw_empty[rstage]);
      next_raw();
    };
    for (int u = pair; ok && u < units; u += pairs) {
      const ExpandUnit w = expand_unit(p, u);
      if (KIND == kExpandW4) {
        // A thread takes four pieces of a tile of 128 inputs: 16 bytes (four words) of a row.  Words 0 and 1 belong to the first
        // step, 2 and 3 to the second.  Lanes of odd rows take the second word of a step first, so that eight
        // lanes always store to eight different 16-byte columns of the swizzled tile.
        const int g = lane >> 2, t = lane & 3, odd = g & 1;
        const uint32_t mask = in_register(0x000f000fu), magic = in_register(Half<T>::magic);
        const int row0 = (tid >> 6) * kW4Rows + 8 * ((tid >> 5) & 1) + g;  // of the first piece; the others 32 rows on
        const uint32_t line0 = row0 * 128 + (((4 * odd + t) ^ g) << 4), line1 = row0 * 128 + (((4 * (1 - odd) + t) ^ g) << 4);
        for (int kk = w.k0; kk < w.k1; kk += 2) {
          turn ^= 1u;
          if (turn == 0) {
            next_raw();
            next_stage();
            next_stage();
            continue;
          }
          if (!raw_ready()) { ok = false; break; }
          const uint32_t from = codes + rstage * kRawBytes + tid * 16;
          const uint32_t table = ptx::smem_u32(tables) + rstage * kTable;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t word[kPieces][2], bias[kPieces][2], scale[kPieces][2];  // [piece][first, second to be stored]
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
              const uint2 c = lds_v2(from + i * (kRawBytes / kPieces) + h * 8);
              word[i][0] = odd ? c.y : c.x;
              word[i][1] = odd ? c.x : c.y;
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                if (PER < 4 && j == 1) { bias[i][1] = bias[i][0]; scale[i][1] = scale[i][0]; continue; }
                const int at = (row0 + (kCtaRows / kPieces) * i) * PER + (PER == 4 ? 2 * h + (j ^ odd) : PER == 2 ? h : 0);
                const uint32_t s = lds_u16(table + 2 * at), z = p.zeros ? lds_u8(table + kCtaRows * 2 * PER + at) : 8u;
                scale[i][j] = __byte_perm(s, 0, 0x1010);
                bias[i][j] = Half<T>::magic + __byte_perm(z, 0, 0x4040);
              }
            }
            if (!acquire()) { ok = false; break; }
            const uint32_t to = left + stage * kStageBytes;
#pragma unroll
            for (int i = 0; i < kPieces; ++i)
#pragma unroll
              for (int j = 0; j < 2; ++j)
                ptx::sts_v4(to + i * (kLeftBytes / kPieces) + (j ? line1 : line0), expand_w4<T>(word[i][j], bias[i][j], scale[i][j], mask, magic));
            publish();
          }
          if (!ok) break;
          raw_done();
        }
      } else {
        // A thread takes four pieces of a step: 16 channels of a token, of the first 64 channels or the second.  Of eight
        // neighbouring lanes four hold the first 64 channels of one token and four the second 64 of the token beside it:
        // loads and stores then touch eight different 16-byte columns.
        const int quarter = tid & 3, block = (tid >> 2) & 1, piece = quarter + 4 * block;
        uint32_t from[2], exponent[2], line[2][2];  // of the first two pieces; the others 32 tokens on
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int token = 2 * (tid >> 3) + (block ^ i);
          from[i] = token * 128 + piece * 16;
          exponent[i] = token * 4 + (piece >> 1);
#pragma unroll
          for (int j = 0; j < 2; ++j) line[i][j] = block * kRightBlock + token * 128 + (((2 * quarter + j) ^ (token & 7)) << 4);
        }
        for (int kk = w.k0; kk < w.k1; ++kk) {
          turn ^= 1u;
          if (turn == 0) {
            next_raw();
            next_stage();
            continue;
          }
          if (!raw_ready()) { ok = false; break; }
          uint4 c[kPieces];
          uint32_t e[kPieces];
#pragma unroll
          for (int i = 0; i < kPieces; ++i) {
            c[i] = ptx::lds_v4(codes + rstage * kRawBytes + from[i & 1] + (i >> 1) * (32 * 128));
            e[i] = lds_u8(ptx::smem_u32(tables) + rstage * kTable + exponent[i & 1] + (i >> 1) * (32 * 4));
          }
          if (!acquire()) { ok = false; break; }
          const uint32_t to = left + stage * kStageBytes;
#pragma unroll
          for (int i = 0; i < kPieces; ++i) {
            const Act8Step<T> step(e[i]);
            ptx::sts_v4(to + line[i & 1][0] + (i >> 1) * (32 * 128), expand_act8<T>(c[i].x, c[i].y, step));
            ptx::sts_v4(to + line[i & 1][1] + (i >> 1) * (32 * 128), expand_act8<T>(c[i].z, c[i].w, step));
          }
          raw_done();
          publish();
        }
      }
    }
  }

  // ---- teardown
  ptx::tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag) {  // copies in flight land before the shared memory goes
    const uint64_t t0 = ptx::globaltimer_ns();
    while (ptx::globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
  }
  ptx::cluster_sync_all();
  if (warp == 1) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc_pair(tmem_base, 512);
  }
}

// out[r][c] = base[r][c] + the slices' parts in order.  A thread adds V neighbours (4 where rows of the parts start on 16 bytes:
// cols a multiple of 4); 2^cols_log2 threads stand along a row.
template <typename Out, int V>
__global__ void __launch_bounds__(256) join_slices_kernel(const float* __restrict__ part, int slices, int rows, int cols, Out* out,
                                                          long long ldo, const Out* base, long long ldbase, int cols_log2,
                                                          int row_parts) {
  const long long r = ((static_cast<long long>(blockIdx.x) / row_parts) << (8 - cols_log2)) + (threadIdx.x >> cols_log2);
  const int c = (((blockIdx.x % row_parts) << cols_log2) + (threadIdx.x & ((1 << cols_log2) - 1))) * V;
  if (r >= rows || c >= cols) return;
  const long long total = static_cast<long long>(rows) * cols;
  const float* from = part + r * cols + c;
  float v[V];
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = base ? to_f32(base[r * ldbase + c + i]) : 0.f;
#pragma unroll 4
  for (int s = 0; s < slices; ++s, from += total) {
    if (V == 4) {
      const float4 x = __ldcs(reinterpret_cast<const float4*>(from));
      v[0] += x.x; v[V > 1 ? 1 : 0] += x.y; v[V > 2 ? 2 : 0] += x.z; v[V > 3 ? 3 : 0] += x.w;
    } else {
      v[0] += __ldcs(from);
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) out[r * ldo + c + i] = from_f32<Out>(v[i]);
}

}  // namespace lowbit
}  // namespace sb200
