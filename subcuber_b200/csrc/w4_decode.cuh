// y = x W^T for up to 64 rows of x (a decoding batch), weights in format W4.
//
// Up to 8 rows a warp's own matrix instruction takes the codes from registers (w4_rows.cuh), but that kernel is bound by the
// instructions it issues, and every 8 rows more add a matrix instruction and the loads of x for each 16 x 16 codes.  Here the
// weights go where tcgen05.mma takes them from without another pass through shared memory: a thread expands a row of
// 128 inputs in its registers and writes it to its lane of tensor memory, which is the left operand (128 rows x 16 inputs
// an instruction); x, the right operand, comes to shared memory by TMA.  What a batch costs is then almost independent of its
// rows: 8192 x 8192, groups of 128: 9 rows 17.9 us, 16 rows 18.4, 32 rows 19.2, 64 rows 21.0 (the bytes: 5.3 us; 1.9 TB/s).  64 rows are
// what its shared memory and 256 columns of tensor memory hold; 65 rows in the next kernel take 36.0 us (4096 x 4096: 11.4 and 17.4).
//
// Bound.  Neither memory nor the tensor cores (16 rows: 6 % busy, 64: 22 %) nor one pipe: the integer pipe is active for 36 % of the
// cycles, issue for half, and the warps wait on one another (load, expand, store to tensor memory, hand over).  About 15 instructions
// for eight weights are the expansion.  The scales are multiplied in here, one rounding to 16 bits for each weight: an accumulator
// gathers groups whose scales differ, and scaling the sums of each group instead, as up to 8 rows, would mean emptying it every 32 to
// 128 inputs.  Against exact weights that costs a third more error in the result (bf16, root mean square: 0.0022 of the result; its own
// rounding alone is 0.0017).
//
// Split.  A CTA holds 128 rows; where rows are few, the CTAs of a cluster divide the inputs and add their sums over
// distributed shared memory, rank by rank, so that results do not change from call to call.  Two CTAs share an SM: one
// starts or ends while the other works.  Two groups of four converter warps take the tiles of 128 inputs in turn; every warp
// fetches the codes of its own 32 rows by asynchronous copies into a ring of its own, kAhead tiles ahead.
#pragma once
#include <cooperative_groups.h>

#include "expand_product.cuh"

namespace sb200 {
namespace lowbit {

struct DecodeParams {
  CUtensorMap right;  // x: boxes of 64 inputs x n16 rows
  const uint8_t* codes;
  const uint8_t* scales;
  const uint8_t* zeros;  // or null
  void* y;
  long long ldy;
  int m, n, blocks;
  int n16;            // rows of x rounded up to 16
  int* status;
  Waits waits;
};

constexpr int kDecodeThreads = 320;  // warps 0 and 1: TMA and MMA, 2-9: converters
constexpr int kDecodeRows = 128, kDecodeMaxRight = 64;
constexpr int kDecodeMaxRanks = 8;   // CTAs of a cluster
// Tiles of 128 inputs that one accumulator takes while a cluster can still be larger: the tensor cores chop when they add (eight
// additions a tile; measured 0.4 units of 2^-23 of the partial sum for each, 2.3 where the terms are far smaller than the sum), and
// there is no room in tensor memory to drain it on the way.  128 tiles that rise and fall back leave 1e-5 of the sum of all
// magnitudes; f16 rounds at 4.9e-4.  16 rows, without and with this rule: 16384 x 53248: 151 us, 159; 9472 x 53248: 96, 119;
// 19072 x 32768: 181, 142; up to 16384 inputs it changes nothing.
constexpr int kDecodeBlocks = 128;
constexpr int kAhead = 3;            // stages of a converter warp's ring
constexpr int kLeftStages = 3;       // of 128 inputs in tensor memory, 64 columns each; the sums take the 64 behind
constexpr int kRightStages = 3;      // of 128 inputs of x in shared memory
__host__ __device__ constexpr int decode_warp_stage(int per) { return 2 * (kW4TileBytes + kW4Rows * 3 * per); }
__host__ __device__ constexpr int decode_smem(int per, int n16) {
  return 1024 + kRightStages * n16 * 256 + 8 * kAhead * decode_warp_stage(per) + 256;
}

__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
      "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
      "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Left operand from tensor memory, right one from shared memory.
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

template <typename T, int PER>
__global__ void __launch_bounds__(kDecodeThreads, 2) w4_decode_kernel(const __grid_constant__ DecodeParams p) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  constexpr int kWarpStage = decode_warp_stage(PER), kTile = kWarpStage / 2;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int right_bytes = p.n16 * 256;
  uint8_t* rings = smem + kRightStages * right_bytes;
  uint64_t* right_full = reinterpret_cast<uint64_t*>(rings + 8 * kAhead * kWarpStage);
  uint64_t* right_empty = right_full + kRightStages;
  uint64_t* left_full = right_empty + kRightStages;
  uint64_t* left_empty = left_full + kLeftStages;
  uint64_t* sums_full = left_empty + kLeftStages;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(sums_full + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row0 = static_cast<int>(blockIdx.x / ranks) * kDecodeRows;
  // this CTA's tiles of 128 inputs
  const int b0 = static_cast<int>(static_cast<long long>(p.blocks) * rank / ranks);
  const int b1 = static_cast<int>(static_cast<long long>(p.blocks) * (rank + 1) / ranks);
  auto give_up_here = [&](int code) {
    if (lane == 0) {
      *abort_flag = 1;
      atomicCAS(p.status, 0, code);
    }
  };

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    if (blockIdx.x == 0) *p.status = 0;
    for (int s = 0; s < kRightStages; ++s) {
      ptx::mbar_init(&right_full[s], 1);
      ptx::mbar_init(&right_empty[s], 1);
    }
    for (int s = 0; s < kLeftStages; ++s) {
      ptx::mbar_init(&left_full[s], 4);  // the warps of a group
      ptx::mbar_init(&left_empty[s], 1);
    }
    ptx::mbar_init(sums_full, 1);
    ptx::fence_mbar_init();
  }
  if (warp == 1) {
    ptx::tmem_alloc(tmem_holder, 256);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_holder, tmem_sums = tmem_base + kLeftStages * 64;

  if (warp == 0) {
    // ---- x by TMA
    if (lane == 0) ptx::prefetch_tmap(&p.right);
    uint32_t stage = 0, phase = 0;
    for (int b = b0; b < b1; ++b) {
      if (!ptx::mbar_wait_warp<false>(&right_empty[stage], phase ^ 1u, abort_flag, p.waits.ns)) {
        give_up_here(101);
        break;
      }
      if (ptx::elect_one()) {
        ptx::mbar_arrive_expect_tx(&right_full[stage], right_bytes);
        ptx::tma_load_2d(smem + stage * right_bytes, &p.right, &right_full[stage], b * kW4Block, 0);
        ptx::tma_load_2d(smem + stage * right_bytes + right_bytes / 2, &p.right, &right_full[stage], b * kW4Block + 64, 0);
      }
      __syncwarp();
      if (++stage == kRightStages) { stage = 0; phase ^= 1u; }
    }
  } else if (warp == 1) {
    // ---- MMA issuer
    const uint32_t idesc = (1u << 4) | (Half<T>::fmt << 7) | (Half<T>::fmt << 10) | (static_cast<uint32_t>(p.n16 >> 3) << 17) |
                           (static_cast<uint32_t>(kDecodeRows >> 4) << 24);
    uint32_t rs = 0, rphase = 0, ls = 0, lphase = 0;
    bool ok = true;
    for (int b = b0; b < b1; ++b) {
      if (!ptx::mbar_wait_warp<false>(&right_full[rs], rphase, abort_flag, p.waits.ns) ||
          !ptx::mbar_wait_warp<false>(&left_full[ls], lphase, abort_flag, p.waits.ns)) {
        give_up_here(102);
        ok = false;
        break;
      }
      ptx::tc_fence_after_sync();
      const uint64_t bd = ptx::umma_desc_sw128(ptx::smem_u32(smem + rs * right_bytes), 16, 1024);
      const uint64_t half_step = static_cast<uint64_t>(right_bytes / 2) >> 4;
      if (ptx::elect_one()) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          umma_f16_ts(tmem_sums, tmem_base + ls * 64 + i * 8, bd + (i >> 2) * half_step + (i & 3) * 2, idesc, (b > b0 || i > 0) ? 1u : 0u);
        ptx::umma_commit(&left_empty[ls]);
        ptx::umma_commit(&right_empty[rs]);
      }
      __syncwarp();
      if (++rs == kRightStages) { rs = 0; rphase ^= 1u; }
      if (++ls == kLeftStages) { ls = 0; lphase ^= 1u; }
    }
    if (ok && ptx::elect_one()) ptx::umma_commit(sums_full);
    __syncwarp();
  } else {
    // ---- converters: a warp has the 32 rows of its lane quarter, two row tiles
    const int cw = warp - 2, group = cw >> 2, quarter = warp & 3;
    const uint32_t ring = ptx::smem_u32(rings) + cw * (kAhead * kWarpStage);
    const int tiles = w4_row_tiles(p.n);
    const int tile0 = row0 / kW4Rows + quarter * 2;
    auto fetch = [&](int b, int stage) {
      if (b < b1) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          // row tiles behind the weights read the last one and are not stored
          const long long tile = static_cast<long long>(min(tile0 + r, tiles - 1)) * p.blocks + b;
          const uint32_t to = ring + stage * kWarpStage + r * kTile;
          const uint8_t* from = p.codes + tile * kW4TileBytes + lane * 16;
          // piece t of a row lies at t ^ (row / 2 & 3): eight lanes that read the same piece of eight rows then touch
          // eight different 16-byte columns
#pragma unroll
          for (int h = 0; h < 2; ++h)
            copy_async_16(to + h * 512 + (((lane & ~3) | ((lane & 3) ^ ((lane >> 3) & 3))) << 4), from + h * 512, true);
          if (lane < 3 * PER) {  // 2 PER pieces of scales, PER of zeros
            const bool zero = lane >= 2 * PER;
            const uint8_t* table = zero ? p.zeros + tile * (kW4Rows * PER) + (lane - 2 * PER) * 16
                                        : p.scales + tile * (kW4Rows * 2 * PER) + lane * 16;
            if (!zero || p.zeros) copy_async_16(to + kW4TileBytes + lane * 16, table, true);
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    const int first = b0 + group;
#pragma unroll
    for (int a = 0; a < kAhead - 1; ++a) fetch(first + 2 * a, a);
    int stage = 0, fill = kAhead - 1;
    // tiles of both groups take the left stages in order: this group starts at stage `group` and moves on by two
    uint32_t ls = group, lphase = 0;
    const int r16 = lane & 15;
    const uint32_t mask = in_register(0x000f000fu), magic = in_register(Half<T>::magic);
    for (int b = first; b < b1; b += 2) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 2) : "memory");
      __syncwarp();  // every lane's copies of this stage are there, and all have read the stage that is filled next
      fetch(b + 2 * (kAhead - 1), fill);
      fill = fill + 1 == kAhead ? 0 : fill + 1;
      const uint32_t at = ring + stage * kWarpStage + (lane >> 4) * kTile;
      stage = stage + 1 == kAhead ? 0 : stage + 1;
      uint32_t w[4][4];  // [piece][word]
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const uint4 v = ptx::lds_v4(at + r16 * 64 + ((t ^ ((r16 >> 1) & 3)) << 4));
        w[t][0] = v.x; w[t][1] = v.y; w[t][2] = v.z; w[t][3] = v.w;
      }
      uint32_t scale[PER], bias[PER];
#pragma unroll
      for (int q = 0; q < PER; ++q) {
        scale[q] = __byte_perm(lds_u16(at + kW4TileBytes + 2 * (r16 * PER + q)), 0, 0x1010);
        const uint32_t z = p.zeros ? lds_u8(at + kW4TileBytes + kW4Rows * 2 * PER + r16 * PER + q) : 8u;
        bias[q] = Half<T>::magic + __byte_perm(z, 0, 0x4040);
      }
      if (!ptx::mbar_wait_warp<false>(&left_empty[ls], lphase ^ 1u, abort_flag, p.waits.ns)) {
        give_up_here(104);
        break;
      }
      ptx::tc_fence_after_sync();
      const uint32_t to = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + ls * 64;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t r[32];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const int q = (2 * h + j) * PER / 4;
            const uint4 v = expand_w4<T>(w[t][2 * h + j], bias[q], scale[q], mask, magic);
            r[j * 16 + t * 4] = v.x; r[j * 16 + t * 4 + 1] = v.y; r[j * 16 + t * 4 + 2] = v.z; r[j * 16 + t * 4 + 3] = v.w;
          }
        tmem_st_32x32(to + h * 32, r);
      }
      tmem_st_wait();
      ptx::tc_fence_before_sync();
      __syncwarp();
      if (lane == 0 && !p.waits.drop) ptx::mbar_arrive(&left_full[ls]);
      ls += 2;
      if (ls >= kLeftStages) { ls -= kLeftStages; lphase ^= 1u; }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  }

  // ---- the sums: row = lane of tensor memory, column = row of x
  __syncthreads();  // the rings are free (and every role is done, or has given up)
  if (!ptx::mbar_wait_warp<false>(sums_full, 0, abort_flag, p.waits.ns)) give_up_here(103);
  float* part = reinterpret_cast<float*>(smem);  // [rows of x][128]
  __syncthreads();
  const bool whole = !*abort_flag;  // read where no warp writes it any more: the same for all threads of the CTA
  if (whole && b1 > b0 && warp >= 2) {  // two warps to a lane quarter, each takes eight of sixteen columns
    ptx::tc_fence_after_sync();
    const int quarter = warp & 3, row = row0 + quarter * 32 + lane;
    const uint32_t from = tmem_sums + (static_cast<uint32_t>(quarter * 32) << 16);
    for (int c0 = (warp - 2) / 4 * 8; c0 < p.n16; c0 += 16) {
      uint32_t r[8];
      tmem_ld_32x8(from + c0, r);
      ptx::tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (ranks > 1) part[(c0 + i) * kDecodeRows + quarter * 32 + lane] = __uint_as_float(r[i]);
        else if (c0 + i < p.m && row < p.n) static_cast<T*>(p.y)[(c0 + i) * p.ldy + row] = from_f32<T>(__uint_as_float(r[i]));
      }
    }
    ptx::tc_fence_before_sync();
  }
  if (ranks > 1) {
    cluster.sync();
    // Four neighbouring rows for each thread, all CTAs' parts asked for before the first is added.  Rows behind the weights are
    // not fetched.
    constexpr int kJoins = (kDecodeMaxRight * (kDecodeRows / 4) + 2 * kDecodeThreads - 1) / (2 * kDecodeThreads);
    float4 sum[kJoins];
    auto place = [&](int i, int& row, int& col) -> bool {  // of the thread's i-th four values
      const int e = (i * ranks + rank) * kDecodeThreads + static_cast<int>(threadIdx.x);
      row = row0 + e % (kDecodeRows / 4) * 4;
      col = e / (kDecodeRows / 4);
      return col < p.m && row < p.n;
    };
#pragma unroll
    for (int i = 0; i < kJoins; ++i) {
      int row, col;
      if (!place(i, row, col)) continue;
      const float* at = part + col * kDecodeRows + (row - row0);
      float4 v[kDecodeMaxRanks];
#pragma unroll
      for (int c = 0; c < kDecodeMaxRanks; ++c)
        if (c < ranks) v[c] = *reinterpret_cast<const float4*>(cluster.map_shared_rank(at, c));
      sum[i] = v[0];
#pragma unroll
      for (int c = 1; c < kDecodeMaxRanks; ++c)
        if (c < ranks) { sum[i].x += v[c].x; sum[i].y += v[c].y; sum[i].z += v[c].z; sum[i].w += v[c].w; }
    }
    // No CTA leaves while others read its memory: the arrival releases, so that this thread's reads are over before any CTA gets
    // past the wait.  The stores to y come after it, so that it does not wait for them.
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
#pragma unroll
    for (int i = 0; i < kJoins; ++i) {
      int row, col;
      if (!place(i, row, col)) continue;
      T* to = static_cast<T*>(p.y) + col * p.ldy + row;
      const T four[4] = {from_f32<T>(sum[i].x), from_f32<T>(sum[i].y), from_f32<T>(sum[i].z), from_f32<T>(sum[i].w)};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (row + j < p.n) to[j] = four[j];
    }
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  }
  __syncthreads();
  if (*abort_flag) {
    const uint64_t t0 = ptx::globaltimer_ns();
    while (ptx::globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
  }
  if (warp == 1) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc(tmem_base, 256);
  }
}

}  // namespace lowbit
}  // namespace sb200
