// y = x W^T for a few rows of x (a decoding batch), weights in format W4: bound by the bytes of the weights.
//
// Mathematics.  Codes are small whole numbers and exact in 16 bits, so that the matrix instruction multiplies (code -
// zero) with x without any rounding; the sums of one group are scaled in fp32 afterwards:
//     y[m][n] = sum over groups g of scale(n, g) * (sum over k in g of (code - zero) x[m][k])
// A 4-bit code becomes a 16-bit number by bits alone: OR-ed into the last bits of 1024 (f16) or 128 (bf16) it adds exactly
// its value, and one packed subtraction of (1024 | 128) + zero leaves code - zero, for two codes at a time.
//
// Split.  A warp holds RT row tiles (16 weights' rows each) and walks over tiles of 128 inputs, one 16-byte load per lane and
// eight rows; the weights are the left operand of mma.m16n8k16 (16 rows x 16 inputs) and 8 NT rows of x the right one.  The
// order of inputs inside an instruction is free as long as both operands have the same: a lane takes its word's eight
// inputs as they lie in memory.  The warps of a block take the tiles of 128 inputs in turn, and where there are few row
// tiles the CTAs of a cluster divide them further: the sums meet in shared memory, in the order of warps and ranks, so
// that results do not change from call to call.
#pragma once
#include <cooperative_groups.h>

#include "lowbit_format.cuh"

namespace sb200 {
namespace lowbit {

constexpr int kRowWarps = 8;
constexpr int kRowThreads = kRowWarps * 32;

template <typename T> struct Pair16;
template <> struct Pair16<__half> {
  static constexpr uint32_t magic = 0x64006400u;  // 1024, last bit 1
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <> struct Pair16<__nv_bfloat16> {
  static constexpr uint32_t magic = 0x43004300u;  // 128, last bit 1
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

struct RowsParams {
  const void* x;
  long long ldx;
  const uint8_t* codes;
  const void* scales;
  const uint8_t* zeros;  // or null
  void* y;
  long long ldy;
  int m, n, k, blocks;
  bool wide;  // rows of x start on 16 bytes
};

// What a lane needs of one row tile and 128 inputs: rows g and g + 8.
template <int PER>  // groups in 128 inputs
struct TileRaw {
  uint4 w[2];
  uint32_t s[2][(PER + 1) / 2];  // scales, two to a register
  uint32_t z[2];                 // zeros, one to a byte
};

template <typename T, int PER>
__device__ __forceinline__ void load_tile(TileRaw<PER>& t, const RowsParams& p, long long tile, int lane) {
  const uint4* w = reinterpret_cast<const uint4*>(p.codes) + tile * (kW4TileBytes / 16) + lane;
  t.w[0] = __ldcs(w);
  t.w[1] = __ldcs(w + 32);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const long long at = (tile * kW4Rows + 8 * h + (lane >> 2)) * PER;
    const uint16_t* s = static_cast<const uint16_t*>(p.scales) + at;
    if (PER == 1) t.s[h][0] = __ldg(s);
    if (PER == 2) t.s[h][0] = __ldg(reinterpret_cast<const uint32_t*>(s));
    if (PER == 4) {
      const uint2 v = __ldg(reinterpret_cast<const uint2*>(s));
      t.s[h][0] = v.x;
      t.s[h][PER / 4] = v.y;
    }
    t.z[h] = 0x08080808u;
    if (p.zeros) {
      if (PER == 1) t.z[h] = __ldg(p.zeros + at);
      if (PER == 2) t.z[h] = __ldg(reinterpret_cast<const uint16_t*>(p.zeros + at));
      if (PER == 4) t.z[h] = __ldg(reinterpret_cast<const uint32_t*>(p.zeros + at));
    }
  }
}

template <typename T>
__device__ __forceinline__ float scale_of(uint32_t two, int which) {
  const uint16_t bits = static_cast<uint16_t>(two >> (16 * which));
  return to_f32(*reinterpret_cast<const T*>(&bits));
}

// Eight inputs of a row of x, zeros behind its end.
template <typename T>
__device__ __forceinline__ uint4 load_x(const T* row, int k0, int k, bool wide) {
  if (wide && k0 + 8 <= k) return __ldg(reinterpret_cast<const uint4*>(row + k0));
  uint4 r;
  uint16_t v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = k0 + i < k ? __ldg(reinterpret_cast<const uint16_t*>(row) + k0 + i) : uint16_t(0);
  r.x = v[0] | (v[1] << 16); r.y = v[2] | (v[3] << 16); r.z = v[4] | (v[5] << 16); r.w = v[6] | (v[7] << 16);
  return r;
}

template <typename T, int PER, int NT, int RT, int AHEAD>
__global__ void __launch_bounds__(kRowThreads) w4_rows_kernel(const RowsParams p) {
  namespace cg = cooperative_groups;
  __shared__ float part[kRowWarps][NT * 8][RT * 16 + 1];
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int tile0 = static_cast<int>(blockIdx.x / ranks) * RT;  // first row tile
  const int tiles = w4_row_tiles(p.n);
  const int m0 = blockIdx.y * (NT * 8);
  const int first = rank * kRowWarps + warp, stride = ranks * kRowWarps;
  float total[RT][NT][4] = {};
  // a block's last row tiles may lie behind the weights: they read the last one and are not stored
  long long base[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) base[r] = static_cast<long long>(min(tile0 + r, tiles - 1)) * p.blocks;

  TileRaw<PER> raw[AHEAD][RT];
#pragma unroll
  for (int a = 0; a < AHEAD; ++a)
#pragma unroll
    for (int r = 0; r < RT; ++r)
      if (first + a * stride < p.blocks) load_tile<T, PER>(raw[a][r], p, base[r] + first + a * stride, lane);

  for (int b0 = first; b0 < p.blocks; b0 += AHEAD * stride) {
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const int b = b0 + a * stride;
      if (b >= p.blocks) break;
      uint4 xv[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int row = m0 + nt * 8 + g;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          xv[nt][j] = make_uint4(0, 0, 0, 0);
          if (row < p.m) xv[nt][j] = load_x(static_cast<const T*>(p.x) + row * p.ldx, b * kW4Block + 32 * j + 8 * t, p.k, p.wide);
        }
      }
      TileRaw<PER> cur[RT];
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        cur[r] = raw[a][r];
        if (b + AHEAD * stride < p.blocks) load_tile<T, PER>(raw[a][r], p, base[r] + b + AHEAD * stride, lane);
      }
#pragma unroll
      for (int r = 0; r < RT; ++r) {
#pragma unroll
        for (int gr = 0; gr < PER; ++gr) {
          float acc[NT][4] = {};
          uint32_t bias[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t z = (cur[r].z[h] >> (8 * gr)) & 255u;
            bias[h] = Pair16<T>::magic + (z | (z << 16));
          }
#pragma unroll
          for (int jj = 0; jj < 4 / PER; ++jj) {
            const int j = gr * (4 / PER) + jj;
            const uint32_t lo = (&cur[r].w[0].x)[j], hi = (&cur[r].w[1].x)[j];
            uint32_t e[4][2];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              e[q][0] = Pair16<T>::sub(((lo >> (4 * q)) & 0x000f000fu) | Pair16<T>::magic, bias[0]);
              e[q][1] = Pair16<T>::sub(((hi >> (4 * q)) & 0x000f000fu) | Pair16<T>::magic, bias[1]);
            }
#pragma unroll
            for (int q = 0; q < 4; q += 2) {
              const uint32_t a4[4] = {e[q][0], e[q][1], e[q + 1][0], e[q + 1][1]};
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                Pair16<T>::mma(acc[nt], a4, (&xv[nt][j].x)[q], (&xv[nt][j].x)[q + 1]);
            }
          }
          const float s0 = scale_of<T>(cur[r].s[0][gr / 2], gr & 1), s1 = scale_of<T>(cur[r].s[1][gr / 2], gr & 1);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            total[r][nt][0] = fmaf(s0, acc[nt][0], total[r][nt][0]);
            total[r][nt][1] = fmaf(s0, acc[nt][1], total[r][nt][1]);
            total[r][nt][2] = fmaf(s1, acc[nt][2], total[r][nt][2]);
            total[r][nt][3] = fmaf(s1, acc[nt][3], total[r][nt][3]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) part[warp][nt * 8 + 2 * t + (i & 1)][r * 16 + g + 8 * (i >> 1)] = total[r][nt][i];
  __syncthreads();
  if (ranks > 1) {
    // the warps' sums of this CTA first, then rank 0 adds the ranks' in order
    for (int e = threadIdx.x; e < NT * 8 * RT * 16; e += kRowThreads) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < kRowWarps; ++w) s += part[w][e / (RT * 16)][e % (RT * 16)];
      part[0][e / (RT * 16)][e % (RT * 16)] = s;
    }
    cluster.sync();
  }
  if (rank == 0) {
    for (int e = threadIdx.x; e < NT * 8 * RT * 16; e += kRowThreads) {
      const int row = m0 + e / (RT * 16), col = tile0 * 16 + e % (RT * 16);
      float s = 0.f;
      if (ranks > 1) {
        for (int c = 0; c < ranks; ++c) s += *cluster.map_shared_rank(&part[0][e / (RT * 16)][e % (RT * 16)], c);
      } else {
#pragma unroll
        for (int w = 0; w < kRowWarps; ++w) s += part[w][e / (RT * 16)][e % (RT * 16)];
      }
      if (row < p.m && col < p.n) static_cast<T*>(p.y)[row * p.ldy + col] = from_f32<T>(s);
    }
  }
  if (ranks > 1) cluster.sync();  // no CTA leaves while rank 0 reads its memory
}

template <typename T, int PER, int NT, int RT, int AHEAD>
int launch_rows(const RowsParams& p, int ranks, cudaStream_t stream) {
  const long long gx = static_cast<long long>(ceil_div(w4_row_tiles(p.n), RT)) * ranks;
  const int gy = ceil_div(p.m, NT * 8);
  if (gx > 0x7fffffffll || gy > 65535) return kErrNotSupported;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(gx), static_cast<unsigned>(gy));
  cfg.blockDim = dim3(kRowThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {static_cast<unsigned>(ranks), 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, w4_rows_kernel<T, PER, NT, RT, AHEAD>, p));
}

}  // namespace lowbit
}  // namespace sb200
