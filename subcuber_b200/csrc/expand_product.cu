// Host side of the products with an expanded operand: how a product is cut, workspace, launches.
#include "expand_product.cuh"
#include "w4_decode.cuh"

#include <atomic>

#include "lowbit_host.h"
#include "per_device.h"

namespace sb200 {
namespace lowbit {
namespace {

inline size_t align_up(size_t x, size_t a) { return (x + a - 1) / a * a; }

constexpr int kMaxSlices = 16;
// From here on two passes.  On the way and in two passes, in us; rows through 4-bit weights:
//   2048 x 2048:   512: 15 and 17, 1024: 20 and 18, 1280: 21 and 19, 2048: 21 and 20
//   4096 x 4096:   512: 26 and 30, 1024: 33 and 34, 1280: 60 and 48, 2048: 59 and 54
//   8192 x 4096:   512: 34 and 42, 1024: 59 and 62, 1280: 86 and 78, 2048: 112 and 110
//   16384 x 4096:  512: 65 and 85, 1024: 115 and 124, 1280: 142 and 147, 2048: 206 and 202
//   8192 x 8192:   512: 59 and 86, 1024: 111 and 131, 1280: 162 and 157, 2048: 217 and 221
// columns of a gradient, tokens x channels:
//   2048 x 1024:   512: 16 and 20, 1024: 17 and 24, 1280: 20 and 24, 2048: 23 and 25
//   4096 x 4096:   512: 31 and 39, 1024: 39 and 43, 1280: 69 and 60, 2048: 69 and 65
//   16384 x 2048:  512: 42 and 56, 1024: 68 and 76, 1280: 90 and 94, 2048: 118 and 113
constexpr int kDenseColumns = 1280;
constexpr size_t kPartBytes = size_t(64) << 20;  // most that the parts of a divided reduction may take

struct Cut {
  int bn, slices;
};

// Tile width and parts of the reduction.  A step of 64 costs a pair about 2 bn clocks on the tensor cores (256 rows x bn
// columns x 64 at 8192 operations a clock and SM) and never less than what the hand-overs between the roles take (measured:
// 0.37 us at every narrow tile); a unit more than that for filling its pipeline and for its sums; dividing the
// reduction costs a pass over the parts, and a launch.  The cut with the least total of the fullest pair wins; widths
// are what the instruction takes.  (128 rows through 4096 x 4096 4-bit weights: 16 tiles; in one part 38 us, in four 17.5 us.)
Cut cut_of(long long rows, long long cols, int steps, int pairs, bool dense) {
  const double kStepLeast = dense ? 500 : 700, kUnit = 4000, kJoin = 4000, kBytesPerClock = 4000;
  Cut best{kMaxCols, 1};
  double least = 1e300;
  for (int bn = kMaxCols; bn >= 32; bn -= 32) {
    const double tiles = static_cast<double>(ceil_div(static_cast<int>(rows), kPairRows)) * ceil_div(static_cast<int>(cols), bn);
    for (int s = 1; s <= kMaxSlices; ++s) {
      if (s > 1 && (s > (steps + 1) / 2 || static_cast<double>(s) * rows * cols * 4 > kPartBytes)) break;
      const double waves = ceil(tiles * s / pairs);
      const double step = 2 * bn > kStepLeast ? 2 * bn : kStepLeast;
      double t = waves * (2 * ceil((steps + 1) / 2 / static_cast<double>(s)) * step + kUnit);
      if (s > 1) t += kJoin + (2.0 * s + 1) * rows * cols * 4 / kBytesPerClock;
      if (t < least) { least = t; best = Cut{bn, s}; }
    }
  }
  return best;
}

int pairs_of_device() {
  const int sms = sm_count_of_current_device();
  return (sms > 0 ? sms : 148) / 2;
}

size_t part_bytes(long long rows, long long cols) {
  const size_t all = align_up(size_t(kMaxSlices) * rows * cols * 4, 256);
  return all < kPartBytes ? all : kPartBytes;
}

template <typename T, int KIND, int PER, bool DENSE>
int launch(const ExpandParams& p, int pairs, cudaStream_t stream) {
  auto* kernel = expand_product_kernel<T, KIND, PER, DENSE>;
  constexpr int kSmem = DENSE ? kDenseSmem : expand_smem(KIND, PER);
  static PerDeviceOnce once;
  const int rc = once.run_once([&] {
    // the warps trade registers: a block launched with fewer than the trade needs would wait for good
    cudaFuncAttributes a;
    cudaError_t e = cudaFuncGetAttributes(&a, kernel);
    if (e != cudaSuccess) return static_cast<int>(e);
    if (!DENSE && a.numRegs != kRegsLaunch) return static_cast<int>(kErrInternal);
    return static_cast<int>(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
  });
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * pairs));
  cfg.blockDim = dim3(DENSE ? kDenseThreads : kExpandThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {2, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kernel, p));
}

template <typename Out>
int join(const ExpandParams& p, int rows, int cols, cudaStream_t stream) {
  const bool wide = cols % 4 == 0;
  const int pieces = wide ? cols / 4 : cols;
  int cols_log2 = 0;
  while (cols_log2 < 8 && (1 << cols_log2) < pieces) ++cols_log2;
  const int row_parts = ceil_div(pieces, 1 << cols_log2);
  const long long blocks = static_cast<long long>(row_parts) * ceil_div(rows, 256 >> cols_log2);
  if (blocks > 0x7fffffffll) return kErrNotSupported;
  auto* kernel = wide ? join_slices_kernel<Out, 4> : join_slices_kernel<Out, 1>;
  kernel<<<static_cast<unsigned>(blocks), 256, 0, stream>>>(p.part, p.slices, rows, cols, static_cast<Out*>(p.out), p.ldo,
                                                            static_cast<const Out*>(p.base), p.ldbase, cols_log2, row_parts);
  return static_cast<int>(cudaGetLastError());
}

// Fills in the cut; returns the pairs to launch, or 0 when there are too many units.
int place(ExpandParams& p, int pairs, bool dense) {
  const Cut c = cut_of(p.rows, p.cols, p.steps, pairs, dense);
  p.bn = c.bn;
  p.slices = c.slices;
  p.tiles_r = ceil_div(p.rows, kPairRows);
  p.tiles_c = ceil_div(p.cols, p.bn);
  const long long units = static_cast<long long>(p.tiles_r) * p.tiles_c * p.slices;
  if (units > 0x3fffffffll) return 0;
  return units < pairs ? static_cast<int>(units) : pairs;
}

template <typename T>
int run_w4(const ExpandParams& p, int group, bool dense, int pairs, cudaStream_t stream) {
  int rc;
  if (dense) rc = launch<T, kExpandW4, 1, true>(p, pairs, stream);
  else if (group == 32) rc = launch<T, kExpandW4, 4, false>(p, pairs, stream);
  else if (group == 64) rc = launch<T, kExpandW4, 2, false>(p, pairs, stream);
  else rc = launch<T, kExpandW4, 1, false>(p, pairs, stream);
  if (rc || p.slices == 1) return rc;
  return join<T>(p, p.cols, p.rows, stream);
}

template <typename T>
int run_act8(const ExpandParams& p, bool dense, int pairs, cudaStream_t stream) {
  if (p.steps > 0) {
    const int rc = dense ? launch<T, kExpandAct8, 1, true>(p, pairs, stream) : launch<T, kExpandAct8, 1, false>(p, pairs, stream);
    if (rc || p.slices == 1) return rc;
  }
  return p.out_f32 ? join<float>(p, p.rows, p.cols, stream) : join<T>(p, p.rows, p.cols, stream);
}

// Whether the left operand is expanded once, before the product: from so many columns on that the pass over memory (2.5 or 3
// bytes a value) costs less than expanding every tile again for each tile of columns.
bool dense_w4(int m) { return m >= kDenseColumns; }
bool dense_act8(int n) { return n >= kDenseColumns; }
size_t dense_bytes(long long rows, long long ld) { return align_up(size_t(rows) * ld * 2, 256); }

}  // namespace

size_t expand_w4_workspace(int m, int n, int k, bool x_aligned) {
  return kStatusBytes + (x_aligned ? 0 : copy_bytes(m, k)) + (dense_w4(m) ? dense_bytes(n, align_up(k, 8)) : 0) +
         (m > kDecodeMaxRows ? part_bytes(m, n) : 0);
}

int expand_w4(const W4& w, const void* x, long long ldx, void* y, long long ldy, int m, void* workspace, size_t workspace_bytes,
              const Waits& waits, cudaStream_t stream) {
  ExpandParams p = {};
  p.scales = w.scales;
  p.zeros = static_cast<const uint8_t*>(w.zeros);
  p.rows = w.n;
  p.cols = m;
  p.depth = w.k;
  p.steps = dense_w4(m) ? ceil_div(w.k, kStep) : 2 * w4_blocks(w.k);
  p.out = y;
  p.ldo = ldy;
  p.waits = waits;
  p.status = static_cast<int*>(workspace);
  const bool dense = dense_w4(m);
  char* part = static_cast<char*>(workspace) + (workspace_bytes - part_bytes(m, w.n)) / 256 * 256;
  p.part = reinterpret_cast<float*>(part);
  const int pairs = place(p, pairs_of_device(), dense);
  if (!pairs) return kErrNotSupported;
  int rc;
  if ((rc = tc::map_rows_16bit(&p.right, x, m, w.k, ldx, p.bn / 2))) return rc;
  if (dense) {
    const long long ld = static_cast<long long>(align_up(w.k, 8));
    char* left = part - dense_bytes(w.n, ld);
    if ((rc = dequantize_w4(w, left, ld, stream))) return rc;
    if ((rc = tc::map_rows_16bit(&p.left, left, w.n, w.k, ld, kCtaRows))) return rc;
  } else if ((rc = tc::map_rows_plain(&p.left, w.codes, 8, w4_row_tiles(w.n), 128ll * w4_blocks(w.k), 1024ll * w4_blocks(w.k),
                                      8, 128))) {  // a row tile's codes are one row of words; a box is 128 inputs of eight row tiles
    return rc;
  }
  return w.dtype == kF16 ? run_w4<__half>(p, w.group, dense, pairs, stream)
                         : run_w4<__nv_bfloat16>(p, w.group, dense, pairs, stream);
}

namespace {

template <typename T, int PER>
int launch_decode(const DecodeParams& p, cudaStream_t stream) {
  auto* kernel = w4_decode_kernel<T, PER>;
  static PerDeviceOnce attr;
  const int rc = attr.run_once([&] {
    return static_cast<int>(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, decode_smem(PER, kDecodeMaxRight)));
  });
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kDecodeThreads);
  cfg.dynamicSmemBytes = decode_smem(PER, p.n16);
  cfg.stream = stream;
  cudaLaunchAttribute attrs[1];
  attrs[0].id = cudaLaunchAttributeClusterDimension;
  cfg.attrs = attrs;
  cfg.numAttrs = 1;
  // CTAs that divide the inputs of 128 rows: as many as fit on the device at once, one for each SM, or two where they have eight
  // tiles or more to go through (the runtime counts one).  A cluster lies within one group of SMs, which leaves some of
  // them over.  16 rows, clusters of 1, 2, 4 and 8 CTAs in us: 128 x 4096: 16.6, 11.2, 8.2, 6.8; 4096 x 4096: 17.5, 11.8, 9.3,
  // 10.2; 8192 x 1024: 7.4, 6.7, 8.2, 13.8; 8192 x 8192: 31.8, 19.6, 18.4, 24.0; 9472 x 4096: 18.2, 12.8, 18.4, 22.8;
  // 16384 x 512: 6.3, 8.1, 13.1, 13.1 (no more than four, the tiles); 16384 x 4096: 18.7, 17.8, 22.8, 33.3.
  static std::atomic<int> room[kMaxDevices][kDecodeMaxRight / 16][4];  // clusters at once, plus one
  const int groups = ceil_div(p.n, kDecodeRows);
  int dev = -1, log2 = 3, least = 0;
  while (least < 3 && p.blocks > (kDecodeBlocks << least)) ++least;
  if (cudaError_t e = cudaGetDevice(&dev)) return static_cast<int>(e);
  for (; log2 > least; --log2) {
    const int ranks = 1 << log2;
    if (ranks > p.blocks || groups > 0x7fffffff / ranks) continue;
    attrs[0].val.clusterDim = {static_cast<unsigned>(ranks), 1, 1};
    cfg.gridDim = dim3(static_cast<unsigned>(groups) * ranks);
    std::atomic<int>* cached = dev < kMaxDevices ? &room[dev][p.n16 / 16 - 1][log2] : nullptr;
    int fit = cached ? cached->load(std::memory_order_relaxed) - 1 : -1;
    if (fit < 0) {
      if (cudaError_t e = cudaOccupancyMaxActiveClusters(&fit, kernel, &cfg)) return static_cast<int>(e);
      if (cached) cached->store(fit + 1, std::memory_order_relaxed);
    }
    if (groups <= fit || (groups <= 2 * fit && p.blocks >= 8 * ranks)) break;
  }
  attrs[0].val.clusterDim = {1u << log2, 1, 1};
  cfg.gridDim = dim3(static_cast<unsigned>(groups) << log2);
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kernel, p));
}

template <typename T>
int run_decode(const DecodeParams& p, int group, cudaStream_t stream) {
  if (group == 32) return launch_decode<T, 4>(p, stream);
  if (group == 64) return launch_decode<T, 2>(p, stream);
  return launch_decode<T, 1>(p, stream);
}

}  // namespace

int decode_w4(const W4& w, const void* x, long long ldx, void* y, long long ldy, int m, void* status, const Waits& waits,
              cudaStream_t stream) {
  DecodeParams p = {};
  p.codes = static_cast<const uint8_t*>(w.codes);
  p.scales = static_cast<const uint8_t*>(w.scales);
  p.zeros = static_cast<const uint8_t*>(w.zeros);
  p.y = y;
  p.ldy = ldy;
  p.m = m;
  p.n = w.n;
  p.blocks = w4_blocks(w.k);
  p.n16 = ceil_div(m, 16) * 16;
  p.status = static_cast<int*>(status);
  p.waits = waits;
  if (int rc = tc::map_rows_16bit(&p.right, x, m, w.k, ldx, p.n16)) return rc;
  return w.dtype == kF16 ? run_decode<__half>(p, w.group, stream) : run_decode<__nv_bfloat16>(p, w.group, stream);
}

size_t expand_act8_workspace(int m, int n, int k, bool dy_aligned) {
  return kStatusBytes + (dy_aligned ? 0 : copy_bytes(m, n)) + (dense_act8(n) ? dense_bytes(m, align_up(k, 64)) : 0) + part_bytes(k, n);
}

int expand_act8(const Act8& a, const void* dy, long long lddy, bool out_f32, const void* base, long long ldbase, void* dw,
                long long lddw, int n, void* workspace, const Waits& waits, cudaStream_t stream) {
  ExpandParams p = {};
  p.exps = static_cast<const uint8_t*>(a.exps);
  p.exp_pitch = static_cast<int>(a.exp_pitch);
  p.rows = a.k;
  p.cols = n;
  p.depth = a.m;
  p.steps = ceil_div(a.m, kStep);
  p.out = dw;
  p.ldo = lddw;
  p.base = base;
  p.ldbase = ldbase;
  p.out_f32 = out_f32;
  p.waits = waits;
  char* ws = static_cast<char*>(workspace);
  p.status = reinterpret_cast<int*>(ws);
  ws += kStatusBytes;
  int pairs = 0;
  const bool dense = dense_act8(n);
  if (p.steps > 0) {
    int rc;
    if (!tma_rows(dy, lddy)) {
      const int cols = static_cast<int>(align_up(n, 8));
      if ((rc = copy_rows_16bit(ws, cols, dy, a.m, n, lddy, stream))) return rc;
      dy = ws;
      lddy = cols;
      ws += copy_bytes(a.m, n);
    }
    if (!(pairs = place(p, pairs_of_device(), dense))) return kErrNotSupported;
    // one load for a CTA's half of the columns where that is whole blocks of 64, and the matrix too (a partial last block
    // would be read past the end of the row)
    p.right_blocked = n % 64 == 0 && p.bn % 128 == 0;
    if ((rc = p.right_blocked ? tc::map_blocks_16bit(&p.right, dy, a.m, n, lddy, kStep, p.bn / 128)
                              : tc::map_rows_16bit(&p.right, dy, a.m, n, lddy, kStep)))
      return rc;
    if (dense) {
      // (channels behind k are not written: they reach rows of the result that are not stored)
      const int ld = static_cast<int>(align_up(a.k, 64));
      if ((rc = restore_act8(a, ws, ld, stream))) return rc;
      if ((rc = tc::map_blocks_16bit(&p.left, ws, a.m, ld, ld, kStep, kCtaRows / 64))) return rc;
      ws += dense_bytes(a.m, ld);
    } else if ((rc = tc::map_rows_plain(&p.left, a.codes, 1, a.m, static_cast<long long>(align_up(a.k, 16)), a.pitch, kStep,
                                        kCtaRows))) {
      return rc;
    }
    p.part = reinterpret_cast<float*>(ws);
  }
  return a.dtype == kF16 ? run_act8<__half>(p, dense, pairs, stream) : run_act8<__nv_bfloat16>(p, dense, pairs, stream);
}

}  // namespace lowbit
}  // namespace sb200
