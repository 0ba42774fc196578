// C = A B (+ C0) with operands that are read element by element through functors, in fp32 on the CUDA cores.
#pragma once
#include "lowbit_format.cuh"

namespace sb200 {
namespace lowbit {

template <typename T>
struct DenseLeft {
  const T* p;
  long long ld;
  int rows, cols;
  __device__ float operator()(int i, int k) const { return i < rows && k < cols ? to_f32(p[i * ld + k]) : 0.f; }
};

template <typename Out, typename L, typename R>
__global__ void __launch_bounds__(256) simple_product_kernel(L left, R right, Out* __restrict__ c, long long ldc, const Out* c0,
                                                             long long ldc0, int m, int n, int k) {
  __shared__ float a[16][65], b[16][65];
  const int tiles_n = ceil_div(n, 64);
  const int i0 = static_cast<int>(blockIdx.x / tiles_n) * 64, j0 = static_cast<int>(blockIdx.x % tiles_n) * 64;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < k; k0 += 16) {
    for (int e = threadIdx.x; e < 1024; e += 256) {
      a[e & 15][e >> 4] = left(i0 + (e >> 4), k0 + (e & 15));
      b[e & 15][e >> 4] = right(k0 + (e & 15), j0 + (e >> 4));
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < 16; ++kk)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += a[kk][ty + 16 * i] * b[kk][tx + 16 * j];
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int r = i0 + ty + 16 * i, s = j0 + tx + 16 * j;
      if (r < m && s < n) c[r * ldc + s] = from_f32<Out>(acc[i][j] + (c0 ? to_f32(c0[r * ldc0 + s]) : 0.f));
    }
}

template <typename Out, typename L, typename R>
int simple_product(const L& left, const R& right, Out* c, long long ldc, const Out* c0, long long ldc0, int m, int n, int k,
                   cudaStream_t stream) {
  const long long grid = static_cast<long long>(ceil_div(m, 64)) * ceil_div(n, 64);
  if (grid > 0x7fffffffll) return 5;
  simple_product_kernel<Out><<<static_cast<unsigned>(grid), 256, 0, stream>>>(left, right, c, ldc, c0, ldc0, m, n, k);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace lowbit
}  // namespace sb200
