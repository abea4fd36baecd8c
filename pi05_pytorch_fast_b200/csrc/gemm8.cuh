// Matrix product in 8-bit integers with a scale for each token and each
// output channel:
//   y[m, n] = (sum_k a[m, k] w[n, k]) * sa[m] * sw[n] + bias[n]
// a int8 [m, k] (rows8.cuh), w int8 [n, k].  The sum is exact in int32 (k <=
// 131072); the scaling is fp32, rounded once to the output's type.
#pragma once

#include "rows8.cuh"

namespace w4a4 {

struct Gemm8Params {
  const int8_t* a;
  const int8_t* w;
  const float* sa;
  const float* sw;
  const void* bias;  // output type, or NULL
  void* y;           // contiguous [m, n]
  long long lda, ldw;
  long long m;
  int n, k;
};

// A 32 x 32 tile of y per CTA of 256 threads, K in steps of 64 bytes through
// shared memory, four products per dp4a: right for every case.
template <typename T>
__global__ void __launch_bounds__(256) gemm8_simple_kernel(const __grid_constant__ Gemm8Params p) {
  __shared__ __align__(16) int8_t as[32][68], ws[32][68];
  pdl_launch_dependents();
  pdl_wait();
  const long long m0 = static_cast<long long>(blockIdx.y) * 32;
  const int n0 = blockIdx.x * 32;
  const int tm = threadIdx.x >> 5, tn = threadIdx.x & 31;
  int acc[4] = {};
  for (int k0 = 0; k0 < p.k; k0 += 64) {
    for (int i = threadIdx.x; i < 32 * 64; i += 256) {
      const int r = i >> 6, c = i & 63;
      as[r][c] = m0 + r < p.m && k0 + c < p.k ? p.a[(m0 + r) * p.lda + k0 + c] : int8_t(0);
      ws[r][c] = n0 + r < p.n && k0 + c < p.k ? p.w[static_cast<long long>(n0 + r) * p.ldw + k0 + c] : int8_t(0);
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 64; c += 4) {
      const int wv = *reinterpret_cast<const int*>(&ws[tn][c]);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = __dp4a(*reinterpret_cast<const int*>(&as[tm + 8 * i][c]), wv, acc[i]);
    }
    __syncthreads();
  }
  const int n = n0 + tn;
  if (n >= p.n) return;
  const float b = p.bias ? to_float(static_cast<const T*>(p.bias)[n]) : 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long long m = m0 + tm + 8 * i;
    if (m < p.m)
      static_cast<T*>(p.y)[m * p.n + n] = from_float<T>(fmaf(static_cast<float>(acc[i]) * p.sa[m], p.sw[n], b));
  }
}

}  // namespace w4a4
