// Products with 4-bit weights: C[m,n] = a_scale[m] * sum_k A[m,k] * (q[n,k] - zero[n,k/group]) * scale[n,k/group].
// W is [N][K/2] bytes, the even k in the low half.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "softmax.cuh"

namespace tsm100 {
namespace w4 {

struct Params {
  const void* a;
  const float* a_scales;   // rows in 8 bits
  const uint8_t* w;
  const void* scales;
  const uint8_t* zeros;    // or null: 8
  void* c;
  int64_t m, n;
  int32_t k, group;
};

// A warp per output.
template <typename T, typename A>
__global__ void __launch_bounds__(256)
gemm_w4_kernel(const Params p) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (i >= p.m * p.n) return;
  const int64_t row = i / p.n, col = i % p.n;
  const int groups = p.k / p.group;
  float acc = 0.f;
  for (int k = 2 * (threadIdx.x & 31); k < p.k; k += 64) {
    const int64_t g = col * groups + k / p.group;
    const int z = p.zeros ? p.zeros[g] : 8, b = p.w[col * (p.k / 2) + k / 2];
    const float s = softmax::Elem<T>::load1(static_cast<const T*>(p.scales) + g);
    const A* a = static_cast<const A*>(p.a) + row * p.k + k;
    acc = fmaf(static_cast<float>(a[0]), s * ((b & 15) - z), acc);
    acc = fmaf(static_cast<float>(a[1]), s * ((b >> 4) - z), acc);
  }
  acc = softmax::warp_sum(acc);
  if ((threadIdx.x & 31) == 0) softmax::Elem<T>::store1(static_cast<T*>(p.c) + i, p.a_scales ? acc * p.a_scales[row] : acc);
}

}  // namespace w4
}  // namespace tsm100
