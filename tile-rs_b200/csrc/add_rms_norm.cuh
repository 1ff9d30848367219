// RMS normalisation with the residual's addition, a weight, and an output in storage type or 8 bits:
//   h = x + residual,  sum = h,  y = h * rsqrt(mean(h^2) + eps) * weight
// all in f32 and each result rounded once.  8 bits: z = h * weight, step s = max|z| / 127, q = z / s rounded to nearest even, and the
// row's scale is s * rsqrt(..): the whole numbers do not depend on the order in which the squares were summed.
#pragma once

#include "softmax.cuh"

namespace tsm100 {
namespace addnorm {

using softmax::Elem;

constexpr int kThreads = 256;

template <typename T>
struct Params {
  const T* x;
  const T* residual;  // or null
  T* sum;             // or null; may be x or residual
  const T* weight;    // or null
  void* y;
  float* scales;      // 8 bits
  int64_t rows;
  int32_t cols;
  float eps;
};

// Sum and maximum over the CTA; every thread gets both.
__device__ __forceinline__ float2 block_sum_max(float2 v, float2* red) {
  v.x = softmax::warp_sum(v.x);
  v.y = softmax::warp_max(v.y);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
  for (int w = 1; w < kThreads / 32; ++w) v.x += red[w].x, v.y = fmaxf(v.y, red[w].y);
  return v;
}

// A CTA per row, which reads it twice, the second time from the caches; sum is written on the second way, so that it may be x or residual.
template <typename T, bool kI8>
__global__ void __launch_bounds__(kThreads)
add_rms_norm_kernel(const Params<T> p) {
  __shared__ float2 red[kThreads / 32];
  const int64_t at = static_cast<int64_t>(blockIdx.x) * p.cols;
  auto h_of = [&](int c) { return Elem<T>::load1(p.x + at + c) + (p.residual ? Elem<T>::load1(p.residual + at + c) : 0.f); };
  auto w_of = [&](int c) { return p.weight ? Elem<T>::load1(p.weight + c) : 1.f; };
  float2 acc = make_float2(0.f, 0.f);
  for (int c = threadIdx.x; c < p.cols; c += kThreads) {
    const float h = h_of(c);
    acc.x = fmaf(h, h, acc.x);
    if (kI8) acc.y = fmaxf(acc.y, fabsf(h * w_of(c)));
  }
  acc = block_sum_max(acc, red);
  const float r = rsqrtf(acc.x / p.cols + p.eps), step = acc.y * static_cast<float>(1.0 / 127.0);
  for (int c = threadIdx.x; c < p.cols; c += kThreads) {
    const float h = h_of(c), z = h * w_of(c);
    if (p.sum) Elem<T>::store1(p.sum + at + c, h);
    if (kI8) static_cast<int8_t*>(p.y)[at + c] = static_cast<int8_t>(step > 0.f ? __float2int_rn(z / step) : 0);
    else Elem<T>::store1(static_cast<T*>(p.y) + at + c, z * r);
  }
  if (kI8 && threadIdx.x == 0) p.scales[blockIdx.x] = step * r;
}

}  // namespace addnorm
}  // namespace tsm100
