// RMS normalisation with the residual's addition, a weight, and an output in storage type or 8 bits:
//   h = x + residual,  sum = h,  y = h * rsqrt(mean(h^2) + eps) * weight
// all in f32 and each result rounded once.  8 bits: z = h * weight, step s = max|z| / 127, q = z / s rounded to nearest even, and the
// row's scale is s * rsqrt(..): the whole numbers do not depend on the order in which the squares were summed.
//
// Bound: HBM.  A row is read once and held in registers as h, by a warp (up to 1024 elements of 16 bits) or a CTA that takes a row and goes; its sum of squares and
// its largest |z| are reduced together.  Rows that start anywhere are held the same way, an element at a time, up to 8192; wider ones are read twice, the second
// time from the caches.
#pragma once

#include "quantise.cuh"
#include "softmax.cuh"

namespace tsm100 {
namespace addnorm {

using softmax::Elem;
using softmax::Vec16;

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

// Sum and maximum over the LANES threads of a row (a warp or the CTA); each gets both.
template <int LANES>
__device__ __forceinline__ float2 row_sum_max(float2 v, float2* red) {
  v.x = softmax::warp_sum(v.x);
  v.y = softmax::warp_max(v.y);
  if (LANES == 32) return v;
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int w = 1; w < LANES / 32; ++w) v.x += red[w].x, v.y = fmaxf(v.y, red[w].y);
  return v;
}
// Every buffer and row on 16-byte boundaries (y in 8 bits: on as many bytes as a vector has elements); VPT vectors a thread.
template <typename T, bool kI8, int LANES, int VPT>
__global__ void __launch_bounds__(kThreads)
add_rms_norm_vec_kernel(const Params<T> p) {
  constexpr int PV = Elem<T>::kPerVec;
  __shared__ float2 red[kThreads / 32];
  ptx::launch_dependents_if_few();
  ptx::wait_prior_grid();
  const int lane = threadIdx.x % LANES;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / LANES) + threadIdx.x / LANES;
  if (row >= p.rows) return;  // rows of a CTA are all there, or each has a warp
  const int nvec = p.cols / PV;
  const Vec16* x = reinterpret_cast<const Vec16*>(p.x + row * p.cols);
  const Vec16* residual = reinterpret_cast<const Vec16*>(p.residual + (p.residual ? row * p.cols : 0));
  const Vec16* weight = reinterpret_cast<const Vec16*>(p.weight);
  Vec16 a[VPT], b[VPT];
#pragma unroll
  for (int k = 0; k < VPT; ++k)
    if (k * LANES + lane < nvec) a[k] = softmax::ld_stream(x + k * LANES + lane);
  if (p.residual) {
#pragma unroll
    for (int k = 0; k < VPT; ++k)
      if (k * LANES + lane < nvec) b[k] = softmax::ld_stream(residual + k * LANES + lane);
  }
  float h[VPT][PV];
  float2 acc = make_float2(0.f, 0.f);
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    const int i = k * LANES + lane;
    if (i >= nvec) continue;
    Elem<T>::unpack(a[k], h[k]);
    if (p.residual) {
      float r[PV];
      Elem<T>::unpack(b[k], r);
#pragma unroll
      for (int e = 0; e < PV; ++e) h[k][e] += r[e];
    }
    if (p.sum) softmax::st_stream(reinterpret_cast<Vec16*>(p.sum + row * p.cols) + i, Elem<T>::pack(h[k]));
#pragma unroll
    for (int e = 0; e < PV; ++e) acc.x = fmaf(h[k][e], h[k][e], acc.x);
    if (p.weight) {
      float w[PV];
      Elem<T>::unpack(softmax::ld_keep(weight + i), w);
#pragma unroll
      for (int e = 0; e < PV; ++e) h[k][e] *= w[e];
    }
    if (kI8) {
#pragma unroll
      for (int e = 0; e < PV; ++e) acc.y = fmaxf(acc.y, fabsf(h[k][e]));
    }
  }
  acc = row_sum_max<LANES>(acc, red);
  const float r = rsqrtf(acc.x / p.cols + p.eps);
  const quant::Step step = kI8 ? quant::step_of(acc.y) : quant::Step{};
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    const int i = k * LANES + lane;
    if (i >= nvec) continue;
    if constexpr (kI8) {
      uint32_t q[PV / 4];
#pragma unroll
      for (int j = 0; j < PV / 4; ++j) q[j] = quant::quantise4(h[k] + 4 * j, step);
      uint8_t* to = static_cast<uint8_t*>(p.y) + row * p.cols + static_cast<int64_t>(i) * PV;
      if constexpr (PV == 8) *reinterpret_cast<uint2*>(to) = make_uint2(q[0], q[PV / 4 - 1]);
      else *reinterpret_cast<uint32_t*>(to) = q[0];
    } else {
#pragma unroll
      for (int e = 0; e < PV; ++e) h[k][e] *= r;
      softmax::st_stream(reinterpret_cast<Vec16*>(static_cast<T*>(p.y) + row * p.cols) + i, Elem<T>::pack(h[k]));
    }
  }
  if (kI8 && lane == 0) p.scales[row] = step.step * r;
}

// Rows that start anywhere.  EPT > 0: that many elements a thread in registers; 0: any width, read twice (sum is written on the second way, so that it may be x or
// residual).
template <typename T, bool kI8, int EPT>
__global__ void __launch_bounds__(kThreads)
add_rms_norm_any_kernel(const Params<T> p) {
  __shared__ float2 red[kThreads / 32];
  ptx::launch_dependents_if_few();
  ptx::wait_prior_grid();
  const int64_t at = static_cast<int64_t>(blockIdx.x) * p.cols;
  auto h_of = [&](int c) { return Elem<T>::load1(p.x + at + c) + (p.residual ? Elem<T>::load1(p.residual + at + c) : 0.f); };
  auto w_of = [&](int c) { return p.weight ? Elem<T>::load1(p.weight + c) : 1.f; };
  float2 acc = make_float2(0.f, 0.f);
  float h[EPT > 0 ? EPT : 1];
  if constexpr (EPT > 0) {
#pragma unroll
    for (int k = 0; k < EPT; ++k) {
      const int c = k * kThreads + threadIdx.x;
      h[k] = c < p.cols ? Elem<T>::load1(p.x + at + c) : 0.f;
    }
    if (p.residual) {
      float b[EPT];
#pragma unroll
      for (int k = 0; k < EPT; ++k) {
        const int c = k * kThreads + threadIdx.x;
        b[k] = c < p.cols ? Elem<T>::load1(p.residual + at + c) : 0.f;
      }
#pragma unroll
      for (int k = 0; k < EPT; ++k) h[k] += b[k];
    }
#pragma unroll
    for (int k = 0; k < EPT; ++k) {
      const int c = k * kThreads + threadIdx.x;
      if (c >= p.cols) continue;
      acc.x = fmaf(h[k], h[k], acc.x);
      if (p.sum) Elem<T>::store1(p.sum + at + c, h[k]);
      if (p.weight) h[k] *= w_of(c);
      if (kI8) acc.y = fmaxf(acc.y, fabsf(h[k]));
    }
  } else {
    for (int c = threadIdx.x; c < p.cols; c += kThreads) {
      const float v = h_of(c);
      acc.x = fmaf(v, v, acc.x);
      if (kI8) acc.y = fmaxf(acc.y, fabsf(v * w_of(c)));
    }
  }
  acc = row_sum_max<kThreads>(acc, red);
  const float r = rsqrtf(acc.x / p.cols + p.eps);
  const quant::Step step = kI8 ? quant::step_of(acc.y) : quant::Step{};
  auto put = [&](int c, float z) {
    if (kI8) static_cast<int8_t*>(p.y)[at + c] = static_cast<int8_t>(step.step > 0.f ? __float2int_rn(z / step.step) : 0);
    else Elem<T>::store1(static_cast<T*>(p.y) + at + c, z * r);
  };
  if constexpr (EPT > 0) {
#pragma unroll
    for (int k = 0; k < EPT; ++k) {
      const int c = k * kThreads + threadIdx.x;
      if (c < p.cols) put(c, h[k]);
    }
  } else {
    for (int c = threadIdx.x; c < p.cols; c += kThreads) {
      const float v = h_of(c), z = v * w_of(c);
      if (p.sum) Elem<T>::store1(p.sum + at + c, v);
      put(c, z);
    }
  }
  if (kI8 && threadIdx.x == 0) p.scales[blockIdx.x] = step.step * r;
}

}  // namespace addnorm
}  // namespace tsm100
