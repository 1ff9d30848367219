// Rows as 8-bit whole numbers and a step for each: v = x, or silu(x) * up with silu(x) = x / (1 + exp(-x)), in f32; step = max|v| / 127, q = v / step
// rounded to nearest even (quantise.cuh).  A row that is not finite has a step of NaN.
//
// Bound: HBM.  A row is read once and held in registers as f32, by a warp or a CTA that takes a row and goes.  Rows that start anywhere are held the
// same way, an element at a time; wider ones are read twice, the second time from the caches.
#pragma once

#include "ptx.cuh"
#include "quantise.cuh"
#include "softmax.cuh"

namespace tsm100 {
namespace rows_i8 {

using softmax::Elem;
using softmax::Vec16;

template <typename T>
struct Params {
  const T* x;
  const T* up;        // or null
  int8_t* y;          // [rows][cols]
  float* scales;      // [rows]
  int64_t rows, pitch;
  int32_t cols;
};

// |v| of which is the larger, NaN above all: as bits.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// The largest magnitude over a row's threads (a warp or the CTA); each gets it.
template <bool kWarp>
__device__ __forceinline__ float row_max(uint32_t top, uint32_t* red) {
  top = __reduce_max_sync(0xffffffffu, top);
  if (kWarp) return __uint_as_float(top);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
  __syncthreads();
  top = (threadIdx.x & 31) < (blockDim.x >> 5) ? red[threadIdx.x & 31] : 0u;
  return __uint_as_float(__reduce_max_sync(0xffffffffu, top));
}
// silu(x) * up, off by 2^-20 of itself and for a negative x another |x| 2^-23.6 of itself at most: x * log2(e) is rounded to f32 (|x| 1.25 2^-24 of the exponential, with the constant), the
// exponential and the reciprocal are the approximate ones, 2^-22 and 2^-23 off, because exact ones are twenty more instructions and 8192 rows of 14336 bf16 took 170 us with them,
// 114 so (5.1 TB/s).  rcp.approx makes 0 of results below 2^-126, which 1 / (1 + exp(-x)) is from x = -87.3 down while exp(-x) is finite (-88.7): so it is
// taken of 2^-32 (1 + exp(-x)), and 2^-32 times that still has 21 bits there.  Further down the exponential overflows and the value is 0, as the formula's is in f32.
__device__ __forceinline__ float gated(float x, float up) {
  const float e = ptx::ex2_approx(x * -1.4426950408889634f);
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fmaf(e, 0x1p-32f, 0x1p-32f)));
  return x * (r * 0x1p-32f) * up;
}

// Every row on 16-byte boundaries (y: on as many bytes as a vector has elements); VPT vectors a thread, a warp a row (kWarp) or a CTA of as many warps as the row fills.
constexpr int kMaxThreads = 1024;
template <typename T, bool kGated, bool kWarp, int VPT>
__global__ void __launch_bounds__(kWarp ? 256 : kMaxThreads)
rows_i8_vec_kernel(const Params<T> p) {
  constexpr int PV = Elem<T>::kPerVec;
  __shared__ uint32_t red[32];
  ptx::launch_dependents_if_few();
  ptx::wait_prior_grid();
  const int lanes = kWarp ? 32 : blockDim.x, lane = kWarp ? threadIdx.x & 31 : threadIdx.x;
  const int64_t row = kWarp ? static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5) : blockIdx.x;
  if (row >= p.rows) return;  // a warp's
  const int nvec = p.cols / PV;
  const Vec16* x = reinterpret_cast<const Vec16*>(p.x + row * p.pitch);
  const Vec16* up = reinterpret_cast<const Vec16*>(p.up + (kGated ? row * p.pitch : 0));
  Vec16 a[VPT], b[kGated ? VPT : 1];
#pragma unroll
  for (int k = 0; k < VPT; ++k)
    if (k * lanes + lane < nvec) a[k] = softmax::ld_stream(x + k * lanes + lane);
  if constexpr (kGated) {
#pragma unroll
    for (int k = 0; k < VPT; ++k)
      if (k * lanes + lane < nvec) b[k] = softmax::ld_stream(up + k * lanes + lane);
  }
  float v[VPT][PV];
  uint32_t top = 0u;
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    if (k * lanes + lane >= nvec) continue;
    Elem<T>::unpack(a[k], v[k]);
    if constexpr (kGated) {
      float u[PV];
      Elem<T>::unpack(b[k], u);
#pragma unroll
      for (int e = 0; e < PV; ++e) v[k][e] = gated(v[k][e], u[e]);
    }
#pragma unroll
    for (int e = 0; e < PV; ++e) top = max(top, magnitude(v[k][e]));
  }
  const quant::Step step = quant::step_of(row_max<kWarp>(top, red));
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    const int i = k * lanes + lane;
    if (i >= nvec) continue;
    uint32_t q[PV / 4];
#pragma unroll
    for (int j = 0; j < PV / 4; ++j) q[j] = quant::quantise4(v[k] + 4 * j, step);
    int8_t* to = p.y + row * p.cols + static_cast<int64_t>(i) * PV;
    if constexpr (PV == 8) *reinterpret_cast<uint2*>(to) = make_uint2(q[0], q[PV / 4 - 1]);
    else *reinterpret_cast<uint32_t*>(to) = q[0];
  }
  if (lane == 0) p.scales[row] = step.step;
}

// Rows that start anywhere.  EPT > 0: that many elements a thread in registers; 0: any width, read twice.
constexpr int kThreads = 256;
template <typename T, bool kGated, int EPT>
__global__ void __launch_bounds__(kThreads)
rows_i8_any_kernel(const Params<T> p) {
  __shared__ uint32_t red[32];
  ptx::launch_dependents_if_few();
  ptx::wait_prior_grid();
  const int64_t from = static_cast<int64_t>(blockIdx.x) * p.pitch, to = static_cast<int64_t>(blockIdx.x) * p.cols;
  auto value = [&](int c) {
    const float x = Elem<T>::load1(p.x + from + c);
    return kGated ? gated(x, Elem<T>::load1(p.up + from + c)) : x;
  };
  uint32_t top = 0u;
  float v[EPT > 0 ? EPT : 1];
  if constexpr (EPT > 0) {
#pragma unroll
    for (int k = 0; k < EPT; ++k) {
      const int c = k * kThreads + threadIdx.x;
      v[k] = c < p.cols ? value(c) : 0.f;
    }
#pragma unroll
    for (int k = 0; k < EPT; ++k) top = max(top, magnitude(v[k]));
  } else {
    for (int c = threadIdx.x; c < p.cols; c += kThreads) top = max(top, magnitude(value(c)));
  }
  const quant::Step step = quant::step_of(row_max<false>(top, red));
  auto put = [&](int c, float x) { p.y[to + c] = static_cast<int8_t>(step.step > 0.f ? __float2int_rn(x / step.step) : 0); };
  if constexpr (EPT > 0) {
#pragma unroll
    for (int k = 0; k < EPT; ++k) {
      const int c = k * kThreads + threadIdx.x;
      if (c < p.cols) put(c, v[k]);
    }
  } else {
    for (int c = threadIdx.x; c < p.cols; c += kThreads) put(c, value(c));
  }
  if (threadIdx.x == 0) p.scales[blockIdx.x] = step.step;
}

}  // namespace rows_i8
}  // namespace tsm100
