// 4-bit weights as 16-bit ones, for products with so many rows of A that making the weights once and multiplying them as a 16-bit matrix takes
// less time than making them for every 128 or 256 rows (gemm_w4.cuh): each weight times its scale, rounded once, as there.  A C with rows off 16-byte
// boundaries is copied from one with rows on them.  And rows of A in 8 bits as 16-bit numbers, exactly.
// Bound: memory, writing the weights (16 bytes a thread and access); the product after it is bound as the 16-bit one.
#pragma once

#include "gemm_w4.cuh"

namespace tsm100 {
namespace w4 {

constexpr int kDenseThreads = 256;

// A CTA per row of W; rows beyond the n of W, up to the grid's, are zeros.
template <typename T>
__global__ void __launch_bounds__(kDenseThreads)
w4_expand_kernel(const uint8_t* __restrict__ w, const uint16_t* __restrict__ scales, const uint8_t* __restrict__ zeros, uint16_t* __restrict__ out, int32_t n, int32_t k,
                 int32_t group_log2) {
  constexpr bool kBf16 = !std::is_same<T, __half>::value;
  ptx::launch_dependents_if_few();
  w = ptx::wait_prior_grid(w);
  scales = ptx::wait_prior_grid(scales);
  if (zeros) zeros = ptx::wait_prior_grid(zeros);
  const int64_t row = blockIdx.x;
  const int words = k / 8, groups = k >> group_log2;
  if (row >= n) {
    for (int i = threadIdx.x; i < words; i += kDenseThreads) reinterpret_cast<uint4*>(out + row * k)[i] = make_uint4(0, 0, 0, 0);
    return;
  }
  const uint32_t* from = reinterpret_cast<const uint32_t*>(w + row * (k / 2));
  uint4* to = reinterpret_cast<uint4*>(out + row * k);
#pragma unroll 4
  for (int i = threadIdx.x; i < words; i += kDenseThreads) {
    const uint32_t x = __ldcs(from + i);
    const int64_t g = row * groups + ((8 * i) >> group_log2);
    const uint32_t zero = (zeros ? zeros[g] : 8u) * 0x10001u + kMagic<kBf16>, scale = scales[g] * 0x10001u;
    const uint32_t even = x & 0x0f0f0f0fu, odd = (x >> 4) & 0x0f0f0f0fu;  // bytes
    uint32_t y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t pair = (__byte_perm(even, odd, j | (4 + j) << 8) & 0x00ff00ffu) | kMagic<kBf16>;
      y[j] = mul2<kBf16>(sub2<kBf16>(pair, zero), scale);
    }
    to[i] = make_uint4(y[0], y[1], y[2], y[3]);
  }
}
// 8-bit numbers as 16-bit ones, eight a thread.
template <typename T>
__global__ void __launch_bounds__(kDenseThreads)
w4_widen_kernel(const uint2* __restrict__ a, uint4* __restrict__ out, int64_t vecs) {
  ptx::launch_dependents_if_few();
  a = ptx::wait_prior_grid(a);
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kDenseThreads + threadIdx.x;
  if (i >= vecs) return;
  const uint2 x = a[i];
  auto two = [&](uint32_t v, int lo) {  // bytes lo and lo + 1
    return i8_to_16<T>(v >> (8 * lo), v >> (8 * lo + 8), 0);
  };
  out[i] = make_uint4(two(x.x, 0), two(x.x, 2), two(x.y, 0), two(x.y, 2));
}
// Rows of `pitch` elements, a multiple of eight, to rows of n: four elements a thread and access.
template <typename T>
__global__ void __launch_bounds__(kDenseThreads)
w4_rows_kernel(const T* __restrict__ from, T* __restrict__ c, int32_t n, int32_t pitch) {
  ptx::launch_dependents_if_few();
  from = ptx::wait_prior_grid(from);
  from += static_cast<int64_t>(blockIdx.x) * pitch;
  c += static_cast<int64_t>(blockIdx.x) * n;
  const bool vectors = reinterpret_cast<uintptr_t>(c) % 8 == 0;
  for (int i = 4 * (blockIdx.y * kDenseThreads + threadIdx.x); i < n; i += 4 * gridDim.y * kDenseThreads) {
    alignas(8) T y[4];
    *reinterpret_cast<uint2*>(y) = *reinterpret_cast<const uint2*>(from + i);
    if (vectors && i + 4 <= n) {
      *reinterpret_cast<uint2*>(c + i) = *reinterpret_cast<const uint2*>(y);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i + j < n) c[i + j] = y[j];
    }
  }
}

}  // namespace w4
}  // namespace tsm100
