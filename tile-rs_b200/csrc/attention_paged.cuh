// Attention of new tokens over the pages of their sequences: a token at position p sees positions 0 .. p.
#pragma once

#include "kv_pages.cuh"
#include "ptx.cuh"

namespace tsm100 {
namespace paged {

struct Params {
  pages::Cache cache;
  pages::Batch step;
  int32_t heads_q;
  float scale_log2;  // log2(e) / sqrt(d)
  uint32_t* status;
};

// A warp per (token, head), a position at a time.
template <typename T, bool kI8, int D>
__global__ void __launch_bounds__(256)
attention_paged_kernel(const T* __restrict__ q, T* __restrict__ o, const Params p) {
  constexpr int N = D / 32;
  using H = typename std::conditional<kI8, int8_t, T>::type;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (i >= static_cast<int64_t>(p.step.tokens) * p.heads_q) return;
  const int head = static_cast<int>(i % p.heads_q), token = static_cast<int>(i / p.heads_q), g = head / (p.heads_q / p.cache.heads);
  const int b = pages::sequence_of(p.step, token);
  int first, count, len;
  if (b < 0 || !pages::sequence(p.step, p.cache.page_size, b, first, count, len, p.status, 3)) return;
  const int last = len - count + token - first;
  float qv[N], acc[N] = {}, m = -INFINITY, l = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j) qv[j] = softmax::Elem<T>::load1(q + i * D + j * 32 + lane) * p.scale_log2;
  for (int pos = 0; pos <= last; ++pos) {
    const int page = pages::page_of(p.cache, p.step, b, pos, p.status, 4);
    if (page < 0) return;
    const int64_t row = (static_cast<int64_t>(page) * p.cache.heads + g) * p.cache.page_size + pos % p.cache.page_size;
    const H* k = static_cast<const H*>(p.cache.kv[0]) + row * D;
    const H* v = static_cast<const H*>(p.cache.kv[1]) + row * D;
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) s = fmaf(qv[j], static_cast<float>(k[j * 32 + lane]), s);
    s = softmax::warp_sum(s);
    if (kI8) s *= p.cache.scales[0][row];
    const float n = fmaxf(m, s), a = ptx::ex2_approx(m - n), w = ptx::ex2_approx(s - n);
    l = fmaf(l, a, w);
    m = n;
    const float wv = kI8 ? w * p.cache.scales[1][row] : w;
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = fmaf(acc[j], a, wv * static_cast<float>(v[j * 32 + lane]));
  }
#pragma unroll
  for (int j = 0; j < N; ++j) softmax::Elem<T>::store1(o + i * D + j * 32 + lane, acc[j] / l);
}

}  // namespace paged
}  // namespace tsm100
