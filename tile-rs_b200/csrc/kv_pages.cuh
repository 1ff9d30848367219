// A KV cache in pages: where the tokens of a call lie, writing them (quantised on the way if the cache holds 8 bits) and reading them back.
//
// k, v: [pages][heads][page_size][d]; in 8 bits a row is whole numbers -127 .. 127 and an f32 step, max|x| / 127.
#pragma once

#include <type_traits>

#include "ptx.cuh"
#include "quantise.cuh"
#include "softmax.cuh"

namespace tsm100 {
namespace pages {

constexpr uint32_t kStatusOutside = 0x2000u;  // | site: a page, a position or a sequence outside what the call described

struct Cache {
  int32_t heads, d, page_size;
  int64_t pages;
  void* kv[2];      // k, v
  float* scales[2];
};
struct Batch {
  int32_t batch, tokens, max_new, pitch;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* starts;
};

__device__ __forceinline__ void report(uint32_t* status, uint32_t site) {
  if (status) atomicCAS(status, 0u, kStatusOutside | site);
}

// The tokens and positions of sequence b; false, and reported, if they contradict each other or the call.
__device__ __forceinline__ bool sequence(const Batch& s, int64_t page_size, int b, int& first, int& count, int& len, uint32_t* status, uint32_t site) {
  first = s.starts[b];
  count = s.starts[b + 1] - first;
  len = s.lens[b];
  if (count == 0) return false;
  if (first < 0 || count < 0 || count > s.max_new || first > s.tokens - count || len < count || len > page_size * s.pitch) {
    report(status, site);
    return false;
  }
  return true;
}
// The page that holds a position of sequence b, or -1 (reported).
__device__ __forceinline__ int page_of(const Cache& c, const Batch& s, int b, int pos, uint32_t* status, uint32_t site) {
  const int page = s.table[static_cast<int64_t>(b) * s.pitch + pos / c.page_size];
  if (page >= 0 && page < c.pages) return page;
  report(status, site);
  return -1;
}
// The sequence that has a token: the last one that starts at it or before, and so not an empty one.  -1: none.
__device__ __forceinline__ int sequence_of(const Batch& s, int token) {
  int lo = 0, hi = s.batch;
  while (lo < hi) {  // the first sequence that starts behind the token
    const int mid = (lo + hi) >> 1;
    if (s.starts[mid] > token) hi = mid;
    else lo = mid + 1;
  }
  return lo > 0 && token < s.starts[lo] ? lo - 1 : -1;
}

// A CTA has `per_cta` tokens.  Where those lie is found first, a token to a thread; then LANES threads have a row of a token (k or v, head), eight numbers each
// (LANES times 8 is d or the next power of two), and kPasses rows in turn, all of whose loads are on their way before the first is used.
// Bound: HBM.
constexpr int kThreads = 256, kPasses = 4, kMaxTokens = 32;

template <typename T, bool kI8, bool kRead, int LANES>
__global__ void __launch_bounds__(kThreads)
kv_page_rows_kernel(const Cache c, const Batch s, T* k, T* v, int32_t per_cta, uint32_t* status) {
  constexpr int kRows = kThreads / LANES;  // of a pass
  using softmax::Elem;
  using softmax::Vec16;
  __shared__ int64_t place[kMaxTokens];    // of a token in its page's first head, in rows of the cache; -1: it has none
  ptx::launch_dependents_if_few();
  ptx::wait_prior_grid();
  const int token0 = static_cast<int>(blockIdx.x) * per_cta;
  if (static_cast<int>(threadIdx.x) < per_cta) {
    const int token = token0 + threadIdx.x;
    int64_t at = -1;
    const int b = token < s.tokens ? sequence_of(s, token) : -1;
    int first, count, len;
    if (b >= 0 && sequence(s, c.page_size, b, first, count, len, status, 141)) {
      const int pos = len - count + token - first, page = page_of(c, s, b, pos, status, 142);
      if (page >= 0) at = static_cast<int64_t>(page) * c.heads * c.page_size + pos % c.page_size;
    }
    place[threadIdx.x] = at;
  }
  __syncthreads();
  const int lane = threadIdx.x % LANES, e = lane * 8, per_token = 2 * c.heads;
  const bool inside = e < c.d;
  int row = threadIdx.x / LANES, token = row / per_token;  // of the CTA's
  row -= token * per_token;
  const int rounds = (per_cta * per_token + kRows * kPasses - 1) / (kRows * kPasses);
  for (int round = 0; round < rounds; ++round) {
    T* mine[kPasses];
    int64_t at[kPasses];  // -1: none
    bool second[kPasses];
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      at[i] = token < per_cta ? place[token] : -1;
      second[i] = row >= c.heads;
      const int head = second[i] ? row - c.heads : row;
      if (at[i] >= 0) at[i] += static_cast<int64_t>(head) * c.page_size;
      mine[i] = (second[i] ? v : k) + (static_cast<int64_t>(token0 + token) * c.heads + head) * c.d + e;
      row += kRows;
      while (row >= per_token) row -= per_token, ++token;
    }
    auto held = [&](int i) { return static_cast<uint8_t*>(second[i] ? c.kv[1] : c.kv[0]) + (at[i] * c.d + e) * (kI8 ? 1 : 2); };
    auto step_at = [&](int i) { return (second[i] ? c.scales[1] : c.scales[0]) + at[i]; };
    if constexpr (!kI8) {
      Vec16 x[kPasses];
#pragma unroll
      for (int i = 0; i < kPasses; ++i)
        if (at[i] >= 0 && inside) x[i] = softmax::ld_stream(kRead ? reinterpret_cast<const Vec16*>(held(i)) : reinterpret_cast<const Vec16*>(mine[i]));
#pragma unroll
      for (int i = 0; i < kPasses; ++i)
        if (at[i] >= 0 && inside) *(kRead ? reinterpret_cast<Vec16*>(mine[i]) : reinterpret_cast<Vec16*>(held(i))) = x[i];
    } else if constexpr (kRead) {
      uint2 x[kPasses];
      float step[kPasses];
#pragma unroll
      for (int i = 0; i < kPasses; ++i)
        if (at[i] >= 0 && inside) x[i] = __ldcs(reinterpret_cast<const uint2*>(held(i))), step[i] = *step_at(i);
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        if (at[i] < 0 || !inside) continue;
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = quant::number(j < 4 ? x[i].x : x[i].y, j & 3) * step[i];
        softmax::st_stream(reinterpret_cast<Vec16*>(mine[i]), Elem<T>::pack(f));
      }
    } else {
      Vec16 x[kPasses];
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        x[i] = Vec16{};
        if (at[i] >= 0 && inside) x[i] = softmax::ld_stream(reinterpret_cast<const Vec16*>(mine[i]));
      }
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        float f[8], top = 0.f;
        Elem<T>::unpack(x[i], f);
#pragma unroll
        for (int j = 0; j < 8; ++j) top = ptx::fmax_nan(top, fabsf(f[j]));
#pragma unroll
        for (int off = LANES / 2; off > 0; off >>= 1) top = ptx::fmax_nan(top, __shfl_xor_sync(0xffffffffu, top, off));
        if (at[i] < 0 || !inside) continue;
        const quant::Step step = quant::step_of(top);
        *reinterpret_cast<uint2*>(held(i)) = make_uint2(quant::quantise4(f, step), quant::quantise4(f + 4, step));
        if (lane == 0) *step_at(i) = step.step;
      }
    }
  }
}

}  // namespace pages
}  // namespace tsm100
