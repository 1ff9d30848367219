// A KV cache in pages: where the tokens of a call lie, writing them (quantised on the way if the cache holds 8 bits) and reading them back.
//
// k, v: [pages][heads][page_size][d]; in 8 bits a row is whole numbers -127 .. 127 and an f32 step, max|x| / 127.
#pragma once

#include <type_traits>

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

// A warp per row of a token: (token, k or v, head).
template <typename T, bool kI8, bool kRead>
__global__ void __launch_bounds__(256)
kv_page_rows_kernel(const Cache c, const Batch s, T* k, T* v, uint32_t* status) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (i >= static_cast<int64_t>(s.tokens) * 2 * c.heads) return;
  const int head = static_cast<int>(i % c.heads), which = static_cast<int>(i / c.heads & 1), token = static_cast<int>(i / c.heads / 2);
  const int b = sequence_of(s, token);
  int first, count, len;
  if (b < 0 || !sequence(s, c.page_size, b, first, count, len, status, 1)) return;
  const int pos = len - count + token - first;
  const int page = page_of(c, s, b, pos, status, 2);
  if (page < 0) return;
  T* mine = (which ? v : k) + (static_cast<int64_t>(token) * c.heads + head) * c.d;
  const int64_t row = (static_cast<int64_t>(page) * c.heads + head) * c.page_size + pos % c.page_size;
  if constexpr (!kI8) {
    T* held = static_cast<T*>(c.kv[which]) + row * c.d;
    for (int j = lane; j < c.d; j += 32) (kRead ? mine : held)[j] = (kRead ? held : mine)[j];
  } else {
    int8_t* held = static_cast<int8_t*>(c.kv[which]) + row * c.d;
    if constexpr (kRead) {
      const float step = c.scales[which][row];
      for (int j = lane; j < c.d; j += 32) softmax::Elem<T>::store1(mine + j, held[j] * step);
    } else {
      float top = 0.f;
      for (int j = lane; j < c.d; j += 32) top = fmaxf(top, fabsf(softmax::Elem<T>::load1(mine + j)));
      const float step = softmax::warp_max(top) * static_cast<float>(1.0 / 127.0);
      for (int j = lane; j < c.d; j += 32) held[j] = static_cast<int8_t>(step > 0.f ? __float2int_rn(softmax::Elem<T>::load1(mine + j) / step) : 0);
      if (lane == 0) c.scales[which][row] = step;
    }
  }
}

}  // namespace pages
}  // namespace tsm100
