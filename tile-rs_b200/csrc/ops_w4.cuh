// Host-side launch logic of products with 4-bit weights (gemm_w4.cuh); as ops_serving.cuh.
#pragma once

#include <algorithm>

#include "gemm_w4.cuh"
#include "launch.cuh"
#include "w4_dense.cuh"

namespace tsm100 {
namespace ops {

// CTAs of a cluster along K: until the GPU has its `places`, each with two steps of K or more.
inline int gemm_w4_splits(int64_t n, int64_t k, int64_t token_blocks, int64_t places) {
  const int64_t steps = (k + w4::kStepK - 1) / w4::kStepK, tiles = (n + w4::kRows - 1) / w4::kRows * token_blocks;
  int splits = 1;
  while (splits < 8 && tiles * splits * 2 <= places && steps / (2 * splits) >= 2) splits *= 2;
  return splits;
}

template <typename T, int N, int GC, bool kScaled = false>
inline int32_t gemm_w4_launch(std::string* err, const CUtensorMap& map, w4::Params p, int sms, cudaStream_t s) {
  using S = w4::Shape<N, GC, kScaled>;
  const int blocks = (p.m + N - 1) / N;
  p.tokens = ((p.m + blocks - 1) / blocks + 15) / 16 * 16;
  p.splits = gemm_w4_splits(p.n, p.k, blocks, S::kTwo ? 2ll * sms : sms);
  CUtensorMap map_a{};
  if (kScaled) {
    const int32_t st = make_tmap_16bit_3d(err, &map_a, p.a, p.k, p.m, 1, p.k, static_cast<uint64_t>(p.m) * p.k, 64, static_cast<uint32_t>(p.tokens),
                                          std::is_same<T, __nv_bfloat16>::value);
    if (st != TSM100_OK) return st;
  }
  auto kern = w4::gemm_w4_kernel<T, N, GC, kScaled, false>;
  if constexpr (!kScaled)
    if (p.a_scales) kern = w4::gemm_w4_kernel<T, N, GC, kScaled, true>;
  cudaError_t e = set_dyn_smem_once(kern, S::kSmem);
  const dim3 grid(static_cast<unsigned>((p.n + w4::kRows - 1) / w4::kRows * p.splits), static_cast<unsigned>((p.m + p.tokens - 1) / p.tokens));
  if (e == cudaSuccess) e = launch_chained(kern, grid, w4::kThreads, S::kSmem, s, p.splits > 1 ? p.splits : 0, map, map_a, p);
  return cuda_ok(err, e, "gemm_w4_kernel launch");
}
template <typename T, int GC>
inline int32_t gemm_w4_grouped(std::string* err, const CUtensorMap& map, const w4::Params& p, int sms, cudaStream_t s) {
  if (p.m <= 16) return gemm_w4_launch<T, 16, GC>(err, map, p, sms, s);
  // Tiles of 256 rows make half the weights but have more to a CTA: where those of 128 are more than a wave.  bf16, us with 128, 256: 200 x 16384 x 4096 44, 30;
  // 400 x 8192 x 4096 43, 29; 400 x 4096 x 4096 (128 tiles of 128) 22, 28; 200 x 8192 x 4096 (128) 22, 28.  Left out: fewer tiles whose K
  // is split, 200 x 4096 x 16384 (64, in two) 39, 32.
  const int64_t tiles = static_cast<int64_t>((p.m + 127) / 128) * ((p.n + w4::kRows - 1) / w4::kRows);
  if (p.m > 128 && tiles > sms) return gemm_w4_launch<T, 256, GC, true>(err, map, p, sms, s);
  if (p.m > w4::kExactTokens) return gemm_w4_launch<T, 128, GC, true>(err, map, p, sms, s);
  if constexpr (GC <= 2)
    if (p.m > 32) return gemm_w4_launch<T, 64, GC>(err, map, p, sms, s);
  return gemm_w4_launch<T, 32, GC>(err, map, p, sms, s);
}
template <typename T>
int32_t gemm_w4_typed(std::string* err, const tsm100_gemm_w4_desc* d, const uint8_t* w, const w4::Params& p, cudaStream_t s) {
  int sms = 0;
  int32_t st = sm_count(err, &sms);
  if (st != TSM100_OK) return st;
  if (d->k == 0) return cuda_ok(err, cudaMemsetAsync(p.c, 0, static_cast<size_t>(d->m) * d->n * sizeof(T), s), "cudaMemsetAsync");
  CUtensorMap map;
  st = make_tmap_3d(err, &map, w, d->k / 2, d->n, 1, d->k / 2, static_cast<uint64_t>(d->n) * (d->k / 2), w4::kStepK / 2, w4::kRows,
                    CU_TENSOR_MAP_DATA_TYPE_UINT8, 1);
  if (st != TSM100_OK) return st;
  switch (d->group) {
    case 32: return gemm_w4_grouped<T, 4>(err, map, p, sms, s);
    case 64: return gemm_w4_grouped<T, 2>(err, map, p, sms, s);
    default: return gemm_w4_grouped<T, 1>(err, map, p, sms, s);
  }
}
// one translation unit each: serving_w4_bf16.cu, serving_w4_f16.cu
extern template int32_t gemm_w4_typed<__nv_bfloat16>(std::string*, const tsm100_gemm_w4_desc*, const uint8_t*, const w4::Params&, cudaStream_t);
extern template int32_t gemm_w4_typed<__half>(std::string*, const tsm100_gemm_w4_desc*, const uint8_t*, const w4::Params&, cudaStream_t);

// Whether the weights are made 16-bit ones first.  The kernel of gemm_w4.cuh makes each of them for every 128 or 256 rows; made once they are written
// and read again, by a launch more.  bf16, us with the weights made in the kernel, made first:
//   N = K = 4096, 640 rows: 30, 35     1000: 32, 37     1500: 61, 55     3000: 97, 81         N = 16384, K = 4096: 94, 106     130, 132     193, 187     353, 313
//   N = 16384, K = 512: 34, 28     48, 32     71, 44     130, 79                              N = 1024, K = 4096: 15, 20     15, 24     23, 31     32, 42
//   N = 672, K = 864, 3000 rows: 10, 15
// The rule is one bound for all, and not the better of both everywhere.  1024 rows in the kernel and 1025 made first: N = 2048, K = 2048 15, 19,
// K = 4096 22, 30; 3000 x 2048 21, 21; 4096 x 4096 31, 54 (1025 rows are a second wave of tiles in the kernel too); 5003 x 2048 56, 38; 8192 x 512 23, 20; 16384 x 512 47, 32;
// 16384 x 4096 130, 154.  So short K and N off vectors would gain from fewer rows on, and N of 2048 from more.
// Rows that came in 8 bits have the steps to multiply besides, in another pass over an f32 result: 3000 x 16384 x 4096 took 416 so, 95 more than with 16 bits,
// and 410 in the kernel.  (With K = 512 the kernel takes 165, three times the 16-bit form.)
inline bool gemm_w4_dense_pays(const tsm100_gemm_w4_desc* d) { return d->a_dtype == d->dtype && d->m > 1024 && d->n >= 2048 && d->k >= 512; }

// `gemm` is the library's own 16-bit product, (desc, a, b, c) on this stream.  kNoScratch: no memory for the weights.
template <typename T, typename Gemm>
inline int32_t gemm_w4_dense(std::string* err, const tsm100_gemm_w4_desc* d, const uint8_t* w, const w4::Params& p, cudaStream_t s, Gemm gemm) {
  const int64_t n8 = (d->n + 7) / 8 * 8;  // rows of C, and of W's last tiles, as the tensor cores' product takes them
  const bool apart = n8 != d->n || !aligned16(p.c);
  const size_t w_bytes = (static_cast<size_t>(n8) * d->k * 2 + 255) / 256 * 256, c_bytes = apart ? static_cast<size_t>(d->m) * n8 * 2 : 0;
  uint8_t* ws = nullptr;
  int32_t st = take_scratch(err, reinterpret_cast<void**>(&ws), w_bytes + c_bytes, s);
  if (st != TSM100_OK) return st;
  T* rows = reinterpret_cast<T*>(ws + w_bytes);
  const int group_log2 = d->group == 32 ? 5 : d->group == 64 ? 6 : 7;
  cudaError_t e = launch_chained(w4::w4_expand_kernel<T>, static_cast<unsigned>(n8), w4::kDenseThreads, 0, s, 0, w, static_cast<const uint16_t*>(p.scales),
                                 p.zeros, reinterpret_cast<uint16_t*>(ws), p.n, p.k, static_cast<int32_t>(group_log2));
  st = cuda_ok(err, e, "w4_expand_kernel launch");
  if (st == TSM100_OK) {
    tsm100_gemm_desc g = {};
    g.dtype = d->dtype, g.out_dtype = d->dtype;
    g.b_transposed = 1, g.batch = 1;
    g.m = d->m, g.n = n8, g.k = d->k;
    st = gemm(&g, p.a, static_cast<const void*>(ws), apart ? static_cast<void*>(rows) : p.c);
  }
  if (st == TSM100_OK && apart) {
    const dim3 grid(static_cast<unsigned>(d->m), static_cast<unsigned>(std::min<int64_t>((d->n + 2047) / 2048, 64)));
    e = launch_chained(w4::w4_rows_kernel<T>, grid, w4::kDenseThreads, 0, s, 0, static_cast<const T*>(rows), static_cast<T*>(p.c), p.n, static_cast<int32_t>(n8));
    st = cuda_ok(err, e, "w4_rows_kernel launch");
  }
  e = cudaFreeAsync(ws, s);
  if (st == TSM100_OK && e != cudaSuccess) st = cuda_ok(err, e, "cudaFreeAsync");
  return st;
}

// Rows in 8 bits as rows of T, in scratch; without memory for them the product is refused.
template <typename T>
inline int32_t gemm_w4_widen(std::string* err, const tsm100_gemm_w4_desc* d, const void* a, void** wide, cudaStream_t s) {
  const int32_t st = take_scratch(err, wide, static_cast<size_t>(d->m) * d->k * 2, s);
  if (st == kNoScratch) return op_fail(err, TSM100_ERR_MEMORY, "gemm_w4: no device memory for the rows in 16 bits");
  if (st != TSM100_OK) return st;
  const int64_t vecs = d->m * d->k / 8;
  return cuda_ok(err, launch_chained(w4::w4_widen_kernel<T>, static_cast<unsigned>((vecs + w4::kDenseThreads - 1) / w4::kDenseThreads), w4::kDenseThreads, 0, s, 0,
                                     static_cast<const uint2*>(a), static_cast<uint4*>(*wide), vecs),
                 "w4_widen_kernel launch");
}

template <typename Gemm>
inline int32_t gemm_w4(std::string* err, const tsm100_gemm_w4_desc* d, const void* a, const float* a_scales, const uint8_t* w, const void* w_scales,
                       const uint8_t* w_zeros, void* c, uint32_t* status, void* stream, Gemm gemm) {
  if (!d) return op_fail(err, TSM100_ERR_INVALID, "gemm_w4: null descriptor");
  if (!dtype_16bit(d->dtype)) return op_fail(err, TSM100_ERR_INVALID, "gemm_w4: dtype must be TSM100_F16 or TSM100_BF16");
  if (d->a_dtype != d->dtype && d->a_dtype != TSM100_I8) return op_fail(err, TSM100_ERR_INVALID, "gemm_w4: a_dtype must be dtype or TSM100_I8");
  if (d->group != 32 && d->group != 64 && d->group != 128) return op_fail(err, TSM100_ERR_INVALID, "gemm_w4: group must be 32, 64 or 128");
  if (d->m < 0 || d->n < 0 || d->k < 0 || d->m > 0x7fffffff || d->n > 0x7fffffff || d->k > 0x7fffffff)
    return op_fail(err, TSM100_ERR_INVALID, "gemm_w4: bad shape");
  if (d->k % d->group != 0) return op_fail(err, TSM100_ERR_INVALID, "gemm_w4: k must be a multiple of group");
  if (d->m == 0 || d->n == 0) return TSM100_OK;
  if (d->m > 64 * 65535) return op_fail(err, TSM100_ERR_INVALID, "gemm_w4: too many rows for one launch");
  if (!c || (d->k > 0 && (!a || !w || !w_scales))) return op_fail(err, TSM100_ERR_INVALID, "gemm_w4: null buffer");
  if (d->a_dtype == TSM100_I8 && !a_scales) return op_fail(err, TSM100_ERR_INVALID, "gemm_w4: rows in 8 bits need a_scales");
  if (!aligned16(a) || !aligned16(w)) return op_fail(err, TSM100_ERR_INVALID, "gemm_w4: a and w must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(w_scales) | reinterpret_cast<uintptr_t>(c)) & 1u || reinterpret_cast<uintptr_t>(a_scales) & 3u)
    return op_fail(err, TSM100_ERR_INVALID, "gemm_w4: a buffer does not start on an element boundary");
  w4::Params p;
  p.a = a;
  p.a_scales = d->a_dtype == TSM100_I8 ? a_scales : nullptr;
  p.scales = w_scales;
  p.zeros = w_zeros;
  p.c = c;
  p.m = static_cast<int32_t>(d->m), p.n = static_cast<int32_t>(d->n), p.k = static_cast<int32_t>(d->k);
  p.groups = static_cast<int32_t>(d->k / d->group);
  p.status = status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int32_t st = TSM100_OK;
  void* wide = nullptr;
  if (p.a_scales && d->m > w4::kExactTokens && d->k > 0) {
    st = d->dtype == TSM100_BF16 ? gemm_w4_widen<__nv_bfloat16>(err, d, p.a, &wide, s) : gemm_w4_widen<__half>(err, d, p.a, &wide, s);
    p.a = wide;
  }
  if (st == TSM100_OK) {
    st = kNoScratch;
    if (gemm_w4_dense_pays(d))
      st = d->dtype == TSM100_BF16 ? gemm_w4_dense<__nv_bfloat16>(err, d, w, p, s, gemm) : gemm_w4_dense<__half>(err, d, w, p, s, gemm);
    if (st == kNoScratch) st = d->dtype == TSM100_BF16 ? gemm_w4_typed<__nv_bfloat16>(err, d, w, p, s) : gemm_w4_typed<__half>(err, d, w, p, s);
  }
  if (wide) {
    const cudaError_t e = cudaFreeAsync(wide, s);
    if (st == TSM100_OK && e != cudaSuccess) st = cuda_ok(err, e, "cudaFreeAsync");
  }
  return st;
}

}  // namespace ops
}  // namespace tsm100
