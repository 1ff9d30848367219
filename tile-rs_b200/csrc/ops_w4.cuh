// Host-side launch logic of products with 4-bit weights (gemm_w4.cuh); as ops_serving.cuh.
#pragma once

#include <algorithm>

#include "gemm_w4.cuh"
#include "launch.cuh"

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
  auto kern = p.a_scales ? w4::gemm_w4_kernel<T, N, GC, kScaled, true> : w4::gemm_w4_kernel<T, N, GC, kScaled, false>;
  cudaError_t e = set_dyn_smem_once(kern, S::kSmem);
  const dim3 grid(static_cast<unsigned>((p.n + w4::kRows - 1) / w4::kRows * p.splits), static_cast<unsigned>((p.m + p.tokens - 1) / p.tokens));
  if (e == cudaSuccess) e = launch_chained(kern, grid, w4::kThreads, S::kSmem, s, p.splits > 1 ? p.splits : 0, map, p);
  return cuda_ok(err, e, "gemm_w4_kernel launch");
}
template <typename T, int GC>
inline int32_t gemm_w4_grouped(std::string* err, const CUtensorMap& map, const w4::Params& p, int sms, cudaStream_t s) {
  if (p.m <= 16) return gemm_w4_launch<T, 16, GC>(err, map, p, sms, s);
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

inline int32_t gemm_w4(std::string* err, const tsm100_gemm_w4_desc* d, const void* a, const float* a_scales, const uint8_t* w, const void* w_scales,
                       const uint8_t* w_zeros, void* c, uint32_t* status, void* stream) {
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
  return d->dtype == TSM100_BF16 ? gemm_w4_typed<__nv_bfloat16>(err, d, w, p, s) : gemm_w4_typed<__half>(err, d, w, p, s);
}

}  // namespace ops
}  // namespace tsm100
