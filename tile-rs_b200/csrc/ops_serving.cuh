// Host-side launch logic of the serving operators (residual norm, 4-bit weights, paged KV cache and its attention): argument checks, kernel
// selection, launch.  As in ops.cuh nothing here synchronises and every function answers a TSM100_* status with a message in *err.
#pragma once

#include <algorithm>
#include <cmath>

#include "add_rms_norm.cuh"
#include "attention_paged.cuh"
#include "gemm_w4.cuh"
#include "kv_pages.cuh"
#include "launch.cuh"

namespace tsm100 {
namespace ops {

inline bool dtype_16bit(int32_t dtype) { return dtype == TSM100_F16 || dtype == TSM100_BF16; }

// ---------------------------------------------------------------------------
// residual norm
// ---------------------------------------------------------------------------
template <typename T>
inline int32_t add_rms_norm_typed(std::string* err, const tsm100_add_rms_norm_desc* d, const void* x, const void* residual, void* sum, const void* weight,
                                  void* y, float* scales, cudaStream_t s) {
  addnorm::Params<T> p;
  p.x = static_cast<const T*>(x);
  p.residual = static_cast<const T*>(residual);
  p.sum = static_cast<T*>(sum);
  p.weight = static_cast<const T*>(weight);
  p.y = y;
  p.scales = scales;
  p.rows = d->rows;
  p.cols = static_cast<int32_t>(d->cols);
  p.eps = d->eps;
  const unsigned grid = static_cast<unsigned>(d->rows);
  if (d->out_dtype == TSM100_I8) addnorm::add_rms_norm_kernel<T, true><<<grid, addnorm::kThreads, 0, s>>>(p);
  else addnorm::add_rms_norm_kernel<T, false><<<grid, addnorm::kThreads, 0, s>>>(p);
  return cuda_ok(err, cudaGetLastError(), "add_rms_norm launch");
}

inline int32_t add_rms_norm(std::string* err, const tsm100_add_rms_norm_desc* d, const void* x, const void* residual, void* sum, const void* weight, void* y,
                            float* scales, void* stream) {
  if (!d) return op_fail(err, TSM100_ERR_INVALID, "add_rms_norm: null descriptor");
  if (!dtype_valid(d->dtype)) return op_fail(err, TSM100_ERR_INVALID, "add_rms_norm: unknown dtype");
  if (d->out_dtype != d->dtype && d->out_dtype != TSM100_I8) return op_fail(err, TSM100_ERR_INVALID, "add_rms_norm: out_dtype must be dtype or TSM100_I8");
  if (d->rows < 0 || d->cols < 0 || d->rows > 0x7fffffff || d->cols > 0x7fffffff) return op_fail(err, TSM100_ERR_INVALID, "add_rms_norm: bad shape");
  if (d->rows == 0 || d->cols == 0) return TSM100_OK;
  if (!x || !y) return op_fail(err, TSM100_ERR_INVALID, "add_rms_norm: null buffer");
  if (d->out_dtype == TSM100_I8 && !scales) return op_fail(err, TSM100_ERR_INVALID, "add_rms_norm: an output in 8 bits needs scales");
  if (sum && sum == y) return op_fail(err, TSM100_ERR_INVALID, "add_rms_norm: sum and y are the same buffer");
  if (d->out_dtype == TSM100_I8 && (y == x || y == residual)) return op_fail(err, TSM100_ERR_INVALID, "add_rms_norm: y in 8 bits cannot be x or residual");
  const size_t mask = dtype_size(d->dtype) - 1;
  for (const void* q : {x, residual, static_cast<const void*>(sum), weight, d->out_dtype == TSM100_I8 ? nullptr : static_cast<const void*>(y)})
    if (reinterpret_cast<uintptr_t>(q) & mask) return op_fail(err, TSM100_ERR_INVALID, "add_rms_norm: a buffer does not start on an element boundary");
  if (reinterpret_cast<uintptr_t>(scales) & 3u) return op_fail(err, TSM100_ERR_INVALID, "add_rms_norm: scales do not start on an element boundary");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (d->dtype) {
    case TSM100_F32: return add_rms_norm_typed<float>(err, d, x, residual, sum, weight, y, scales, s);
    case TSM100_BF16: return add_rms_norm_typed<__nv_bfloat16>(err, d, x, residual, sum, weight, y, scales, s);
    default: return add_rms_norm_typed<__half>(err, d, x, residual, sum, weight, y, scales, s);
  }
}

// ---------------------------------------------------------------------------
// 4-bit weights
// ---------------------------------------------------------------------------
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
  auto kern = w4::gemm_w4_kernel<T, N, GC, kScaled>;
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
inline int32_t gemm_w4_typed(std::string* err, const tsm100_gemm_w4_desc* d, const uint8_t* w, const w4::Params& p, cudaStream_t s) {
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

// ---------------------------------------------------------------------------
// paged KV cache
// ---------------------------------------------------------------------------
// What every operator on pages asks of its descriptors.  *nothing: there are no tokens.
inline int32_t paged_args(std::string* err, const char* op, const tsm100_paged_kv* kv, const tsm100_paged_batch* b, int32_t dtype, pages::Cache* c,
                          pages::Batch* s, bool* nothing) {
  auto no = [&](const char* what) { return op_fail(err, TSM100_ERR_INVALID, std::string(op) + ": " + what); };
  *nothing = false;
  if (!kv || !b) return no("null descriptor");
  if (!dtype_16bit(dtype)) return no("dtype must be TSM100_F16 or TSM100_BF16");
  if (kv->dtype != dtype && kv->dtype != TSM100_I8) return no("the cache must hold dtype or TSM100_I8");
  if (kv->heads_kv <= 0 || kv->page_size <= 0 || kv->page_size > 4096 || kv->pages < 0 || kv->pages > 0x7fffffff) return no("bad cache shape");
  if (kv->head_dim <= 0 || kv->head_dim > 256 || kv->head_dim % 16 != 0) return no("head_dim must be a multiple of 16, up to 256");
  if (static_cast<int64_t>(kv->heads_kv) * kv->pages > 0x7fffffff) return no("too many pages times heads");
  if (b->batch < 0 || b->tokens < 0 || b->max_new < 0 || b->max_len < 0 || b->table_pitch < 0) return no("bad batch shape");
  if (static_cast<int64_t>(b->table_pitch) * kv->page_size > 0x7fffffff) return no("a row of the table covers too many positions");
  if (b->batch == 0 || b->tokens == 0 || b->max_new == 0) {
    *nothing = true;
    return TSM100_OK;
  }
  if (!b->table || !b->lens || !b->starts) return no("null table, lens or starts");
  if ((reinterpret_cast<uintptr_t>(b->table) | reinterpret_cast<uintptr_t>(b->lens) | reinterpret_cast<uintptr_t>(b->starts)) & 3u)
    return no("table, lens or starts do not start on an element boundary");
  if (kv->pages == 0) return no("the cache has no pages");
  if (!kv->k || !kv->v) return no("null cache");
  if (!aligned16(kv->k) || !aligned16(kv->v)) return no("the cache must be 16-byte aligned");
  if (kv->dtype == TSM100_I8 && (!kv->k_scales || !kv->v_scales)) return no("a cache of 8 bits needs scales");
  if ((reinterpret_cast<uintptr_t>(kv->k_scales) | reinterpret_cast<uintptr_t>(kv->v_scales)) & 3u) return no("scales do not start on an element boundary");
  c->heads = kv->heads_kv, c->d = kv->head_dim, c->page_size = kv->page_size, c->pages = kv->pages;
  c->kv[0] = kv->k, c->kv[1] = kv->v;
  c->scales[0] = kv->k_scales, c->scales[1] = kv->v_scales;
  s->batch = b->batch, s->tokens = b->tokens, s->max_new = b->max_new, s->pitch = b->table_pitch;
  s->table = b->table, s->lens = b->lens, s->starts = b->starts;
  return TSM100_OK;
}

template <typename T, bool kRead>
inline cudaError_t kv_page_rows_launch(const pages::Cache& c, const pages::Batch& b, bool i8, void* k, void* v, uint32_t* status, cudaStream_t s) {
  const unsigned grid = static_cast<unsigned>((static_cast<int64_t>(b.tokens) * 2 * c.heads + 7) / 8);
  if (i8) pages::kv_page_rows_kernel<T, true, kRead><<<grid, 256, 0, s>>>(c, b, static_cast<T*>(k), static_cast<T*>(v), status);
  else pages::kv_page_rows_kernel<T, false, kRead><<<grid, 256, 0, s>>>(c, b, static_cast<T*>(k), static_cast<T*>(v), status);
  return cudaGetLastError();
}

template <bool kRead>
inline int32_t kv_page_rows(std::string* err, const tsm100_paged_kv* kv, const tsm100_paged_batch* b, int32_t dtype, void* k, void* v, uint32_t* status,
                            void* stream) {
  const char* op = kRead ? "kv_page_read" : "kv_page_append";
  pages::Cache c;
  pages::Batch step;
  bool nothing;
  const int32_t st = paged_args(err, op, kv, b, dtype, &c, &step, &nothing);
  if (st != TSM100_OK || nothing) return st;
  if (!k || !v) return op_fail(err, TSM100_ERR_INVALID, std::string(op) + ": null buffer");
  if (!aligned16(k) || !aligned16(v)) return op_fail(err, TSM100_ERR_INVALID, std::string(op) + ": k and v must be 16-byte aligned");
  if (static_cast<int64_t>(step.tokens) * 2 * c.heads / 8 >= 0x7fffffff) return op_fail(err, TSM100_ERR_INVALID, std::string(op) + ": too many tokens for one launch");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool i8 = kv->dtype == TSM100_I8;
  return cuda_ok(err, dtype == TSM100_BF16 ? kv_page_rows_launch<__nv_bfloat16, kRead>(c, step, i8, k, v, status, s)
                                           : kv_page_rows_launch<__half, kRead>(c, step, i8, k, v, status, s), op);
}

// ---------------------------------------------------------------------------
// attention over pages
// ---------------------------------------------------------------------------
// The tiles of all sequences' caches dealt out evenly over the SMs, and what several of them have a part of merged (attention_paged.cuh).
template <typename T, bool kI8, int D>
inline int32_t attention_paged_launch(std::string* err, paged::Params p, const void* q, void* o, cudaStream_t s) {
  using L = paged::Tile<kI8, D>;
  int sms = 0;
  int32_t st = sm_count(err, &sms);
  if (st != TSM100_OK) return st;
  const unsigned ctas = static_cast<unsigned>(std::min(sms, paged::kMaxCtas));
  const int64_t rows = std::min<int64_t>(paged::kRows, static_cast<int64_t>(p.step.max_new) * p.group);
  const size_t part = static_cast<size_t>(ctas) * 2 * paged::kRows * L::kRec * sizeof(float);
  st = take_scratch(err, reinterpret_cast<void**>(&p.part), part + ctas * sizeof(int4), s);
  if (st == kNoScratch) return op_fail(err, TSM100_ERR_MEMORY, "attention_paged: no device memory for partial results");
  if (st != TSM100_OK) return st;
  p.info = reinterpret_cast<int4*>(reinterpret_cast<uint8_t*>(p.part) + part);
  // boxes of a power of two of positions that a page is a multiple of; 8-bit steps come by copies of 16 bytes and more
  int run_log2 = 0;
  while ((2 << run_log2) <= L::kPos && p.cache.page_size % (2 << run_log2) == 0) ++run_log2;
  const bool boxes = run_log2 >= 3 && (!kI8 || (aligned16(p.cache.scales[0]) && aligned16(p.cache.scales[1])));
  p.run_log2 = boxes ? run_log2 : L::kPos == 32 ? 5 : 6;
  CUtensorMap map[2];
  std::memset(map, 0, sizeof map);
  for (int i = 0; i < 2 && boxes && st == TSM100_OK; ++i) {
    TmapKey key;
    std::memset(&key, 0, sizeof key);
    constexpr bool kTwo = L::kRowBytes == 256;  // rows of two 128-byte groups
    key.base = p.cache.kv[i];
    const uint64_t rows = static_cast<uint64_t>(p.cache.page_size), units = static_cast<uint64_t>(p.cache.pages) * p.cache.heads;
    if (kTwo) {
      key.dim[0] = 64, key.dim[1] = rows, key.dim[2] = 2, key.dim[3] = units;
      key.stride[0] = 256, key.stride[1] = 128, key.stride[2] = rows * 256;
      key.box[0] = 64, key.box[1] = 1u << run_log2, key.box[2] = 2, key.box[3] = 1;
    } else {
      key.dim[0] = kI8 ? D : 64, key.dim[1] = rows, key.dim[2] = units;
      key.stride[0] = L::kRowBytes, key.stride[1] = rows * L::kRowBytes;
      key.box[0] = kI8 ? D : 64, key.box[1] = 1u << run_log2, key.box[2] = 1;
    }
    key.dtype = static_cast<int32_t>(kI8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16);
    key.rank = kTwo ? 4 : 3;
    st = make_tmap(err, &map[i], key, kI8 ? 1 : 2);
  }
  if (st == TSM100_OK) {
    auto kern = boxes ? paged::attention_paged_kernel<T, kI8, D, true> : paged::attention_paged_kernel<T, kI8, D, false>;
    cudaError_t e = set_dyn_smem_once(kern, L::kSmem);
    if (e == cudaSuccess) e = launch_chained(kern, ctas, paged::kThreads, L::kSmem, s, 0, map[0], map[1], static_cast<const T*>(q), static_cast<T*>(o), p);
    if (e == cudaSuccess) e = launch_chained(paged::attention_paged_merge_kernel<T, D>, dim3(ctas, static_cast<unsigned>((rows + 3) / 4)), 128, 0, s, 0, static_cast<T*>(o), p);
    st = cuda_ok(err, e, "attention_paged_kernel launch");
  }
  const cudaError_t e = cudaFreeAsync(p.part, s);
  if (st == TSM100_OK && e != cudaSuccess) st = cuda_ok(err, e, "cudaFreeAsync");
  return st;
}

template <typename T>
inline int32_t attention_paged_typed(std::string* err, const paged::Params& p, bool i8, const void* q, void* o, cudaStream_t s) {
  if (p.cache.d == 128) return i8 ? attention_paged_launch<T, true, 128>(err, p, q, o, s) : attention_paged_launch<T, false, 128>(err, p, q, o, s);
  return i8 ? attention_paged_launch<T, true, 64>(err, p, q, o, s) : attention_paged_launch<T, false, 64>(err, p, q, o, s);
}

inline int32_t attention_paged(std::string* err, const tsm100_paged_kv* kv, const tsm100_paged_batch* b, const tsm100_attention_paged_desc* d, const void* q,
                               void* o, uint32_t* status, void* stream) {
  if (!d) return op_fail(err, TSM100_ERR_INVALID, "attention_paged: null descriptor");
  paged::Params p;
  bool nothing;
  const int32_t st = paged_args(err, "attention_paged", kv, b, d->dtype, &p.cache, &p.step, &nothing);
  if (st != TSM100_OK) return st;
  if (kv->head_dim != 64 && kv->head_dim != 128) return op_fail(err, TSM100_ERR_INVALID, "attention_paged: head_dim must be 64 or 128");
  if (d->heads_q <= 0 || d->heads_q % kv->heads_kv != 0)
    return op_fail(err, TSM100_ERR_INVALID, "attention_paged: heads_q must be a positive multiple of heads_kv");
  if (nothing) return TSM100_OK;
  if (!q || !o) return op_fail(err, TSM100_ERR_INVALID, "attention_paged: null buffer");
  if (!aligned16(q) || !aligned16(o)) return op_fail(err, TSM100_ERR_INVALID, "attention_paged: q and o must be 16-byte aligned");
  if (static_cast<int64_t>(b->tokens) * d->heads_q > 0x7fffffff) return op_fail(err, TSM100_ERR_INVALID, "attention_paged: too many tokens times heads");
  p.heads_q = d->heads_q;
  p.group = d->heads_q / kv->heads_kv;
  p.scale_log2 = static_cast<float>((1.0 / std::sqrt(static_cast<double>(kv->head_dim))) * 1.4426950408889634);
  p.status = status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool i8 = kv->dtype == TSM100_I8;
  return d->dtype == TSM100_BF16 ? attention_paged_typed<__nv_bfloat16>(err, p, i8, q, o, s) : attention_paged_typed<__half>(err, p, i8, q, o, s);
}

}  // namespace ops
}  // namespace tsm100
