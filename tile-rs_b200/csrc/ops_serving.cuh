// Host-side launch logic of the serving operators (residual norm, paged KV cache and its attentions, whose kernels ops_paged.cuh launches): argument checks, kernel
// selection, launch.  As in ops.cuh nothing here synchronises and every function answers a TSM100_* status with a message in *err.
#pragma once

#include <algorithm>
#include <cmath>

#include "add_rms_norm.cuh"
#include "kv_pages.cuh"
#include "launch.cuh"
#include "ops_paged.cuh"
#include "route.hpp"

namespace tsm100 {
namespace ops {

// ---------------------------------------------------------------------------
// residual norm
// ---------------------------------------------------------------------------
template <typename T, bool kI8>
inline cudaError_t add_rms_norm_launch(const addnorm::Params<T>& p, cudaStream_t s) {
  namespace an = addnorm;
  constexpr int PV = softmax::Elem<T>::kPerVec;
  const int64_t vecs = p.cols / PV;
  bool vec = p.cols % PV == 0 && vecs <= 8 * an::kThreads;
  for (const void* q : {static_cast<const void*>(p.x), static_cast<const void*>(p.residual), static_cast<const void*>(p.sum), static_cast<const void*>(p.weight)})
    vec = vec && aligned16(q);
  vec = vec && (kI8 ? reinterpret_cast<uintptr_t>(p.y) % PV == 0 : aligned16(p.y));
  const unsigned rows = static_cast<unsigned>(p.rows);
  auto go = [&](auto kern, unsigned grid) { return launch_chained(kern, grid, an::kThreads, 0, s, 0, p); };
  if (vec) {
    // a warp a row as long as that is four vectors a lane, and there are rows for its lanes
    const unsigned warps = (rows + 7) / 8;
    if (vecs <= 32) return go(an::add_rms_norm_vec_kernel<T, kI8, 32, 1>, warps);
    if (vecs <= 64) return go(an::add_rms_norm_vec_kernel<T, kI8, 32, 2>, warps);
    if (vecs <= 128) return go(an::add_rms_norm_vec_kernel<T, kI8, 32, 4>, warps);
    if (vecs <= an::kThreads) return go(an::add_rms_norm_vec_kernel<T, kI8, an::kThreads, 1>, rows);
    if (vecs <= 2 * an::kThreads) return go(an::add_rms_norm_vec_kernel<T, kI8, an::kThreads, 2>, rows);
    if (vecs <= 4 * an::kThreads) return go(an::add_rms_norm_vec_kernel<T, kI8, an::kThreads, 4>, rows);
    return go(an::add_rms_norm_vec_kernel<T, kI8, an::kThreads, 8>, rows);
  }
  // as few elements a thread as hold the row: registers decide how many CTAs an SM has (3000 x 5001 f32 66 us with 32 a thread, 45 with 20); wider rows are read twice
  if (p.cols <= 4 * an::kThreads) return go(an::add_rms_norm_any_kernel<T, kI8, 4>, rows);
  if (p.cols <= 12 * an::kThreads) return go(an::add_rms_norm_any_kernel<T, kI8, 12>, rows);
  if (p.cols <= 20 * an::kThreads) return go(an::add_rms_norm_any_kernel<T, kI8, 20>, rows);
  if (p.cols <= 32 * an::kThreads) return go(an::add_rms_norm_any_kernel<T, kI8, 32>, rows);
  return go(an::add_rms_norm_any_kernel<T, kI8, 0>, rows);
}

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
  return cuda_ok(err, d->out_dtype == TSM100_I8 ? add_rms_norm_launch<T, true>(p, s) : add_rms_norm_launch<T, false>(p, s), "add_rms_norm launch");
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
// paged KV cache
// ---------------------------------------------------------------------------
template <typename T, bool kI8, bool kRead, int LANES>
inline cudaError_t kv_page_rows_launch(const pages::Cache& c, const pages::Batch& b, T* k, T* v, uint32_t* status, cudaStream_t s) {
  if constexpr (LANES < 32)
    if (c.d > 8 * LANES) return kv_page_rows_launch<T, kI8, kRead, 2 * LANES>(c, b, k, v, status, s);
  // eight rounds of rows to a CTA, so that finding their places counts for little, unless that left SMs without one
  constexpr int kRows = pages::kThreads / LANES * pages::kPasses;
  int sms = 148;
  (void)sm_count(nullptr, &sms);
  const int per_cta = std::max(1, std::min({pages::kMaxTokens, (8 * kRows + 2 * c.heads - 1) / (2 * c.heads), b.tokens / (4 * sms)}));
  return launch_chained(pages::kv_page_rows_kernel<T, kI8, kRead, LANES>, static_cast<unsigned>((b.tokens + per_cta - 1) / per_cta), pages::kThreads, 0, s, 0, c, b, k, v,
                        static_cast<int32_t>(per_cta), status);
}
template <typename T, bool kRead>
inline cudaError_t kv_page_rows_typed(const pages::Cache& c, const pages::Batch& b, bool i8, void* k, void* v, uint32_t* status, cudaStream_t s) {
  return i8 ? kv_page_rows_launch<T, true, kRead, 2>(c, b, static_cast<T*>(k), static_cast<T*>(v), status, s)
            : kv_page_rows_launch<T, false, kRead, 2>(c, b, static_cast<T*>(k), static_cast<T*>(v), status, s);
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
  return cuda_ok(err, dtype == TSM100_BF16 ? kv_page_rows_typed<__nv_bfloat16, kRead>(c, step, i8, k, v, status, s)
                                           : kv_page_rows_typed<__half, kRead>(c, step, i8, k, v, status, s), op);
}

// ---------------------------------------------------------------------------
// attention over pages
// ---------------------------------------------------------------------------
inline int32_t attention_paged_any(std::string* err, const paged::Params& p, bool bf16, bool i8, const void* q, void* o, cudaStream_t s) {
  return bf16 ? attention_paged_typed<__nv_bfloat16>(err, p, i8, q, o, s) : attention_paged_typed<__half>(err, p, i8, q, o, s);
}

inline int32_t attention_paged(std::string* err, const tsm100_paged_kv* kv, const tsm100_paged_batch* b, const tsm100_attention_paged_desc* d, const void* q,
                               void* o, uint32_t* status, void* stream) {
  if (!d) return op_fail(err, TSM100_ERR_INVALID, "attention_paged: null descriptor");
  paged::Params p;
  bool nothing;
  const int32_t st = attention_paged_args(err, "attention_paged", kv, b, d->dtype, d->heads_q, q, o, status, &p, &nothing);
  if (st != TSM100_OK || nothing) return st;
  return attention_paged_any(err, p, d->dtype == TSM100_BF16, kv->dtype == TSM100_I8, q, o, static_cast<cudaStream_t>(stream));
}

// Records, and routes, by max_new: no sequence has more tokens than the call, whatever the caller allows.
inline void bound_new(paged::Params* p) { p->step.max_new = std::min(p->step.max_new, p->step.tokens); }

inline int32_t attention_paged_cross(std::string* err, const tsm100_paged_kv* kv, const tsm100_paged_batch* b, const tsm100_attention_paged_desc* d, const void* q,
                                     void* o, uint32_t* status, void* stream) {
  if (!d) return op_fail(err, TSM100_ERR_INVALID, "attention_paged_cross: null descriptor");
  paged::Params p;
  bool nothing;
  const int32_t st = attention_paged_args(err, "attention_paged_cross", kv, b, d->dtype, d->heads_q, q, o, status, &p, &nothing);
  if (st != TSM100_OK || nothing) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf16 = d->dtype == TSM100_BF16;
  bound_new(&p);
  return kv->dtype == TSM100_I8 ? attention_cross_held<true>(err, p, bf16, q, o, s) : attention_cross_held<false>(err, p, bf16, q, o, s);
}

inline int32_t attention_paged_prefix(std::string* err, const tsm100_paged_kv* kv, const tsm100_paged_batch* b, const tsm100_attention_paged_prefix_desc* d, const void* q,
                                      void* o, uint32_t* status, void* stream) {
  auto no = [&](const char* what) { return op_fail(err, TSM100_ERR_INVALID, std::string("attention_paged_prefix: ") + what); };
  if (!d) return no("null descriptor");
  paged::Params p;
  bool nothing;
  int32_t st = attention_paged_args(err, "attention_paged_prefix", kv, b, d->dtype, d->heads_q, q, o, status, &p, &nothing);
  if (st != TSM100_OK) return st;
  if (d->prefix_len < 0 || d->prefix_len % kv->page_size != 0) return no("prefix_len must be a multiple of page_size");
  if (d->prefix_len > static_cast<int64_t>(b->table_pitch) * kv->page_size) return no("prefix_len is more than a row of the table covers");
  if (nothing) return TSM100_OK;
  if (d->prefix_len > 0 && !d->prefix) return no("null prefix");
  if (reinterpret_cast<uintptr_t>(d->prefix) & 3u) return no("prefix does not start on an element boundary");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf16 = d->dtype == TSM100_BF16, i8 = kv->dtype == TSM100_I8;
  if (d->prefix_len == 0) return attention_paged_any(err, p, bf16, i8, q, o, s);
  bound_new(&p);
  PrefixPlan plan;
  plan.run_log2 = page_run_log2(kv->page_size, 7);
  const bool tc = paged_fits_tcgen05(p.group, i8, plan.run_log2);
  plan.shared_tc = tc && route::prefix_on_tcgen05(static_cast<int64_t>(b->tokens) * p.group, d->prefix_len, kv->heads_kv, kv->head_dim, i8);
  plan.rest_tc = tc && static_cast<int64_t>(p.step.max_new) * p.group > route::kPrefixFewRows;
  PrefixArgs more = {};
  more.large = plan.rest_tc ? static_cast<int32_t>(route::kPrefixFewRows) : 0;
  more.prefix = d->prefix_len, more.table = d->prefix;
  p.step.table += d->prefix_len / kv->page_size;
  if (kv->head_dim == 128) return i8 ? attention_prefix_held<true, 128>(err, p, bf16, plan, more, q, o, s) : attention_prefix_held<false, 128>(err, p, bf16, plan, more, q, o, s);
  return i8 ? attention_prefix_held<true, 64>(err, p, bf16, plan, more, q, o, s) : attention_prefix_held<false, 64>(err, p, bf16, plan, more, q, o, s);
}

}  // namespace ops
}  // namespace tsm100
