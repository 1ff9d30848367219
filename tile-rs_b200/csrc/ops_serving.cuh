// Host-side launch logic of the serving operators (residual norm, paged KV cache and its attention): argument checks, kernel
// selection, launch.  As in ops.cuh nothing here synchronises and every function answers a TSM100_* status with a message in *err.
#pragma once

#include <algorithm>
#include <cmath>

#include "add_rms_norm.cuh"
#include "attention_paged.cuh"
#include "attention_paged_tc.cuh"
#include "kv_pages.cuh"
#include "launch.cuh"

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
// Positions that a TMA box of a page may have, as a power of two: one that the page is a multiple of, at most 2^top.
inline int page_run_log2(int page_size, int top) {
  int n = 0;
  while (n < top && page_size % (2 << n) == 0) ++n;
  return n;
}
// Boxes of 64 columns and 2^run_log2 positions of the pages.
inline int32_t page_tmap(std::string* err, CUtensorMap* map, const pages::Cache& c, const void* base, int run_log2, bool is_bf16) {
  const uint64_t d = static_cast<uint64_t>(c.d), rows = static_cast<uint64_t>(c.page_size);
  return make_tmap_16bit_3d(err, map, base, d, rows, static_cast<uint64_t>(c.pages) * c.heads, d, rows * d, 64, 1u << run_log2, is_bf16);
}

// Chunks of tokens: tcgen05 (attention_paged_tc.cuh).
template <typename T, bool kI8, int D>
inline int32_t attention_paged_tc_launch(std::string* err, const paged::Params& base, int run_log2, const void* q, void* o, cudaStream_t s) {
  namespace tc = paged::tc;
  constexpr bool kIsBf16 = !std::is_same<T, __half>::value;
  using S = tc::Shape<kI8, D>;
  int sms = 0;
  int32_t st = sm_count(err, &sms);
  if (st != TSM100_OK) return st;
  const unsigned ctas = static_cast<unsigned>(sms);
  tc::Params p;
  p.cache = base.cache, p.step = base.step;
  p.heads_q = base.heads_q, p.group = base.group;
  p.tokens = tc::kTileRows / base.group;
  p.run_log2 = run_log2;
  p.scale_log2 = base.scale_log2;
  p.status = base.status;
  CUtensorMap tq, tk, tv;
  TmapKey key;
  std::memset(&key, 0, sizeof key);
  key.base = q;
  key.dim[0] = D, key.dim[1] = static_cast<uint64_t>(p.heads_q), key.dim[2] = static_cast<uint64_t>(p.step.tokens);
  key.stride[0] = D * 2, key.stride[1] = static_cast<uint64_t>(p.heads_q) * D * 2;
  key.box[0] = 64, key.box[1] = static_cast<uint32_t>(p.group), key.box[2] = static_cast<uint32_t>(p.tokens);
  key.dtype = static_cast<int32_t>(kIsBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16), key.rank = 3;
  st = make_tmap(err, &tq, key, 2);
  if (kI8) {
    tk = tv = tq;  // not used
  } else {
    if (st == TSM100_OK) st = page_tmap(err, &tk, p.cache, p.cache.kv[0], run_log2, kIsBf16);
    if (st == TSM100_OK) st = page_tmap(err, &tv, p.cache, p.cache.kv[1], run_log2, kIsBf16);
  }
  if (st != TSM100_OK) return st;
  const size_t rows = static_cast<size_t>(ctas) * 2 * 256, part = rows * D * sizeof(float), ml = rows * sizeof(float2);
  uint8_t* ws = nullptr;
  st = take_scratch(err, reinterpret_cast<void**>(&ws), part + ml + ctas * sizeof(int4), s);
  if (st == kNoScratch) return op_fail(err, TSM100_ERR_MEMORY, "attention_paged: no device memory for partial results");
  if (st != TSM100_OK) return st;
  p.part = reinterpret_cast<float4*>(ws);
  p.part_ml = reinterpret_cast<float2*>(ws + part);
  p.info = reinterpret_cast<int4*>(ws + part + ml);
  auto kern = tc::attention_paged_tc_kernel<kIsBf16, kI8, D>;
  constexpr int smem = tc::smem_bytes<kI8, D>();
  cudaError_t e = set_dyn_smem_once(kern, smem);
  if (e == cudaSuccess) e = launch_chained(kern, ctas, S::kThreads, smem, s, 0, tq, tk, tv, static_cast<uint16_t*>(o), p);
  if (e == cudaSuccess) e = launch_chained(tc::attention_paged_tc_merge_kernel<kIsBf16, D>, dim3(ctas, D / 16), 256, 0, s, 0, static_cast<uint16_t*>(o), p);
  st = cuda_ok(err, e, "attention_paged_tc_kernel launch");
  e = cudaFreeAsync(ws, s);
  if (st == TSM100_OK && e != cudaSuccess) st = cuda_ok(err, e, "cudaFreeAsync");
  return st;
}

// The tiles of all sequences' caches dealt out evenly over the SMs, and what several of them have a part of merged (attention_paged.cuh).
template <typename T, bool kI8, int D, bool kWide>
inline int32_t attention_paged_few_launch(std::string* err, paged::Params p, const void* q, void* o, cudaStream_t s) {
  using L = paged::Tile<kI8, D, kWide>;
  int sms = 0;
  int32_t st = sm_count(err, &sms);
  if (st != TSM100_OK) return st;
  const unsigned ctas = static_cast<unsigned>(std::min(sms, paged::kMaxCtas));
  const int64_t rows = std::min<int64_t>(L::kHeld, static_cast<int64_t>(p.step.max_new) * p.group);
  const size_t part = static_cast<size_t>(ctas) * 2 * L::kHeld * L::kRec * sizeof(float);
  st = take_scratch(err, reinterpret_cast<void**>(&p.part), part + ctas * sizeof(int4), s);
  if (st == kNoScratch) return op_fail(err, TSM100_ERR_MEMORY, "attention_paged: no device memory for partial results");
  if (st != TSM100_OK) return st;
  p.info = reinterpret_cast<int4*>(reinterpret_cast<uint8_t*>(p.part) + part);
  // boxes of a power of two of positions that a page is a multiple of; 8-bit steps come by copies of 16 bytes and more
  constexpr int kTop = L::kPos == 16 ? 4 : L::kPos == 32 ? 5 : 6;
  const int run_log2 = page_run_log2(p.cache.page_size, kTop);
  const bool boxes = run_log2 >= 3 && (!kI8 || (aligned16(p.cache.scales[0]) && aligned16(p.cache.scales[1])));
  p.run_log2 = boxes ? run_log2 : kTop;
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
    auto kern = boxes ? paged::attention_paged_kernel<T, kI8, D, true, kWide> : paged::attention_paged_kernel<T, kI8, D, false, kWide>;
    cudaError_t e = set_dyn_smem_once(kern, L::kSmem);
    if (e == cudaSuccess) e = launch_chained(kern, ctas, L::kThreads, L::kSmem, s, 0, map[0], map[1], static_cast<const T*>(q), static_cast<T*>(o), p);
    if (e == cudaSuccess) e = launch_chained(paged::attention_paged_merge_kernel<T, D, L::kHeld>, dim3(ctas, static_cast<unsigned>((rows + 3) / 4)), 128, 0, s, 0, static_cast<T*>(o), p);
    st = cuda_ok(err, e, "attention_paged_kernel launch");
  }
  const cudaError_t e = cudaFreeAsync(p.part, s);
  if (st == TSM100_OK && e != cudaSuccess) st = cuda_ok(err, e, "cudaFreeAsync");
  return st;
}

// More rows than a tile of mma.sync has would go over their keys again: those take tcgen05, as long as a group's heads fit a tile and boxes of eight positions a page.
template <typename T, bool kI8, int D>
inline int32_t attention_paged_launch(std::string* err, const paged::Params& p, const void* q, void* o, cudaStream_t s) {
  const int64_t rows = static_cast<int64_t>(p.step.max_new) * p.group;
  const int wide = page_run_log2(p.cache.page_size, 7);
  if (rows > paged::kRows && p.group <= paged::tc::kMaxGroup && (kI8 || wide >= 3)) return attention_paged_tc_launch<T, kI8, D>(err, p, wide, q, o, s);
  return rows > 8 ? attention_paged_few_launch<T, kI8, D, true>(err, p, q, o, s) : attention_paged_few_launch<T, kI8, D, false>(err, p, q, o, s);
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
