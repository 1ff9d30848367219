// Host-side launch logic of the attentions over pages: arguments that they have in common and the kernels' launches, as templates, so that a translation unit compiles those that it
// instantiates (serving.cu, serving_cross_*.cu, serving_prefix_*.cu).  As ops.cuh: nothing here synchronises and every function answers a TSM100_* status with a message in *err.
#pragma once

#include <algorithm>
#include <cmath>
#include <utility>

#include "attention_paged.cuh"
#include "attention_paged_rows.cuh"
#include "attention_paged_tc.cuh"
#include "kv_pages.cuh"
#include "launch.cuh"
#include "route.hpp"

namespace tsm100 {
namespace ops {

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

// What the attentions over pages ask of their arguments.  *nothing: there are no tokens.
inline int32_t attention_paged_args(std::string* err, const char* op, const tsm100_paged_kv* kv, const tsm100_paged_batch* b, int32_t dtype, int32_t heads_q, const void* q,
                                    const void* o, uint32_t* status, paged::Params* p, bool* nothing) {
  auto no = [&](const char* what) { return op_fail(err, TSM100_ERR_INVALID, std::string(op) + ": " + what); };
  const int32_t st = paged_args(err, op, kv, b, dtype, &p->cache, &p->step, nothing);
  if (st != TSM100_OK) return st;
  if (kv->head_dim != 64 && kv->head_dim != 128) return no("head_dim must be 64 or 128");
  if (heads_q <= 0 || heads_q % kv->heads_kv != 0) return no("heads_q must be a positive multiple of heads_kv");
  if (*nothing) return TSM100_OK;
  if (!q || !o) return no("null buffer");
  if (!aligned16(q) || !aligned16(o)) return no("q and o must be 16-byte aligned");
  if (static_cast<int64_t>(b->tokens) * heads_q > 0x7fffffff) return no("too many tokens times heads");
  p->heads_q = heads_q;
  p->group = heads_q / kv->heads_kv;
  p->scale_log2 = static_cast<float>((1.0 / std::sqrt(static_cast<double>(kv->head_dim))) * 1.4426950408889634);
  p->status = status;
  return TSM100_OK;
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
struct PrefixArgs {  // of the attentions that leave records (attention_paged_rows.cuh)
  int32_t prefix, large;
  const int32_t* table;
  paged::Records shared, rest;
};
template <typename T, bool kI8, int D, paged::Keys kKeys>
inline int32_t attention_paged_tc_launch(std::string* err, const paged::Params& base, int run_log2, const void* q, void* o, cudaStream_t s, const PrefixArgs& more = PrefixArgs()) {
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
  p.prefix = more.prefix, p.large = more.large, p.prefix_table = more.table;
  p.records = kKeys == paged::kShared ? more.shared : more.rest;
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
  auto kern = tc::attention_paged_tc_kernel<kIsBf16, kI8, D, kKeys>;
  constexpr int smem = tc::smem_bytes<kI8, D>();
  cudaError_t e = set_dyn_smem_once(kern, smem);
  if constexpr (paged::leaves_records(kKeys)) {
    p.part = nullptr, p.part_ml = nullptr, p.info = nullptr;
    if (e == cudaSuccess) e = launch_chained(kern, ctas, S::kThreads, smem, s, 0, tq, tk, tv, static_cast<uint16_t*>(o), p);
    return cuda_ok(err, e, "attention_paged_tc_kernel launch");
  } else {
    const size_t rows = static_cast<size_t>(ctas) * 2 * 256, part = rows * D * sizeof(float), ml = rows * sizeof(float2);
    uint8_t* ws = nullptr;
    st = take_scratch(err, reinterpret_cast<void**>(&ws), part + ml + ctas * sizeof(int4), s);
    if (st == kNoScratch)
      return op_fail(err, TSM100_ERR_MEMORY, kKeys == paged::kAll ? "attention_paged_cross: no device memory for partial results" : "attention_paged: no device memory for partial results");
    if (st != TSM100_OK) return st;
    p.part = reinterpret_cast<float4*>(ws);
    p.part_ml = reinterpret_cast<float2*>(ws + part);
    p.info = reinterpret_cast<int4*>(ws + part + ml);
    if (e == cudaSuccess) e = launch_chained(kern, ctas, S::kThreads, smem, s, 0, tq, tk, tv, static_cast<uint16_t*>(o), p);
    if (e == cudaSuccess) e = launch_chained(tc::attention_paged_tc_merge_kernel<kIsBf16, D, kKeys>, dim3(ctas, D / 16), 256, 0, s, 0, static_cast<uint16_t*>(o), p);
    st = cuda_ok(err, e, "attention_paged_tc_kernel launch");
    e = cudaFreeAsync(ws, s);
    if (st == TSM100_OK && e != cudaSuccess) st = cuda_ok(err, e, "cudaFreeAsync");
    return st;
  }
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
inline bool paged_fits_tcgen05(int group, bool i8, int run_log2) { return group <= paged::tc::kMaxGroup && (i8 || run_log2 >= 3); }
template <typename T, bool kI8, int D>
inline int32_t attention_paged_launch(std::string* err, const paged::Params& p, const void* q, void* o, cudaStream_t s) {
  const int64_t rows = static_cast<int64_t>(p.step.max_new) * p.group;
  const int wide = page_run_log2(p.cache.page_size, 7);
  if (rows > paged::kRows && paged_fits_tcgen05(p.group, kI8, wide)) return attention_paged_tc_launch<T, kI8, D, paged::kPast>(err, p, wide, q, o, s);
  return rows > 8 ? attention_paged_few_launch<T, kI8, D, true>(err, p, q, o, s) : attention_paged_few_launch<T, kI8, D, false>(err, p, q, o, s);
}

template <typename T>
inline int32_t attention_paged_typed(std::string* err, const paged::Params& p, bool i8, const void* q, void* o, cudaStream_t s) {
  if (p.cache.d == 128) return i8 ? attention_paged_launch<T, true, 128>(err, p, q, o, s) : attention_paged_launch<T, false, 128>(err, p, q, o, s);
  return i8 ? attention_paged_launch<T, true, 64>(err, p, q, o, s) : attention_paged_launch<T, false, 64>(err, p, q, o, s);
}

// ---------------------------------------------------------------------------
// records of rows, joined: cross attention of few rows, and sequences that begin with the same pages
// ---------------------------------------------------------------------------
template <typename T, bool kI8, int D, bool kWide, paged::Keys kKeys>
inline int32_t attention_rows_launch(std::string* err, const paged::Params& base, const PrefixArgs& more, const void* q, cudaStream_t s) {
  using L = paged::RowsTile<kI8, D, kWide>;
  int sms = 0;
  int32_t st = sm_count(err, &sms);
  if (st != TSM100_OK) return st;
  paged::RowsParams p;
  p.cache = base.cache, p.step = base.step;
  p.heads_q = base.heads_q, p.group = base.group;
  p.scale_log2 = base.scale_log2;
  p.prefix = more.prefix, p.large = more.large, p.prefix_table = more.table;
  p.shared = more.shared, p.rest = more.rest;
  p.status = base.status;
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
  if (st != TSM100_OK) return st;
  auto kern = boxes ? paged::attention_paged_rows_kernel<T, kI8, D, true, kWide, kKeys> : paged::attention_paged_rows_kernel<T, kI8, D, false, kWide, kKeys>;
  cudaError_t e = set_dyn_smem_once(kern, L::kSmem);
  if (e == cudaSuccess)
    e = launch_chained(kern, static_cast<unsigned>(std::min(sms, paged::kMaxCtas)), L::kThreads, L::kSmem, s, 0, map[0], map[1], static_cast<const T*>(q), p);
  return cuda_ok(err, e, "attention_paged_rows_kernel launch");
}
// `records`: about how many a row has.
template <typename T, int D>
inline int32_t attention_join_launch(std::string* err, const paged::Join& join, int64_t records, void* o, cudaStream_t s) {
  int sms = 0;
  const int32_t st = sm_count(err, &sms);
  if (st != TSM100_OK) return st;
  auto go = [&](auto kern, int splits, int threads) {
    const int64_t at_once = threads / (D / 4) / splits, rows = static_cast<int64_t>(join.step.max_new) * join.heads_q;
    const dim3 grid(static_cast<unsigned>(join.step.batch), static_cast<unsigned>(route::join_ctas(rows, at_once, join.step.batch, 1024 / threads, sms)));
    return cuda_ok(err, launch_chained(kern, grid, threads, 0, s, 0, static_cast<T*>(o), join), "attention_paged_join_kernel launch");
  };
  return records > 40 ? go(paged::attention_paged_join_kernel<T, D, 16>, 16, paged::kJoinThreads<16>) : go(paged::attention_paged_join_kernel<T, D, 4>, 4, paged::kJoinThreads<4>);
}
// What both need: scratch for `whole` arrays of records, `part` bytes of cut ones and `cuts` places.
struct RecordSpace {
  uint8_t *base = nullptr, *at = nullptr;
  float* floats(size_t bytes) { return reinterpret_cast<float*>(std::exchange(at, at + bytes)); }
  int2* places(size_t n) { return reinterpret_cast<int2*>(std::exchange(at, at + n * sizeof(int2))); }
};
inline int32_t take_records(std::string* err, const char* op, RecordSpace* x, size_t bytes, cudaStream_t s) {
  const int32_t st = take_scratch(err, reinterpret_cast<void**>(&x->base), bytes, s);
  if (st == kNoScratch) return op_fail(err, TSM100_ERR_MEMORY, std::string(op) + ": no device memory for partial results");
  x->at = x->base;
  return st;
}
inline int32_t give_records(std::string* err, const RecordSpace& x, cudaStream_t s, int32_t st) {
  const cudaError_t e = cudaFreeAsync(x.base, s);
  return st == TSM100_OK && e != cudaSuccess ? cuda_ok(err, e, "cudaFreeAsync") : st;
}
// Bytes of the places that shares of the warps of all CTAs have for what they cut.
template <bool kI8, int D, bool kWide>
inline size_t rows_part_bytes(int64_t ctas) {
  using L = paged::RowsTile<kI8, D, kWide>;
  return static_cast<size_t>(ctas) * L::kWarps * 2 * L::kHeld * L::kRec * sizeof(float);
}
inline paged::Join join_of(const paged::Params& p) {
  paged::Join x;
  std::memset(&x, 0, sizeof x);
  x.cache = p.cache, x.step = p.step;
  x.heads_q = p.heads_q, x.group = p.group;
  return x;
}

// Every token against all positions of its sequence (serving_cross_16bit.cu, serving_cross_i8.cu).
template <typename T, bool kI8, int D, bool kWide>
inline int32_t attention_cross_rows(std::string* err, const paged::Params& p, const void* q, void* o, cudaStream_t s) {
  using L = paged::RowsTile<kI8, D, kWide>;
  int sms = 0;
  int32_t st = sm_count(err, &sms);
  if (st != TSM100_OK) return st;
  const int64_t ctas = std::min(sms, paged::kMaxCtas), units = (static_cast<int64_t>(p.step.max_new) * p.group + L::kHeld - 1) / L::kHeld;
  const size_t whole = static_cast<size_t>(p.step.tokens) * p.heads_q * L::kRec * sizeof(float), part = rows_part_bytes<kI8, D, kWide>(ctas);
  const size_t cuts = static_cast<size_t>(p.step.batch) * p.cache.heads * units;
  RecordSpace space;
  st = take_records(err, "attention_paged_cross", &space, whole + part + cuts * sizeof(int2), s);
  if (st != TSM100_OK) return st;
  PrefixArgs more = {};
  more.rest.whole = space.floats(whole), more.rest.part = space.floats(part), more.rest.cut = space.places(cuts);
  more.rest.units = static_cast<int32_t>(units), more.rest.shares = static_cast<int32_t>(ctas * L::kWarps);
  paged::Join join = join_of(p);
  join.all = 1, join.rest = more.rest, join.rest_held = L::kHeld;
  st = attention_rows_launch<T, kI8, D, kWide, paged::kAll>(err, p, more, q, s);
  if (st == TSM100_OK) st = attention_join_launch<T, D>(err, join, ctas * L::kWarps / static_cast<int64_t>(cuts), o, s);
  return give_records(err, space, s, st);
}
template <typename T, bool kI8, int D>
inline int32_t attention_cross_launch(std::string* err, const paged::Params& p, const void* q, void* o, cudaStream_t s) {
  const int64_t rows = static_cast<int64_t>(p.step.max_new) * p.group;
  const int wide = page_run_log2(p.cache.page_size, 7);
  if (rows > paged::kRows && paged_fits_tcgen05(p.group, kI8, wide)) return attention_paged_tc_launch<T, kI8, D, paged::kAll>(err, p, wide, q, o, s);
  return rows > 8 ? attention_cross_rows<T, kI8, D, true>(err, p, q, o, s) : attention_cross_rows<T, kI8, D, false>(err, p, q, o, s);
}
template <bool kI8>
int32_t attention_cross_held(std::string* err, const paged::Params& p, bool bf16, const void* q, void* o, cudaStream_t s) {
  if (p.cache.d == 128) return bf16 ? attention_cross_launch<__nv_bfloat16, kI8, 128>(err, p, q, o, s) : attention_cross_launch<__half, kI8, 128>(err, p, q, o, s);
  return bf16 ? attention_cross_launch<__nv_bfloat16, kI8, 64>(err, p, q, o, s) : attention_cross_launch<__half, kI8, 64>(err, p, q, o, s);
}
extern template int32_t attention_cross_held<false>(std::string*, const paged::Params&, bool, const void*, void*, cudaStream_t);
extern template int32_t attention_cross_held<true>(std::string*, const paged::Params&, bool, const void*, void*, cudaStream_t);

// All tokens against the prefix and each against its own positions, both as records, and then those joined.  Translation units by cache and head size
// (serving_prefix*.cu).
struct PrefixPlan {
  bool shared_tc;  // the prefix on tcgen05, else in one stream with the rest
  bool rest_tc;    // so are sequences of many rows
  int run_log2;    // boxes of pages for tcgen05
};
template <typename T, bool kI8, int D>
inline int32_t attention_prefix_launch(std::string* err, const paged::Params& p, const PrefixPlan& plan, PrefixArgs more, const void* q, void* o, cudaStream_t s) {
  namespace pg = paged;
  constexpr size_t REC = pg::kRecord<D>;
  int sms = 0;
  int32_t st = sm_count(err, &sms);
  if (st != TSM100_OK) return st;
  const int64_t ctas = std::min(sms, pg::kMaxCtas), heads = p.cache.heads;
  const int32_t tile_tokens = pg::tc::kTileRows / p.group;
  // the rows of a unit: what a sequence has, unless the prefix's, which are all tokens', are in the same stream
  const bool wide = !plan.shared_tc || static_cast<int64_t>(p.step.max_new) * p.group > 8;
  const int held = wide ? 16 : 8;
  pg::Join join = join_of(p);
  join.prefix = more.prefix, join.large = more.large;
  join.shared_tokens = plan.shared_tc ? tile_tokens : 0, join.large_tokens = tile_tokens;
  join.shared_held = join.rest_held = held;
  auto units = [&](bool tc, int64_t tokens) { return tc ? (tokens + 2 * tile_tokens - 1) / (2 * tile_tokens) : (tokens * p.group + held - 1) / held; };
  const int64_t shared_units = units(plan.shared_tc, p.step.tokens), rest_units = units(false, plan.rest_tc ? more.large / p.group : p.step.max_new);
  const int64_t large_units = plan.rest_tc ? units(true, p.step.max_new) : 0;
  const size_t rows_part = wide ? rows_part_bytes<kI8, D, true>(ctas) : rows_part_bytes<kI8, D, false>(ctas), tc_part = static_cast<size_t>(ctas) * 2 * 256 * REC * sizeof(float);
  const size_t whole = static_cast<size_t>(p.step.tokens) * p.heads_q * REC * sizeof(float), cuts = heads * (shared_units + p.step.batch * (rest_units + large_units));
  RecordSpace space;
  st = take_records(err, "attention_paged_prefix", &space, 2 * whole + rows_part + (plan.shared_tc ? tc_part : 0) + (plan.rest_tc ? tc_part : 0) + cuts * sizeof(int2), s);
  if (st != TSM100_OK) return st;
  join.shared.whole = space.floats(whole), join.rest.whole = join.rest_large.whole = space.floats(whole);
  join.rest.part = space.floats(rows_part);
  join.shared.part = plan.shared_tc ? space.floats(tc_part) : join.rest.part;  // a share's two places are for whatever it has cut
  join.rest_large.part = plan.rest_tc ? space.floats(tc_part) : nullptr;
  join.shared.cut = space.places(heads * shared_units), join.rest.cut = space.places(heads * p.step.batch * rest_units);
  join.rest_large.cut = space.places(heads * p.step.batch * large_units);
  join.shared.units = static_cast<int32_t>(shared_units), join.rest.units = static_cast<int32_t>(rest_units), join.rest_large.units = static_cast<int32_t>(large_units);
  join.rest.shares = static_cast<int32_t>(ctas) * (wide ? pg::RowsTile<kI8, D, true>::kWarps : pg::RowsTile<kI8, D, false>::kWarps);
  join.shared.shares = plan.shared_tc ? static_cast<int32_t>(ctas) : join.rest.shares, join.rest_large.shares = static_cast<int32_t>(ctas);
  more.shared = join.shared, more.rest = join.rest;
  if (plan.shared_tc) {
    st = attention_paged_tc_launch<T, kI8, D, pg::kShared>(err, p, plan.run_log2, q, o, s, more);
    if (st == TSM100_OK) st = wide ? attention_rows_launch<T, kI8, D, true, pg::kRest>(err, p, more, q, s) : attention_rows_launch<T, kI8, D, false, pg::kRest>(err, p, more, q, s);
  } else {
    st = attention_rows_launch<T, kI8, D, true, pg::kBoth>(err, p, more, q, s);
  }
  if (st == TSM100_OK && plan.rest_tc) {
    more.rest = join.rest_large;
    st = attention_paged_tc_launch<T, kI8, D, pg::kRest>(err, p, plan.run_log2, q, o, s, more);
  }
  const int64_t tiles = more.prefix / pg::RowsTile<kI8, D, true>::kPos;
  const int64_t records = plan.shared_tc ? ctas / (heads * shared_units) : std::min<int64_t>(ctas * 8 / (heads * shared_units), tiles / pg::kRowsMinShare);
  if (st == TSM100_OK) st = attention_join_launch<T, D>(err, join, records, o, s);
  return give_records(err, space, s, st);
}
template <bool kI8, int D>
int32_t attention_prefix_held(std::string* err, const paged::Params& p, bool bf16, const PrefixPlan& plan, const PrefixArgs& more, const void* q, void* o, cudaStream_t s) {
  return bf16 ? attention_prefix_launch<__nv_bfloat16, kI8, D>(err, p, plan, more, q, o, s) : attention_prefix_launch<__half, kI8, D>(err, p, plan, more, q, o, s);
}
extern template int32_t attention_prefix_held<false, 64>(std::string*, const paged::Params&, bool, const PrefixPlan&, const PrefixArgs&, const void*, void*, cudaStream_t);
extern template int32_t attention_prefix_held<false, 128>(std::string*, const paged::Params&, bool, const PrefixPlan&, const PrefixArgs&, const void*, void*, cudaStream_t);
extern template int32_t attention_prefix_held<true, 64>(std::string*, const paged::Params&, bool, const PrefixPlan&, const PrefixArgs&, const void*, void*, cudaStream_t);
extern template int32_t attention_prefix_held<true, 128>(std::string*, const paged::Params&, bool, const PrefixPlan&, const PrefixArgs&, const void*, void*, cudaStream_t);

}  // namespace ops
}  // namespace tsm100
