// Host-side launch logic of 8-bit products and the rows they take (gemm_i8.cuh, rows_i8.cuh); as ops_serving.cuh.
#pragma once

#include <algorithm>
#include <type_traits>

#include "args_i8.hpp"
#include "gemm_i8.cuh"
#include "launch.cuh"
#include "route.hpp"
#include "rows_i8.cuh"

namespace tsm100 {
namespace ops {

// ---------------------------------------------------------------------------
// rows in 8 bits
// ---------------------------------------------------------------------------
template <typename T, bool kGated>
inline cudaError_t rows_i8_launch(const rows_i8::Params<T>& p, cudaStream_t s) {
  namespace r8 = rows_i8;
  constexpr int PV = softmax::Elem<T>::kPerVec;
  const int64_t vecs = p.cols / PV;
  const bool vec = p.cols % PV == 0 && p.pitch % PV == 0 && aligned16(p.x) && (!kGated || aligned16(p.up)) && reinterpret_cast<uintptr_t>(p.y) % PV == 0;
  const unsigned rows = static_cast<unsigned>(p.rows);
  auto go = [&](auto kern, unsigned grid, int threads) { return launch_chained(kern, grid, threads, 0, s, 0, p); };
  // a CTA of as many warps as leave no more than VPT vectors to a thread
  const auto threads = [&](int vpt) { return static_cast<int>((vecs + 32 * vpt - 1) / (32 * vpt) * 32); };
  if (vec) {
    const unsigned warps = (rows + 7) / 8;
    if (vecs <= 32) return go(r8::rows_i8_vec_kernel<T, kGated, true, 1>, warps, 256);
    if (vecs <= 64) return go(r8::rows_i8_vec_kernel<T, kGated, true, 2>, warps, 256);
    if (vecs <= 2 * 256) return go(r8::rows_i8_vec_kernel<T, kGated, false, 2>, rows, threads(2));
    if (vecs <= 4 * r8::kMaxThreads) return go(r8::rows_i8_vec_kernel<T, kGated, false, 4>, rows, threads(4));
  }
  if (p.cols <= 4 * r8::kThreads) return go(r8::rows_i8_any_kernel<T, kGated, 4>, rows, r8::kThreads);
  if (p.cols <= 16 * r8::kThreads) return go(r8::rows_i8_any_kernel<T, kGated, 16>, rows, r8::kThreads);
  if (p.cols <= 32 * r8::kThreads) return go(r8::rows_i8_any_kernel<T, kGated, 32>, rows, r8::kThreads);
  return go(r8::rows_i8_any_kernel<T, kGated, 0>, rows, r8::kThreads);
}

template <typename T>
inline int32_t rows_i8_typed(std::string* err, const tsm100_quantise_rows_desc* d, int64_t pitch, const void* x, const void* up, int8_t* y, float* scales, cudaStream_t s) {
  rows_i8::Params<T> p;
  p.x = static_cast<const T*>(x), p.up = static_cast<const T*>(up);
  p.y = y, p.scales = scales;
  p.rows = d->rows, p.pitch = pitch, p.cols = static_cast<int32_t>(d->cols);
  return cuda_ok(err, up ? rows_i8_launch<T, true>(p, s) : rows_i8_launch<T, false>(p, s), "rows_i8 launch");
}

inline int32_t quantise_rows(std::string* err, const tsm100_quantise_rows_desc* d, const void* x, const void* up, void* y, float* scales, void* stream) {
  bool nothing;
  if (const char* what = args::quantise_rows(d, x, up, y, scales, &nothing)) return op_fail(err, TSM100_ERR_INVALID, std::string("quantise_rows: ") + what);
  if (nothing) return TSM100_OK;
  const int64_t pitch = d->pitch ? d->pitch : d->cols;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (d->dtype) {
    case TSM100_F32: return rows_i8_typed<float>(err, d, pitch, x, up, static_cast<int8_t*>(y), scales, s);
    case TSM100_BF16: return rows_i8_typed<__nv_bfloat16>(err, d, pitch, x, up, static_cast<int8_t*>(y), scales, s);
    default: return rows_i8_typed<__half>(err, d, pitch, x, up, static_cast<int8_t*>(y), scales, s);
  }
}

// ---------------------------------------------------------------------------
// 8-bit products
// ---------------------------------------------------------------------------
// What the kernels get: operands whose rows start on 16-byte boundaries.
struct GemmI8 {
  const void *a, *w;
  int64_t lda, ldw, ldc;
  int64_t m, n, k;
  const float *a_scales, *w_scales;
  uint32_t* status;
};
inline int32_t gemm_i8_tmap(std::string* err, CUtensorMap* out, const void* base, int64_t k, int64_t rows, int64_t pitch, uint32_t box_rows) {
  return make_tmap_3d(err, out, base, k, rows, 1, pitch, static_cast<uint64_t>(rows) * pitch, gemm_i8::kBK, box_rows, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1);
}

template <typename OutT, int NT>
inline int32_t gemm_i8_few_launch(std::string* err, const GemmI8& g, const route::GemmI8& plan, OutT* c, cudaStream_t s) {
  namespace k8 = gemm_i8;
  CUtensorMap ta, tw;
  int32_t st = gemm_i8_tmap(err, &ta, g.a, g.k, g.m, g.lda, NT);
  if (st == TSM100_OK) st = gemm_i8_tmap(err, &tw, g.w, g.k, g.n, g.ldw, k8::kBN);
  if (st != TSM100_OK) return st;
  k8::Params p;
  p.a_scales = g.a_scales, p.w_scales = g.w_scales;
  p.m = static_cast<int32_t>(g.m), p.n = static_cast<int32_t>(g.n), p.k = static_cast<int32_t>(g.k);
  p.m_blocks = static_cast<int32_t>(route::div_up(g.m, NT)), p.n_blocks = static_cast<int32_t>(route::div_up(g.n, k8::kBN));
  p.kb_per_cta = static_cast<int32_t>(plan.k_blocks_per_cta);
  p.ldc = g.ldc;
  p.vectors = g.n % 4 == 0 && g.ldc * sizeof(OutT) % 16 == 0 && aligned16(c);
  p.status = g.status;
  const int64_t tiles = static_cast<int64_t>(p.m_blocks) * p.n_blocks, splits = route::div_up(route::div_up(g.k, k8::kBK), p.kb_per_cta);  // a last CTA without work is dropped
  auto kern = k8::gemm_i8_few_kernel<OutT, NT>;
  constexpr int smem = k8::smem_bytes<NT>();
  cudaError_t e = set_dyn_smem_once(kern, smem);
  if (e == cudaSuccess) e = launch_chained(kern, static_cast<unsigned>(tiles * splits), k8::kThreads, smem, s, static_cast<unsigned>(splits), ta, tw, c, p);
  return cuda_ok(err, e, "gemm_i8_few_kernel launch");
}

template <typename OutT, bool kLoose>
inline int32_t gemm_i8_pairs_launch(std::string* err, const GemmI8& g, int bn, OutT* c, int sms, cudaStream_t s) {
  namespace k8 = gemm_i8::pairs;
  CUtensorMap ta, tw, tc = {};
  int32_t st = gemm_i8_tmap(err, &ta, g.a, g.k, g.m, g.lda, k8::kCtaM);
  if (st == TSM100_OK) st = gemm_i8_tmap(err, &tw, g.w, g.k, g.n, g.ldw, static_cast<uint32_t>(bn / 2));
  if (st == TSM100_OK && !kLoose)
    st = make_tmap_3d(err, &tc, c, g.n, g.m, 1, g.ldc, static_cast<uint64_t>(g.m) * g.ldc, gemm_tc::kBoxCols<OutT>, 32,
                      sizeof(OutT) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                        : std::is_same<OutT, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, sizeof(OutT));
  if (st != TSM100_OK) return st;
  k8::Params p;
  p.a_scales = g.a_scales, p.w_scales = g.w_scales;
  p.m = static_cast<int32_t>(g.m), p.n = static_cast<int32_t>(g.n), p.k = static_cast<int32_t>(g.k);
  p.bn = bn;
  p.m_blocks = static_cast<int32_t>(route::div_up(g.m, k8::kPairM)), p.n_blocks = static_cast<int32_t>(route::div_up(g.n, bn));
  p.ldc = g.ldc;
  p.status = g.status;
  auto kern = k8::gemm_i8_pairs_kernel<OutT, kLoose>;
  cudaError_t e = set_dyn_smem_once(kern, k8::kSmemBytes);
  if (e != cudaSuccess) return cuda_ok(err, e, "cudaFuncSetAttribute(gemm_i8_pairs_kernel)");
  const int max_clusters = resident_clusters(kern, k8::kThreads, k8::kSmemBytes, 2, static_cast<unsigned>(sms & ~1), sms / 2);
  const int64_t pairs = std::min<int64_t>(static_cast<int64_t>(p.m_blocks) * p.n_blocks, std::min<int64_t>(max_clusters, sms / 2));
  return cuda_ok(err, launch_chained(kern, static_cast<unsigned>(2 * pairs), k8::kThreads, k8::kSmemBytes, s, 2, ta, tw, tc, c, p), "gemm_i8_pairs_kernel launch");
}

template <typename OutT>
inline int32_t gemm_i8_typed(std::string* err, const GemmI8& g, void* c, int sms, cudaStream_t s) {
  const bool loose = !aligned16(c) || g.ldc * sizeof(OutT) % 16 != 0;
  const route::GemmI8 plan = route::gemm_i8(g.m, g.n, g.k, loose || sizeof(OutT) == 4 ? 32 : 64, sms);
  OutT* out = static_cast<OutT*>(c);
  if (plan.pairs)
    return loose ? gemm_i8_pairs_launch<OutT, true>(err, g, plan.width, out, sms, s) : gemm_i8_pairs_launch<OutT, false>(err, g, plan.width, out, sms, s);
  switch (plan.rows) {
    case 16: return gemm_i8_few_launch<OutT, 16>(err, g, plan, out, s);
    case 32: return gemm_i8_few_launch<OutT, 32>(err, g, plan, out, s);
    case 64: return gemm_i8_few_launch<OutT, 64>(err, g, plan, out, s);
    default: return gemm_i8_few_launch<OutT, 128>(err, g, plan, out, s);
  }
}

inline int32_t gemm_i8(std::string* err, const tsm100_gemm_i8_desc* d, const void* a, const float* a_scales, const void* w, const float* w_scales, void* c,
                       uint32_t* status, void* stream) {
  bool nothing;
  if (const char* what = args::gemm_i8(d, a, a_scales, w, w_scales, c, &nothing)) return op_fail(err, TSM100_ERR_INVALID, std::string("gemm_i8: ") + what);
  if (nothing) return TSM100_OK;
  GemmI8 g;
  g.m = d->m, g.n = d->n, g.k = d->k;
  g.lda = d->lda ? d->lda : d->k, g.ldw = d->ldw ? d->ldw : d->k, g.ldc = d->ldc ? d->ldc : d->n;
  g.a = a, g.w = w, g.a_scales = a_scales, g.w_scales = w_scales, g.status = status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (g.k == 0) {
    const size_t e = dtype_size(d->dtype);
    return cuda_ok(err, cudaMemset2DAsync(c, g.ldc * e, 0, g.n * e, g.m, s), "cudaMemset2DAsync");
  }
  int sms = 0;
  int32_t st = sm_count(err, &sms);
  if (st != TSM100_OK) return st;
  // rows that do not start on 16-byte boundaries are copied to where they do
  gemm_i8::Operand pa = {}, pw = {};
  uint8_t* ws = nullptr;
  const int64_t pitch = (g.k + 15) / 16 * 16;
  const bool copy_a = !aligned16(a) || g.lda % 16 != 0, copy_w = !aligned16(w) || g.ldw % 16 != 0;
  if (copy_a || copy_w) {
    const size_t a_bytes = copy_a ? static_cast<size_t>(g.m) * pitch : 0, w_bytes = copy_w ? static_cast<size_t>(g.n) * pitch : 0;
    st = take_scratch(err, reinterpret_cast<void**>(&ws), a_bytes + w_bytes, s);
    if (st == kNoScratch) return op_fail(err, TSM100_ERR_MEMORY, "gemm_i8: no device memory for rows that start on 16-byte boundaries");
    if (st != TSM100_OK) return st;
    auto operand = [&](gemm_i8::Operand& o, const void* src, void* dst, int64_t rows, int64_t ld) {
      o.src = static_cast<const uint8_t*>(src), o.dst = static_cast<uint4*>(dst), o.ld = ld;
      o.rows = static_cast<int32_t>(rows), o.cols = static_cast<int32_t>(g.k), o.pitch = static_cast<int32_t>(pitch);
      o.blocks = static_cast<int32_t>(std::min<int64_t>(route::div_up(rows * (pitch / 16), gemm_i8::kPadThreads), 8ll * sms));
    };
    if (copy_a) operand(pa, a, ws, g.m, g.lda), g.a = ws, g.lda = pitch;
    if (copy_w) operand(pw, w, ws + a_bytes, g.n, g.ldw), g.w = ws + a_bytes, g.ldw = pitch;
    st = cuda_ok(err, launch_chained(gemm_i8::gemm_i8_pad_kernel, static_cast<unsigned>(pa.blocks + pw.blocks), gemm_i8::kPadThreads, 0, s, 0, pa, pw), "gemm_i8_pad_kernel launch");
  }
  if (st == TSM100_OK) {
    switch (d->dtype) {
      case TSM100_F32: st = gemm_i8_typed<float>(err, g, c, sms, s); break;
      case TSM100_BF16: st = gemm_i8_typed<__nv_bfloat16>(err, g, c, sms, s); break;
      default: st = gemm_i8_typed<__half>(err, g, c, sms, s); break;
    }
  }
  if (ws) {
    const cudaError_t e = cudaFreeAsync(ws, s);
    if (st == TSM100_OK && e != cudaSuccess) st = cuda_ok(err, e, "cudaFreeAsync");
  }
  return st;
}

}  // namespace ops
}  // namespace tsm100
