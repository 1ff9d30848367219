// C-ABI operators around the intrinsics in a serving step: tsm100_add_rms_norm / _gemm_w4 / _kv_page_append / _kv_page_read / _attention_paged.
#include "common.hpp"
#include "ops_serving.cuh"
#include "ops_w4.cuh"

using namespace tsm100;

namespace {

// Runs `op` with dev's CUDA device current; an exception (memory for a message) ends here.
template <typename F>
int32_t on_device(tsm100_device_t dev, F op) {
  const int32_t st = use_device(dev);
  if (st != TSM100_OK) return st;
  try {
    std::string err;
    const int32_t r = op(&err);
    if (r != TSM100_OK && !err.empty()) last_error_ref() = err;  // an operator called on the way has left its own
    return r;
  } catch (...) {
    return TSM100_ERR_RUNTIME;
  }
}

}  // namespace

extern "C" {

int32_t tsm100_add_rms_norm(tsm100_device_t dev, const tsm100_add_rms_norm_desc* desc, const void* x, const void* residual, void* sum,
                            const void* weight, void* y, float* scales, void* stream) {
  return on_device(dev, [&](std::string* err) { return ops::add_rms_norm(err, desc, x, residual, sum, weight, y, scales, stream); });
}

int32_t tsm100_gemm_w4(tsm100_device_t dev, const tsm100_gemm_w4_desc* desc, const void* a, const float* a_scales, const uint8_t* w, const void* w_scales,
                       const uint8_t* w_zeros, void* c, void* stream) {
  return on_device(dev, [&](std::string* err) {
    return ops::gemm_w4(err, desc, a, a_scales, w, w_scales, w_zeros, c, dev->status, stream,
                        [&](const tsm100_gemm_desc* g, const void* x, const void* y, void* z) { return tsm100_gemm(dev, g, x, y, z, stream); });
  });
}

int32_t tsm100_kv_page_append(tsm100_device_t dev, const tsm100_paged_kv* kv, const tsm100_paged_batch* batch, int32_t dtype, const void* k, const void* v,
                              void* stream) {
  return on_device(dev, [&](std::string* err) {
    return ops::kv_page_rows<false>(err, kv, batch, dtype, const_cast<void*>(k), const_cast<void*>(v), dev->status, stream);
  });
}

int32_t tsm100_kv_page_read(tsm100_device_t dev, const tsm100_paged_kv* kv, const tsm100_paged_batch* batch, int32_t dtype, void* k, void* v, void* stream) {
  return on_device(dev, [&](std::string* err) { return ops::kv_page_rows<true>(err, kv, batch, dtype, k, v, dev->status, stream); });
}

int32_t tsm100_attention_paged(tsm100_device_t dev, const tsm100_paged_kv* kv, const tsm100_paged_batch* batch, const tsm100_attention_paged_desc* desc,
                               const void* q, void* o, void* stream) {
  return on_device(dev, [&](std::string* err) { return ops::attention_paged(err, kv, batch, desc, q, o, dev->status, stream); });
}

}  // extern "C"
