// C-ABI operators of 8-bit products: tsm100_quantise_rows / _gemm_i8.
#include "common.hpp"
#include "on_device.hpp"
#include "ops_i8.cuh"

using namespace tsm100;

extern "C" {

int32_t tsm100_quantise_rows(tsm100_device_t dev, const tsm100_quantise_rows_desc* desc, const void* x, const void* up, void* y, float* scales, void* stream) {
  return on_device(dev, [&](std::string* err) { return ops::quantise_rows(err, desc, x, up, y, scales, stream); });
}

int32_t tsm100_gemm_i8(tsm100_device_t dev, const tsm100_gemm_i8_desc* desc, const void* a, const float* a_scales, const void* w, const float* w_scales,
                       void* c, void* stream) {
  return on_device(dev, [&](std::string* err) { return ops::gemm_i8(err, desc, a, a_scales, w, w_scales, c, dev->status, stream); });
}

}  // extern "C"
