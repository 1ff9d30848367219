// Products with 4-bit weights, scales and results in bf16 (ops_w4.cuh).
#include "ops_w4.cuh"

template int32_t tsm100::ops::gemm_w4_typed<__nv_bfloat16>(std::string*, const tsm100_gemm_w4_desc*, const uint8_t*, const w4::Params&, cudaStream_t);
