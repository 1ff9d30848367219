// Attention over pages of all positions of a sequence (ops_serving.cuh).
#include "ops_serving.cuh"

using namespace tsm100;

template int32_t tsm100::ops::attention_paged_keys<paged::kAll>(std::string*, const paged::Params&, bool, bool, const void*, void*, cudaStream_t);
