// Attention over pages of the positions behind a shared prefix (ops_serving.cuh).
#include "ops_serving.cuh"

using namespace tsm100;

template int32_t tsm100::ops::attention_paged_keys<paged::kRest>(std::string*, const paged::Params&, bool, bool, const void*, void*, cudaStream_t);
