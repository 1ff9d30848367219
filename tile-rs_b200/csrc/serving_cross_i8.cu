// Attention over all positions of a sequence's pages: a cache of 8 bits (ops_paged.cuh).
#include "ops_paged.cuh"

template int32_t tsm100::ops::attention_cross_held<true>(std::string*, const paged::Params&, bool, const void*, void*, cudaStream_t);
