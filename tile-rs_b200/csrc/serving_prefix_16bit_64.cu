// Attention of sequences that begin with the same pages: a cache of 16 bits, heads of 64 (ops_paged.cuh).
#include "ops_paged.cuh"

template int32_t tsm100::ops::attention_prefix_held<false, 64>(std::string*, const paged::Params&, bool, const PrefixPlan&, const PrefixArgs&, const void*, void*, cudaStream_t);
