// Paged decode attention over an Q8_0 cache.
#include "paged_attn.cuh"

namespace tb2 {
int paged_attend_q8(const PagedAttnArgs& a, cudaStream_t st) { return attn::launch_type<kCacheQ8, 2>(a, st); }
int paged_prepare_q8() { return attn::prepare_type<kCacheQ8, 2>(); }
}  // namespace tb2
