// Paged decode attention over an f16 cache.
#include "paged_attn.cuh"

namespace tb2 {
int paged_attend_f16(const PagedAttnArgs& a, cudaStream_t st) { return attn::launch_type<kCacheF16, 2>(a, st); }
int paged_prepare_f16() { return attn::prepare_type<kCacheF16, 2>(); }
}  // namespace tb2
