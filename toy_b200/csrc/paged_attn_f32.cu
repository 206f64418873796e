// Paged decode attention over an f32 cache.
#include "paged_attn.cuh"

namespace tb2 {
int paged_attend_f32(const PagedAttnArgs& a, cudaStream_t st) { return attn::launch_type<kCacheF32, 2>(a, st); }
int paged_prepare_f32() { return attn::prepare_type<kCacheF32, 2>(); }
}  // namespace tb2
