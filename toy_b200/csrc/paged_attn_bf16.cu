// Paged decode attention over a bf16 cache: three planes of q and of the
// weights for f32 rows (24 bits), two for 16-bit rows, whose values and
// results have no more than 11.
#include "paged_attn.cuh"

namespace tb2 {
int paged_attend_bf16(const PagedAttnArgs& a, cudaStream_t st) {
  return a.row_type == kTypeF32 ? attn::launch_type<kCacheBF16, 3>(a, st) : attn::launch_type<kCacheBF16, 2>(a, st);
}
int paged_prepare_bf16() { return attn::prepare_type<kCacheBF16, 3>() || attn::prepare_type<kCacheBF16, 2>() ? -3 : 0; }
}  // namespace tb2
