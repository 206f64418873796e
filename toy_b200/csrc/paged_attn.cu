// C entries of the paged decode attention: argument checks, the workspace and
// the choice of the cache type's kernels (paged_attn.cuh).
#include <cmath>

#include "paged_attn.cuh"

namespace tb2 {

// The factor of a score in powers of two.
static float scale_log2e(float scale) { return (float)(scale * 1.4426950408889634); }

int paged_attend_launch(const tb2_paged_kv& c, const tb2_paged_attend_args& a, int* err, cudaStream_t st) {
  PagedAttnArgs k;
  k.kv = paged_kv_of(&c);
  k.q = a.q;
  k.out = a.out;
  k.ldq = a.ldq;
  k.ldo = a.ldo;
  k.table = a.table;
  k.table_stride = a.table_stride;
  k.lens = a.lens;
  k.lse = a.lse;
  k.tickets = static_cast<unsigned*>(a.workspace);
  k.slots = reinterpret_cast<float*>(static_cast<uint8_t*>(a.workspace) + kAttnTicketBytes);
  k.err = err;
  k.c = scale_log2e(a.scale);
  k.q_vec = aligned(a.q, 16) && (a.ldq * type_bytes(a.row_type)) % 16 == 0;
  k.out_vec = aligned(a.out, 16) && (a.ldo * type_bytes(a.row_type)) % 16 == 0;
  k.n_req = a.n_req;
  k.n_heads = a.n_heads;
  k.group = a.n_heads / c.n_kv;
  k.width = a.table_width;
  k.row_type = a.row_type;
  k.page_shift = -1;
  for (int s = 0; s < 31; ++s)
    if (c.page_size == 1 << s) k.page_shift = s;
  switch (c.kv_type) {
    case kTypeF32: return paged_attend_f32(k, st);
    case kTypeF16: return paged_attend_f16(k, st);
    case kTypeBF16: return paged_attend_bf16(k, st);
    default: return paged_attend_q8(k, st);
  }
}

}  // namespace tb2

extern "C" {

size_t tb2_paged_attend_workspace(void) { return tb2::kAttnWorkspace; }

int tb2_paged_attend_workspace_init(void* workspace, size_t bytes, void* stream) {
  if (!workspace || bytes < tb2::kAttnWorkspace || !tb2::aligned(workspace, 16)) return -1;
  // the tickets are what a call expects to find at 0
  return cudaMemsetAsync(workspace, 0, tb2::kAttnTicketBytes, static_cast<cudaStream_t>(stream)) == cudaSuccess ? 0 : -3;
}

int tb2_paged_attend(const tb2_paged_kv* kv, const tb2_paged_attend_args* a, void* stream) {
  if (!tb2::paged_kv_ok(kv) || !a || a->n_req < 0 || !tb2::row_type_ok(a->row_type)) return -1;
  if (a->n_req == 0) return 0;
  const long long width = (long long)a->n_heads * kv->d_head;
  if (a->n_heads < 1 || a->n_heads % kv->n_kv || width > (1 << 24) || a->n_req > (1 << 20)) return -1;
  if (!a->q || !a->out || !a->lens || !a->table || a->ldq < width || a->ldo < width) return -1;
  const size_t e = (size_t)tb2::type_bytes(a->row_type);
  if (!tb2::aligned(a->q, e) || !tb2::aligned(a->out, e)) return -1;
  if (!tb2::all_aligned(4, {a->table, a->lens, a->lse})) return -1;
  // (positions, rounded up to whole units, are 32 bits wide)
  if (a->table_width < 1 || a->table_stride < a->table_width ||
      (long long)a->table_width * kv->page_size > 0x7fffff00LL)
    return -1;
  // (the units of every table row filled, at the smallest unit, are numbered in 31 bits)
  const long long tiles_h = (a->n_heads / kv->n_kv + 7) / 8;
  if ((((long long)a->table_width * kv->page_size + 31) / 32) * kv->n_kv * tiles_h > 0x7fffffffLL / a->n_req) return -1;
  if (!std::isfinite(a->scale) || !std::isfinite(tb2::scale_log2e(a->scale))) return -1;
  if (!a->workspace || a->workspace_bytes < tb2::kAttnWorkspace || !tb2::aligned(a->workspace, 16)) return -1;
  int* err = tb2::device_error_word();
  if (!err) return -3;
  return tb2::paged_attend_launch(*kv, *a, err, static_cast<cudaStream_t>(stream));
}

int tb2_paged_prepare(void) {
  using namespace tb2;
  if (!device_error_word() || paged_plan_prepare() || paged_append_prepare()) return -3;
  return paged_prepare_f32() || paged_prepare_f16() || paged_prepare_bf16() || paged_prepare_q8() ? -3 : 0;
}

}  // extern "C"
