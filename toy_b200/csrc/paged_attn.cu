// Attention of one new token per request over a paged key-value cache.
//
//   out[b][h] = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale q . k_t - m),
//
// t over the request's history through its block table, m a running maximum,
// j = h / (H / KV) the key head of query head h. The sums are f32.
#include <cmath>

#include "paged.cuh"
#include "pdl.cuh"
#include "runtime.cuh"

namespace tb2 {
namespace {

constexpr int kKeys = 128;   // keys per pass of a CTA, one per thread

template <class C>
__device__ __forceinline__ float cache_val(const void* x, const uint16_t* s, long long at) {
  if constexpr (sizeof(C) > 1)
    return to_f32<C>(static_cast<const C*>(x)[at]);
  else
    return __half2float(__ushort_as_half(s[at / 32])) * (float)static_cast<const int8_t*>(x)[at];
}

// One CTA per (request, query head), its keys 128 at a time.
template <class T, class C>
__global__ void __launch_bounds__(kKeys) paged_attend_kernel(const PagedKv kv, const tb2_paged_attend_args a,
                                                             int* err) {
  __shared__ float qs[128], ps[kKeys], red[kKeys / 32];
  __shared__ long long at[kKeys];
  griddep_wait_release();
  const int b = blockIdx.x / a.n_heads, h = blockIdx.x % a.n_heads, j = h / (a.n_heads / kv.n_kv);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, dh = kv.dh;
  const long long most = (long long)a.table_width * kv.page_size;
  const int len = (int)min(most, (long long)max(0, a.lens[b]));
  if (tid < dh) qs[tid] = to_f32<T>(static_cast<const T*>(a.q)[b * a.ldq + h * dh + tid]);
  float m = -INFINITY, l = 0.f, o = 0.f;
  __syncthreads();
  for (int t0 = 0; t0 < len; t0 += kKeys) {
    const int t = t0 + tid;
    float s = -INFINITY;
    long long row = -1;
    if (t < len) {
      const int page = a.table[b * a.table_stride + t / kv.page_size];
      if (page >= 0 && page < kv.n_pages) {
        row = page * kv.page_stride + j * kv.head_stride + (t % kv.page_size) * kv.tok_stride;
        float acc = 0.f;
        for (int d = 0; d < dh; ++d) acc = fmaf(qs[d], cache_val<C>(kv.k, kv.ks, row + d), acc);
        s = acc * a.scale;
      } else {
        *err = kErrPagedPage;
      }
    }
    at[tid] = row;
    float x = s;
    for (int w = 16; w; w >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, w));
    if (lane == 0) red[warp] = x;
    __syncthreads();
    float mt = m;
    for (int w = 0; w < kKeys / 32; ++w) mt = fmaxf(mt, red[w]);
    const float p = s == -INFINITY ? 0.f : expf(s - mt);
    ps[tid] = p;
    x = p;
    for (int w = 16; w; w >>= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
    __syncthreads();
    if (lane == 0) red[warp] = x;
    __syncthreads();
    const float keep = m == -INFINITY ? 0.f : expf(m - mt);
    l *= keep;
    for (int w = 0; w < kKeys / 32; ++w) l += red[w];
    o *= keep;
    if (tid < dh)
      for (int k = 0; k < min(kKeys, len - t0); ++k)
        if (at[k] >= 0) o = fmaf(ps[k], cache_val<C>(kv.v, kv.vs, at[k] + tid), o);
    m = mt;
    __syncthreads();
  }
  if (tid < dh) static_cast<T*>(a.out)[b * a.ldo + h * dh + tid] = from_f32<T>(l == 0.f ? 0.f : o / l);
  if (tid == 0 && a.lse) a.lse[(long long)b * a.n_heads + h] = l == 0.f ? -INFINITY : m + logf(l);
}

template <class T, class C>
int launch(const tb2_paged_kv& c, const tb2_paged_attend_args& a, int* err, cudaStream_t st) {
  return launch_pdl(paged_attend_kernel<T, C>, dim3(a.n_req * a.n_heads), dim3(kKeys), 0, st, paged_kv_of(&c), a, err);
}

template <class T>
int launch_cache(const tb2_paged_kv& c, const tb2_paged_attend_args& a, int* err, cudaStream_t st) {
  switch (c.kv_type) {
    case kTypeF32: return launch<T, float>(c, a, err, st);
    case kTypeF16: return launch<T, __half>(c, a, err, st);
    case kTypeBF16: return launch<T, __nv_bfloat16>(c, a, err, st);
    default: return launch<T, int8_t>(c, a, err, st);
  }
}

constexpr size_t kWorkspace = 16;

}  // namespace

int paged_attend_launch(const tb2_paged_kv& c, const tb2_paged_attend_args& a, int* err, cudaStream_t st) {
  switch (a.row_type) {
    case kTypeF32: return launch_cache<float>(c, a, err, st);
    case kTypeF16: return launch_cache<__half>(c, a, err, st);
    default: return launch_cache<__nv_bfloat16>(c, a, err, st);
  }
}

}  // namespace tb2

extern "C" {

size_t tb2_paged_attend_workspace(void) { return tb2::kWorkspace; }

int tb2_paged_attend_workspace_init(void* workspace, size_t bytes, void* stream) {
  if (!workspace || bytes < tb2::kWorkspace || !tb2::aligned(workspace, 16)) return -1;
  return cudaMemsetAsync(workspace, 0, tb2::kWorkspace, static_cast<cudaStream_t>(stream)) == cudaSuccess ? 0 : -3;
}

int tb2_paged_attend(const tb2_paged_kv* kv, const tb2_paged_attend_args* a, void* stream) {
  if (!tb2::paged_kv_ok(kv) || !a || a->n_req < 0 || !tb2::row_type_ok(a->row_type)) return -1;
  if (a->n_req == 0) return 0;
  const long long width = (long long)a->n_heads * kv->d_head;
  if (a->n_heads < 1 || a->n_heads % kv->n_kv || width > (1 << 24) || a->n_req > (1 << 20)) return -1;
  if (!a->q || !a->out || !a->lens || !a->table || a->ldq < width || a->ldo < width) return -1;
  const size_t e = (size_t)tb2::type_bytes(a->row_type);
  if (!tb2::aligned(a->q, e) || !tb2::aligned(a->out, e)) return -1;
  if (a->table_width < 1 || a->table_stride < a->table_width ||
      (long long)a->table_width * kv->page_size > 0x7fffffffLL)
    return -1;
  if (!std::isfinite(a->scale)) return -1;
  if (!a->workspace || a->workspace_bytes < tb2::kWorkspace || !tb2::aligned(a->workspace, 16)) return -1;
  int* err = tb2::device_error_word();
  if (!err) return -3;
  return tb2::paged_attend_launch(*kv, *a, err, static_cast<cudaStream_t>(stream));
}

int tb2_paged_prepare(void) { return tb2::device_error_word() ? 0 : -3; }

}  // extern "C"
