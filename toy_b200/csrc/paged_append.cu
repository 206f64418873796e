// A step's new rows into the paged cache: bias, NEOX RoPE on q and k, k and v
// into their slots' page rows in the cache's type.
//
// Arithmetic (the same for every type): x + bias, then for the pair
// (a, b) = (x_e, x_{e + d_head / 2}) and the table's (c, s)
//   a' = a c - b s,   b' = a s + b c,
// products and sums rounded to f32 one by one (no contraction, so that a host
// can reproduce the Q8_0 bytes), then one rounding to the row's or the cache's
// type; Q8_0 as ggml's quantiser: d = amax / 127 per 32 values, kept as fp16,
// q = round-half-away(x * (1 / d)).
#include "paged.cuh"
#include "pdl.cuh"
#include "runtime.cuh"

namespace tb2 {
namespace {

// ggml's Q8_0 rounding: round half away from zero
__device__ __forceinline__ int round_away(float v) {
  const float t = truncf(v);
  const int ti = (int)t;
  return fabsf(__fsub_rn(v, t)) >= 0.5f ? (v < 0.f ? ti - 1 : ti + 1) : ti;
}

// grid (tokens, n_heads + n_kv), one thread per element of a head: q heads,
// then key heads, each with its value head.
template <class T, class C>
__global__ void paged_append_kernel(const PagedKv kv, const tb2_paged_append_args a, int* err) {
  __shared__ float sh[128];
  griddep_wait_release();
  const int i = blockIdx.x, t = threadIdx.x, dh = kv.dh, half = dh / 2;
  const int H = a.q ? a.n_heads : 0;
  const bool is_q = (int)blockIdx.y < H;
  const int j = is_q ? blockIdx.y : blockIdx.y - H;
  const int c0 = is_q ? j * dh : (a.n_heads + j) * dh;   // bias column
  const T* row = is_q ? static_cast<const T*>(a.q) + i * a.ldq : static_cast<const T*>(a.k) + i * a.ldk;
  float x = to_f32<T>(row[j * dh + t]);
  if (a.bias) x = __fadd_rn(x, a.bias[c0 + t]);
  if (a.rope) {
    const int p = a.positions[i];
    if (p < 0 || p >= a.rope_rows) {
      if (t == 0) *err = kErrPagedPosition;
      return;
    }
    sh[t] = x;
    __syncthreads();
    const int e = t < half ? t : t - half;
    const float2 cs = reinterpret_cast<const float2*>(a.rope)[(long long)p * half + e];
    x = t < half ? __fsub_rn(__fmul_rn(sh[t], cs.x), __fmul_rn(sh[t + half], cs.y))
                 : __fadd_rn(__fmul_rn(sh[t - half], cs.y), __fmul_rn(sh[t], cs.x));
  }
  if (is_q) {
    (static_cast<T*>(a.q_out) + i * a.ldqo)[j * dh + t] = from_f32<T>(x);
    return;
  }
  float v = to_f32<T>((static_cast<const T*>(a.v) + i * a.ldv)[j * dh + t]);
  if (a.bias) v = __fadd_rn(v, a.bias[(a.n_heads + kv.n_kv + j) * dh + t]);
  const long long slot = a.slots[i];
  if (slot < 0) return;
  const long long page = slot / kv.page_size;
  if (page >= kv.n_pages) {
    if (t == 0) *err = kErrPagedSlot;
    return;
  }
  const long long at =
      page * kv.page_stride + j * kv.head_stride + (slot - page * kv.page_size) * kv.tok_stride + t;
  if constexpr (sizeof(C) > 1) {
    static_cast<C*>(kv.k)[at] = from_f32<C>(x);
    static_cast<C*>(kv.v)[at] = from_f32<C>(v);
  } else {
    for (int w = 0; w < 2; ++w) {
      const float val = w ? v : x;
      float amax = fabsf(val);
#pragma unroll
      for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      const float d = __fdiv_rn(amax, 127.0f);
      const float id = d != 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
      static_cast<int8_t*>(w ? kv.v : kv.k)[at] = (int8_t)round_away(__fmul_rn(val, id));
      if ((t & 31) == 0) (w ? kv.vs : kv.ks)[at / 32] = __half_as_ushort(__float2half_rn(d));
    }
  }
}

template <class T, class C>
int launch(const tb2_paged_kv& c, const tb2_paged_append_args& a, int* err, cudaStream_t st) {
  return launch_pdl(paged_append_kernel<T, C>, dim3(a.n_tokens, (a.q ? a.n_heads : 0) + c.n_kv), dim3(c.d_head), 0, st,
                    paged_kv_of(&c), a, err);
}

template <class T>
int launch_cache(const tb2_paged_kv& c, const tb2_paged_append_args& a, int* err, cudaStream_t st) {
  switch (c.kv_type) {
    case kTypeF32: return launch<T, float>(c, a, err, st);
    case kTypeF16: return launch<T, __half>(c, a, err, st);
    case kTypeBF16: return launch<T, __nv_bfloat16>(c, a, err, st);
    default: return launch<T, int8_t>(c, a, err, st);
  }
}

}  // namespace

int paged_append_launch(const tb2_paged_kv& c, const tb2_paged_append_args& a, int* err, cudaStream_t st) {
  switch (a.row_type) {
    case kTypeF32: return launch_cache<float>(c, a, err, st);
    case kTypeF16: return launch_cache<__half>(c, a, err, st);
    default: return launch_cache<__nv_bfloat16>(c, a, err, st);
  }
}

}  // namespace tb2

extern "C" {

int tb2_paged_append(const tb2_paged_kv* kv, const tb2_paged_append_args* a, void* stream) {
  if (!tb2::paged_kv_ok(kv) || !a || a->n_tokens < 0 || !tb2::row_type_ok(a->row_type)) return -1;
  if (a->n_tokens == 0) return 0;
  const int e = tb2::type_bytes(a->row_type), dh = kv->d_head;
  if (!a->k || !a->v || !a->slots) return -1;
  if (a->n_heads < 0 || (a->q && a->n_heads < 1) || (a->n_heads + 2LL * kv->n_kv) * dh > (1 << 24)) return -1;
  if (a->q && (!a->q_out || a->ldq < (long long)a->n_heads * dh || a->ldqo < (long long)a->n_heads * dh ||
               !tb2::aligned(a->q, 16) || !tb2::aligned(a->q_out, 16) || (a->ldq * e) % 16 || (a->ldqo * e) % 16))
    return -1;
  if (a->q && a->q == a->q_out && a->ldq != a->ldqo) return -1;
  if (a->ldk < (long long)kv->n_kv * dh || a->ldv < (long long)kv->n_kv * dh || !tb2::aligned(a->k, 16) ||
      !tb2::aligned(a->v, 16) || (a->ldk * e) % 16 || (a->ldv * e) % 16)
    return -1;
  if (a->rope && (!a->positions || a->rope_rows < 1 || !tb2::aligned(a->rope, 16))) return -1;
  if (a->bias && !tb2::aligned(a->bias, 16)) return -1;
  int* err = tb2::device_error_word();
  if (!err) return -3;
  return tb2::paged_append_launch(*kv, *a, err, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
