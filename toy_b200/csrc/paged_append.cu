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
#include <algorithm>
#include <cstring>

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

// A thread's share of a row: V values of the head's first half and the V they
// are turned with, 16 bytes each.
template <class T>
struct Row {
  static constexpr int V = 16 / sizeof(T);
};

template <class T>
__device__ __forceinline__ void load_chunk(const T* p, float* x) {
  constexpr int V = Row<T>::V;
  T v[V];
  const uint4 w = *reinterpret_cast<const uint4*>(p);
  memcpy(v, &w, 16);
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = to_f32<T>(v[i]);
}
template <int V>
__device__ __forceinline__ void load_f32(const float* p, float* x) {
#pragma unroll
  for (int i = 0; i < V; i += 4) {
    const float4 v = *reinterpret_cast<const float4*>(p + i);
    x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
  }
}
// V values of type C at p (16, 8 or 4 bytes a store)
template <class C, int V>
__device__ __forceinline__ void store_chunk(C* p, const C (&v)[V]) {
  constexpr int B = V * sizeof(C);
  if constexpr (B >= 16) {
#pragma unroll
    for (int i = 0; i < B / 16; ++i) {
      uint4 w;
      memcpy(&w, &v[i * (16 / sizeof(C))], 16);
      *reinterpret_cast<uint4*>(p + i * (16 / sizeof(C))) = w;
    }
  } else if constexpr (B == 8) {
    uint2 w;
    memcpy(&w, v, 8);
    *reinterpret_cast<uint2*>(p) = w;
  } else {
    uint32_t w;
    memcpy(&w, v, 4);
    *reinterpret_cast<uint32_t*>(p) = w;
  }
}

// Bound: HBM (a prompt's rows in, q and the cache rows out; the slots,
// positions and table rows are re-read from the caches), or the launch for a
// decode step. A CTA takes a token, a thread a chunk of a head of it. Units of
// a token: q heads, k heads, v heads. A Q8_0 block of 32 values lies in 32 / V
// neighbouring lanes (d_head 64 and 128: in one half; d_head 32: both halves of
// 16 / V lanes).
template <class T, class C>
__global__ void __launch_bounds__(512) paged_append_kernel(const PagedKv kv, const tb2_paged_append_args a, int* err) {
  constexpr int V = Row<T>::V;
  constexpr bool kQ8 = sizeof(C) == 1;
  griddep_wait_release();
  const int dh = kv.dh, half = dh / 2, per_head = half / V;
  const int H = a.q ? a.n_heads : 0, units = H + 2 * kv.n_kv, items = units * per_head;
  const long long t = blockIdx.x;
  for (int base = 0; base < items; base += blockDim.x) {
    // (lanes past the end stay for the shuffles and repeat the last item)
    const int item = min(base + (int)threadIdx.x, items - 1);
    bool on = base + (int)threadIdx.x < items;
    const int unit = item / per_head, e = (item - unit * per_head) * V;
    const int kind = unit < H ? 0 : unit < H + kv.n_kv ? 1 : 2;
    const int j = kind == 0 ? unit : kind == 1 ? unit - H : unit - H - kv.n_kv;
    const T* row = static_cast<const T*>(kind == 0 ? a.q : kind == 1 ? a.k : a.v) +
                   t * (kind == 0 ? a.ldq : kind == 1 ? a.ldk : a.ldv) + j * dh + e;
    // (a padded token's row is read too: waiting for its slot first would put two reads one after the other)
    float lo[V], hi[V];
    load_chunk<T>(row, lo);
    load_chunk<T>(row + half, hi);
    long long pos = 0;
    if (a.rope) {
      pos = a.positions[t];
      if (pos < 0 || pos >= a.rope_rows) {
        if (on) *err = kErrPagedPosition;
        on = false;
        pos = 0;
      }
    }
    long long at = -1;   // element of the cache (of q_out) that the chunk goes to; -1: none
    if (kind == 0) {
      if (on) at = t * a.ldqo + j * dh + e;
    } else {
      const long long slot = a.slots[t];
      if (on && slot >= 0) {
        const long long page =
            (unsigned long long)slot >> 32 ? slot / kv.page_size : (unsigned)slot / (unsigned)kv.page_size;
        if (page < kv.n_pages)
          at = page * kv.page_stride + j * kv.head_stride + (slot - page * kv.page_size) * kv.tok_stride + e;
        else
          *err = kErrPagedSlot;
      }
    }
    if (a.bias) {
      const int first = kind == 0 ? 0 : kind == 1 ? a.n_heads : a.n_heads + kv.n_kv;
      float b0[V], b1[V];
      load_f32<V>(a.bias + (first + j) * dh + e, b0);
      load_f32<V>(a.bias + (first + j) * dh + e + half, b1);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        lo[v] = __fadd_rn(lo[v], b0[v]);
        hi[v] = __fadd_rn(hi[v], b1[v]);
      }
    }
    if (a.rope && kind < 2) {
      float cs[2 * V];
      load_f32<2 * V>(a.rope + (pos * half + e) * 2, cs);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float x = lo[v], y = hi[v], c = cs[2 * v], s = cs[2 * v + 1];
        lo[v] = __fsub_rn(__fmul_rn(x, c), __fmul_rn(y, s));
        hi[v] = __fadd_rn(__fmul_rn(x, s), __fmul_rn(y, c));
      }
    }
    if (kind == 0 && at >= 0) {
      T c0[V], c1[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        c0[v] = from_f32<T>(lo[v]);
        c1[v] = from_f32<T>(hi[v]);
      }
      T* out = static_cast<T*>(a.q_out) + at;
      store_chunk<T, V>(out, c0);
      store_chunk<T, V>(out + half, c1);
    }
    if constexpr (kQ8) {
      // (every lane of a warp takes part: blocks of a warp may belong to q, which has none)
      float m0 = 0.f, m1 = 0.f;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        m0 = fmaxf(m0, fabsf(lo[v]));
        m1 = fmaxf(m1, fabsf(hi[v]));
      }
      if (dh == 32) m0 = m1 = fmaxf(m0, m1);
      for (int o = (dh == 32 ? 16 : 32) / V / 2; o; o >>= 1) {
        m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, o));
        m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, o));
      }
      if (kind > 0 && at >= 0) {
        const float d0 = __fdiv_rn(m0, 127.0f), d1 = __fdiv_rn(m1, 127.0f);
        const float r0 = d0 != 0.0f ? __fdiv_rn(1.0f, d0) : 0.0f, r1 = d1 != 0.0f ? __fdiv_rn(1.0f, d1) : 0.0f;
        int8_t q0[V], q1[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
          q0[v] = (int8_t)round_away(__fmul_rn(lo[v], r0));
          q1[v] = (int8_t)round_away(__fmul_rn(hi[v], r1));
        }
        int8_t* pool = static_cast<int8_t*>(kind == 1 ? kv.k : kv.v) + at;
        store_chunk<int8_t, V>(pool, q0);
        store_chunk<int8_t, V>(pool + half, q1);
        uint16_t* sc = kind == 1 ? kv.ks : kv.vs;
        if (e % 32 == 0) {
          sc[at / 32] = __half_as_ushort(__float2half_rn(d0));
          if (dh > 32) sc[(at + half) / 32] = __half_as_ushort(__float2half_rn(d1));
        }
      }
    } else if (kind > 0 && at >= 0) {
      C c0[V], c1[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        c0[v] = from_f32<C>(lo[v]);
        c1[v] = from_f32<C>(hi[v]);
      }
      C* pool = static_cast<C*>(kind == 1 ? kv.k : kv.v) + at;
      store_chunk<C, V>(pool, c0);
      store_chunk<C, V>(pool + half, c1);
    }
  }
}

// Q8_0 at d_head 96, whose blocks straddle the halves: one thread per element
// of a head, q heads, then key heads, each with its value head. Right for a
// decode step (16 tokens of 32 / 8 heads 2.7 us, as at d_head 64 and 128), bound
// by its instructions and small CTAs for a prompt: 16384 tokens 675 us, 0.8
// TB/s, where the kernel above takes 61 us at d_head 64 and 115 at 128.
template <class T>
__global__ void paged_append_96_kernel(const PagedKv kv, const tb2_paged_append_args a, int* err) {
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

template <class T, class C>
int launch(const tb2_paged_kv& c, const tb2_paged_append_args& a, int* err, cudaStream_t st) {
  const int heads = a.q ? a.n_heads : 0;
  if (sizeof(C) == 1 && c.d_head == 96)
    return launch_pdl(paged_append_96_kernel<T>, dim3(a.n_tokens, heads + c.n_kv), dim3(96), 0, st, paged_kv_of(&c), a,
                      err);
  const int items = (heads + 2 * c.n_kv) * (c.d_head / 2 / Row<T>::V);
  // A decode step has its whole token in one round: 28 / 4 bf16 heads of 128 with 512 (256) threads, 8 tokens 2.2 (2.8)
  // us, 250 2.6 (3.2), 400 3.5 (3.5), 1000 5.4 (5.6). A prompt keeps more CTAs on an SM: 2000 tokens 11.9 (10.5), 4000
  // 21.4 (19.0); f32 rows of 32 / 8 heads of 64 into bf16: 250 2.3 (2.8), 400 3.4 (3.0), 1000 4.4 (5.4), 2000 9.7
  // (9.5), 16384 61.7 (57.9; 6.4 TB/s). The bound is two such CTAs to an SM; between
  // 300 and 1500 tokens either is right within a microsecond.
  const int most = a.n_tokens <= 2 * 148 ? 512 : 256;
  const int rounds = (items + most - 1) / most, threads = ((items + rounds - 1) / rounds + 31) / 32 * 32;
  return launch_pdl(paged_append_kernel<T, C>, dim3(a.n_tokens), dim3(threads), 0, st, paged_kv_of(&c), a, err);
}

template <class T>
int load_kernels() {   // (asking for its attributes loads a kernel)
  cudaFuncAttributes at;
  return cudaFuncGetAttributes(&at, paged_append_kernel<T, float>) == cudaSuccess &&
                 cudaFuncGetAttributes(&at, paged_append_kernel<T, __half>) == cudaSuccess &&
                 cudaFuncGetAttributes(&at, paged_append_kernel<T, __nv_bfloat16>) == cudaSuccess &&
                 cudaFuncGetAttributes(&at, paged_append_kernel<T, int8_t>) == cudaSuccess &&
                 cudaFuncGetAttributes(&at, paged_append_96_kernel<T>) == cudaSuccess
             ? 0
             : -3;
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

int paged_append_prepare() {
  static DeviceOnce setup;
  return setup.ensure(
      [](int) { return load_kernels<float>() || load_kernels<__half>() || load_kernels<__nv_bfloat16>() ? -3 : 0; });
}

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
  if (!tb2::aligned(a->positions, 4) || !tb2::aligned(a->slots, 8)) return -1;
  int* err = tb2::device_error_word();
  if (!err) return -3;
  return tb2::paged_append_launch(*kv, *a, err, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
