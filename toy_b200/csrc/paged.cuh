// What the paged KV-cache operators (paged_plan.cu, paged_append.cu,
// paged_attn.cu) and the decode engine share: the descriptor of a layer's page
// pools, its host-side checks, and the codes the kernels record in the device
// error word.
#pragma once
#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <initializer_list>

#include "toy_b200.h"

namespace tb2 {

enum PagedError : int {
  kErrPagedPage = 0x5001,      // a page id outside [0, n_pages)
  kErrPagedSlot = 0x5002,      // a slot past the pool
  kErrPagedPosition = 0x5003,  // a position outside the RoPE table
};

// ggml type ids of the values a cache or a row may hold
constexpr int kTypeF32 = 0, kTypeF16 = 1, kTypeQ8_0 = 8, kTypeBF16 = 30;

inline int type_bytes(int t) { return t == kTypeF32 ? 4 : t == kTypeQ8_0 ? 1 : 2; }
inline bool row_type_ok(int t) { return t == kTypeF32 || t == kTypeF16 || t == kTypeBF16; }
inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
inline bool all_aligned(size_t a, std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (!aligned(p, a)) return false;
  return true;
}

// What a descriptor is checked for: rows of d_head values (a multiple of 32,
// at most 128) that start on 16-byte boundaries, strides of a row at least, and
// for Q8_0 of whole rows. (That rows do not overlap is the caller's word:
// every access stays inside the strides' extent either way.)
inline bool paged_kv_ok(const tb2_paged_kv* c) {
  if (!c || !c->k || !c->v || c->n_pages < 1 || c->page_size < 1 || c->n_kv < 1) return false;
  if (!row_type_ok(c->kv_type) && c->kv_type != kTypeQ8_0) return false;
  if (c->d_head < 32 || c->d_head > 128 || c->d_head % 32) return false;
  if ((long long)c->page_size > (1 << 20)) return false;
  const long long e = type_bytes(c->kv_type);
  for (long long s : {c->page_stride, c->head_stride, c->tok_stride})
    if (s < c->d_head || (s * e) % 16) return false;
  if (!aligned(c->k, 16) || !aligned(c->v, 16)) return false;
  if (c->kv_type == kTypeQ8_0) {
    const size_t row = c->d_head == 128 ? 8 : c->d_head == 64 ? 4 : 2;   // a row's scales in one aligned read
    if (!c->k_scale || !c->v_scale || !aligned(c->k_scale, row) || !aligned(c->v_scale, row)) return false;
    if (c->page_stride % c->d_head || c->head_stride % c->d_head || c->tok_stride % c->d_head) return false;
  }
  return true;
}

// The descriptor as the kernels take it.
struct PagedKv {
  void *k, *v;
  uint16_t *ks, *vs;
  long long page_stride, head_stride, tok_stride;
  int n_pages, page_size, n_kv, dh;
};

inline PagedKv paged_kv_of(const tb2_paged_kv* c) {
  return {c->k, c->v, static_cast<uint16_t*>(c->k_scale), static_cast<uint16_t*>(c->v_scale), c->page_stride,
          c->head_stride, c->tok_stride, c->n_pages, c->page_size, c->n_kv, c->d_head};
}

template <class T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Kernels loaded and set up on the current device, so that a first launch may be captured into a graph.
int paged_plan_prepare();
int paged_append_prepare();

// Launches behind the C entries (arguments already checked).
int paged_plan_launch(const tb2_paged_plan_args& a, int* err, cudaStream_t st);
int paged_release_launch(const tb2_paged_release_args& a, int* err, cudaStream_t st);
int paged_append_launch(const tb2_paged_kv& kv, const tb2_paged_append_args& a, int* err, cudaStream_t st);
int paged_attend_launch(const tb2_paged_kv& kv, const tb2_paged_attend_args& a, int* err, cudaStream_t st);

}  // namespace tb2
