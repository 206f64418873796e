// What the operators over a caller's rows (logprobs.cu, experts.cu,
// multi_adamw.cu) share: 16-byte pieces of f32, f16 or bf16 values as f32, the
// launch shape, and the codes the kernels record in the device error word.
#pragma once
#include "paged.cuh"
#include "pdl.cuh"

namespace tb2 {

enum RowsError : int {
  kErrToken = 0x5101,     // a token or alternative outside the vocabulary
  kErrExpert = 0x5102,    // an expert id outside [0, n_experts)
  kErrExpertRow = 0x5103  // a sorted row outside the buffer
};

constexpr int kSMs = 148;

// A kernel loaded on the current device, so that its first launch may be captured.
template <class K>
int load_kernel(K* k) {
  cudaFuncAttributes at;
  return cudaFuncGetAttributes(&at, k) == cudaSuccess ? 0 : -3;
}
// The slots of ids [n] (0 .. E - 1, or negative: none) by expert: see tb2_expert_sort. order may be NULL.
int expert_sort_launch(const tb2_expert_sort_args& a, int* err, cudaStream_t st);

int logprobs_prepare();
int experts_prepare();
int multi_adamw_prepare();

// 16 bytes of T as f32, and back (one rounding)
template <class T>
struct Piece {
  static constexpr int kN = 16 / (int)sizeof(T);
  static __device__ __forceinline__ void get(const uint4& u, float (&f)[kN]) {
    T t[kN];
    memcpy(t, &u, 16);
#pragma unroll
    for (int i = 0; i < kN; ++i) f[i] = to_f32<T>(t[i]);
  }
  static __device__ __forceinline__ uint4 put(const float (&f)[kN]) {
    T t[kN];
#pragma unroll
    for (int i = 0; i < kN; ++i) t[i] = from_f32<T>(f[i]);
    uint4 u;
    memcpy(&u, t, 16);
    return u;
  }
};

// Whether na rows at a and nb rows at b, of d values each, share no memory. Rows may lie between one another's; of
// unlike strides that is left to the caller.
inline bool rows_apart(const void* a, long long lda, long long na, const void* b, long long ldb, long long nb, int d,
                       int type) {
  if (!a || !b || na < 1 || nb < 1) return true;
  typedef unsigned long long u64;
  const u64 e = type_bytes(type), row = d * e, x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  const u64 la = (na > 1 ? lda : nb > 1 ? ldb : d) * e, lb = (nb > 1 ? ldb : na > 1 ? lda : d) * e;
  if (x + (na - 1) * la + row <= y || y + (nb - 1) * lb + row <= x) return true;
  if (la != lb) return true;
  const u64 off = x < y ? (y - x) % la : (x - y) % la;   // where the later one's rows begin in the earlier one's
  return off >= row && la - off >= row;
}

template <class F>
int by_row_type(int type, F&& f) {
  switch (type) {
    case kTypeF32: return f(float());
    case kTypeF16: return f(__half());
    case kTypeBF16: return f(__nv_bfloat16());
    default: return -1;
  }
}

}  // namespace tb2
