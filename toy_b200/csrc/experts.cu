// Tokens sorted by expert and back.
//
// A slot is token * n_used + choice. sort: the slots of each expert behind one
// another, in slot order (order), where each expert's begin (offsets), and
// each slot's place (pos, the inverse of order; -1 for a slot of no expert).
// dispatch: every token's row to its slots' places. combine: y_t = r_t + sum_k
// w_tk z[pos_tk], k ascending, in f32, rounded once. combine_grad: dz[pos] =
// w dy_t and dw = <dy_t, z[pos]>. Rows past the last expert's are left alone.
#include <algorithm>
#include <climits>

#include "rows.cuh"
#include "runtime.cuh"

namespace tb2 {
namespace {

constexpr int kMaxExperts = 1024, kSortThreads = 1024;

__device__ __forceinline__ int expert_of(const void* ids, int wide, long long i, int E, int* err) {
  const long long e = wide ? static_cast<const long long*>(ids)[i] : static_cast<const int*>(ids)[i];
  if (e >= E) atomicExch(err, (int)kErrExpert);
  return e >= 0 && e < E ? (int)e : -1;
}

// One CTA: expert e's slots are counted and then placed by thread e.
__global__ void __launch_bounds__(kSortThreads) sort_kernel(const void* ids, int wide, int n, int E, int* offsets,
                                                            int* order, int* pos, int* err) {
  griddep_wait();
  __shared__ int count[kMaxExperts + 1];
  const int e = threadIdx.x;
  if (e < E) {
    int c = 0;
    for (int i = 0; i < n; ++i) c += expert_of(ids, wide, i, E, err) == e;
    count[e] = c;
  }
  __syncthreads();
  int at = 0;
  for (int j = 0; j < e && j < E; ++j) at += count[j];
  if (e < E) {
    offsets[e] = at;
    if (e == E - 1) count[E] = offsets[E] = at + count[e];
    for (int i = 0; i < n; ++i)
      if (expert_of(ids, wide, i, E, err) == e) {
        order[at] = i;
        pos[i] = at++;
      }
  }
  __syncthreads();
  for (int i = e; i < n; i += kSortThreads) {
    if (expert_of(ids, wide, i, E, err) < 0) pos[i] = -1;
    if (i >= count[E]) order[i] = -1;
  }
}

struct RowsArgs {
  const void *x, *z, *res;
  void *y, *dz;
  const float* w;
  float* dw;
  const int *pos, *n_sorted;
  long long ldx, ldz, ldr, ldy, lddz;
  int* err;
  int T, K, d, rows;
};

__device__ __forceinline__ int place(const RowsArgs& a, long long slot) {
  const int p = a.pos[slot];
  if (p >= a.rows) atomicExch(a.err, (int)kErrExpertRow);
  return p < a.rows ? p : -1;
}

// Rows past the sorted ones set to 0 (where that is wanted).
template <class T>
__device__ void clear_rest(const RowsArgs& a, T* y, long long ld) {
  if (!a.n_sorted) return;
  for (long long r = (long long)max(*a.n_sorted, 0) + blockIdx.x; r < a.rows; r += gridDim.x)
    for (int c = threadIdx.x; c < a.d; c += blockDim.x) y[r * ld + c] = from_f32<T>(0.f);
}

template <class T>
__global__ void __launch_bounds__(256) dispatch_kernel(RowsArgs a) {
  griddep_wait();
  for (long long t = blockIdx.x; t < a.T; t += gridDim.x)
    for (int k = 0; k < a.K; ++k) {
      const int p = place(a, t * a.K + k);
      if (p < 0) continue;
      for (int c = threadIdx.x; c < a.d; c += 256)
        static_cast<T*>(a.y)[p * a.ldy + c] = static_cast<const T*>(a.x)[t * a.ldx + c];
    }
  clear_rest(a, static_cast<T*>(a.y), a.ldy);
}

template <class T>
__global__ void __launch_bounds__(256) combine_kernel(RowsArgs a) {
  griddep_wait();
  for (long long t = blockIdx.x; t < a.T; t += gridDim.x)
    for (int c = threadIdx.x; c < a.d; c += 256) {
      float y = a.res ? to_f32(static_cast<const T*>(a.res)[t * a.ldr + c]) : 0.f;
      for (int k = 0; k < a.K; ++k) {
        const int p = place(a, t * a.K + k);
        if (p < 0) continue;
        const float z = to_f32(static_cast<const T*>(a.z)[p * a.ldz + c]);
        y += a.w ? a.w[t * a.K + k] * z : z;
      }
      static_cast<T*>(a.y)[t * a.ldy + c] = from_f32<T>(y);
    }
}

// a warp per slot
template <class T>
__global__ void __launch_bounds__(256) combine_grad_kernel(RowsArgs a) {
  griddep_wait();
  const int lane = threadIdx.x % 32;
  const long long slots = (long long)a.T * a.K;
  for (long long s = blockIdx.x * 8 + threadIdx.x / 32; s < slots; s += gridDim.x * 8) {
    const int p = place(a, s);
    const long long t = s / a.K;
    float dot = 0.f;
    if (p >= 0) {
      const float w = a.w ? a.w[s] : 1.f;
      for (int c = lane; c < a.d; c += 32) {
        const float g = to_f32(static_cast<const T*>(a.x)[t * a.ldx + c]);
        dot += g * to_f32(static_cast<const T*>(a.z)[p * a.ldz + c]);
        if (a.dz) static_cast<T*>(a.dz)[p * a.lddz + c] = from_f32<T>(w * g);
      }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    if (lane == 0 && a.dw) a.dw[s] = dot;
  }
  if (a.dz) clear_rest(a, static_cast<T*>(a.dz), a.lddz);
}

bool shape_ok(int T, int K, int d, int rows, int type) {
  return T >= 0 && K >= 1 && d >= 1 && rows >= 0 && row_type_ok(type) && (long long)T * K <= INT_MAX;
}
bool row_ok(const void* p, long long ld, int d, int type) { return p && ld >= d && aligned(p, type_bytes(type)); }

template <class T>
int prepare_type() {
  return load_kernel(dispatch_kernel<T>) || load_kernel(combine_kernel<T>) || load_kernel(combine_grad_kernel<T>) ? -3
                                                                                                                  : 0;
}

}  // namespace

int experts_prepare() {
  if (load_kernel(sort_kernel)) return -3;
  return prepare_type<float>() || prepare_type<__half>() || prepare_type<__nv_bfloat16>() ? -3 : 0;
}

}  // namespace tb2

extern "C" {

int tb2_expert_sort(const tb2_expert_sort_args* a, void* stream) {
  using namespace tb2;
  if (!a || a->n_slots < 0 || a->n_experts < 1 || a->n_experts > kMaxExperts || (a->id_bytes != 4 && a->id_bytes != 8))
    return -1;
  if (!a->offsets || (a->n_slots && (!a->ids || !a->order || !a->pos))) return -1;
  if (!aligned(a->ids, a->id_bytes) || !all_aligned(4, {a->offsets, a->order, a->pos})) return -1;
  int* err = device_error_word();
  if (!err) return -3;
  return launch_pdl(sort_kernel, dim3(1), dim3(kSortThreads), 0, static_cast<cudaStream_t>(stream), a->ids,
                    (int)(a->id_bytes == 8), a->n_slots, a->n_experts, a->offsets, a->order, a->pos, err);
}

int tb2_expert_dispatch(const tb2_expert_rows_args* a, void* stream) {
  using namespace tb2;
  if (!a || !shape_ok(a->n_tokens, a->n_used, a->d, a->n_rows, a->row_type)) return -1;
  if (a->n_tokens == 0) return 0;
  if (!row_ok(a->x, a->ldx, a->d, a->row_type) || !row_ok(a->xs, a->ldxs, a->d, a->row_type)) return -1;
  if (!a->pos || !all_aligned(4, {a->pos, a->n_sorted})) return -1;
  RowsArgs k = {};
  k.x = a->x; k.ldx = a->ldx; k.y = a->xs; k.ldy = a->ldxs; k.pos = a->pos; k.n_sorted = a->n_sorted;
  k.T = a->n_tokens; k.K = a->n_used; k.d = a->d; k.rows = a->n_rows;
  if (!(k.err = device_error_word())) return -3;
  return by_row_type(a->row_type, [&](auto t) {
    return launch_pdl(dispatch_kernel<decltype(t)>, dim3(a->n_tokens), dim3(256), 0, static_cast<cudaStream_t>(stream), k);
  });
}

int tb2_expert_combine(const tb2_expert_rows_args* a, void* stream) {
  using namespace tb2;
  if (!a || !shape_ok(a->n_tokens, a->n_used, a->d, a->n_rows, a->row_type)) return -1;
  if (a->n_tokens == 0) return 0;
  if (!row_ok(a->x, a->ldx, a->d, a->row_type) || !row_ok(a->xs, a->ldxs, a->d, a->row_type)) return -1;
  if (a->residual && !row_ok(a->residual, a->ldr, a->d, a->row_type)) return -1;
  if (!a->pos || !all_aligned(4, {a->pos, a->weights})) return -1;
  RowsArgs k = {};
  k.z = a->xs; k.ldz = a->ldxs; k.y = a->x; k.ldy = a->ldx; k.res = a->residual; k.ldr = a->ldr; k.pos = a->pos;
  k.w = a->weights;
  k.T = a->n_tokens; k.K = a->n_used; k.d = a->d; k.rows = a->n_rows;
  if (!(k.err = device_error_word())) return -3;
  return by_row_type(a->row_type, [&](auto t) {
    return launch_pdl(combine_kernel<decltype(t)>, dim3(a->n_tokens), dim3(256), 0, static_cast<cudaStream_t>(stream), k);
  });
}

int tb2_expert_combine_grad(const tb2_expert_rows_args* a, void* stream) {
  using namespace tb2;
  if (!a || !shape_ok(a->n_tokens, a->n_used, a->d, a->n_rows, a->row_type)) return -1;
  if (a->n_tokens == 0) return 0;
  if (!row_ok(a->x, a->ldx, a->d, a->row_type) || !row_ok(a->xs, a->ldxs, a->d, a->row_type)) return -1;
  if (a->d_xs && !row_ok(a->d_xs, a->ldd, a->d, a->row_type)) return -1;
  if (!a->pos || !all_aligned(4, {a->pos, a->weights, a->d_weights, a->n_sorted})) return -1;
  RowsArgs k = {};
  k.x = a->x; k.ldx = a->ldx; k.z = a->xs; k.ldz = a->ldxs; k.dz = a->d_xs; k.lddz = a->ldd; k.pos = a->pos;
  k.w = a->weights; k.dw = a->d_weights; k.n_sorted = a->n_sorted;
  k.T = a->n_tokens; k.K = a->n_used; k.d = a->d; k.rows = a->n_rows;
  if (!(k.err = device_error_word())) return -3;
  const long long ctas = ((long long)k.T * k.K + 7) / 8;
  return by_row_type(a->row_type, [&](auto t) {
    return launch_pdl(combine_grad_kernel<decltype(t)>, dim3((unsigned)std::min<long long>(ctas, 1 << 20)), dim3(256),
                      0, static_cast<cudaStream_t>(stream), k);
  });
}

}  // extern "C"
