// Tokens sorted by expert and back.
//
// A slot is token * n_used + choice. sort: the slots of each expert behind one
// another, in slot order (order), where each expert's begin (offsets), and
// each slot's place (pos, the inverse of order; -1 for a slot of no expert).
// dispatch: every token's row to its slots' places. combine: y_t = r_t + sum_k
// w_tk z[pos_tk], k ascending, in f32, rounded once. combine_grad: dz[pos] =
// w dy_t and dw = <dy_t, z[pos]>. Rows past the last expert's are left alone.
#include <cooperative_groups.h>

#include <algorithm>
#include <climits>
#include <cstring>

#include "rows.cuh"
#include "runtime.cuh"

namespace tb2 {
namespace {

namespace cg = cooperative_groups;

constexpr int kMaxExperts = 1024, kSortThreads = 1024, kSortWarps = kSortThreads / 32, kSortCtas = 8;

__device__ __forceinline__ int expert_of(const void* ids, int wide, long long i, int E) {
  const long long e = wide ? static_cast<const long long*>(ids)[i] : static_cast<const int*>(ids)[i];
  return e >= E ? kMaxExperts : e < 0 ? -1 : (int)e;   // kMaxExperts: no expert's
}

// A stable counting sort in one launch of a cluster. Every warp has a run of
// the slots. It counts its run's experts in shared memory, one atomic-free
// update per distinct expert of 32 slots (match_any); the runs' counts are
// summed over warps and CTAs (distributed shared memory), which gives every
// warp the place of its first slot of each expert, and the second walk of the
// run hands out the places in slot order. No workspace, no second launch.
__global__ void __launch_bounds__(kSortThreads) sort_kernel(const void* ids, int wide, int n, int E, int* offsets,
                                                            int* order, int* pos, int* err) {
  extern __shared__ int count[];                   // [kSortWarps][E]: then each warp's next place
  __shared__ int total[kMaxExperts];               // this CTA's slots of each expert
  __shared__ int warp_sum[kSortWarps];
  __shared__ int live;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  for (int i = tid; i < kSortWarps * E; i += kSortThreads) count[i] = 0;
  // runs of a multiple of 32 slots
  const long long run = ((long long)n + 32 * C * kSortWarps - 1) / (32 * C * kSortWarps) * 32;
  const long long i0 = min((long long)n, run * (part * kSortWarps + warp)), i1 = min((long long)n, i0 + run);
  griddep_wait();
  __syncthreads();
  int* mine = count + warp * E;
  bool bad = false;
  for (long long b = i0; b < i1; b += 32) {
    const int e = b + lane < i1 ? expert_of(ids, wide, b + lane, E) : -1;
    bad |= e == kMaxExperts;
    const unsigned same = __match_any_sync(0xffffffffu, e);
    if (e >= 0 && e < E && (same & ((1u << lane) - 1)) == 0) mine[e] += __popc(same);
    __syncwarp();
  }
  if (bad) atomicExch(err, (int)kErrExpert);
  __syncthreads();
  // a thread an expert: its warps' counts become their offsets in this CTA
  int sum = 0;
  if (tid < E)
    for (int w = 0; w < kSortWarps; ++w) {
      const int c = count[w * E + tid];
      count[w * E + tid] = sum;
      sum += c;
    }
  if (tid < E) total[tid] = sum;
  cluster.sync();
  int before = 0, all = 0;   // this expert's slots in earlier CTAs, and in all
  if (tid < E)
    for (int k = 0; k < C; ++k) {
      const int c = cluster.map_shared_rank(total, k)[tid];
      before += k < part ? c : 0;
      all += c;
    }
  // the experts before this one
  int incl = all;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int q = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += q;
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  int base = incl - all;
  for (int w = 0; w < kSortWarps; ++w) base += w < warp ? warp_sum[w] : 0;
  if (tid == E - 1) live = base + all;
  if (part == 0 && tid < E) {
    offsets[tid] = base;
    if (tid == E - 1) offsets[E] = base + all;
  }
  if (tid < E)
    for (int w = 0; w < kSortWarps; ++w) count[w * E + tid] += base + before;
  __syncthreads();
  for (long long b = i0; b < i1; b += 32) {
    const int e = b + lane < i1 ? expert_of(ids, wide, b + lane, E) : -1;
    const unsigned same = __match_any_sync(0xffffffffu, e), lower = same & ((1u << lane) - 1);
    const bool on = e >= 0 && e < E;
    const int at = on ? mine[e] + __popc(lower) : -1;
    __syncwarp();
    if (on && lower == 0) mine[e] += __popc(same);
    __syncwarp();
    if (b + lane < i1) pos[b + lane] = at;
    if (on) order[at] = (int)(b + lane);
  }
  for (long long i = (long long)live + part * kSortThreads + tid; i < n; i += (long long)C * kSortThreads) order[i] = -1;
  cluster.sync();   // (the totals are read until here)
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
  int per;   // pieces to a row
};

__device__ __forceinline__ int place(const RowsArgs& a, long long slot) {
  const int p = a.pos[slot];
  if (p >= a.rows) atomicExch(a.err, (int)kErrExpertRow);
  return p < a.rows ? p : -1;
}

// A piece of a row: 16 bytes where every row starts on 16 bytes and is made of them (V = uint4), else one value.
template <class T, class V>
struct Chunk {
  static constexpr int kN = sizeof(V) / sizeof(T);
  static __device__ __forceinline__ V load(const void* base, long long row, long long ld, int c) {
    return *reinterpret_cast<const V*>(static_cast<const T*>(base) + row * ld + (long long)c * kN);
  }
  static __device__ __forceinline__ V load_once(const void* base, long long row, long long ld, int c) {
    return __ldcs(reinterpret_cast<const V*>(static_cast<const T*>(base) + row * ld + (long long)c * kN));
  }
  static __device__ __forceinline__ void store(void* base, long long row, long long ld, int c, V v) {
    *reinterpret_cast<V*>(static_cast<T*>(base) + row * ld + (long long)c * kN) = v;
  }
  static __device__ __forceinline__ void get(const V& v, float (&f)[kN]) {
    T t[kN];
    memcpy(t, &v, sizeof(V));
#pragma unroll
    for (int i = 0; i < kN; ++i) f[i] = to_f32<T>(t[i]);
  }
  static __device__ __forceinline__ V put(const float (&f)[kN]) {
    T t[kN];
#pragma unroll
    for (int i = 0; i < kN; ++i) t[i] = from_f32<T>(f[i]);
    V v;
    memcpy(&v, t, sizeof(V));
    return v;
  }
};

// Rows past the sorted ones set to 0 (where that is wanted).
template <class T, class V>
__device__ void clear_rest(const RowsArgs& a, void* y, long long ld) {
  if (!a.n_sorted) return;
  const long long from = max(*a.n_sorted, 0), all = ((long long)a.rows - from) * a.per;
  V zero;
  memset(&zero, 0, sizeof zero);
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < all; i += gridDim.x * 256LL)
    Chunk<T, V>::store(y, from + i / a.per, ld, (int)(i % a.per), zero);
}

// A thread has one piece of one token's row: read once, written to the token's places (one place read ahead).
template <class T, class V>
__global__ void __launch_bounds__(256) dispatch_kernel(RowsArgs a) {
  griddep_wait();
  const long long all = (long long)a.T * a.per;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < all; i += gridDim.x * 256LL) {
    const long long t = i / a.per;
    const int c = (int)(i - t * a.per);
    const V v = Chunk<T, V>::load_once(a.x, t, a.ldx, c);
#pragma unroll 8
    for (int k = 0; k < a.K; ++k) {
      const int p = place(a, t * a.K + k);
      if (p >= 0) Chunk<T, V>::store(a.y, p, a.ldy, c, v);
    }
  }
  clear_rest<T, V>(a, a.y, a.ldy);
}

// A thread has one piece of one token's row; the places' pieces are read eight at a time.
template <class T, class V>
__global__ void __launch_bounds__(256) combine_kernel(RowsArgs a) {
  using H = Chunk<T, V>;
  constexpr int kAhead = 8;
  griddep_wait();
  const long long all = (long long)a.T * a.per;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < all; i += gridDim.x * 256LL) {
    const long long t = i / a.per;
    const int c = (int)(i - t * a.per);
    float y[H::kN];
#pragma unroll
    for (int e = 0; e < H::kN; ++e) y[e] = 0.f;
    if (a.res) H::get(H::load_once(a.res, t, a.ldr, c), y);
    for (int k0 = 0; k0 < a.K; k0 += kAhead) {
      V z[kAhead];
      int p[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        p[k] = k0 + k < a.K ? place(a, t * a.K + k0 + k) : -1;
        if (p[k] >= 0) z[k] = H::load_once(a.z, p[k], a.ldz, c);
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (p[k] >= 0) {
          const float w = a.w ? a.w[t * a.K + k0 + k] : 1.f;
          float f[H::kN];
          H::get(z[k], f);
#pragma unroll
          for (int e = 0; e < H::kN; ++e) y[e] = fmaf(w, f[e], y[e]);
        }
    }
    H::store(a.y, t, a.ldy, c, H::put(y));
  }
}

// A warp has a slot: its token's gradient and its row are read once (the token's other slots, next in line, find the
// gradient in the caches).
template <class T, class V>
__global__ void __launch_bounds__(256) combine_grad_kernel(RowsArgs a) {
  using H = Chunk<T, V>;
  griddep_wait();
  const int lane = threadIdx.x % 32;
  const long long slots = (long long)a.T * a.K;
  for (long long s = blockIdx.x * 8LL + threadIdx.x / 32; s < slots; s += gridDim.x * 8LL) {
    const int p = place(a, s);
    const long long t = s / a.K;
    float dot = 0.f;
    if (p >= 0) {
      const float w = a.w ? a.w[s] : 1.f;
#pragma unroll 4
      for (int c = lane; c < a.per; c += 32) {
        float g[H::kN], f[H::kN];
        H::get(H::load(a.x, t, a.ldx, c), g);
        if (a.dw) {
          H::get(H::load_once(a.z, p, a.ldz, c), f);
#pragma unroll
          for (int e = 0; e < H::kN; ++e) dot = fmaf(g[e], f[e], dot);
        }
        if (a.dz) {
#pragma unroll
          for (int e = 0; e < H::kN; ++e) f[e] = w * g[e];
          H::store(a.dz, p, a.lddz, c, H::put(f));
        }
      }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    if (lane == 0 && a.dw) a.dw[s] = dot;
  }
  if (a.dz) clear_rest<T, V>(a, a.dz, a.lddz);
}

bool shape_ok(int T, int K, int d, int rows, int type) {
  return T >= 0 && K >= 1 && d >= 1 && rows >= 0 && row_type_ok(type) && (long long)T * K <= INT_MAX;
}
bool row_ok(const void* p, long long ld, int d, int type) { return p && ld >= d && aligned(p, type_bytes(type)); }

template <class T, class V>
int prepare_type() {
  return load_kernel(dispatch_kernel<T, V>) || load_kernel(combine_kernel<T, V>) || load_kernel(combine_grad_kernel<T, V>)
             ? -3
             : 0;
}

// The kernel's shared-memory limit on the current device, and the largest portable cluster.
int sort_setup() {
  static DeviceOnce once;
  return once.ensure([](int) {
    return cudaFuncSetAttribute(sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                kSortWarps * kMaxExperts * (int)sizeof(int)) == cudaSuccess
               ? 0
               : -3;
  });
}

// f(a value of the row type, a piece): 16-byte pieces where all the rows given consist of them.
template <class F>
int by_piece(RowsArgs& k, int type, std::initializer_list<std::pair<const void*, long long>> rows, F&& f) {
  const long long e = type_bytes(type);
  bool whole = k.d * e % 16 == 0;
  for (const auto& r : rows) whole = whole && aligned(r.first, 16) && r.second * e % 16 == 0;
  k.per = whole ? (int)(k.d * e / 16) : k.d;
  return by_row_type(type, [&](auto t) { return whole ? f(t, uint4()) : f(t, t); });
}
unsigned grid_of(long long threads) {
  return (unsigned)std::max(1LL, std::min((threads + 255) / 256, (long long)INT_MAX));
}

}  // namespace

int experts_prepare() {
  if (sort_setup() || load_kernel(sort_kernel)) return -3;
  if (prepare_type<float, uint4>() || prepare_type<__half, uint4>() || prepare_type<__nv_bfloat16, uint4>()) return -3;
  return prepare_type<float, float>() || prepare_type<__half, __half>() || prepare_type<__nv_bfloat16, __nv_bfloat16>()
             ? -3
             : 0;
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
  if (sort_setup()) return -3;
  // one CTA where 32 slots a warp do
  const int ctas = a->n_slots <= kSortThreads ? 1 : kSortCtas;
  return launch_pdl_cluster(sort_kernel, dim3(ctas), dim3(kSortThreads), (size_t)kSortWarps * a->n_experts * sizeof(int),
                            static_cast<cudaStream_t>(stream), ctas, a->ids, (int)(a->id_bytes == 8), a->n_slots,
                            a->n_experts, a->offsets, a->order, a->pos, err);
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
  return by_piece(k, a->row_type, {{k.x, k.ldx}, {k.y, k.ldy}}, [&](auto t, auto v) {
    return launch_pdl(dispatch_kernel<decltype(t), decltype(v)>, dim3(grid_of((long long)k.T * k.per)), dim3(256), 0,
                      static_cast<cudaStream_t>(stream), k);
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
  return by_piece(k, a->row_type, {{k.z, k.ldz}, {k.y, k.ldy}, {k.res, k.ldr}}, [&](auto t, auto v) {
    return launch_pdl(combine_kernel<decltype(t), decltype(v)>, dim3(grid_of((long long)k.T * k.per)), dim3(256), 0,
                      static_cast<cudaStream_t>(stream), k);
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
  return by_piece(k, a->row_type, {{k.x, k.ldx}, {k.z, k.ldz}, {k.dz, k.lddz}}, [&](auto t, auto v) {
    return launch_pdl(combine_grad_kernel<decltype(t), decltype(v)>, dim3(grid_of((long long)k.T * k.K * 32)), dim3(256),
                      0, static_cast<cudaStream_t>(stream), k);
  });
}

}  // extern "C"
