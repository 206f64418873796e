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
#include "warp_reduce.cuh"

namespace tb2 {
namespace {

namespace cg = cooperative_groups;

constexpr int kOneCta = 256;         // slots that one CTA sorts
// Slots above which order, scattered 4-byte writes, is left to a kernel of all SMs. In the sort's own kernel, and in
// the other: 16384 slots 7.3 and 7.6 us, 32768 of 128 experts 8.8 and 9.3, 65536 10.9 and 10.4, 262144 30 and 27.
constexpr int kOrderApart = 32768;
constexpr int kMaxExperts = 1024, kSortThreads = 1024, kSortWarps = kSortThreads / 32, kSortCtas = 8;

// A slot's expert, or E: none (past: the id is no expert's).
__device__ __forceinline__ int expert_of(const void* ids, int wide, long long i, int E, bool& past) {
  const long long e = wide ? static_cast<const long long*>(ids)[i] : static_cast<const int*>(ids)[i];
  past |= e >= E;
  return e >= E || e < 0 ? E : (int)e;
}

// The lanes with this lane's value of BITS bits. (A ballot a bit; __match_any_sync took longer: sorting 262144 slots 67
// us instead of 44.)
template <int BITS>
__device__ __forceinline__ unsigned same_lanes(int e) {
  unsigned same = 0xffffffffu;
#pragma unroll
  for (int b = 0; b < BITS; ++b) same &= __ballot_sync(0xffffffffu, e >> b & 1) ^ ((unsigned)(e >> b & 1) - 1u);
  return same;
}

// A stable counting sort in one launch of a cluster. Every warp has a run of
// the slots. It counts its run's experts in shared memory; the runs' counts are
// summed over warps and CTAs (distributed shared memory), which gives every
// warp the place of its first slot of each expert; and the second walk of the
// run hands out the places in slot order, 32 slots at a time by the lanes that
// share an expert. No workspace. What it takes is latency where slots are few
// (ids are read eight times 32 at once and kept where a run is no longer, and
// as many warps take part as have 32 slots, so that few counts are summed) and
// the instructions of eight SMs where they are many: 128 slots 2.7 us, 4096 4.5,
// 32768 8.4, 262144 27 (in whose time a tenth of their rows, 2048 bf16 each, is
// moved).
constexpr int kAhead = 8;
template <int BITS>
__global__ void __launch_bounds__(kSortThreads) sort_kernel(const void* ids, int wide, int n, int E, int warps,
                                                            int* offsets, int* order, int* pos, int* err) {
  // order NULL: a launch of its own writes it
  extern __shared__ int count[];                   // [warps][E]: then each warp's next place
  __shared__ int total[kMaxExperts];               // this CTA's slots of each expert
  __shared__ int warp_sum[kSortWarps];
  __shared__ int live;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, threads = blockDim.x;
  for (int i = tid; i < warps * E; i += threads) count[i] = 0;
  // runs of a multiple of 32 slots
  const long long run = ((long long)n + 32 * C * warps - 1) / (32 * C * warps) * 32;
  const long long i0 = warp < warps ? min((long long)n, run * (part * warps + warp)) : n;
  const long long i1 = min((long long)n, i0 + run);
  griddep_wait();
  int e[kAhead];
  bool past = false;
  auto read = [&](long long b) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      e[k] = b + 32 * k + lane < i1 ? expert_of(ids, wide, b + 32 * k + lane, E, past) : E;
  };
  read(i0);
  __syncthreads();
  int* mine = count + warp * E;
  for (long long b = i0; b < i1; b += 32 * kAhead) {
    if (b > i0) read(b);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (e[k] < E) atomicAdd(&mine[e[k]], 1);
    }
  }
  if (past) atomicExch(err, (int)kErrExpert);
  __syncthreads();
  // a thread an expert: its warps' counts become their offsets in this CTA
  for (int x = tid; x < E; x += threads) {
    int sum = 0;
#pragma unroll 8
    for (int w = 0; w < warps; ++w) {
      const int c = count[w * E + x];
      count[w * E + x] = sum;
      sum += c;
    }
    total[x] = sum;
  }
  if (C > 1) cluster.sync();
  else __syncthreads();
  // the experts in blocks of a CTA's threads
  for (int x0 = 0, base0 = 0; x0 < E; x0 += threads) {
    const int x = x0 + tid;
    int before = 0, all = 0;   // this expert's slots in earlier CTAs, and in all
    if (x < E) {
      int c[kSortCtas];
#pragma unroll
      for (int k = 0; k < kSortCtas; ++k) c[k] = k < C ? cluster.map_shared_rank(total, k)[x] : 0;
#pragma unroll
      for (int k = 0; k < kSortCtas; ++k) {
        before += k < part ? c[k] : 0;
        all += c[k];
      }
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
    int ahead = lane < threads / 32 && lane < warp ? warp_sum[lane] : 0, sum = lane < threads / 32 ? warp_sum[lane] : 0;
    ahead = __reduce_add_sync(0xffffffffu, ahead);
    sum = __reduce_add_sync(0xffffffffu, sum);
    const int base = base0 + ahead + incl - all;
    if (x < E) {
      if (part == 0) offsets[x] = base;
      if (x == E - 1) {
        live = base + all;
        if (part == 0) offsets[E] = base + all;
      }
#pragma unroll 8
      for (int w = 0; w < warps; ++w) count[w * E + x] += base + before;
    }
    base0 += sum;
    __syncthreads();
  }
  for (long long b = i0; b < i1; b += 32 * kAhead) {
    if (run > 32 * kAhead) read(b);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const long long i = b + 32 * k + lane;
      if (b + 32 * k >= i1) break;
      const unsigned same = same_lanes<BITS>(e[k]), lower = same & ((1u << lane) - 1);
      const bool on = e[k] < E;
      const int at = on ? mine[e[k]] + __popc(lower) : -1;
      __syncwarp();
      if (on && lower == 0) mine[e[k]] += __popc(same);
      __syncwarp();
      if (i < i1) pos[i] = at;
      if (on && order) order[at] = (int)i;
    }
  }
  if (order)
    for (long long i = (long long)live + part * threads + tid; i < n; i += (long long)C * threads) order[i] = -1;
  if (C > 1) cluster.sync();   // (the totals are read until here)
}

// order from its inverse, over the whole GPU: the eight SMs of the sort have enough to do.
__global__ void __launch_bounds__(256) order_kernel(const int* pos, const int* live, int n, int* order) {
  griddep_wait();
  const int from = *live;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < n; i += gridDim.x * 256LL) {   // (past n may be past 2^31)
    const int p = pos[i];
    if (p >= 0) order[p] = (int)i;
    if (i >= from) order[i] = -1;
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
  int per;             // pieces to a row
  unsigned magic;      // ceil(2^(31 + shift) / per), 2^shift >= per: i / per = i magic >> (31 + shift) for i < 2^31
  int shift;
};
__device__ __forceinline__ long long row_of(const RowsArgs& a, long long i) {
  return i >> 31 ? i / a.per : (long long)((unsigned long long)(unsigned)i * a.magic >> (31 + a.shift));
}

__device__ __forceinline__ int place(const RowsArgs& a, long long slot) {
  const int p = a.pos[slot];
  if (p >= a.rows) atomicExch(a.err, (int)kErrExpertRow);
  return p < a.rows ? p : -1;
}

// A piece of a row of T: the most bytes (16, 8, 4 or 2) that every row given starts on and consists of.
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
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < all; i += gridDim.x * 256LL) {
    const long long r = row_of(a, i);
    Chunk<T, V>::store(y, from + r, ld, (int)(i - r * a.per), zero);
  }
}

// A thread has one piece of a token's row: read once, written to the token's places. Bound by writing: 4096 tokens of 8
// bf16 rows of 2048 26.3 us (23.2 for the bytes), 8192 of 4 f32 rows 54 (52).
template <class T, class V>
__global__ void __launch_bounds__(256, 5) dispatch_kernel(RowsArgs a) {
  griddep_wait();
  const long long all = (long long)a.T * a.per;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < all; i += gridDim.x * 256LL) {
    const long long t = row_of(a, i);
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

// A slot or two to a token: P pieces to a thread, 256 apart among all, so that enough of them are on their way (31672
// tokens of one bf16 row of 1024 22.6 us instead of 26.9, the bytes' 19.9; of two 32.2, 34.4, 29.9; four pieces 23.8).
template <class T, class V, int P>
__global__ void __launch_bounds__(256) dispatch_few_kernel(RowsArgs a) {
  griddep_wait();
  const long long all = (long long)a.T * a.per;
  for (long long i0 = blockIdx.x * (256LL * P) + threadIdx.x; i0 < all; i0 += gridDim.x * (256LL * P)) {
    long long t[P];
    int c[P];
    V v[P];
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const long long i = min(i0 + 256 * j, all - 1);
      t[j] = row_of(a, i);
      c[j] = (int)(i - t[j] * a.per);
      v[j] = Chunk<T, V>::load_once(a.x, t[j], a.ldx, c[j]);
    }
    for (int k = 0; k < a.K; ++k) {
      int p[P];
#pragma unroll
      for (int j = 0; j < P; ++j) p[j] = i0 + 256 * j < all ? place(a, t[j] * a.K + k) : -1;
#pragma unroll
      for (int j = 0; j < P; ++j)
        if (p[j] >= 0) Chunk<T, V>::store(a.y, p[j], a.ldy, c[j], v[j]);
    }
  }
  clear_rest<T, V>(a, a.y, a.ldy);
}

// Pieces of less than 16 bytes: a warp has kCols of a token's, eight to a lane, so that the places and the rows'
// addresses are found once for eight. (A thread a piece was bound by its instructions: combine of 9902 tokens of 3 f32
// rows of 3395 220 us instead of 104.)
constexpr int kCols = 256;
template <class T, class V>
__global__ void __launch_bounds__(256) dispatch_narrow_kernel(RowsArgs a) {
  griddep_wait();
  const int lane = threadIdx.x % 32, groups = (a.per + kCols - 1) / kCols;
  const long long all = (long long)a.T * groups;
  for (long long i = blockIdx.x * 8LL + threadIdx.x / 32; i < all; i += gridDim.x * 8LL) {
    const long long t = i / groups;
    const int c = (int)(i - t * groups) * kCols + lane;
    V v[kCols / 32];
#pragma unroll
    for (int q = 0; q < kCols / 32; ++q)
      if (c + 32 * q < a.per) v[q] = Chunk<T, V>::load_once(a.x, t, a.ldx, c + 32 * q);
    for (int k = 0; k < a.K; ++k) {
      const int p = place(a, t * a.K + k);
      if (p < 0) continue;
#pragma unroll
      for (int q = 0; q < kCols / 32; ++q)
        if (c + 32 * q < a.per) Chunk<T, V>::store(a.y, p, a.ldy, c + 32 * q, v[q]);
    }
  }
  clear_rest<T, V>(a, a.y, a.ldy);
}

// A thread has one piece of a token's row; its places' pieces are read eight at a time. 4096 tokens of 8 bf16 rows of
// 2048 and a residual 28.5 us (25.8).
template <class T, class V>
__global__ void __launch_bounds__(256) combine_kernel(RowsArgs a) {
  constexpr int K = 8;
  using H = Chunk<T, V>;
  griddep_wait();
  const long long all = (long long)a.T * a.per;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < all; i += gridDim.x * 256LL) {
    const long long t = row_of(a, i);
    const int c = (int)(i - t * a.per);
    V r;
    if (a.res) r = H::load_once(a.res, t, a.ldr, c);
    float y[H::kN];
    for (int k0 = 0; k0 < a.K; k0 += K) {
      V z[K];
      int p[K];
#pragma unroll
      for (int k = 0; k < K; ++k) {
        p[k] = k0 + k < a.K ? place(a, t * a.K + k0 + k) : -1;
        if (p[k] >= 0) z[k] = H::load_once(a.z, p[k], a.ldz, c);
      }
      if (k0 == 0) {
        if (a.res) {
          H::get(r, y);
        } else {
#pragma unroll
          for (int e = 0; e < H::kN; ++e) y[e] = 0.f;
        }
      }
#pragma unroll
      for (int k = 0; k < K; ++k)
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

// K slots to a token, and P pieces to a thread, 256 apart among all. With the slots known the addresses cost less,
// and one slot leaves room for four pieces: 31672 tokens of one bf16 row of 1024 and a residual 30.4 us (29.9 for the
// bytes) instead of 46.6 by slots in a loop; 16384 of two f32 rows of 2048 83 instead of 105 (82.5; two pieces 88),
// 8192 of four 61 instead of 66, 2696 of five f16 rows 14.4 instead of 16.6. (Eight slots are too many at once, 512
// tokens of bf16 rows 6.8 instead of 5.7.)
template <class T, class V, int K, int P>
__global__ void __launch_bounds__(256) combine_slots_kernel(RowsArgs a) {
  using H = Chunk<T, V>;
  griddep_wait();
  const long long all = (long long)a.T * a.per;
  for (long long i0 = blockIdx.x * (256LL * P) + threadIdx.x; i0 < all; i0 += gridDim.x * (256LL * P)) {
    long long t[P];
    int c[P], p[P][K];
    V r[P], z[P][K];
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const long long i = min(i0 + 256 * j, all - 1);
      t[j] = row_of(a, i);
      c[j] = (int)(i - t[j] * a.per);
      if (a.res) r[j] = H::load_once(a.res, t[j], a.ldr, c[j]);
#pragma unroll
      for (int k = 0; k < K; ++k) p[j][k] = place(a, t[j] * K + k);
    }
#pragma unroll
    for (int j = 0; j < P; ++j)
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (p[j][k] >= 0) z[j][k] = H::load_once(a.z, p[j][k], a.ldz, c[j]);
#pragma unroll
    for (int j = 0; j < P; ++j) {
      if (i0 + 256 * j >= all) continue;
      float y[H::kN];
      if (a.res) {
        H::get(r[j], y);
      } else {
#pragma unroll
        for (int e = 0; e < H::kN; ++e) y[e] = 0.f;
      }
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (p[j][k] >= 0) {
          const float w = a.w ? a.w[t[j] * K + k] : 1.f;
          float f[H::kN];
          H::get(z[j][k], f);
#pragma unroll
          for (int e = 0; e < H::kN; ++e) y[e] = fmaf(w, f[e], y[e]);
        }
      H::store(a.y, t[j], a.ldy, c[j], H::put(y));
    }
  }
}

template <class T, class V, int K>
__global__ void __launch_bounds__(256) combine_narrow_kernel(RowsArgs a) {
  using H = Chunk<T, V>;
  constexpr int Q = kCols / 32;
  griddep_wait();
  const int lane = threadIdx.x % 32, groups = (a.per + kCols - 1) / kCols;
  const long long all = (long long)a.T * groups;
  for (long long i = blockIdx.x * 8LL + threadIdx.x / 32; i < all; i += gridDim.x * 8LL) {
    const long long t = i / groups;
    const int c = (int)(i - t * groups) * kCols + lane;
    float y[Q][H::kN];
#pragma unroll
    for (int q = 0; q < Q; ++q)
#pragma unroll
      for (int e = 0; e < H::kN; ++e) y[q][e] = 0.f;
    if (a.res) {
      V r[Q];
#pragma unroll
      for (int q = 0; q < Q; ++q)
        if (c + 32 * q < a.per) r[q] = H::load_once(a.res, t, a.ldr, c + 32 * q);
#pragma unroll
      for (int q = 0; q < Q; ++q)
        if (c + 32 * q < a.per) H::get(r[q], y[q]);
    }
    for (int k0 = 0; k0 < a.K; k0 += K) {
      V z[K][Q];
      float w[K];
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int p = k0 + k < a.K ? place(a, t * a.K + k0 + k) : -1;
        w[k] = p < 0 ? 0.f : a.w ? a.w[t * a.K + k0 + k] : 1.f;
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          memset(&z[k][q], 0, sizeof(V));
          if (p >= 0 && c + 32 * q < a.per) z[k][q] = H::load_once(a.z, p, a.ldz, c + 32 * q);
        }
      }
#pragma unroll
      for (int k = 0; k < K; ++k)   // (a slot that takes no part adds 0 times 0)
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          float f[H::kN];
          H::get(z[k][q], f);
#pragma unroll
          for (int e = 0; e < H::kN; ++e) y[q][e] = fmaf(w[k], f[e], y[q][e]);
        }
    }
#pragma unroll
    for (int q = 0; q < Q; ++q)
      if (c + 32 * q < a.per) H::store(a.y, t, a.ldy, c + 32 * q, H::put(y[q]));
  }
}

// A warp has K slots of a token (its last ones may be fewer), Q pieces to a lane at a time: the token's gradient is
// read once for them, and all their pieces are on their way together. (4096 tokens of 8 bf16 rows of 2048: a warp a
// slot 62 us, a warp eight 54, with the gradient's pieces read behind the rows' 54, now 50, the bytes' 44. A CTA a
// token, its warps' parts added up through shared memory, 63.)
template <class T, class V, int K, int Q>
__global__ void __launch_bounds__(256) combine_grad_kernel(RowsArgs a) {
  using H = Chunk<T, V>;
  // a piece's products are summed by themselves, so that a lane's 64 of a row of 2048 are no chain of 64 roundings
  // (f32: dw off by 1.1e-7 instead of 1.6e-7, in the same time); of small pieces the Q that are read together (for
  // large ones that took 51.6 us instead of 49.1)
  constexpr bool kPieces = H::kN >= 4;
  griddep_wait();
  const int lane = threadIdx.x % 32, parts = (a.K + K - 1) / K;
  const long long all = (long long)a.T * parts;
  for (long long i = blockIdx.x * 8LL + threadIdx.x / 32; i < all; i += gridDim.x * 8LL) {
    const long long t = i / parts, s = t * a.K + i % parts * K;
    const int n = (int)min((long long)K, (t + 1) * a.K - s);
    int p[K];
    float w[K], dot[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      p[k] = k < n ? place(a, s + k) : -1;
      w[k] = p[k] >= 0 && a.w ? a.w[s + k] : 1.f;
      dot[k] = 0.f;
    }
    for (int c0 = lane; c0 < a.per; c0 += 32 * Q) {
      V z[K][Q], x[Q];
      float part[K] = {};
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int c = c0 + 32 * q;
        if (c >= a.per) continue;
        x[q] = H::load(a.x, t, a.ldx, c);
        if (a.dw) {
#pragma unroll
          for (int k = 0; k < K; ++k)
            if (p[k] >= 0) z[k][q] = H::load_once(a.z, p[k], a.ldz, c);
        }
      }
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int c = c0 + 32 * q;
        if (c >= a.per) continue;
        float g[H::kN];
        H::get(x[q], g);
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (p[k] >= 0) {
            float f[H::kN];
            if (a.dw) {
              H::get(z[k][q], f);
              if (kPieces) part[k] = 0.f;
#pragma unroll
              for (int e = 0; e < H::kN; ++e) part[k] = fmaf(g[e], f[e], part[k]);
              if (kPieces) dot[k] += part[k];
            }
            if (a.dz) {
#pragma unroll
              for (int e = 0; e < H::kN; ++e) f[e] = w[k] * g[e];
              H::store(a.dz, p[k], a.lddz, c, H::put(f));
            }
          }
      }
      if (!kPieces) {
#pragma unroll
        for (int k = 0; k < K; ++k) dot[k] += part[k];
      }
    }
    if (a.dw) {
      const float d = warp_sum_multi<K>(dot, lane);
      const int k = warp_sum_multi_index<K>(lane);
      if (warp_sum_multi_leader<K>(lane) && k < n) a.dw[s + k] = d;
    }
  }
  if (a.dz) clear_rest<T, V>(a, a.dz, a.lddz);
}

// (a row's pieces are counted in 32 bits up to a group or a step of 256 past its last)
bool shape_ok(int T, int K, int d, int rows, int type) {
  return T >= 0 && K >= 1 && d >= 1 && d <= INT_MAX - 256 && rows >= 0 && row_type_ok(type) &&
         (long long)T * K <= INT_MAX;
}
bool row_ok(const void* p, long long ld, int d, int type) { return p && ld >= d && aligned(p, type_bytes(type)); }
// A result's rows that lie over an operand's and are not that operand in place: other threads read what it writes.
bool over(const tb2_expert_rows_args& a, const void* p, long long ld, int n, const void* q, long long ldq, int m) {
  return !rows_apart(p, ld, n, q, ldq, m, a.d, a.row_type);
}

// Sorted rows; where there are none they have no address either (every slot is of no expert).
bool sorted_ok(const tb2_expert_rows_args& a) { return a.n_rows == 0 || row_ok(a.xs, a.ldxs, a.d, a.row_type); }

// The kernel's shared-memory limit on the current device.
template <int BITS>
int sort_setup() {
  static DeviceOnce once;
  return once.ensure([](int) {
    return cudaFuncSetAttribute(sort_kernel<BITS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                kSortWarps * kMaxExperts * (int)sizeof(int)) == cudaSuccess
               ? 0
               : -3;
  });
}
template <int BITS>
int sort_launch(const tb2_expert_sort_args& a, int* err, cudaStream_t st) {
  if (sort_setup<BITS>()) return -3;
  // one CTA for few slots, and no more warps than have 32 slots
  const int ctas = a.n_slots <= kOneCta ? 1 : kSortCtas;
  const long long groups = ((long long)a.n_slots + 32 * ctas - 1) / (32 * ctas);
  const int warps = (int)std::max(1LL, std::min((long long)kSortWarps, groups));
  const int threads = std::max(warps * 32, std::min(kSortThreads, (a.n_experts + 31) / 32 * 32));
  const bool apart = a.order && a.n_slots > kOrderApart;
  if (launch_pdl_cluster(sort_kernel<BITS>, dim3(ctas), dim3(threads), (size_t)warps * a.n_experts * sizeof(int), st,
                         ctas, a.ids, (int)(a.id_bytes == 8), a.n_slots, a.n_experts, warps, a.offsets,
                         apart ? (int*)nullptr : a.order, a.pos, err))
    return -3;
  if (!apart) return 0;
  return launch_pdl(order_kernel, dim3((unsigned)std::min((a.n_slots + 255LL) / 256, 8LL * kSMs)), dim3(256), 0, st,
                    (const int*)a.pos, (const int*)a.offsets + a.n_experts, a.n_slots, a.order);
}

// f(a value of the row type, a piece): see Chunk.
template <class F>
int by_piece(RowsArgs& k, int type, std::initializer_list<std::pair<const void*, long long>> rows, F&& f) {
  const long long e = type_bytes(type);
  int bytes = 16;
  while (bytes > e) {
    bool fits = k.d * e % bytes == 0;
    for (const auto& r : rows) fits = fits && aligned(r.first, bytes) && (r.second * e % bytes == 0 || !r.first);
    if (fits) break;
    bytes /= 2;
  }
  k.per = (int)(k.d * e / bytes);
  k.shift = 0;
  while ((1LL << k.shift) < k.per) ++k.shift;
  k.magic = (unsigned)(((1ULL << (31 + k.shift)) + k.per - 1) / k.per);
  return by_row_type(type, [&](auto t) {
    if constexpr (sizeof(t) == 2)
      if (bytes == 2) return f(t, (unsigned short)0);
    return bytes == 16 ? f(t, uint4()) : bytes == 8 ? f(t, uint2()) : f(t, 0u);
  });
}

unsigned grid_of(long long threads) {
  return (unsigned)std::max(1LL, std::min((threads + 255) / 256, (long long)INT_MAX));
}
unsigned few_grid(const RowsArgs& k, int pieces) { return grid_of(((long long)k.T * k.per + pieces - 1) / pieces); }
unsigned narrow_grid(const RowsArgs& k) { return grid_of((long long)k.T * ((k.per + kCols - 1) / kCols) * 32); }
template <class T, class V>
int dispatch_by(const RowsArgs& k, cudaStream_t st) {
  if constexpr (sizeof(V) < 16)
    return launch_pdl(dispatch_narrow_kernel<T, V>, dim3(narrow_grid(k)), dim3(256), 0, st, k);
  else
    return k.K <= 2 ? launch_pdl(dispatch_few_kernel<T, V, 2>, dim3(few_grid(k, 2)), dim3(256), 0, st, k)
                    : launch_pdl(dispatch_kernel<T, V>, dim3(grid_of((long long)k.T * k.per)), dim3(256), 0, st, k);
}
template <class T, class V, int K, int P>
int combine_slots(const RowsArgs& k, cudaStream_t st) {
  return launch_pdl(combine_slots_kernel<T, V, K, P>, dim3(few_grid(k, P)), dim3(256), 0, st, k);
}
template <class T, class V>
int combine_by(const RowsArgs& k, cudaStream_t st) {
  if constexpr (sizeof(V) < 16)
    return launch_pdl(k.K <= 2 ? combine_narrow_kernel<T, V, 2> : combine_narrow_kernel<T, V, 4>, dim3(narrow_grid(k)),
                      dim3(256), 0, st, k);
  else
    switch (k.K) {
      case 1: return combine_slots<T, V, 1, 4>(k, st);
      case 2: return combine_slots<T, V, 2, 1>(k, st);
      case 3: return combine_slots<T, V, 3, 1>(k, st);
      case 4: return combine_slots<T, V, 4, 1>(k, st);
      case 5: return combine_slots<T, V, 5, 1>(k, st);
      case 6: return combine_slots<T, V, 6, 1>(k, st);
      case 7: return combine_slots<T, V, 7, 1>(k, st);
      default: return launch_pdl(combine_kernel<T, V>, dim3(few_grid(k, 1)), dim3(256), 0, st, k);
    }
}
// Two slots to a warp, one where that would leave less than 16 warps an SM or pieces are of 4 bytes and less (180 us
// instead of 203 for 9902 tokens of 3 f32 rows of 3395). One slot has four 16-byte pieces to a lane (32768 tokens of
// one bf16 row of 576 25 us, with two 29).
template <class V, int K>
constexpr int kGradCols = sizeof(V) == 16 ? 4 / K : sizeof(V) == 8 ? 4 : 8;
template <class T, class V, int K>
int combine_grad_launch(const RowsArgs& k, cudaStream_t st) {
  const long long warps = (long long)k.T * ((k.K + K - 1) / K);
  return launch_pdl(combine_grad_kernel<T, V, K, kGradCols<V, K>>, dim3(grid_of(32 * warps)), dim3(256), 0, st, k);
}
template <class T, class V>
int combine_grad_by(const RowsArgs& k, cudaStream_t st) {
  if constexpr (sizeof(V) > 4)
    if (k.K > 1 && (long long)k.T * ((k.K + 1) / 2) >= 16LL * kSMs) return combine_grad_launch<T, V, 2>(k, st);
  return combine_grad_launch<T, V, 1>(k, st);
}

template <class T, class V>
int prepare_piece() {
  if (load_kernel(combine_grad_kernel<T, V, 1, kGradCols<V, 1>>)) return -3;
  if constexpr (sizeof(V) > 4)
    if (load_kernel(combine_grad_kernel<T, V, 2, kGradCols<V, 2>>)) return -3;
  if constexpr (sizeof(V) < 16)
    return load_kernel(dispatch_narrow_kernel<T, V>) || load_kernel(combine_narrow_kernel<T, V, 2>) ||
                   load_kernel(combine_narrow_kernel<T, V, 4>)
               ? -3
               : 0;
  else
    return load_kernel(dispatch_kernel<T, V>) || load_kernel(dispatch_few_kernel<T, V, 2>) ||
                   load_kernel(combine_kernel<T, V>) || load_kernel(combine_slots_kernel<T, V, 1, 4>) ||
                   load_kernel(combine_slots_kernel<T, V, 2, 1>) || load_kernel(combine_slots_kernel<T, V, 3, 1>) ||
                   load_kernel(combine_slots_kernel<T, V, 4, 1>) || load_kernel(combine_slots_kernel<T, V, 5, 1>) ||
                   load_kernel(combine_slots_kernel<T, V, 6, 1>) || load_kernel(combine_slots_kernel<T, V, 7, 1>)
               ? -3
               : 0;
}
template <class T>
int prepare_type() {
  if constexpr (sizeof(T) == 2)
    if (prepare_piece<T, unsigned short>()) return -3;
  return prepare_piece<T, uint4>() || prepare_piece<T, uint2>() || prepare_piece<T, unsigned>() ? -3 : 0;
}

}  // namespace

int expert_sort_launch(const tb2_expert_sort_args& a, int* err, cudaStream_t st) {
  return a.n_experts < 16 ? sort_launch<4>(a, err, st)   // (values 0 .. n_experts)
       : a.n_experts < 128 ? sort_launch<7>(a, err, st) : sort_launch<11>(a, err, st);
}

int experts_prepare() {
  if (sort_setup<4>() || sort_setup<7>() || sort_setup<11>() || load_kernel(order_kernel)) return -3;
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
  // (places are scattered while other ids are still read)
  const long long n = a->n_slots;
  const std::pair<const void*, long long> parts[4] = {
      {a->ids, n * a->id_bytes}, {a->offsets, 4LL * (a->n_experts + 1)}, {a->order, 4 * n}, {a->pos, 4 * n}};
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < i; ++j) {
      const char *p = static_cast<const char*>(parts[i].first), *q = static_cast<const char*>(parts[j].first);
      if (parts[i].second && parts[j].second && p < q + parts[j].second && q < p + parts[i].second) return -1;
    }
  int* err = device_error_word();
  if (!err) return -3;
  return expert_sort_launch(*a, err, static_cast<cudaStream_t>(stream));
}

int tb2_expert_dispatch(const tb2_expert_rows_args* a, void* stream) {
  using namespace tb2;
  if (!a || !shape_ok(a->n_tokens, a->n_used, a->d, a->n_rows, a->row_type)) return -1;
  if (a->n_tokens == 0) return 0;
  if (!row_ok(a->x, a->ldx, a->d, a->row_type) || !sorted_ok(*a)) return -1;
  if (!a->pos || !all_aligned(4, {a->pos, a->n_sorted})) return -1;
  if (over(*a, a->xs, a->ldxs, a->n_rows, a->x, a->ldx, a->n_tokens)) return -1;
  RowsArgs k = {};
  k.x = a->x; k.ldx = a->ldx; k.y = a->xs; k.ldy = a->ldxs; k.pos = a->pos; k.n_sorted = a->n_sorted;
  k.T = a->n_tokens; k.K = a->n_used; k.d = a->d; k.rows = a->n_rows;
  if (!(k.err = device_error_word())) return -3;
  return by_piece(k, a->row_type, {{k.x, k.ldx}, {k.y, k.ldy}}, [&](auto t, auto v) {
    return dispatch_by<decltype(t), decltype(v)>(k, static_cast<cudaStream_t>(stream));
  });
}

int tb2_expert_combine(const tb2_expert_rows_args* a, void* stream) {
  using namespace tb2;
  if (!a || !shape_ok(a->n_tokens, a->n_used, a->d, a->n_rows, a->row_type)) return -1;
  if (a->n_tokens == 0) return 0;
  if (!row_ok(a->x, a->ldx, a->d, a->row_type) || !sorted_ok(*a)) return -1;
  if (a->residual && !row_ok(a->residual, a->ldr, a->d, a->row_type)) return -1;
  if (a->residual == a->x && a->ldr != a->ldx && a->n_tokens > 1) return -1;
  if (!a->pos || !all_aligned(4, {a->pos, a->weights})) return -1;
  if (over(*a, a->x, a->ldx, a->n_tokens, a->xs, a->ldxs, a->n_rows)) return -1;
  if (a->residual != a->x && over(*a, a->x, a->ldx, a->n_tokens, a->residual, a->ldr, a->n_tokens)) return -1;
  RowsArgs k = {};
  k.z = a->xs; k.ldz = a->ldxs; k.y = a->x; k.ldy = a->ldx; k.res = a->residual; k.ldr = a->ldr; k.pos = a->pos;
  k.w = a->weights;
  k.T = a->n_tokens; k.K = a->n_used; k.d = a->d; k.rows = a->n_rows;
  if (!(k.err = device_error_word())) return -3;
  return by_piece(k, a->row_type, {{k.z, k.ldz}, {k.y, k.ldy}, {k.res, k.ldr}}, [&](auto t, auto v) {
    return combine_by<decltype(t), decltype(v)>(k, static_cast<cudaStream_t>(stream));
  });
}

int tb2_expert_combine_grad(const tb2_expert_rows_args* a, void* stream) {
  using namespace tb2;
  if (!a || !shape_ok(a->n_tokens, a->n_used, a->d, a->n_rows, a->row_type)) return -1;
  if (a->n_tokens == 0) return 0;
  if (!row_ok(a->x, a->ldx, a->d, a->row_type) || !sorted_ok(*a)) return -1;
  if (a->d_xs && !row_ok(a->d_xs, a->ldd, a->d, a->row_type)) return -1;
  if (a->d_xs == a->xs && a->ldd != a->ldxs && a->n_rows > 1) return -1;
  if (!a->pos || !all_aligned(4, {a->pos, a->weights, a->d_weights, a->n_sorted})) return -1;
  if (over(*a, a->d_xs, a->ldd, a->n_rows, a->x, a->ldx, a->n_tokens)) return -1;
  if (a->d_xs != a->xs && over(*a, a->d_xs, a->ldd, a->n_rows, a->xs, a->ldxs, a->n_rows)) return -1;
  RowsArgs k = {};
  k.x = a->x; k.ldx = a->ldx; k.z = a->xs; k.ldz = a->ldxs; k.dz = a->d_xs; k.lddz = a->ldd; k.pos = a->pos;
  k.w = a->weights; k.dw = a->d_weights; k.n_sorted = a->n_sorted;
  k.T = a->n_tokens; k.K = a->n_used; k.d = a->d; k.rows = a->n_rows;
  if (!(k.err = device_error_word())) return -3;
  return by_piece(k, a->row_type, {{k.x, k.ldx}, {k.z, k.ldz}, {k.dz, k.lddz}}, [&](auto t, auto v) {
    return combine_grad_by<decltype(t), decltype(v)>(k, static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
