// Log probabilities of given tokens, entropy and the most likely alternatives
// of each row of logits, and the gradient back to the logits.
//
// With a the scale, M = max x, d = x - M and s = sum exp(a d):
//   ln p_j = a d_j - ln s,   H = ln s - a sum exp(a d) d / s.
// (Differences first: a row may be full of the type's lowest value.)
//
// Both directions are one pass and bound by reading the logits: the forward
// keeps a running maximum and rescales its sums when that grows, so that a row
// is read once; the gradient reads it again and writes as much.
//
// The alternatives cost no second pass. Every thread keeps the maximum of each
// of its four interleaved shares of the row, which the softmax needs anyway.
// The top-th largest of 64 group maxima is a lower bound of the row's top-th
// largest value, and only shares whose maximum reaches it can hold an
// alternative: of the 1024 shares of 256 threads about 24 at top = 20 (values
// fall into groups like coupons: 20 of 64 groups are hit by the first 64 (H_64
// - H_44) = 24), so some 3 % of the row is read again. Values above the bound are ranked
// by (value, lower index). Bounds that many values equal (flat rows) take the
// lowest indices by a scan in order; what passes the buffers (or holds a NaN)
// takes one round of the row for each alternative.
//
// Measured: 4096 rows of 152064 bf16 208 to 221 us where other work has filled the
// L2 (191 for the bytes at 6506 GB/s; 190 over and over, part of them in the L2),
// of 128256 164, with the entropy 175 (161; two more instructions a value, the
// issue slots are 65 % busy), with 20 alternatives too 214 (the re-read's
// latency, in all the CTAs of a round at once); the gradient 338 (323). One row
// of 49152 f32 3.6, with five alternatives 6.4; 16 of 128256 5.2 and 9.0.
#include <cooperative_groups.h>

#include <algorithm>
#include <cfloat>

#include "rows.cuh"
#include "runtime.cuh"

namespace tb2 {
namespace {

namespace cg = cooperative_groups;
typedef unsigned long long u64;

constexpr int kThreads = 1024;   // an SM's, in CTAs of NT
constexpr int kRound = 4 * kSMs;   // CTAs of 256 threads at once
constexpr int kMaxTop = 32, kGroups = 64, kCand = 1024, kTies = 512, kUnroll = 4;

struct ScoreArgs {
  const void* x;
  long long ld;
  const long long* tokens;
  float *logprob, *stats, *entropy, *top_lp;
  long long* top_ids;
  int* err;
  float scale;
  int n, V, top, whole, split;   // CTAs to a row: one for the first `whole`, then a cluster of `split`
};

// Values in the order of (x, lower index first) as whole numbers: NaN above everything, -0 equal to 0.
__device__ __forceinline__ u64 top_key(float x, int j) {
  x += 0.0f;
  unsigned b = __float_as_uint(x);
  b = x != x ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
  return (u64)b << 32 | (unsigned)(0x7fffffff - j);
}
__device__ __forceinline__ float key_value(u64 k) {
  const unsigned b = (unsigned)(k >> 32);
  return b == 0xffffffffu ? NAN : __uint_as_float((b & 0x80000000u) ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ int key_index(u64 k) { return 0x7fffffff - (int)(unsigned)k; }

// two f32 at a time
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<u64&>(r)) : "l"(reinterpret_cast<u64&>(a)), "l"(reinterpret_cast<u64&>(b)));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<u64&>(r)) : "l"(reinterpret_cast<u64&>(a)), "l"(reinterpret_cast<u64&>(b)));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<u64&>(r))
      : "l"(reinterpret_cast<u64&>(a)), "l"(reinterpret_cast<u64&>(b)), "l"(reinterpret_cast<u64&>(c)));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// The largest of a 16-byte piece (NaN passed over), and its values by twos.
template <class T>
struct Logits;
template <>
struct Logits<float> {
  static __device__ __forceinline__ float top(const uint4& u) {
    return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
  }
  static __device__ __forceinline__ float2 pair(const uint4& u, int i) {
    return i ? make_float2(__uint_as_float(u.z), __uint_as_float(u.w))
             : make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
  }
};
template <>
struct Logits<__nv_bfloat16> {
  static __device__ __forceinline__ __nv_bfloat162 h(unsigned w) { return reinterpret_cast<__nv_bfloat162&>(w); }
  static __device__ __forceinline__ float top(const uint4& u) {
    const __nv_bfloat162 m = __hmax2(__hmax2(h(u.x), h(u.y)), __hmax2(h(u.z), h(u.w)));
    return fmaxf(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ float2 pair(const uint4& u, int i) {
    const unsigned w = i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w;
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
};
template <>
struct Logits<__half> {
  static __device__ __forceinline__ __half2 h(unsigned w) { return reinterpret_cast<__half2&>(w); }
  static __device__ __forceinline__ float top(const uint4& u) {
    const __half2 m = __hmax2(__hmax2(h(u.x), h(u.y)), __hmax2(h(u.z), h(u.w)));
    return fmaxf(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ float2 pair(const uint4& u, int i) {
    return __half22float2(h(i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w));
  }
};

// A share's softmax sums: the maximum m (-inf: nothing yet), s = sum exp(a (x - m)), u = sum exp(a (x - m)) (x - m).
struct Sums {
  float m = -INFINITY, s = 0.f, u = 0.f;
};
// The sums with the reference moved up to m.
template <bool ENT>
__device__ __forceinline__ void move_to(Sums& a, float m, float c) {
  if (a.m == m) return;
  const float d = a.m - m, k = a.m == -INFINITY ? 0.f : ex2(d * c);   // (s and u are 0 where the reference was -inf)
  if (ENT) a.u = k == 0.f ? a.u * k : (a.u + a.s * d) * k;
  a.s *= k;
  a.m = m;
}

template <int NT>
struct ScoreShared {
  alignas(16) float group[kGroups];
  float red[NT / 32 * 3];
  u64 best[NT / 32];
  float tau;
  int n_shares, n_cand, n_ties, n_found;
  unsigned short shares[kUnroll * NT];
  u64 cand[kCand + kMaxTop + 16], ties[kTies];   // (16: the values outside the pieces)
  // what the cluster's first CTA reads
  float m, s, u;
  u64 list[kMaxTop];
};

// A row in memory: h values up to the first 16-byte boundary, P pieces, and the rest.
template <class T>
struct RowShape {
  const T* x;
  int V, h, P, rest;
  __device__ RowShape(const T* p, int v) : x(p), V(v) {
    const int off = (int)(reinterpret_cast<uintptr_t>(p) & 15);
    h = min(V, (16 - off) % 16 / (int)sizeof(T));
    P = (V - h) / Piece<T>::kN;
    rest = V - h - P * Piece<T>::kN;
  }
  __device__ const uint4* pieces() const { return reinterpret_cast<const uint4*>(x + h); }
  // the index of the i-th value outside the pieces (i < h + rest)
  __device__ int edge(int i) const { return i < h ? i : V - rest + (i - h); }
};

// The CTA's lowest `need` indices of pieces [p0, p1) whose value is v, behind cand[n ..).
template <int NT, class T>
__device__ void scan_equal(ScoreShared<NT>& sh, const RowShape<T>& row, int p0, int p1, float v, int need, int n) {
  constexpr int N = Piece<T>::kN;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  int found = 0;
  for (int b = p0; b < p1 && found < need; b += NT) {
    const int i = b + threadIdx.x;
    unsigned hit = 0;
    if (i < p1) {
      float f[N];
      Piece<T>::get(row.pieces()[i], f);
#pragma unroll
      for (int e = 0; e < N; ++e) hit |= (f[e] == v) << e;
    }
    int incl = __popc(hit);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int q = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += q;
    }
    __syncthreads();
    if (lane == 31) sh.red[warp] = __int_as_float(incl);
    __syncthreads();
    int at = found + incl - __popc(hit);
    for (int w = 0; w < NT / 32; ++w) {
      const int q = __float_as_int(sh.red[w]);
      if (w < warp) at += q;
      found += q;
    }
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (hit >> e & 1) {
        if (at < need) sh.cand[n + at] = top_key(v, row.h + i * N + e);
        ++at;
      }
  }
  if (threadIdx.x == 0) sh.n_found = min(found, need);
  __syncthreads();
}

// cand[0 .. n) and ties[0 .. more) by rank: the `top` largest to list, which holds zeros.
template <int NT>
__device__ void rank_keys(ScoreShared<NT>& sh, int n, int more, int top) {
  const int lane = threadIdx.x % 32, all = n + more;
  for (int i = threadIdx.x / 32 * 8; i < all; i += NT / 32 * 8) {   // four lanes to a key
    const int me = i + lane / 4;
    const u64 k = me < n ? sh.cand[me] : me < all ? sh.ties[me - n] : 0;
    int r = 0;
#pragma unroll 4
    for (int j = lane % 4; j < n; j += 4) r += sh.cand[j] > k;
    for (int j = lane % 4; j < more; j += 4) r += sh.ties[j] > k;
    r += __shfl_xor_sync(0xffffffffu, r, 1);
    r += __shfl_xor_sync(0xffffffffu, r, 2);
    if (lane % 4 == 0 && r < top && k) sh.list[r] = k;
  }
  __syncthreads();
}

// The `top` largest keys of C lists in falling order (kMaxTop entries each, 0 past the last) in cand: a key's place is
// the number of larger ones, found in every list by halving.
template <int NT>
__device__ void merge_lists(ScoreShared<NT>& sh, int C, int top) {
  if (threadIdx.x < kMaxTop) sh.list[threadIdx.x] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < C * kMaxTop; i += NT) {
    const u64 k = sh.cand[i];
    if (!k) continue;
    int r = 0;
    for (int l = 0; l < C; ++l) {
      const u64* q = sh.cand + l * kMaxTop;
      int c = 0;   // entries of the list before c are larger
#pragma unroll
      for (int step = kMaxTop / 2; step; step >>= 1)
        if (q[c + step - 1] > k) c += step;
      r += c + (q[c] > k);
    }
    if (r < top) sh.list[r] = k;
  }
  __syncthreads();
}

// One round of the CTA's share of the row for each alternative (-inf left out).
template <int NT, class T>
__device__ void top_by_rounds(ScoreShared<NT>& sh, const RowShape<T>& row, int p0, int p1, int edges, int top) {
  constexpr int N = Piece<T>::kN;
  u64 last = ~0ull;
  for (int k = 0; k < kMaxTop; ++k) {
    u64 b = 0;
    auto take = [&](float x, int j) {
      const u64 key = x == -INFINITY ? 0 : top_key(x, j);
      if (key < last && key > b) b = key;
    };
    if (k < top) {
      for (int i = p0 + threadIdx.x; i < p1; i += NT) {
        float f[N];
        Piece<T>::get(row.pieces()[i], f);
#pragma unroll
        for (int e = 0; e < N; ++e) take(f[e], row.h + i * N + e);
      }
      if ((int)threadIdx.x < edges) take(to_f32(row.x[row.edge(threadIdx.x)]), row.edge(threadIdx.x));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const u64 q = __shfl_xor_sync(0xffffffffu, b, o);
      b = q > b ? q : b;
    }
    __syncthreads();
    if (threadIdx.x % 32 == 0) sh.best[threadIdx.x / 32] = b;
    __syncthreads();
    for (int w = 0; w < NT / 32; ++w) b = sh.best[w] > b ? sh.best[w] : b;
    last = b;
    if (threadIdx.x == 0) sh.list[k] = b;
  }
  __syncthreads();
}

// The CTA's alternatives to list, from the maxima of its threads' shares.
template <int NT, class T>
__device__ void find_top(ScoreShared<NT>& sh, const RowShape<T>& row, int p0, int p1, int edges, int top,
                         const float (&share)[kUnroll], bool odd) {
  constexpr int N = Piece<T>::kN, kLanes = NT / kGroups;
  const int tid = threadIdx.x;
  if (odd) {   // (uniform: the CTA's sum is not a number)
    top_by_rounds(sh, row, p0, p1, edges, top);
    return;
  }
  float g = fmaxf(fmaxf(share[0], share[1]), fmaxf(share[2], share[3]));
#pragma unroll
  for (int o = kLanes / 2; o; o >>= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
  if (tid % kLanes == 0) sh.group[tid / kLanes] = g;
  if (tid == 0) sh.n_shares = sh.n_cand = sh.n_ties = 0;
  if (tid < kMaxTop) sh.list[tid] = 0;
  __syncthreads();
  {   // the group whose maximum is the top-th: every lane of a group compares it with a part of the others
    constexpr int kPart = kGroups / kLanes;
    const int me = tid / kLanes, from = tid % kLanes * kPart;
    int r = 0;
#pragma unroll
    for (int j = from; j < from + kPart; j += 4) {
      const float4 q = *reinterpret_cast<const float4*>(&sh.group[j]);
      r += (q.x > g || (q.x == g && j < me)) + (q.y > g || (q.y == g && j + 1 < me)) +
           (q.z > g || (q.z == g && j + 2 < me)) + (q.w > g || (q.w == g && j + 3 < me));
    }
#pragma unroll
    for (int o = kLanes / 2; o; o >>= 1) r += __shfl_xor_sync(0xffffffffu, r, o);
    if (r == top - 1) sh.tau = g;
  }
  __syncthreads();
  const float tau = sh.tau;
#pragma unroll
  for (int u = 0; u < kUnroll; ++u)
    if (share[u] >= tau && share[u] > -INFINITY) sh.shares[atomicAdd(&sh.n_shares, 1)] = (unsigned short)(u * NT + tid);
  auto take = [&](float x, int j) {
    if (x > tau) {
      const int at = atomicAdd(&sh.n_cand, 1);
      if (at < kCand) sh.cand[at] = top_key(x, j);
    } else if (x == tau && tau > -INFINITY) {
      const int at = atomicAdd(&sh.n_ties, 1);
      if (at < kTies) sh.ties[at] = top_key(x, j);
    }
  };
  if (tid < edges) take(to_f32(row.x[row.edge(tid)]), row.edge(tid));
  __syncthreads();
  // the shares' pieces, dealt to all threads
  const int per = (p1 - p0 + kUnroll * NT - 1) / (kUnroll * NT), items = sh.n_shares * per;
#pragma unroll 2
  for (int i = tid; i < items; i += NT) {
    const int f = i / per, at = p0 + sh.shares[f] + (i - f * per) * (kUnroll * NT);
    if (at >= p1) continue;
    const uint4 q = row.pieces()[at];
    if (Logits<T>::top(q) < tau) continue;
    float v[N];
    Piece<T>::get(q, v);
#pragma unroll
    for (int e = 0; e < N; ++e) take(v[e], row.h + at * N + e);
  }
  __syncthreads();
  const int n = sh.n_cand, ties = sh.n_ties;
  if (n > kCand) {
    top_by_rounds(sh, row, p0, p1, edges, top);
    return;
  }
  if (n >= top) {
    rank_keys(sh, n, 0, top);
  } else if (ties <= kTies) {
    rank_keys(sh, n, ties, top);
  } else {
    scan_equal<NT, T>(sh, row, p0, p1, tau, top - n, n);
    const int more = sh.n_found;
    if (tid < edges) {
      const float x = to_f32(row.x[row.edge(tid)]);
      sh.cand[n + more + tid] = x == tau ? top_key(x, row.edge(tid)) : 0;
    }
    __syncthreads();
    rank_keys(sh, n + more + edges, 0, top);
  }
}

// A row by one CTA, or (CLUSTER) after the first a.whole rows by `split` CTAs of a cluster, each with a run of its
// pieces and the first with the values outside the pieces too. (Without the cluster's code, in CTAs of 256, 8192 rows
// of 32000 bf16 take 94 us, not 100, and 8000 of 4000 f32 37, not 41. CTAs that go on to a next row, read ahead, were
// no faster: 100 and 37, but 4096 of 128256 180, not 168; with a ring of asynchronous copies in shared memory 131, 48
// and 228.)
template <int NT, class T, bool ENT, bool CLUSTER>
__global__ void __launch_bounds__(NT, kThreads / NT) score_kernel(ScoreArgs a) {
  constexpr int N = Piece<T>::kN;
  __shared__ ScoreShared<NT> sh;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const bool one = !CLUSTER || (int)blockIdx.x < a.whole;
  const int C = one ? 1 : a.split, part = one ? 0 : blockIdx.x % C;   // (a.whole is a multiple of a.split)
  const long long r = one ? blockIdx.x : a.whole + (blockIdx.x - a.whole) / C;
  const RowShape<T> row(static_cast<const T*>(a.x) + r * a.ld, a.V);
  const int p0 = (int)((long long)row.P * part / C), p1 = (int)((long long)row.P * (part + 1) / C);
  const int edges = part == 0 ? row.h + row.rest : 0;
  const float c = a.scale * 1.4426950408889634f;
  griddep_wait();
  Sums t;
  float share[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) share[u] = -INFINITY;
  float2 s2 = {0.f, 0.f}, u2 = {0.f, 0.f};
  const float2 c2 = {c, c};
  const uint4* piece = row.pieces();
  long long token = -1;
  float x_token = 0.f;
  if (tid == 0 && part == 0) {   // (on its way while the row is read)
    token = a.tokens[r];
    if (token >= 0 && token < a.V) x_token = to_f32(row.x[token]);
  }
  // q[0 .. n): pieces of the shares from `first` on
  auto absorb = [&](const uint4(&q)[2], int first, int n) {
    float m = -INFINITY;
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (u < n) {
        share[first + u] = fmaxf(share[first + u], Logits<T>::top(q[u]));
        m = fmaxf(m, share[first + u]);
      }
    if (m > t.m) {
      t.s = s2.x + s2.y;
      t.u = u2.x + u2.y;
      move_to<ENT>(t, m, c);
      s2 = {t.s, 0.f};
      u2 = {t.u, 0.f};
    }
    const float ref = t.m == -INFINITY ? 0.f : -t.m;
    const float2 ref2 = {ref, ref};
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (u < n) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
          float2 d = add2(Logits<T>::pair(q[u], i), ref2);
          const float2 z = mul2(d, c2), e = {ex2(z.x), ex2(z.y)};
          s2 = add2(s2, e);
          if (ENT) {
            d = {fmaxf(d.x, -FLT_MAX), fmaxf(d.y, -FLT_MAX)};   // (a word of probability 0 adds 0)
            u2 = fma2(e, d, u2);
          }
        }
      }
  };
  // two pieces are computed while the next two are on their way
  int b = p0 + tid;
  uint4 qa[2], qb[2];
  auto fetch = [&](uint4(&q)[2], int first) {
#pragma unroll
    for (int u = 0; u < 2; ++u) q[u] = __ldcs(piece + b + (first + u) * NT);
  };
  if (b + 3 * NT < p1) {
    fetch(qa, 0);
    fetch(qb, 2);
    while (true) {
      b += kUnroll * NT;
      const bool more = b + 3 * NT < p1;
      absorb(qa, 0, 2);
      if (more) fetch(qa, 0);
      absorb(qb, 2, 2);
      if (!more) break;
      fetch(qb, 2);
    }
  }
#pragma unroll
  for (int f = 0; f < kUnroll; f += 2) {
    uint4(&q)[2] = f ? qb : qa;
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (b + (f + u) * NT < p1) q[u] = piece[b + (f + u) * NT];
  }
  absorb(qa, 0, min(2, (p1 - b + NT - 1) / NT));
  absorb(qb, 2, min(2, (p1 - b + NT - 1) / NT - 2));
  t.s = s2.x + s2.y;
  t.u = u2.x + u2.y;
  if (tid < edges) {   // a value outside the pieces
    const float x = to_f32(row.x[row.edge(tid)]);
    if (x > t.m) move_to<ENT>(t, x, c);
    const float d = x - (t.m == -INFINITY ? 0.f : t.m), e = ex2(d * c);
    t.s += e;
    t.u += e * fmaxf(d, -FLT_MAX);
  }
  // the CTA's sums: the maximum first
  float m = t.m;
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) sh.red[warp] = m;
  __syncthreads();
  m = lane < NT / 32 ? sh.red[lane] : -INFINITY;
#pragma unroll
  for (int o = NT / 64; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  m = __shfl_sync(0xffffffffu, m, 0);
  move_to<ENT>(t, m, c);
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    t.s += __shfl_xor_sync(0xffffffffu, t.s, o);
    if (ENT) t.u += __shfl_xor_sync(0xffffffffu, t.u, o);
  }
  if (lane == 0) {
    sh.red[NT / 32 + warp] = t.s;
    sh.red[2 * (NT / 32) + warp] = t.u;
  }
  __syncthreads();
  t.s = lane < NT / 32 ? sh.red[NT / 32 + lane] : 0.f;
  t.u = ENT && lane < NT / 32 ? sh.red[2 * (NT / 32) + lane] : 0.f;
#pragma unroll
  for (int o = NT / 64; o; o >>= 1) {
    t.s += __shfl_xor_sync(0xffffffffu, t.s, o);
    if (ENT) t.u += __shfl_xor_sync(0xffffffffu, t.u, o);
  }
  t.s = __shfl_sync(0xffffffffu, t.s, 0);
  if (ENT) t.u = __shfl_sync(0xffffffffu, t.u, 0);
  if (a.top) {
    __syncthreads();   // red is free
    find_top<NT, T>(sh, row, p0, p1, edges, a.top, share, t.s != t.s);
  }
  if (C > 1) {   // the row's from its CTAs'
    cg::cluster_group cluster = cg::this_cluster();
    if (tid == 0) {
      sh.m = t.m;
      sh.s = t.s;
      sh.u = t.u;
    }
    cluster.sync();
    if (part == 0) {
      Sums o;
      if (lane < C) {
        o.m = *cluster.map_shared_rank(&sh.m, lane);
        o.s = *cluster.map_shared_rank(&sh.s, lane);
        o.u = *cluster.map_shared_rank(&sh.u, lane);
      }
      m = o.m;
#pragma unroll
      for (int k = 4; k; k >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
      m = __shfl_sync(0xffffffffu, m, 0);
      move_to<ENT>(o, m, c);
#pragma unroll
      for (int k = 4; k; k >>= 1) {
        o.s += __shfl_xor_sync(0xffffffffu, o.s, k);
        o.u += __shfl_xor_sync(0xffffffffu, o.u, k);
      }
      t.m = m;
      t.s = __shfl_sync(0xffffffffu, o.s, 0);
      t.u = __shfl_sync(0xffffffffu, o.u, 0);
      if (a.top) {
        for (int i = tid; i < C * kMaxTop; i += NT)
          sh.cand[i] = cluster.map_shared_rank(&sh, i / kMaxTop)->list[i % kMaxTop];
        __syncthreads();
        merge_lists(sh, C, a.top);
      }
    }
    cluster.sync();   // (what the first CTA reads is there until then)
    if (part) return;
  }
  const float ref = t.m == -INFINITY ? 0.f : t.m, ln = logf(t.s);
  auto ln_p = [&](float x) { return ln == -INFINITY ? -INFINITY : fmaf(x - ref, a.scale, -ln); };
  if (tid == 0) {
    a.stats[2 * r] = ref;
    a.stats[2 * r + 1] = ln;
    if (token >= a.V) atomicExch(a.err, (int)kErrToken);
    a.logprob[r] = token < 0 ? 0.f : token < a.V ? ln_p(x_token) : NAN;
    if (ENT) a.entropy[r] = t.s == 0.f ? 0.f : ln - a.scale * (t.u / t.s);
  }
  if (!a.top) return;
  // fewer words than alternatives: those of probability 0, the lowest indices first
  const int have = __popc(__ballot_sync(0xffffffffu, lane < a.top && sh.list[lane] != 0));
  if (have < a.top) {
    if (tid == 0) sh.n_found = 0;
    __syncthreads();
    const int need = a.top - have;
    for (int b0 = 0; b0 < a.V; b0 += NT) {
      const int at = sh.n_found, j = b0 + tid;
      if (at >= need) break;
      const bool hit = j < a.V && to_f32(row.x[j]) == -INFINITY;
      const unsigned mask = __ballot_sync(0xffffffffu, hit);
      __syncthreads();
      if (lane == 0) sh.red[warp] = __int_as_float(__popc(mask));
      __syncthreads();
      int k = at + __popc(mask & ((1u << lane) - 1)), all = at;
      for (int w = 0; w < NT / 32; ++w) {
        const int q = __float_as_int(sh.red[w]);
        if (w < warp) k += q;
        all += q;
      }
      if (hit && k < need) sh.list[have + k] = top_key(-INFINITY, j);
      if (tid == 0) sh.n_found = all;
      __syncthreads();
    }
    __syncthreads();
  }
  if (tid < a.top) {
    const u64 k = sh.list[tid];
    a.top_ids[r * a.top + tid] = key_index(k);
    a.top_lp[r * a.top + tid] = ln_p(key_value(k));
  }
}

struct GradArgs {
  const void* x;
  long long ld;
  const long long* tokens;
  const float *stats, *entropy, *g_lp, *g_h, *g_top;
  const long long* top_ids;
  void* d;
  long long ldd;
  int* err;
  float scale;
  int n, V, top, whole, split;   // CTAs to a row: one for the first `whole`, then `split`
};

// 16 bytes from byte sh of lo | hi
__device__ __forceinline__ uint4 join_bytes(const uint4& lo, const uint4& hi, int sh) {
  const int b = (sh & 3) * 8;
  auto f = [&](unsigned p, unsigned q) { return __funnelshift_r(p, q, b); };
  switch (sh >> 2) {   // (the same for a whole row)
    case 0: return make_uint4(f(lo.x, lo.y), f(lo.y, lo.z), f(lo.z, lo.w), f(lo.w, hi.x));
    case 1: return make_uint4(f(lo.y, lo.z), f(lo.z, lo.w), f(lo.w, hi.x), f(hi.x, hi.y));
    case 2: return make_uint4(f(lo.z, lo.w), f(lo.w, hi.x), f(hi.x, hi.y), f(hi.y, hi.z));
    default: return make_uint4(f(lo.w, hi.x), f(hi.x, hi.y), f(hi.y, hi.z), f(hi.z, hi.w));
  }
}

// dx = p (A + B log2 p) with A = -a (g + g_H H), g the sum of the words' own gradients, B = -a g_H ln 2; the words with
// a gradient of their own (the token, the alternatives) are put right at the end. A CTA has a run of the 16-byte pieces
// of the result's row; a row of logits that starts elsewhere within its 16 bytes is read in aligned pieces and shifted
// (509 rows of 50303 f16 words that lie so: 27 us where the bytes take 16).
template <int NT, class T, bool ENT>
__global__ void __launch_bounds__(NT, kThreads / NT) score_grad_kernel(GradArgs a) {
  constexpr int N = Piece<T>::kN, kWords = kMaxTop + 1;
  __shared__ float x_at[kWords], g_at[kWords];
  __shared__ int at[kWords];
  const int tid = threadIdx.x, lane = tid % 32, V = a.V;
  const bool alone = (int)blockIdx.x < a.whole;
  const int C = alone ? 1 : a.split, part = alone ? 0 : (blockIdx.x - a.whole) % C;
  const long long r = alone ? blockIdx.x : a.whole + (blockIdx.x - a.whole) / C;
  const T* x = static_cast<const T*>(a.x) + r * a.ld;
  const RowShape<T> row(static_cast<T*>(a.d) + r * a.ldd, V);
  T* d = static_cast<T*>(a.d) + r * a.ldd;
  griddep_wait();
  const float m = a.stats[2 * r], ln = a.stats[2 * r + 1];
  const bool some = ln != -INFINITY;   // (a row without a word has no gradient)
  // the words with a gradient of their own: every warp sums them, the CTA keeps them
  auto word = [&](int k, float& g) {
    const long long j = k == kMaxTop ? a.tokens[r] : k < a.top ? a.top_ids[r * a.top + k] : -1;
    const bool ok = j >= 0 && j < V;
    if (part == 0 && (j >= V || (j < 0 && k < a.top))) atomicExch(a.err, (int)kErrToken);
    g = !ok || !some ? 0.f : k < kMaxTop ? a.g_top[r * a.top + k] : a.g_lp ? a.g_lp[r] : 0.f;
    return ok && some ? (int)j : -1;
  };
  float g, g_token;
  const int j_top = word(lane, g), j_token = word(kMaxTop, g_token);
  if (tid < 32) {
    at[tid] = j_top;
    g_at[tid] = g;
    x_at[tid] = j_top < 0 ? 0.f : to_f32(x[j_top]);
    if (tid == 0) {
      at[kMaxTop] = j_token;
      g_at[kMaxTop] = g_token;
      x_at[kMaxTop] = j_token < 0 ? 0.f : to_f32(x[j_token]);
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) g += __shfl_xor_sync(0xffffffffu, g, o);
  g += g_token;
  if (a.x == a.d) __syncthreads();   // (the words are read before any is overwritten)
  const float gh = ENT && some ? a.g_h[r] : 0.f;
  const float A = -a.scale * (g + (ENT ? gh * a.entropy[r] : 0.f)), B = -a.scale * gh * 0.6931471805599453f;
  const float c = a.scale * 1.4426950408889634f, l2 = ln * 1.4426950408889634f;
  const bool none = g == 0.f && gh == 0.f;
  auto one = [&](float xv) {
    if (none) return 0.f;
    const float t = fmaf(xv - m, c, -l2), e = ex2(t);
    return e * (ENT ? fmaf(fmaxf(t, -1e4f), B, A) : A);
  };
  const int p0 = (int)((long long)row.P * part / C), p1 = (int)((long long)row.P * (part + 1) / C);
  uint4* dp = reinterpret_cast<uint4*>(d + row.h);
  if (none) {
    for (int i = p0 + tid; i < p1; i += NT) dp[i] = make_uint4(0, 0, 0, 0);
  } else {
    const float2 m2 = {-m, -m}, c2 = {c, c}, n2 = {-l2, -l2}, A2 = {A, A}, B2 = {B, B};
    const uint8_t* xs = reinterpret_cast<const uint8_t*>(x + row.h);
    const int sh = (int)(reinterpret_cast<uintptr_t>(xs) & 15);
    const uint4* xp = reinterpret_cast<const uint4*>(xs - sh);
    auto put = [&](int i, const uint4& q) {
      float f[N];
#pragma unroll
      for (int k = 0; k < N / 2; ++k) {
        float2 t = fma2(add2(Logits<T>::pair(q, k), m2), c2, n2);
        float2 o = {ex2(t.x), ex2(t.y)};
        if (ENT) {
          t = {fmaxf(t.x, -1e4f), fmaxf(t.y, -1e4f)};   // (a word of probability 0 gets 0)
          o = mul2(o, fma2(t, B2, A2));
        } else {
          o = mul2(o, A2);
        }
        f[2 * k] = o.x;
        f[2 * k + 1] = o.y;
      }
      dp[i] = Piece<T>::put(f);
    };
    if (sh == 0) {
      int i = p0 + tid;
      if (i + 3 * NT < p1) {   // as in the forward
        uint4 qa[2], qb[2];
        auto fetch = [&](uint4(&q)[2], int at) {
          q[0] = __ldcs(xp + at);
          q[1] = __ldcs(xp + at + NT);
        };
        fetch(qa, i);
        fetch(qb, i + 2 * NT);
        while (true) {
          const int at = i;
          i += kUnroll * NT;
          const bool more = i + 3 * NT < p1;
          put(at, qa[0]);
          put(at + NT, qa[1]);
          if (more) fetch(qa, i);
          put(at + 2 * NT, qb[0]);
          put(at + 3 * NT, qb[1]);
          if (!more) break;
          fetch(qb, i + 2 * NT);
        }
      }
      for (; i < p1; i += NT) put(i, __ldcs(xp + i));
    } else {
      // a piece of the result spans two of the logits; those at the row's ends may reach past it
      const int f0 = row.h * (int)sizeof(T) >= sh ? 0 : 1;
      const long long left = (long long)(V - row.h) * (int)sizeof(T) + sh;   // bytes from xp to the row's end
      const int f1 = (int)min((long long)row.P, (left - 16) / 16);
      for (int i = p0 + tid; i < p1; i += NT) {
        if (i >= f0 && i < f1) {
          put(i, join_bytes(xp[i], xp[i + 1], sh));
        } else {
          for (int e = 0; e < N; ++e) d[row.h + i * N + e] = from_f32<T>(one(to_f32(x[row.h + i * N + e])));
        }
      }
    }
  }
  if (part == 0 && tid < row.h + row.rest) {
    const int j = row.edge(tid);
    d[j] = from_f32<T>(one(to_f32(x[j])));
  }
  __syncthreads();
  const int k0 = tid < kMaxTop ? tid : kMaxTop;
  if (tid <= kMaxTop && at[k0] >= 0) {
    const int j = at[k0], i = (j - row.h) / N;
    const bool edge = j < row.h || j >= V - row.rest;
    if (edge ? part == 0 : i >= p0 && i < p1) {
      float v = 0.f;
      for (int k = 0; k < kWords; ++k)
        if (at[k] == j) v += g_at[k];
      d[j] = from_f32<T>(fmaf(v, a.scale, one(x_at[k0])));
    }
  }
}

// (the factor of a difference in powers of two, and its inverse, are f32 numbers)
bool scale_ok(float s) { return s >= 0x1p-126f && s <= 0x1p126f; }
bool rows_ok(long long ld, int V, const void* p, int type) {
  return p && ld >= V && aligned(p, type_bytes(type));
}

// Threads to a CTA of the gradient: see score_threads (8192 rows by 256, 128 and 64 threads: 1000 bf16 36, 19 and 14
// us, 8000 bf16 80, 59, 53, 18240 bf16 113, 106, 108, 50304 bf16 262, 267, 273; 592 of 4096 bf16 3.5, 3.0, 3.3).
int grad_threads(int n, double bytes) {
  if (n <= kRound) return n > kSMs && bytes <= 8192 ? 128 : 256;
  return bytes <= 16384 ? 64 : bytes <= 49152 ? 128 : 256;
}

// CTAs to a row of the gradient: a CTA reads and writes 5.5 B/ns each and has 2 us to spend besides;
// it has 4 KB at least.
int grad_split(int n, double bytes) {
  double best = 1e300;
  int split = 1;
  for (int c = 1; c <= 64 && (c == 1 || bytes / c >= 4096.0) && (long long)n * c <= 0x7fffffffLL; c *= 2) {
    const long long waves = ((long long)n * c + 4 * kSMs - 1) / (4 * kSMs);
    const double us = waves * (bytes / c / 5.5e3 + 2.0);
    if (us < best) best = us, split = c;
  }
  return split;
}

// f(the number as a type)
template <class F>
int by_threads(int threads, F&& f) {
  return threads == 64 ? f(std::integral_constant<int, 64>()) : threads == 128 ? f(std::integral_constant<int, 128>())
                                                                               : f(std::integral_constant<int, 256>());
}

// Threads to a CTA that has a row: what a row costs besides its bytes is latency and its warps' instructions, so short
// rows are for few warps, and more rows at a time (8192 rows by 256, 128 and 64 threads: 1000 bf16 31, 16 and 10 us,
// 8000 bf16 44, 31, 29, 18240 bf16 64, 53, 58 and with 20 alternatives 123, 96, 124, 50304 bf16 135, 129, 143 and with
// 20 alternatives 200, 203, 271; 592 of 2048 bf16 2.7, 2.3, 2.6, of 4096 2.8, 2.9, 3.1).
int score_threads(int n, double bytes, int top) {
  if (n <= kRound) return bytes <= 4096 ? 128 : 256;
  if (n > 2 * kRound && bytes <= 16384) return 64;
  return bytes <= (top > 8 ? 49152 : 110e3) ? 128 : 256;
}

// CTAs to a row: the split with the shortest time by what was measured. A CTA reads 16-bit rows at 20 B/ns where it has
// the SM alone, at 10 where four share it (instructions), f32 at 21 and 16, HBM gives 6500, and each round of CTAs adds
// 2 us (a cluster 4) and with alternatives 3 us more (4). (CTAs of 1024 threads for a few rows, each with its whole
// share in flight: 4.5 us instead of 3.5 for one row of 49152 f32, and 16 clusters of eight such CTAs do not fit the
// GPU at once, 18.2 us instead of 9.0 for 16 rows of 128256 with 20 alternatives. Nor do 74 clusters of eight of 256:
// 11.7 us, of four 9.0.)
template <class T, bool ENT>
int score_launch(ScoreArgs& k, cudaStream_t st) {
  constexpr double kRate[4] = {sizeof(T) == 4 ? 21e3 : 20e3, sizeof(T) == 4 ? 20.5e3 : 17.5e3,
                               sizeof(T) == 4 ? 18e3 : 13e3, sizeof(T) == 4 ? 16e3 : 10e3};
  const double row = (double)k.V * sizeof(T);
  double best = 1e300;
  for (int c = 1; c <= 8 && (long long)k.n * c <= 0x7fffffffLL; c *= 2) {
    const double bytes = row / c;
    const int room = c == 8 ? 512 : kRound, full = k.n * c / room, rest = k.n * c % room;
    double us = full * std::max(room * bytes / 6500e3, bytes / kRate[3]);
    if (rest) us += std::max(rest * bytes / 6500e3, bytes / kRate[std::min(3, (rest - 1) / kSMs)]);
    us += (full + (rest > 0)) * ((c == 1 ? 2.0 : 4.0) + (!k.top ? 0.0 : c == 1 ? 3.0 : 4.0));
    if (us < best) best = us, k.split = c;
  }
  const int threads = k.split == 1 ? score_threads(k.n, row, k.top) : 256;
  // the last, half empty round's rows by pairs: 600 rows of 128256 bf16 32.4 us instead of 37.3, 1300 57 instead of 60
  // (by fours 39 and 60; with 20 alternatives 2500 of 32000 56, not 52)
  k.whole = k.split == 1 ? k.n : 0;
  const int rest = k.n % kRound;
  if (threads == 256 && k.split == 1 && k.n > kRound && rest && rest <= kRound / 2 && row >= 96e3)
    k.split = 2, k.whole -= rest;
  const int grid = k.whole + (k.n - k.whole) * k.split;
  if (k.split > 1) return launch_pdl_cluster(score_kernel<256, T, ENT, true>, dim3(grid), dim3(256), 0, st, k.split, k);
  return by_threads(threads, [&](auto nt) {
    constexpr int NT = decltype(nt)::value;
    return launch_pdl(score_kernel<NT, T, ENT, false>, dim3(grid), dim3(NT), 0, st, k);
  });
}

template <class T>
int prepare_type() {
  int bad = load_kernel(score_kernel<256, T, false, true>) | load_kernel(score_kernel<256, T, true, true>);
  for (int threads : {64, 128, 256})
    bad |= by_threads(threads, [&](auto nt) {
      constexpr int NT = decltype(nt)::value;
      return load_kernel(score_kernel<NT, T, false, false>) | load_kernel(score_kernel<NT, T, true, false>) |
             load_kernel(score_grad_kernel<NT, T, false>) | load_kernel(score_grad_kernel<NT, T, true>);
    });
  return bad;
}
}  // namespace

int logprobs_prepare() {
  return prepare_type<float>() || prepare_type<__half>() || prepare_type<__nv_bfloat16>() ? -3 : 0;
}

}  // namespace tb2

extern "C" {

int tb2_rows_prepare(void) {
  using namespace tb2;
  return !device_error_word() || logprobs_prepare() || experts_prepare() || multi_adamw_prepare() ? -3 : 0;
}

int tb2_logprobs(const tb2_logprobs_args* a, void* stream) {
  using namespace tb2;
  if (!a || a->n_rows < 0 || a->vocab < 1 || !row_type_ok(a->row_type)) return -1;
  if (a->n_rows == 0) return 0;
  if (!rows_ok(a->ld, a->vocab, a->logits, a->row_type) || !scale_ok(a->scale)) return -1;
  if (!a->tokens || !a->logprob || !a->stats || a->top < 0 || a->top > kMaxTop || a->top > a->vocab) return -1;
  if (a->top && (!a->top_ids || !a->top_logprobs)) return -1;
  if (!all_aligned(8, {a->tokens, a->stats, a->top_ids}) || !all_aligned(4, {a->logprob, a->entropy, a->top_logprobs}))
    return -1;
  int* err = device_error_word();
  if (!err) return -3;
  ScoreArgs k = {a->logits, a->ld, a->tokens, a->logprob, a->stats, a->entropy, a->top_logprobs, a->top_ids, err,
                 a->scale, a->n_rows, a->vocab, a->top, 0, 1};
  return by_row_type(a->row_type, [&](auto t) {
    using T = decltype(t);
    return a->entropy ? score_launch<T, true>(k, static_cast<cudaStream_t>(stream))
                      : score_launch<T, false>(k, static_cast<cudaStream_t>(stream));
  });
}

int tb2_logprobs_grad(const tb2_logprobs_grad_args* a, void* stream) {
  using namespace tb2;
  if (!a || a->n_rows < 0 || a->vocab < 1 || !row_type_ok(a->row_type)) return -1;
  if (a->n_rows == 0) return 0;
  if (!rows_ok(a->ld, a->vocab, a->logits, a->row_type) || !scale_ok(a->scale)) return -1;
  if (!rows_ok(a->ldd, a->vocab, a->d_logits, a->row_type)) return -1;
  if (a->d_logits == a->logits && a->ldd != a->ld && a->n_rows > 1) return -1;
  if (a->d_logits != a->logits &&
      !rows_apart(a->d_logits, a->ldd, a->n_rows, a->logits, a->ld, a->n_rows, a->vocab, a->row_type))
    return -1;
  if (!a->tokens || !a->stats || a->top < 0 || a->top > kMaxTop || a->top > a->vocab) return -1;
  if (a->top && (!a->top_ids || !a->g_top)) return -1;
  if (a->g_entropy && !a->entropy) return -1;
  if (!all_aligned(8, {a->tokens, a->stats, a->top_ids}) ||
      !all_aligned(4, {a->entropy, a->g_logprob, a->g_entropy, a->g_top}))
    return -1;
  int* err = device_error_word();
  if (!err) return -3;
  GradArgs k = {a->logits, a->ld, a->tokens, a->stats, a->entropy, a->g_logprob, a->g_entropy, a->g_top, a->top_ids,
                a->d_logits, a->ldd, err, a->scale, a->n_rows, a->vocab, a->top, 0, 1};
  return by_row_type(a->row_type, [&](auto t) {
    using T = decltype(t);
    const double bytes = (double)k.V * sizeof(T);
    const int threads = grad_threads(k.n, bytes);
    // full rounds take a row to a CTA, and only the rows of the last are split (700 rows of 128256 bf16 63 us, all
    // alike 69); longer rows are better split throughout (600 of 400000 159 us, not 167: CTAs do not end together)
    if (threads < 256) k.whole = k.n;
    else if (k.n > kRound && bytes <= 3e5) k.whole = k.n - k.n % kRound;
    if (k.whole < k.n) k.split = grad_split(k.n - k.whole, bytes);
    return by_threads(threads, [&](auto nt) {
      constexpr int NT = decltype(nt)::value;
      return launch_pdl(k.g_h ? score_grad_kernel<NT, T, true> : score_grad_kernel<NT, T, false>,
                        dim3(k.whole + (k.n - k.whole) * k.split), dim3(NT), 0, static_cast<cudaStream_t>(stream), k);
    });
  });
}

}  // extern "C"
