// An AdamW step over many tensors in one launch, moments in 32 or in 8 bits.
//
// With hp = [a, b1, b2, eps, wd, c1, c2] (the 7-slot row of opt_step_adamw) and
// g the gradient times the factor:
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,
//   p = (1 - a wd) p - a c1 m / (sqrt(c2) sqrt(v) + eps).
// In 8 bits a block of 256 values of a tensor shares a power of two, the
// smallest that brings the block within 448, and each value is its e4m3
// rounding: m itself, v by its square root. A positive root keeps at least the
// smallest code, as a second moment of 0 under a first moment that is not
// would make the next step boundless.
#include <cuda_fp8.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstring>
#include <iterator>
#include <type_traits>

#include "rows.cuh"
#include "runtime.cuh"

namespace tb2 {
namespace {

constexpr int kBlock = 256;        // values that share a scale
constexpr long long kMaxValues = 1LL << 37;   // of a tensor (its blocks, and a launch's, are counted in 30 bits)
constexpr int kMaxTensors = 448;   // tensors a launch: their descriptors travel as its arguments (30.5 of 32 KB)
constexpr int kThreads = 256, kWarps = kThreads / 32, kRun = 4;
constexpr int kStepRun = 2;
constexpr int kCtas8 = 3, kCtas32 = 3;   // CTAs an SM: 80 registers a thread

struct Tensors {
  tb2_adamw_tensor t[kMaxTensors];
  int first[kMaxTensors + 2];             // blocks before tensor i; behind the last one, all
  unsigned whole[(kMaxTensors + 31) / 32];   // bit i: tensor i's arrays are on the boundaries of four values
  int n;
  long long before;                       // blocks of earlier launches
};

// The tensor that block b is of.
__device__ __forceinline__ int tensor_of(const Tensors& ts, int b) {
  int lo = 0, hi = ts.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (ts.first[mid] <= b) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// On from tensor i to the one that block b is of: a step or two, or a search where tensors are small.
__device__ __forceinline__ int tensor_from(const Tensors& ts, int i, int b) {
  if (ts.first[i + 1] > b) return i;
  if (ts.first[i + 2] > b) return i + 1;   // (first has an entry past the last tensor's end)
  return tensor_of(ts, b);
}

// Four values: a lane has values 4 lane .. 4 lane + 3 and 128 more of a block, so that a warp's reads and writes are
// contiguous in every type.
template <class T>
__device__ __forceinline__ void store4(void* p, long long i, const float* f) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = make_float4(f[0], f[1], f[2], f[3]);
  } else {
    uint2 u;
    if constexpr (std::is_same<T, __half>::value) {
      const __half2 h[2] = {__floats2half2_rn(f[0], f[1]), __floats2half2_rn(f[2], f[3])};
      memcpy(&u, h, 8);
    } else {
      const __nv_bfloat162 h[2] = {__floats2bfloat162_rn(f[0], f[1]), __floats2bfloat162_rn(f[2], f[3])};
      memcpy(&u, h, 8);
    }
    *reinterpret_cast<uint2*>(static_cast<T*>(p) + i) = u;
  }
}
__device__ __forceinline__ void load4_e4m3(unsigned u, float* f) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const __half2 h(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(u >> 16 * k), __NV_E4M3));
    f[2 * k] = __low2float(h);
    f[2 * k + 1] = __high2float(h);
  }
}
__device__ __forceinline__ unsigned pack4_e4m3(const float* f) {
  const unsigned lo = __nv_cvt_float2_to_fp8x2(make_float2(f[0], f[1]), __NV_SATFINITE, __NV_E4M3);
  const unsigned hi = __nv_cvt_float2_to_fp8x2(make_float2(f[2], f[3]), __NV_SATFINITE, __NV_E4M3);
  return lo | hi << 16;
}

// The e4m3 code of t >= 0 (within 448), given to 64 bits: rounded once.
__device__ __noinline__ unsigned e4m3_of(double t) {
  const int e = t < 0.015625 ? -6 : ilogb(t);
  const double q = ldexp(rint(ldexp(t, 3 - e)), e - 3);   // eighths of the leading bit; at the bottom, steps of 2^-9
  return __nv_cvt_float_to_fp8((float)q, __NV_SATFINITE, __NV_E4M3);
}

// Within 2^-23. FTZ: a number below 2^-126 is 0, which 8-bit moments allow; second moments in f32 go on below that, and
// their roots are far above it. (With f32 moments the correctly rounded root and quotient took 623 us instead of 562
// for 135M weights: their rare paths cost registers.)
template <bool FTZ>
__device__ __forceinline__ float sqrt_near(float x) {
  float r;
  if (FTZ) asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  else asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float inverse_near(float x) {   // within 2^-23
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// The larger magnitude, NaN above all.
__device__ __forceinline__ float top_of(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
  return r;
}

// A block's largest magnitude, from its lanes', as the bits of an f32.
__device__ __forceinline__ unsigned block_top(float top) {
  return __reduce_max_sync(0xffffffffu, __float_as_uint(top) & 0x7fffffffu);
}
// A block's power of two, from the bits of its largest magnitude, and the factor to it: the smallest 2^e with top <=
// 448 2^e (448 = 1.75 2^8), 2^-100 at least; NaN where top is not finite.
__device__ __forceinline__ float block_scale(unsigned b, float& inverse) {
  const int e = max((int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u), -100);
  const bool ok = b < 0x7f800000u;
  inverse = ok ? __uint_as_float((unsigned)(127 - e) << 23) : NAN;
  return ok ? __uint_as_float((unsigned)(127 + e) << 23) : NAN;
}

// The step's factors; dg is (1 - b1) times the gradients' factor, sb2 sqrt(b2), sd2 sqrt(1 - b2) times that factor.
struct Hyper {
  double b1_64, dg_64;
  float b1, b2, eps, keep, c1, c2, gf, dg, d2, sb2, sd2;
};

// f64 to f32 so that rounding the result to few bits rounds the f64 value once: cut, the last bit set where that left
// something out.
__device__ __forceinline__ float to_odd(double x) {
  const float f = __double2float_rz(x);
  return __uint_as_float(__float_as_uint(f) | ((__double2loint(x) & 0x1fffffff) != 0));
}

// From 64 bits and the operands in memory: a root next to a border, its code, and whether it is above a block's border.
__device__ __forceinline__ double wide_root(float g, float gf, float r0, float b2) {
  const double gw = (double)g * gf, v = (double)r0 * r0 * b2 + gw * gw * (1.0 - (double)b2);
  return sqrt(v);
}
__device__ __noinline__ unsigned root_code(float g, float gf, float r0, float b2, float inverse) {
  return max(e4m3_of(wide_root(g, gf, r0, b2) * inverse), 1u);
}
__device__ __noinline__ bool root_above(float g, float gf, float r0, float b2, float border) {
  return wide_root(g, gf, r0, b2) > (double)border;
}
__device__ __forceinline__ void put_byte(unsigned& w, int at, unsigned q) {
  w = (w & ~(0xffu << 8 * at)) | q << 8 * at;
}

// A warp has a block at a time. Where CTAs end after a few blocks the GPU works in few pages at any time, which is what
// HBM likes best (135M weights: f32 moments 563 us, with a grid that stays and deals the blocks out 586, with a run of
// blocks to each CTA 617; the values of 8-bit moments 210, 240 and 267). The 8-bit step has more to compute, and CTAs
// that start anew with the factors take 475 us: its grid stays, and each CTA has two blocks a warp in a row (429 us;
// one 447, four 443, a run of all its blocks 489).
//
// 8-bit moments without a seed are the exact values rounded once, although the step is f32. m is a sum of two terms of
// either sign, and with few bits in its old value it falls on a border again and again (0.9 of 120 is 108, between 104
// and 112: 0.8 % of the values of a run with b1 = 0.9 are closer to one than f32 tells), so it is computed in f64, two
// products and three conversions a value, and converted so that the code is rounded from all its bits. A root's code is
// taken of both ends of an interval that holds the exact one, and where the two differ (one value in 90000) it is
// rounded from 64 bits. With U = 2^-24: the root's square is a sum of squares, the held root's factor and product 2 + 1
// U, the gradient's 3 + 1, doubled by squaring, 1 for a square and 1 for the sum; the root halves these 10, and is off
// by 2 U itself: 7 U of the 8 allowed. With a seed the step stays in f32, and the random bits take its place (456 us
// instead of 425 for 135M weights; 484 with bits of their own for m and the root).
//
// Bound by HBM in 32 bits. In 8 bits a value is 16 bytes, the time of some 75 instructions at most: a look at the
// distance of every root from a border made it 58 (445 us where the bytes of 135M weights take 332), IEEE quotients and
// roots besides 103 (508 us).
// A lane's values of a block as they lie in memory.
template <class T>
struct Raw4 {
  using Bits = typename std::conditional<sizeof(T) == 2, uint2, unsigned>::type;
  typename std::conditional<sizeof(T) == 4, float4, Bits>::type v;
  __device__ __forceinline__ void load(const void* p, long long i) {
    v = __ldcs(reinterpret_cast<const decltype(v)*>(static_cast<const T*>(p) + i));
  }
  __device__ __forceinline__ void get(float* f) const {
    if constexpr (sizeof(T) == 4) {
      f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
    } else if constexpr (sizeof(T) == 2) {
      T t[4];
      memcpy(t, &v, 8);
#pragma unroll
      for (int k = 0; k < 4; ++k) f[k] = to_f32<T>(t[k]);
    } else {
      load4_e4m3(v, f);
    }
  }
};
template <class P, class G, class S>
struct RawBlock {
  Raw4<P> p[2];
  Raw4<G> g[2];
  Raw4<S> m[2], v[2];
  float ms, vs;
};

// A lane's eight values, stepped: p the new weights, m the new first moments, r the new second moments (32 bits) or
// their roots (8 bits).
template <int BITS, bool RANDOM>
__device__ __forceinline__ void step8(const Hyper& h, float (&p)[8], const float (&g)[8], float (&m)[8], float (&r)[8],
                                      float ms, float vs) {
  const float rs = vs * h.sb2;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float v;
    if (BITS == 8) {
      m[e] = RANDOM ? fmaf(m[e] * ms, h.b1, g[e] * h.dg)
                    : to_odd(fma((double)(m[e] * ms), h.b1_64, (double)g[e] * h.dg_64));
      const float gs = g[e] * h.sd2, r0 = r[e] * rs;
      v = fmaf(gs, gs, r0 * r0);
    } else {
      const float gg = g[e] * h.gf;
      m[e] = fmaf(m[e], h.b1, g[e] * h.dg);
      v = fmaf(r[e], h.b2, gg * gg * h.d2);
    }
    const float root = sqrt_near<BITS == 8>(v);
    p[e] = fmaf(-h.c1 * m[e], inverse_near(fmaf(root, h.c2, h.eps)), p[e] * h.keep);
    r[e] = BITS == 8 ? root : v;
  }
}

// 32 bits that look random, of x: the low-bias integer hash that C. Wellons published (xor, shift and multiply, with
// constants found by search).
__device__ __forceinline__ unsigned mixed(unsigned x) {
  x = (x ^ x >> 16) * 0x7feb352du;
  x = (x ^ x >> 15) * 0x846ca68bu;
  return x ^ x >> 16;
}
// t (|t| <= 448) rounded to an e4m3 value next to it, the upper one with the probability of t's place between the two:
// 16 random bits are added below the three that stay. (Codes below 2^-6 are 2^-9 apart, as they are just above it.)
__device__ __forceinline__ float rounded_by(float t, unsigned bits16) {
  const float low = fabsf(t) < 0.015625f ? 0.015625f : 0.f;
  const unsigned b = (__float_as_uint(fabsf(t) + low) + (bits16 << 4)) & 0xfff00000u;
  return copysignf(__uint_as_float(b) - low, t);
}

// The block's codes and scales. RANDOM: rounded by random bits of `key`; else again(e) gives value e's root code from
// 64 bits, given the factor, and above(e) whether the root is above a border.
template <bool RANDOM, class F, class A>
__device__ __forceinline__ void hold8(float (&m)[8], const float (&r)[8], unsigned (&mq)[2], unsigned (&vq)[2],
                                      float& ms, float& vs, unsigned key, F&& again, A&& above) {
  float top_m = 0.f, top_r = 0.f, mi, ri;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    top_m = top_of(top_m, m[e]);
    top_r = top_of(top_r, r[e]);
  }
  ms = block_scale(block_top(top_m), mi);
  const unsigned top = block_top(top_r);
  vs = block_scale(top, ri);
  if (RANDOM) {
    unsigned bits = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float a[4], z[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (e % 2 == 0) bits = mixed(key + (4 * j + e) * 0x9e3779b9u);   // 16 for each value, m's and the root's
        const unsigned mine = e % 2 ? bits >> 16 : bits & 0xffffu;
        a[e] = rounded_by(m[4 * j + e] * mi, mine);
        z[e] = rounded_by(r[4 * j + e] * ri, mine);
        z[e] = r[4 * j + e] > 0.f ? fmaxf(z[e], 0x1p-9f) : z[e];   // a positive root keeps the smallest code
      }
      mq[j] = pack4_e4m3(a);
      vq[j] = pack4_e4m3(z);
    }
    return;
  }
  const float low = ri * (1.f - 0x1p-21f), high = ri * (1.f + 0x1p-21f);
  unsigned look[2];   // nonzero bytes: roots to be looked at
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    float a[4], z[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      m[4 * j + e] *= mi;
      a[e] = r[4 * j + e] * low;
      z[e] = r[4 * j + e] * high;
    }
    mq[j] = pack4_e4m3(m + 4 * j);
    vq[j] = pack4_e4m3(z);
    // (and those of code 0: a positive root keeps the smallest one)
    look[j] = (vq[j] ^ pack4_e4m3(a)) | (~(vq[j] + 0x7f7f7f7fu) & 0x80808080u);
  }
  // A largest root within 8 U of 448 times a power of two, that is 1.75 times one (U of it is 7 / 8 of its steps), one
  // block in a million: the side that the exact one lies on, and the codes, from 64 bits. (135M weights with bf16
  // gradients 425 us as without this look, with f32 ones 425 instead of 415; ahead of the codes 448 and 460, and with
  // roots returned in 64 bits instead of codes and answers 446 and 422.)
  if ((top & 0x7fffffu) - 0x5ffff0u <= 0x20u && top < 0x7f800000u) {
    const unsigned border = (top & 0xff800000u) | 0x600000u;
    bool over = false;
#pragma unroll 1
    for (int e = 0; e < 8; ++e) over |= above(e, __uint_as_float(border));
    vs = block_scale(border + __any_sync(0xffffffffu, over), ri);
    look[0] = look[1] = ~0u;
  }
  if (look[0] | look[1]) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if ((look[e / 4] >> 8 * (e % 4) & 0xff) && r[e] > 0.f && ri == ri)
        put_byte(vq[e / 4], e % 4, again(e, ri));
  }
}

__device__ __forceinline__ float held_code(const void* v, long long k) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<const uint8_t*>(v)[k], __NV_E4M3)));
}

// The next block is read while one is computed where it lies whole on its boundaries; a tensor's end, or one off its
// boundaries, goes value by value. (Reads staged further ahead, by asynchronous copies to shared memory or in runs of
// four blocks with one address each, took as long in 8 bits, 454 and 467 us: what is left is not the reads' latency.)
template <class P, class G, int BITS, bool RANDOM>
__global__ void __launch_bounds__(kThreads, BITS == 8 ? kCtas8 : kCtas32)
    step_kernel(const __grid_constant__ Tensors ts, int copy_type, const float* hp, const float* factor,
                const long long* seed) {
  using S = typename std::conditional<BITS == 8, uint8_t, float>::type;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  // kStepRun blocks to a warp; then a 32-bit CTA ends, and an 8-bit one goes on behind all the grid's
  constexpr int kCta = kWarps * kStepRun;
  const int all = ts.first[ts.n], first = blockIdx.x * kCta;
  const int end = BITS == 8 ? all : min(all, first + kCta);
  int b = first + warp, left = kStepRun - 1;
  int i = tensor_of(ts, min(b, end - 1));
  griddep_wait();
  Hyper h;
  h.b1 = hp[1]; h.b2 = hp[2]; h.eps = hp[3];
  h.keep = 1.f - hp[0] * hp[4];
  h.c1 = hp[0] * hp[5];
  h.c2 = sqrtf(hp[6]);
  h.gf = factor ? *factor : 1.f;
  h.b1_64 = h.b1;
  h.dg_64 = (1.0 - h.b1_64) * (double)h.gf;
  h.dg = (float)h.dg_64;
  h.d2 = 1.f - h.b2;
  h.sb2 = sqrtf(h.b2);
  h.sd2 = h.gf * sqrtf(h.d2);
  // random bits: of the seed, the block's number among all and the lane
  unsigned key0 = 0, key1 = 0;
  if (RANDOM) {
    const unsigned long long x = (unsigned long long)*seed;
    key0 = mixed((unsigned)x) ^ (unsigned)(ts.before >> 32);
    key1 = mixed((unsigned)(x >> 32) + 0x51ed270bu) + lane * 0x85ebca6bu;
  }
  RawBlock<P, G, S> raw;
  // block b of tensor i on its way; whether it is one that is read so
  auto fetch = [&](int b) {
    const tb2_adamw_tensor& t = ts.t[i];
    const int blk = b - ts.first[i];
    const long long k0 = (long long)blk * kBlock + 4 * lane;
    const bool whole = (ts.whole[i / 32] >> (i % 32) & 1) && (long long)(blk + 1) * kBlock <= t.n;
    if (BITS == 8) raw.ms = t.m_scale[blk], raw.vs = t.v_scale[blk];
    if (whole) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        raw.p[j].load(t.p, k0 + 128 * j);
        raw.g[j].load(t.g, k0 + 128 * j);
        raw.m[j].load(t.m, k0 + 128 * j);
        raw.v[j].load(t.v, k0 + 128 * j);
      }
    }
    return whole;
  };
  if (b >= end) return;
  bool next_whole = fetch(b);
  while (true) {
    const tb2_adamw_tensor& t = ts.t[i];
    const int blk = b - ts.first[i];
    const long long k0 = (long long)blk * kBlock + 4 * lane;
    int stride = kWarps;
    if (BITS == 8 && left-- == 0) {
      stride += ((int)gridDim.x - 1) * kCta;
      left = kStepRun - 1;
    }
    const bool whole = next_whole, more = end - b > stride;
    float p[8], g[8], m[8], r[8];
    const float ms = raw.ms, vs = raw.vs;
    if (whole) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        raw.p[j].get(p + 4 * j);
        raw.g[j].get(g + 4 * j);
        raw.m[j].get(m + 4 * j);
        raw.v[j].get(r + 4 * j);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const long long k = k0 + 128 * (e / 4) + e % 4;
        const bool on = k < t.n;
        p[e] = on ? to_f32(static_cast<const P*>(t.p)[k]) : 0.f;
        g[e] = on ? to_f32(static_cast<const G*>(t.g)[k]) : 0.f;
        if (BITS == 8) {
          m[e] = on ? held_code(t.m, k) : 0.f;
          r[e] = on ? held_code(t.v, k) : 0.f;
        } else {
          m[e] = on ? static_cast<const float*>(t.m)[k] : 0.f;
          r[e] = on ? static_cast<const float*>(t.v)[k] : 0.f;
        }
      }
    }
    if (more) {
      i = tensor_from(ts, i, b + stride);   // (t is still block b's)
      next_whole = fetch(b + stride);
    }
    step8<BITS, RANDOM>(h, p, g, m, r, ms, vs);
    unsigned mq[2], vq[2];
    if (BITS == 8) {
      float nms, nvs;
      const unsigned key = RANDOM ? mixed(mixed((unsigned)(ts.before + b) ^ key0) + key1) : 0;
      auto place = [&](int e) { return k0 + 128 * (e / 4) + e % 4; };
      auto grad = [&](long long k) { return to_f32(static_cast<const G*>(t.g)[k]); };
      hold8<RANDOM>(
          m, r, mq, vq, nms, nvs, key,
          [&](int e, float ri) {
            const long long k = place(e);
            return k < t.n ? root_code(grad(k), h.gf, held_code(t.v, k) * vs, h.b2, ri) : 0u;
          },
          [&](int e, float border) {
            const long long k = place(e);
            return k < t.n && root_above(grad(k), h.gf, held_code(t.v, k) * vs, h.b2, border);
          });
      if (lane == 0) t.m_scale[blk] = nms, t.v_scale[blk] = nvs;
    }
    if (whole) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        store4<P>(t.p, k0 + 128 * j, p + 4 * j);
        if (t.copy) {
          if (sizeof(P) == 2) {
#pragma unroll
            for (int e = 0; e < 4; ++e) p[4 * j + e] = to_f32(from_f32<P>(p[4 * j + e]));
          }
          if (copy_type == kTypeF16) store4<__half>(t.copy, k0 + 128 * j, p + 4 * j);
          else store4<__nv_bfloat16>(t.copy, k0 + 128 * j, p + 4 * j);
        }
        if (BITS == 8) {
          *reinterpret_cast<unsigned*>(static_cast<uint8_t*>(t.m) + k0 + 128 * j) = mq[j];
          *reinterpret_cast<unsigned*>(static_cast<uint8_t*>(t.v) + k0 + 128 * j) = vq[j];
        } else {
          store4<float>(t.m, k0 + 128 * j, m + 4 * j);
          store4<float>(t.v, k0 + 128 * j, r + 4 * j);
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const long long k = k0 + 128 * (e / 4) + e % 4;
        if (k >= t.n) continue;
        const P q = from_f32<P>(p[e]);
        static_cast<P*>(t.p)[k] = q;
        if (t.copy) {
          if (copy_type == kTypeF16) static_cast<__half*>(t.copy)[k] = from_f32<__half>(to_f32(q));
          else static_cast<__nv_bfloat16*>(t.copy)[k] = from_f32<__nv_bfloat16>(to_f32(q));
        }
        if (BITS == 8) {
          static_cast<uint8_t*>(t.m)[k] = (uint8_t)(mq[e / 4] >> 8 * (e % 4));
          static_cast<uint8_t*>(t.v)[k] = (uint8_t)(vq[e / 4] >> 8 * (e % 4));
        } else {
          static_cast<float*>(t.m)[k] = m[e];
          static_cast<float*>(t.v)[k] = r[e];
        }
      }
    }
    if (!more) return;
    b += stride;
  }
}

// The values that 8-bit moments stand for (p: m's, copy: v's, f32), or (PUT) the moments from those values.
template <bool PUT>
__global__ void __launch_bounds__(kThreads) moments_kernel(const __grid_constant__ Tensors ts) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int all = ts.first[ts.n];
  // a warp has kRun blocks in a row: so many reads are on their way at once
  long long b = ((long long)blockIdx.x * kWarps + warp) * kRun;
  const long long end = min(b + kRun, (long long)all);
  int i = tensor_of(ts, (int)min(b, all - 1LL));
  griddep_wait();
  while (b < end) {
    i = tensor_from(ts, i, (int)b);
    const tb2_adamw_tensor& t = ts.t[i];
    const int blk = (int)(b - ts.first[i]);
    const long long k0 = (long long)blk * kBlock + 4 * lane;
    const bool aligned = ts.whole[i / 32] >> (i % 32) & 1, whole = aligned && (long long)(blk + 1) * kBlock <= t.n;
    const bool run = !PUT && aligned && b + kRun <= end && (long long)(blk + kRun) * kBlock <= t.n;
    b += run ? kRun : 1;
    if (run) {
      unsigned mq[2 * kRun], vq[2 * kRun];
      float ms[kRun], vs[kRun];
#pragma unroll
      for (int j = 0; j < 2 * kRun; ++j) {
        mq[j] = __ldcs(reinterpret_cast<const unsigned*>(static_cast<uint8_t*>(t.m) + k0 + 128 * j));
        vq[j] = __ldcs(reinterpret_cast<const unsigned*>(static_cast<uint8_t*>(t.v) + k0 + 128 * j));
      }
#pragma unroll
      for (int j = 0; j < kRun; ++j) ms[j] = t.m_scale[blk + j], vs[j] = t.v_scale[blk + j];
#pragma unroll
      for (int j = 0; j < 2 * kRun; ++j) {
        float m[4], r[4];
        load4_e4m3(mq[j], m);
        load4_e4m3(vq[j], r);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          m[e] *= ms[j / 2];
          r[e] *= vs[j / 2];
          r[e] *= r[e];
        }
        store4<float>(t.p, k0 + 128 * j, m);
        store4<float>(t.copy, k0 + 128 * j, r);
      }
      continue;
    }
    uint8_t *mp = static_cast<uint8_t*>(t.m), *vp = static_cast<uint8_t*>(t.v);
    float *mo = static_cast<float*>(t.p), *vo = static_cast<float*>(t.copy);
    float m[8], r[8];
    if (!PUT) {
      const float ms = t.m_scale[blk], vs = t.v_scale[blk];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        unsigned mq = 0, vq = 0;
        if (whole) {
          mq = *reinterpret_cast<const unsigned*>(mp + k0 + 128 * j);
          vq = *reinterpret_cast<const unsigned*>(vp + k0 + 128 * j);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (k0 + 128 * j + e < t.n) {
              mq |= (unsigned)mp[k0 + 128 * j + e] << 8 * e;
              vq |= (unsigned)vp[k0 + 128 * j + e] << 8 * e;
            }
        }
        load4_e4m3(mq, m + 4 * j);
        load4_e4m3(vq, r + 4 * j);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        m[e] *= ms;
        r[e] *= vs;
        r[e] *= r[e];
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (whole) {
          store4<float>(mo, k0 + 128 * j, m + 4 * j);
          store4<float>(vo, k0 + 128 * j, r + 4 * j);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (k0 + 128 * j + e < t.n) {
              mo[k0 + 128 * j + e] = m[4 * j + e];
              vo[k0 + 128 * j + e] = r[4 * j + e];
            }
        }
      }
      continue;
    }
    float top_m = 0.f, top_r = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const long long k = k0 + 128 * (e / 4) + e % 4;
      m[e] = k < t.n ? mo[k] : 0.f;
      r[e] = k < t.n ? vo[k] : 0.f;
      top_m = top_of(top_m, m[e]);
      top_r = top_of(top_r, r[e] < FLT_MIN && r[e] >= 0.f ? 0.f : sqrtf(r[e]));
    }
    float mi, ri;
    const float ms = block_scale(block_top(top_m), mi), vs = block_scale(block_top(top_r), ri);
    if (lane == 0) t.m_scale[blk] = ms, t.v_scale[blk] = vs;
#pragma unroll 1
    for (int e = 0; e < 8; ++e) {
      const long long k = k0 + 128 * (e / 4) + e % 4;
      if (k >= t.n) continue;
      const float x = mo[k], y = vo[k] < FLT_MIN ? 0.f : vo[k];
      mp[k] = mi == mi ? (uint8_t)(e4m3_of(fabs((double)x * mi)) | (x < 0.f ? 0x80 : 0)) : 0x7f;
      vp[k] = ri == ri ? (uint8_t)max(e4m3_of(sqrt((double)y) * ri), y > 0.f ? 1u : 0u) : 0x7f;
    }
  }
}

bool tensor_ok(const tb2_adamw_tensor& t, int p_type, int g_type, int copy_type, int bits) {
  if (t.n < 0 || t.n > kMaxValues) return false;
  if (t.n == 0) return true;
  if (!t.p || !t.g || !t.m || !t.v || (t.copy && !aligned(t.copy, type_bytes(copy_type)))) return false;
  if (!aligned(t.p, type_bytes(p_type)) || !aligned(t.g, type_bytes(g_type))) return false;
  if (bits == 32) return all_aligned(4, {t.m, t.v});
  return t.m_scale && t.v_scale && all_aligned(4, {t.m_scale, t.v_scale});
}

unsigned ctas_of(long long blocks, int run) { return (unsigned)((blocks + kWarps * run - 1) / (kWarps * run)); }

// The tensors in groups of what a launch takes, empty ones left out. whole(tensor): see Tensors.
template <class W, class F>
int in_groups(const tb2_adamw_tensor* t, int n, W&& whole, F&& launch) {
  Tensors g;
  g.before = 0;
  for (int i = 0; i < n;) {
    g.n = 0;
    std::fill(std::begin(g.whole), std::end(g.whole), 0u);
    long long blocks = 0;
    for (; i < n && g.n < kMaxTensors; ++i) {
      if (t[i].n == 0) continue;
      const long long b = (t[i].n + kBlock - 1) / kBlock;
      if (blocks + b > 0x3fffffffLL) break;
      if (whole(t[i])) g.whole[g.n / 32] |= 1u << (g.n % 32);
      g.first[g.n] = (int)blocks;
      g.t[g.n++] = t[i];
      blocks += b;
    }
    g.first[g.n] = g.first[g.n + 1] = (int)blocks;
    if (g.n)
      if (int rc = launch(g, blocks)) return rc;
    g.before += blocks;
  }
  return 0;
}

template <class P, class G>
int prepare_types() {
  return load_kernel(step_kernel<P, G, 8, false>) || load_kernel(step_kernel<P, G, 8, true>) ||
                 load_kernel(step_kernel<P, G, 32, false>)
             ? -3
             : 0;
}
template <class P>
int prepare_type() {
  return prepare_types<P, float>() || prepare_types<P, __half>() || prepare_types<P, __nv_bfloat16>() ? -3 : 0;
}

}  // namespace

int multi_adamw_prepare() {
  if (load_kernel(moments_kernel<true>) || load_kernel(moments_kernel<false>)) return -3;
  return prepare_type<float>() || prepare_type<__half>() || prepare_type<__nv_bfloat16>() ? -3 : 0;
}

}  // namespace tb2

extern "C" {

int tb2_adamw_multi(const tb2_adamw_multi_args* a, void* stream) {
  using namespace tb2;
  if (!a || a->n_tensors < 0 || (a->n_tensors && !a->tensors) || (a->state_bits != 8 && a->state_bits != 32)) return -1;
  if (!row_type_ok(a->p_type) || !row_type_ok(a->g_type)) return -1;
  if (a->copy_type != kTypeF16 && a->copy_type != kTypeBF16) return -1;
  if (!a->hp || !all_aligned(4, {a->hp, a->grad_scale}) || !aligned(a->seed, 8)) return -1;
  for (int i = 0; i < a->n_tensors; ++i)
    if (!tensor_ok(a->tensors[i], a->p_type, a->g_type, a->copy_type, a->state_bits)) return -1;
  const size_t pb = 4 * type_bytes(a->p_type), gb = 4 * type_bytes(a->g_type), cb = 4 * type_bytes(a->copy_type);
  const size_t sb = a->state_bits == 8 ? 4 : 16;
  auto whole = [&](const tb2_adamw_tensor& t) {
    return aligned(t.p, pb) && aligned(t.g, gb) && aligned(t.copy, cb) && all_aligned(sb, {t.m, t.v});
  };
  return in_groups(a->tensors, a->n_tensors, whole, [&](const Tensors& g, long long blocks) {
    const unsigned most = a->state_bits == 8 ? kCtas8 * kSMs : ~0u, ctas = std::min(ctas_of(blocks, kStepRun), most);
    return by_row_type(a->p_type, [&](auto p) {
      return by_row_type(a->g_type, [&](auto q) {
        using P = decltype(p);
        using G = decltype(q);
        auto* kernel = a->state_bits == 32 ? step_kernel<P, G, 32, false>
                       : a->seed           ? step_kernel<P, G, 8, true>
                                           : step_kernel<P, G, 8, false>;
        return launch_pdl(kernel, dim3(ctas), dim3(kThreads), 0, static_cast<cudaStream_t>(stream), g, a->copy_type,
                          a->hp, a->grad_scale, a->seed);
      });
    });
  });
}

int tb2_adamw_moments(const tb2_adamw_tensor* tensors, int n_tensors, int put, void* stream) {
  using namespace tb2;
  if (n_tensors < 0 || (n_tensors && !tensors)) return -1;
  for (int i = 0; i < n_tensors; ++i) {
    const tb2_adamw_tensor& t = tensors[i];
    if (t.n < 0 || t.n > kMaxValues) return -1;
    if (t.n && (!t.p || !t.copy || !t.m || !t.v || !t.m_scale || !t.v_scale ||
                !all_aligned(4, {t.p, t.copy, t.m_scale, t.v_scale})))
      return -1;
  }
  auto whole = [](const tb2_adamw_tensor& t) {
    return all_aligned(16, {t.p, t.copy}) && all_aligned(4, {t.m, t.v});
  };
  return in_groups(tensors, n_tensors, whole, [&](const Tensors& g, long long blocks) {
    return launch_pdl(put ? moments_kernel<true> : moments_kernel<false>, dim3(ctas_of(blocks, kRun)), dim3(kThreads),
                      0, static_cast<cudaStream_t>(stream), g);
  });
}

}  // extern "C"
