// Attention of one new token per request over a paged key-value cache: the
// kernel, instantiated per cache type in paged_attn_*.cu.
//
//   out[b][h] = sum_t p_t v_t / sum_t p_t,  p_t = 2^(c q . k_t - m),
//
// c = scale log2(e), t over the request's history through its block table,
// m a running maximum, h one of the G = H / KV query heads of key head j.
//
// Bound: every K and V byte is read once, so HBM: at 6.5 TB/s an SM receives
// 23 bytes a clock. A 16-bit cache is then 11.5 values a clock, each multiplied
// by G heads: at G = 8 that is most of what the FMA units can do with the
// conversions and loads on top, so the products run on the tensor cores. One
// token has at most 16 heads to a key head, far below the 128 rows of a
// tcgen05 tile, and its operands would cross shared memory and TMEM twice; the
// warp-level m16n8k16 shape fits and is 3 to 4 times faster than the memory.
//
// f32 accuracy from 16-bit operands: K and V of an f16 / bf16 / Q8_0 cache are
// exact tensor-core operands (int8 quants as f16; their block scales are
// applied to the scores and folded into P); q and P are split into planes that
// sum to them (f16: 2 planes of 11 bits after a power-of-two scaling, bf16: 3
// planes of 8 bits, 2 when the result is rounded to 16 bits anyway). Rows 8..15
// of the 16-row operand hold the second plane of rows 0..7 (HT = 8 heads), so
// two planes cost one instruction; with G > 8 (HT = 16) each plane is one. An
// f32 cache is split the same way into tf32 hi + lo, q and P too. An infinity
// has no such planes (it meets one that is 0, or of the other sign): heads
// whose sums are not finite take their CTA's part of the history again in
// plain f32 (plain_part), so that such keys and values count as the formula
// says.
//
// Split: the work is a list of units (kWarps tiles of TK keys of one request
// and key head), cut into equal ranges, one per CTA, whatever the lengths. A
// CTA's warps take the tiles of a range in turn, each through a ring of its own
// in shared memory filled by cp.async (no barrier between warps inside a
// history), the next history's tiles already in flight while the last one's
// sums are joined. A history that one CTA holds whole is written at once;
// pieces go to the workspace and the CTA that finishes last adds them up in
// order (a ticket per history), so the result does not depend on timing.
//
// Measured on one B200 (cold inputs): 131072 tokens of one request, 32 / 8
// heads of 128, bf16: 101 us, 5.3 TB/s with the launch and 6.3 TB/s between
// 65536 and 131072 tokens; 64 histories up to 8191 (28 / 4 heads of 128, f32
// rows over bf16): 112 us, 4.9 TB/s; 16 up to 2048 (16 / 16 of 128, f32): 73
// us, 5.1 TB/s; 128 up to 4096 (9 / 3 of 64, Q8_0): 42 us, 2.6 TB/s; 77 tokens:
// 6.8 us. A 16-bit or f32 cache waits for the memory (a third of the issue
// slots used). Q8_0 at d_head 64 has 770 instructions per 32 keys, half of them
// the conversions of quants and scales, and fills 58 % of the issue slots: its
// warps wait for one another's results (convert, product, scale) more than for
// the memory or for a slot.
#pragma once
#include <algorithm>
#include <type_traits>

#include "paged.cuh"
#include "pdl.cuh"
#include "runtime.cuh"

namespace tb2 {

constexpr int kAttnWarps = 4;
// Units that are worth another CTA on a history, and a place in its join: one request of 4096 tokens (32 / 8 heads of
// 128, bf16) took 19.0, 15.9, 16.7 and 21.3 us at 1, 2, 4 and 8.
constexpr int kMinUnits = 2;
constexpr int kAttnMaxCtas = 4 * 148;
// workspace: three tickets per CTA (0 between calls; its range may end one history and begin another, and be a group's
// first in both), two partial slots per CTA
constexpr size_t kAttnTicketBytes = (3 * kAttnMaxCtas * sizeof(unsigned) + 255) / 256 * 256;
constexpr size_t kAttnWorkspace =
    kAttnTicketBytes + (size_t)2 * 148 * 2 * sizeof(float) * (16 * 128 + 2 * 16);   // (two CTAs of 16 heads an SM)

enum AttnCache : int { kCacheF32 = 0, kCacheF16 = 1, kCacheBF16 = 2, kCacheQ8 = 3 };

struct PagedAttnArgs {
  PagedKv kv;
  const void* q;
  void* out;
  long long ldq, ldo, table_stride;
  const int* table;
  const int* lens;
  float* lse;
  unsigned* tickets;
  float* slots;
  int* err;
  float c;             // scale * log2(e)
  bool q_vec, out_vec; // rows of q, of out start on 16-byte boundaries
  int n_req, n_heads, group, width, row_type, page_shift;   // page_shift < 0: page_size is no power of two
};

namespace attn {

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool on) {
  const int n = on ? 16 : 0;   // 0: the 16 bytes are zeros and nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
template <int B>
__device__ __forceinline__ void cp_small(uint32_t dst, const void* src, bool on) {
  const int n = on ? B : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(dst), "l"(src), "r"(n), "n"(B) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ uint16_t lds16(uint32_t a) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ void sts16(uint32_t a, uint16_t v) { asm volatile("st.shared.u16 [%0], %1;" ::"r"(a), "h"(v) : "memory"); }

__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a));
}

// D += A B: A [16 x k] (rows g and g + 8 of lane group g), B [k x 8]; FIRST:
// D = A B, without registers of zeros to start from.
#define TB2_MMA(name, shape_types)                                                                                   \
  template <bool FIRST = false>                                                                                      \
  __device__ __forceinline__ void name(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {                    \
    if constexpr (FIRST) {                                                                                           \
      asm("mma.sync.aligned." shape_types " {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"     \
          : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])                                                           \
          : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "f"(0.f));                                     \
    } else {                                                                                                         \
      asm("mma.sync.aligned." shape_types " {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"         \
          : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])                                                           \
          : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));                                               \
    }                                                                                                                \
  }
TB2_MMA(mma_f16, "m16n8k16.row.col.f32.f16.f16.f32")
TB2_MMA(mma_bf16, "m16n8k16.row.col.f32.bf16.bf16.f32")
TB2_MMA(mma_tf32, "m16n8k8.row.col.f32.tf32.tf32.f32")
#undef TB2_MMA
template <int CT>
__device__ __forceinline__ void mma16(bool first, float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  // (`first` is a constant once the loops around it are unrolled)
  if constexpr (CT == kCacheBF16) {
    if (first) mma_bf16<true>(d, a, b0, b1);
    else mma_bf16(d, a, b0, b1);
  } else {
    if (first) mma_f16<true>(d, a, b0, b1);
    else mma_f16(d, a, b0, b1);
  }
}
__device__ __forceinline__ void mma8(bool first, float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  if (first) mma_tf32<true>(d, a, b0, b1);
  else mma_tf32(d, a, b0, b1);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// An f32 value as two tf32 ones: rounded to 11 bits, and what is left, which
// has 12 at most and is cut to 11: no more than a unit of the value's last
// place is left out (2^-23 of it). NaN may end in `lo` alone (the carry turns
// its `hi` into a 0), an infinity makes `lo` NaN.
struct Split {
  uint32_t hi, lo;
};
__device__ __forceinline__ Split tf32x2(float x) {
  const uint32_t hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  return {hi, __float_as_uint(x - __uint_as_float(hi)) & 0xffffe000u};
}
// Two f32 operations in one instruction.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n.reg .b64 x, y;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nadd.rn.f32x2 x, x, y;\nmov.b64 {%0, %1}, x;\n}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n.reg .b64 x, y;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmul.rn.f32x2 x, x, y;\nmov.b64 {%0, %1}, x;\n}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n.reg .b64 x, y, z;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmov.b64 z, {%6, %7};\n"
      "fma.rn.f32x2 x, x, y, z;\nmov.b64 {%0, %1}, x;\n}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}

// Two values as one register of plane values (lower half first), what is left
// of them going on to the next plane.
__device__ __forceinline__ uint32_t plane_f16(float& x, float& y) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h), r = fma2(f, make_float2(-1.f, -1.f), make_float2(x, y));
  x = r.x;
  y = r.y;
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t plane_bf16(float& x, float& y) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  const float2 f = __bfloat1622float2(h), r = fma2(f, make_float2(-1.f, -1.f), make_float2(x, y));
  x = r.x;
  y = r.y;
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <int CT>
__device__ __forceinline__ uint32_t plane16(float& x, float& y) {
  if constexpr (CT == kCacheBF16) return plane_bf16(x, y);
  else return plane_f16(x, y);
}

// Four int8 (as u8 words after ^ 0x80808080, i.e. value + 128) in the bytes
// (s0, s1) selected from w: f16 of 1024 + u has u in its low bits, so the pair
// is 0x64u0 | 0x64u1 minus 1152, exact.
__device__ __forceinline__ uint32_t i8pair_f16(uint32_t w, uint32_t sel) {
  const uint32_t p = __byte_perm(w, 0x64646464u, sel);
  const uint32_t k = 0x64806480u;   // 1152
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&p), *reinterpret_cast<const __half2*>(&k));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// The fp16 block scales of two neighbouring rows.
template <int NB>
struct ScalePair {
  uint32_t w[NB];
  __device__ __forceinline__ void load(uint32_t a) {   // a: a multiple of 4 NB bytes
    if constexpr (NB == 4) {
      const uint4 v = lds128(a);
      w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else if constexpr (NB == 2) {
      const uint2 v = lds64(a);
      w[0] = v.x; w[1] = v.y;
    } else {
#pragma unroll
      for (int i = 0; i < NB; ++i) w[i] = lds32(a + 4 * i);
    }
  }
  __device__ __forceinline__ float at(int row, int blk) const {
    const int i = row * NB + blk;
    const __half2 h = *reinterpret_cast<const __half2*>(&w[i / 2]);
    return i & 1 ? __high2float(h) : __low2float(h);
  }
};

template <int CT, int DH, int HT, int PL>
struct Cfg {
  static constexpr int E = CT == kCacheF32 ? 4 : CT == kCacheQ8 ? 1 : 2;
  static constexpr int CR = DH * E / 16;   // 16-byte chunks of a row
  // keys of a tile: about 8 KB of K and V together (a multiple of 16 keys for
  // 16-bit products, 8 for tf32)
  static constexpr int TK = CT == kCacheF32    ? (DH == 32 ? 32 : DH == 64 ? 16 : 8)
                            : CT == kCacheQ8 ? (DH == 32 ? 64 : 32)
                                               : (DH == 32 ? 64 : DH == 64 ? 32 : 16);
  static constexpr int UK = TK * kAttnWarps;   // keys of a unit
  static constexpr int ST = 2;
  static constexpr int OCC = HT == 16 ? 2 : CT == kCacheQ8 && DH <= 64 ? 4 : 3;   // CTAs on an SM
  // Row pitches in shared memory, so that the lanes that read at once meet no
  // bank twice. 16-bit and f32 rows: 16 bytes of padding (a read covers chunks
  // 2 c + e of rows g and g + 1, or one chunk of eight rows). Q8_0: K is read 8
  // bytes at a time over four rows, V 4 bytes over every other row: rows of 128
  // and 64 bytes are swizzled (k_swz, v_swz), narrow V rows padded.
  static constexpr int KP = CT == kCacheQ8 ? DH : DH * E + 16;
  static constexpr int VP = CT == kCacheQ8 ? (DH == 128 ? DH : DH + 16) : DH * E + 16;
  static constexpr int NB = DH / 32;   // Q8_0 blocks of a row
  static constexpr int SB = CT == kCacheQ8 ? TK * NB * 2 : 0;
  static constexpr int kOffV = TK * KP, kOffKS = kOffV + TK * VP, kOffVS = kOffKS + SB;
  static constexpr int kStage = (kOffVS + SB + 15) / 16 * 16;
  static constexpr int RPL = TK > 32 ? TK / 32 : 1;   // rows of a tile per lane
  static constexpr int NT = TK / 8;
  static constexpr int OT = DH / 8;                   // 8-column tiles of the output
  static constexpr int R = HT / 8;                    // heads per lane group
  // weights are kept times 2^14 where they are rounded to f16, so that small
  // ones keep their bits (the factor is in the sums too and cancels)
  static constexpr float kLift = CT == kCacheF16 || CT == kCacheQ8 ? 14.f : 0.f;
  static constexpr int KS = 2 * (CT == kCacheF32 ? DH / 16 : DH / 32);   // k steps of q . k
  // register sets of q: planes that do not share an instruction
  static constexpr int QS = CT == kCacheBF16 ? (HT == 8 ? PL - 1 : PL) : (HT == 8 ? 1 : 2);
  // (the third bf16 plane alone in its rows: half a set)
  static constexpr bool kHalf = CT == kCacheBF16 && HT == 8 && PL == 3;
  static constexpr int kQBytes = kHalf ? KS * 768 : QS * KS * 512;
  static constexpr int kBufs = HT == 8 && DH < 128 ? 2 : 1;   // join buffers (one where three CTAs just fit)
  // separate score accumulators (short chains of dependent products; an f32
  // cache's small products apart from its large ones)
  static constexpr int A = CT == kCacheF32 ? (NT >= 4 ? 2 : 4) : NT >= 8 ? 1 : 2;
  static constexpr int kBufFloats = (OT * 2 + 2) * R * 32;
  static constexpr int kJoinBytes = kBufs * kBufFloats * 4;
  static constexpr int kRegion = kQBytes > kJoinBytes ? kQBytes : kJoinBytes;
  static constexpr int kSmem = kAttnWarps * ST * kStage + kRegion;

  // Q8_0: what the 16-byte chunks of row r are exchanged by.
  static __device__ __forceinline__ int k_swz(int r) {
    return CT != kCacheQ8 ? 0 : DH == 128 ? (r & 3) << 1 : DH == 64 ? ((r >> 1) & 1) << 1 : 0;
  }
  static __device__ __forceinline__ int v_swz(int r) { return CT == kCacheQ8 && DH == 128 ? ((r >> 1) & 3) << 1 : 0; }
  // The 16-byte chunk of a key row that lane c of a group takes for step pair
  // sp of q . k (for Q8_0 the 8 bytes c of block sp, in units of 8 bytes).
  static __device__ __forceinline__ int chunk(int sp, int c) {
    if constexpr (CT == kCacheQ8) return 4 * sp + c;
    else return sp / 2 * 8 + (sp / 2 * 8 + 8 <= CR ? 2 * c + sp % 2 : c);
  }
  static constexpr int QW = CT == kCacheF32 ? 4 : 8;   // values of q in such a chunk
  static constexpr int SP = DH / (4 * QW);              // step pairs
  // Rows of a tile that lie in one page when the page size is a multiple of 16.
  static constexpr int PR = TK < 16 ? TK : 16;
  static constexpr int NP = TK / PR;
};

__device__ __forceinline__ float load_row(const void* p, int type, long long at) {
  if (type == kTypeF32) return static_cast<const float*>(p)[at];
  if (type == kTypeF16) return __half2float(static_cast<const __half*>(p)[at]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[at]);
}
// W values from element `at`; vec: they start on a 16-byte (8 for 4 16-bit ones) boundary.
template <int W>
__device__ __forceinline__ void load_rows(const void* p, int type, bool vec, long long at, float* x) {
  if (!vec) {
#pragma unroll
    for (int k = 0; k < W; ++k) x[k] = load_row(p, type, at + k);
  } else if (type == kTypeF32) {
#pragma unroll
    for (int k = 0; k < W; k += 4) {
      const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + at + k);
      x[k] = v.x; x[k + 1] = v.y; x[k + 2] = v.z; x[k + 3] = v.w;
    }
  } else {
    uint32_t w[W / 2];
    if constexpr (W == 8) {
      const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + at);
      w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else {
      const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + at);
      w[0] = v.x; w[1] = v.y;
    }
#pragma unroll
    for (int k = 0; k < W / 2; ++k) {
      const float2 f = type == kTypeF16 ? __half22float2(*reinterpret_cast<const __half2*>(&w[k]))
                                        : __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[k]));
      x[2 * k] = f.x;
      x[2 * k + 1] = f.y;
    }
  }
}
__device__ __forceinline__ void store_row(void* p, int type, long long at, float x) {
  if (type == kTypeF32) static_cast<float*>(p)[at] = x;
  else if (type == kTypeF16) static_cast<__half*>(p)[at] = __float2half_rn(x);
  else static_cast<__nv_bfloat16*>(p)[at] = __float2bfloat16_rn(x);
}

// N values times f from element `at` on (a multiple of N); vec: rows start on 16-byte boundaries.
template <int N>
__device__ __forceinline__ void store_rows(void* p, int type, bool vec, long long at, const float* v, float f) {
  if (!vec) {
#pragma unroll
    for (int k = 0; k < N; ++k) store_row(p, type, at + k, v[k] * f);
  } else if (type == kTypeF32) {
    float* d = static_cast<float*>(p) + at;
    if constexpr (N == 2) {
      *reinterpret_cast<float2*>(d) = make_float2(v[0] * f, v[1] * f);
    } else {
#pragma unroll
      for (int k = 0; k < N; k += 4)
        *reinterpret_cast<float4*>(d + k) = make_float4(v[k] * f, v[k + 1] * f, v[k + 2] * f, v[k + 3] * f);
    }
  } else {
    uint32_t w[N / 2];
#pragma unroll
    for (int k = 0; k < N / 2; ++k) {
      const float x = v[2 * k] * f, y = v[2 * k + 1] * f;
      const __half2 h = __floats2half2_rn(x, y);
      const __nv_bfloat162 b = __floats2bfloat162_rn(x, y);
      w[k] = type == kTypeF16 ? *reinterpret_cast<const uint32_t*>(&h) : *reinterpret_cast<const uint32_t*>(&b);
    }
    uint16_t* d = static_cast<uint16_t*>(p) + at;
    if constexpr (N == 2) *reinterpret_cast<uint32_t*>(d) = w[0];
    else if constexpr (N == 4) *reinterpret_cast<uint2*>(d) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint4*>(d) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// A place in the list of units: unit t of key head (and head tile) jt of
// request b, whose history has len keys.
struct Cursor {
  int b, jt, t, len;
};

// Value e of a cache's rows of K (of V) as f32.
template <int CT>
__device__ __forceinline__ float load_cache(const PagedKv& kv, bool v, long long e) {
  const void* p = v ? kv.v : kv.k;
  if constexpr (CT == kCacheF32) return static_cast<const float*>(p)[e];
  else if constexpr (CT == kCacheF16) return __half2float(static_cast<const __half*>(p)[e]);
  else if constexpr (CT == kCacheBF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[e]);
  else return (float)static_cast<const int8_t*>(p)[e] * __half2float(__ushort_as_half((v ? kv.vs : kv.ks)[e / 32]));
}

// Units t0 .. t1 - 1 of a history in plain f32, by one warp, a head and four
// keys at a time: the running maximum, the sum of the weights and of the
// weighted values, to `buf` as the warps' sums are exchanged. For parts that
// hold infinities or NaN only: keys whose score is -inf weigh 0, and an
// infinite value of positive weight makes its column infinite. (The sums of
// the whole part are taken again, by one warp: this is rare, and less of it
// in the kernel keeps the registers of the rest.)
template <int CT, int DH, int HT, int PL>
__device__ __noinline__ void plain_part(const PagedAttnArgs& a, int b, int jt, int t0, int t1, float* buf) {
  using C = Cfg<CT, DH, HT, PL>;
  constexpr int W = DH / 32;   // columns of a lane: lane, lane + 32, ..
  constexpr int U = 4;
  const int lane = threadIdx.x & 31, P = a.kv.page_size;
  const int tiles_h = (a.group + HT - 1) / HT, jh = jt / tiles_h, h0 = (jt - jh * tiles_h) * HT;
  const int* pages = a.table + b * a.table_stride;
  const long long len = min((long long)a.width * P, (long long)a.lens[b]);
  const long long begin = (long long)t0 * C::UK, end = min((long long)t1 * C::UK, len);
#pragma unroll 1
  for (int h = 0; h < HT; ++h) {
    float m = -INFINITY, l = 0.f, q[W], o[W];
    const bool on = h0 + h < a.group;
    const long long row = b * a.ldq + ((long long)jh * a.group + h0 + h) * DH + lane;
#pragma unroll
    for (int k = 0; k < W; ++k) {
      q[k] = on ? load_row(a.q, a.row_type, row + 32 * k) : 0.f;
      o[k] = 0.f;
    }
#pragma unroll 1
    for (long long key0 = begin; on && key0 < end; key0 += U) {
      long long at[U];   // -1: no key
      float s[U], v[U][W];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int key = (int)(key0 + u), id = key0 + u < end ? pages[key / P] : -1;
        at[u] = id >= 0 && id < a.kv.n_pages
                    ? id * a.kv.page_stride + jh * a.kv.head_stride + key % P * a.kv.tok_stride + lane
                    : -1;
        s[u] = 0.f;
#pragma unroll
        for (int k = 0; k < W; ++k) {
          if (at[u] >= 0) s[u] = fmaf(q[k], load_cache<CT>(a.kv, false, at[u] + 32 * k), s[u]);
          v[u][k] = at[u] >= 0 ? load_cache<CT>(a.kv, true, at[u] + 32 * k) : 0.f;
        }
      }
      float top = m;
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int w = 16; w; w >>= 1) s[u] += __shfl_xor_sync(0xffffffffu, s[u], w);
        s[u] = at[u] >= 0 ? s[u] * a.c : -INFINITY;
        top = fmaxf(top, s[u]);
      }
      const float keep = m == -INFINITY ? 0.f : ex2(m - top);
      m = top;
      l *= keep;
#pragma unroll
      for (int k = 0; k < W; ++k) o[k] *= keep;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float p = ex2(top == -INFINITY ? s[u] : s[u] - top);
        l += p;
#pragma unroll
        for (int k = 0; k < W; ++k) o[k] = fmaf(p, v[u][k], o[k]);
      }
    }
    const float lift = C::kLift == 0.f ? 1.f : 16384.f;
    const int r = h >> 3, g = h & 7;
#pragma unroll
    for (int k = 0; k < W; ++k) {
      const int col = lane + 32 * k, w = col % 32;
      // the output tile, lane of a group and half of its pair that column `col` belongs to
      constexpr bool kRuns = CT == kCacheF32 || CT == kCacheQ8;
      const int i = kRuns ? col / 32 * 4 + w % 4 : col / 8, c = kRuns ? w / 8 : w % 8 / 2;
      const int y = kRuns ? w % 8 / 4 : w & 1;
      buf[((r * (C::OT / 2) + i / 2) * 32 + g * 4 + c) * 4 + (i & 1) * 2 + y] = o[k] * lift;
    }
    float2* ml = reinterpret_cast<float2*>(buf + C::OT * 2 * C::R * 32) + r * 32 + g * 4;
    if (lane < 4) ml[lane] = make_float2(m, l * lift);
  }
}

template <int CT, int DH, int HT, int PL>
__global__ void __launch_bounds__(kAttnWarps * 32, Cfg<CT, DH, HT, PL>::OCC)
    paged_attend_kernel(const __grid_constant__ PagedAttnArgs a) {
  using C = Cfg<CT, DH, HT, PL>;
  constexpr int TK = C::TK, UK = C::UK, NT = C::NT, OT = C::OT, R = C::R, ST = C::ST;
  constexpr float kLift = C::kLift;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ uint64_t valid[kAttnWarps][ST];   // keys of a staged tile that count
  __shared__ int last_flag;
  __shared__ int pre[kAttnWarps * 32];   // units (of one key head) before each thread's run of requests
  __shared__ float qmax[kAttnWarps][HT];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
  uint8_t* region = smem + kAttnWarps * ST * C::kStage;
  const uint32_t ring = smem_u32(smem) + warp * ST * C::kStage;
  griddep_wait_release();

  const int n = a.n_req, P = a.kv.page_size;
  const long long most = (long long)a.width * P;
  const int tiles_h = (a.group + HT - 1) / HT, KVH = a.kv.n_kv * tiles_h;
  // (lengths, tables and scales may be written by the kernel before, beside which this one may have been launched: read
  // after the grid wait and not through the read-only path)
  auto length = [&](int b) { return (int)min(most, (long long)max(0, a.lens[b])); };

  // ---- the list's length (below 2^31 by the host's limit), each thread a run of requests
  auto units_of = [](int len) { return (len + UK - 1) / UK; };
  int total, histories = 0, longest = 0;   // (of one key head)
  const int per = (n + kAttnWarps * 32 - 1) / (kAttnWarps * 32);
  {
    const int b0 = min(n, tid * per), b1 = min(n, b0 + per);
    int s = 0, live = 0, top = 0;
    for (int b = b0; b < b1; ++b) {
      const int len = length(b);
      s += units_of(len);
      live += len > 0;
      top = max(top, units_of(len));
    }
    live = __reduce_add_sync(0xffffffffu, live);
    top = __reduce_max_sync(0xffffffffu, top);
    int inc = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += x;
    }
    __shared__ int wsum[kAttnWarps], wlive[kAttnWarps], wtop[kAttnWarps];
    if (lane == 31) {
      wsum[warp] = inc;
      wlive[warp] = live;
      wtop[warp] = top;
    }
    __syncthreads();
    int base = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kAttnWarps; ++w) {
      if (w < warp) base += wsum[w];
      total += wsum[w];
      histories += wlive[w];
      longest = max(longest, wtop[w]);
    }
    pre[tid] = base + inc - s;
    __syncthreads();
  }
  // requests without a key: zeros
  for (int b = blockIdx.x; b < n; b += gridDim.x) {
    if (length(b) > 0) continue;
    for (int i = tid; i < a.n_heads * DH; i += blockDim.x) store_row(a.out, a.row_type, b * a.ldo + i, 0.f);
    if (a.lse)
      for (int h = tid; h < a.n_heads; h += blockDim.x) a.lse[(long long)b * a.n_heads + h] = -INFINITY;
  }
  const int units = total * KVH;
  if (units == 0) return;
  // Equal ranges of the list (a unit more or less), kMinUnits at least. (The memory does not serve all SMs alike: on a
  // long bf16 history the first CTA is done after 62 us and the last after 92. Smaller ranges, handed out as CTAs
  // become free, did not make the last one earlier: the memory is busy to the end, and every range costs 2 us.)
  // A CTA for each history where there are as many (eight of one unit: 6.1 us, 8.9 when four CTAs take two each); more
  // only for kMinUnits each.
  // Equal histories and several CTAs to each: a whole number of them, where that leaves three quarters of the CTAs, so
  // that none has the end of one and the start of the next, whose share it would do several us later. Of 444 CTAs,
  // bf16, 32 / 8 heads of 128, with (without): all used, 1 x 8192 tokens 19.4 (25.1) us; 392, 7 x 2000 20.6 (23.6); 384, 8 x
  // 1024 15.5 (20.4); 360, 15 x 1000 21.5 (25.4). With fewer, short histories would gain still (320 CTAs, 20 x 512 17.5
  // (22.4)) and long ones lose (20 x 4096 71.5 (68.2), 40 x 4096 126.6 (122.8)).
  int G = min((int)gridDim.x, max(units / kMinUnits, histories * KVH));
  const int even = G / (histories * KVH) * (histories * KVH);
  if ((long long)longest * histories == total && even * 4 >= G * 3) G = even;
  if (blockIdx.x >= G) return;
  auto range = [&](int i) { return (int)((long long)i * units / G); };
  auto cta_of = [&](int u) { return (int)(((u + 1LL) * G - 1) / units); };   // whose range holds unit u

  // the place of list index u, and the list index at which its request starts
  auto locate = [&](int u, Cursor& k, int& first) {
    const int key = u / KVH;
    int lo = 0, hi = kAttnWarps * 32;   // the last thread whose run starts at or before key
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pre[mid] <= key) lo = mid;
      else hi = mid;
    }
    int base = pre[lo], b = lo * per;
    for (;;) {   // (32 requests of the run at a time)
      const int i = b + lane, nt = i < n && lane < per ? units_of(length(i)) : 0;
      int inc = nt;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += x;
      }
      const unsigned past = __ballot_sync(0xffffffffu, base + inc > key);
      if (past) {
        const int f = __ffs(past) - 1;
        k.b = b + f;
        base += __shfl_sync(0xffffffffu, inc - nt, f);
        break;
      }
      base += __shfl_sync(0xffffffffu, inc, 31);
      b += 32;
    }
    k.len = length(k.b);
    first = base * KVH;
    const int nt = units_of(k.len);
    k.jt = (u - first) / nt;
    k.t = u - first - k.jt * nt;
  };

  // the next (request, head) of the list; the caller knows that there is one
  auto next_history = [&](Cursor& k, int& first) {
    k.t = 0;
    if (++k.jt < KVH) return;
    k.jt = 0;
    first += units_of(k.len) * KVH;
    do {
      ++k.b;
      k.len = length(k.b);
    } while (k.len == 0);
  };

  Cursor cur;                  // this CTA's place
  int u = range(blockIdx.x), cur_first;
  const int u_hi = range(blockIdx.x + 1);
  locate(u, cur, cur_first);
  Cursor pc = cur;             // and the producer's
  int pu = u;

  // ---- the ring: tiles of this warp in list order
  // Where the page size is a multiple of 16, the 16 rows (or the tile, if it
  // has fewer) from a multiple of 16 on lie in one page: the lanes read the
  // page ids of the next tiles' pieces together, and a full tile of good pages
  // is copied with an address per piece. Other page sizes, and the last tile
  // of a history, take an address per row.
  constexpr bool kEven = 32 % C::CR == 0;   // a lane copies the same chunk of every row it has (not at d_head 96)
  constexpr int kWin = 32 / C::NP;          // tiles whose page ids are read at once
  const bool pieces16 = kEven && P % 16 == 0;
  int win = 0, win_t = 0;      // lane's page id; the unit that the window starts at
  const int* pages = nullptr;  // the history's row of the block table
  long long head = 0;          // and its key head's offset in a page
  auto page_of = [&](int key) { return a.page_shift >= 0 ? key >> a.page_shift : key / P; };
  auto tile_key = [&]() { return (pc.t * kAttnWarps + warp) * TK; };
  auto read_page = [&](int key) { return key < pc.len ? pages[page_of(key)] : -1; };
  auto read_window = [&]() {
    win_t = pc.t;
    // (units past the history have no page)
    const long long key = ((long long)(win_t + lane / C::NP) * kAttnWarps + warp) * TK + lane % C::NP * C::PR;
    win = key < pc.len ? read_page((int)key) : -1;
  };
  auto enter = [&]() {
    pages = a.table + pc.b * a.table_stride;
    head = pc.jt / tiles_h * a.kv.head_stride;
    if (pieces16) read_window();
  };
  auto next_unit = [&]() {
    ++pu;
    if (++pc.t * UK >= pc.len && pu < u_hi) {
      int unused = 0;
      next_history(pc, unused);
      enter();
    }
  };
  // whether there is a tile to fetch (the last unit of a history may hold none of this warp's)
  auto has_tile = [&]() {
    while (pu < u_hi && tile_key() >= pc.len) next_unit();
    return pu < u_hi;
  };
  // this lane's part of a copy: 16-byte chunk lc of rows lr, lr + kStep, ..
  constexpr int kIter = TK * C::CR / 32;
  constexpr int kStep = kEven ? 32 / C::CR : 1;
  const int lr = lane / C::CR, lc = lane % C::CR;
  const long long row_bytes = a.kv.tok_stride * C::E;
  const long long lane_off = lr * row_bytes + lc * 16;
  const long long scale_off = lane % C::PR * (a.kv.tok_stride / 32);
  const bool dense = a.kv.tok_stride == DH;   // a page's rows of a head are one run of bytes
  auto scales = [&](uint32_t s, int r, long long at, bool on) {   // Q8_0: the scales of row r, from block `at`
    const uint32_t dk = s + C::kOffKS + r * C::NB * 2, dv = s + C::kOffVS + r * C::NB * 2;
    if constexpr (CT == kCacheQ8 && (DH == 128 || DH == 64)) {
      cp_small<C::NB * 2>(dk, a.kv.ks + at, on);
      cp_small<C::NB * 2>(dv, a.kv.vs + at, on);
    } else if constexpr (CT == kCacheQ8) {
#pragma unroll
      for (int e = 0; e < C::NB; ++e) {
        sts16(dk + 2 * e, on ? a.kv.ks[at + e] : 0);
        sts16(dv + 2 * e, on ? a.kv.vs[at + e] : 0);
      }
    }
  };
  int used = 0, staged = 0;   // tiles consumed; tiles fetched and not consumed
  auto issue = [&]() {        // fetch the next tile into the stage that is free
    const int stage = (used + staged) & 1;
    const uint32_t s = ring + stage * C::kStage;
    const int key0 = tile_key();
    if (pieces16 && pc.t - win_t >= kWin) read_window();
    int page = -1;
    if (pieces16) page = __shfl_sync(0xffffffffu, win, (pc.t - win_t) * C::NP + lane % C::NP);
    const bool fast = pieces16 && key0 + TK <= pc.len && __all_sync(0xffffffffu, page >= 0 && page < a.kv.n_pages);
    if (fast) {
      const int pk = key0 + lane % C::NP * C::PR;
      const long long piece = page * a.kv.page_stride + head + (pk - page_of(pk) * P) * a.kv.tok_stride;
      if (lane == 0) valid[warp][stage] = ~0ull;
      constexpr int kPer = kIter / C::NP;   // copies of a piece
      const uint32_t dk = s + lr * C::KP + (lc ^ C::k_swz(lr)) * 16;
      auto dv = [&](int r) { return s + C::kOffV + lr * C::VP + (lc ^ C::v_swz(lr + r)) * 16 + r * C::VP; };
#pragma unroll
      for (int p = 0; p < C::NP; ++p) {
        const long long base = __shfl_sync(0xffffffffu, piece, p) * C::E + lane_off;
        const uint8_t* sk = static_cast<const uint8_t*>(a.kv.k) + base;
        const uint8_t* sv = static_cast<const uint8_t*>(a.kv.v) + base;
        if (dense) {   // (addresses of one register and constants)
#pragma unroll
          for (int i = 0; i < kPer; ++i) {
            const int r = (p * kPer + i) * kStep;
            cp16(dk + r * C::KP, sk + i * kStep * (DH * C::E));
            cp16(dv(r), sv + i * kStep * (DH * C::E));
          }
        } else {
#pragma unroll 1
          for (int i = 0; i < kPer; ++i) {
            const int r = (p * kPer + i) * kStep;
            cp16(dk + r * C::KP, sk + i * kStep * row_bytes);
            cp16(dv(r), sv + i * kStep * row_bytes);
          }
        }
      }
      if constexpr (CT == kCacheQ8) {
#pragma unroll
        for (int i = 0; i < C::RPL; ++i) {
          const int r = lane + 32 * i;
          scales(s, r, (long long)((unsigned long long)__shfl_sync(0xffffffffu, piece, r / C::PR) >> 5) + scale_off,
                 true);
        }
      }
    } else {
      long long off[C::RPL];
      uint64_t ok = 0;
#pragma unroll
      for (int i = 0; i < C::RPL; ++i) {
        const int key = key0 + (TK < 32 ? lane % TK : lane + 32 * i), id = read_page(key);
        const bool in = key < pc.len, good = in && id >= 0 && id < a.kv.n_pages;
        if (in && !good) *a.err = kErrPagedPage;
        off[i] = good ? id * a.kv.page_stride + head + (key - page_of(key) * P) * a.kv.tok_stride : -1;
        ok |= (uint64_t)__ballot_sync(0xffffffffu, good) << (32 * i);
      }
      if (lane == 0) valid[warp][stage] = ok;
      // (rolled: this path is rare and the code of the others has to stay in the instruction cache)
#pragma unroll 1
      for (int it = 0; it < kIter; ++it) {
        const int i = it * 32 + lane, r = i / C::CR, ch = i % C::CR;
        const long long lo = __shfl_sync(0xffffffffu, off[0], r & 31);
        const long long hi = C::RPL > 1 ? __shfl_sync(0xffffffffu, off[C::RPL - 1], r & 31) : lo;
        const long long o = r < 32 ? lo : hi;
        const bool on = o >= 0;
        const long long at = on ? o * C::E + ch * 16 : 0;
        cp16(s + r * C::KP + (ch ^ C::k_swz(r)) * 16, static_cast<const uint8_t*>(a.kv.k) + at, on);
        cp16(s + C::kOffV + r * C::VP + (ch ^ C::v_swz(r)) * 16, static_cast<const uint8_t*>(a.kv.v) + at, on);
      }
      if constexpr (CT == kCacheQ8) {
#pragma unroll
        for (int i = 0; i < C::RPL; ++i) scales(s, lane + 32 * i, off[i] >= 0 ? off[i] / 32 : 0, off[i] >= 0);
      }
    }
    cp_commit();
    ++staged;
    next_unit();
  };
  enter();

  // this warp's share of a history's q: step pairs are dealt to the warps
  constexpr int kOwn = (C::SP + kAttnWarps - 1) / kAttnWarps;
  float qv[kOwn][R][C::QW];   // the chunks of the lane's rows that its key rows are read by
  auto load_q = [&](const Cursor& k) {
    const int jh = k.jt / tiles_h, h0 = (k.jt - jh * tiles_h) * HT, heads = min(HT, a.group - h0);
    const long long row = (long long)k.b * a.ldq + ((long long)jh * a.group + h0) * DH;
#pragma unroll
    for (int own = 0; own < kOwn; ++own)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int sp = warp + own * kAttnWarps;
        if (g + 8 * r < heads && sp < C::SP) {
          load_rows<C::QW>(a.q, a.row_type, a.q_vec, row + (long long)(g + 8 * r) * DH + C::chunk(sp, c) * C::QW,
                           qv[own][r]);
        } else {
#pragma unroll
          for (int k = 0; k < C::QW; ++k) qv[own][r][k] = 0.f;
        }
      }
  };
  load_q(cur);

  // ---- this warp's sums over the current history
  float2 o[OT][R];
  float m[R], l[R], fac[R];
  float2 l2[CT == kCacheQ8 ? R : 1];   // Q8_0: the sums of the weights in pairs, NaN once a score was not finite
  // Q8_0: the weights carry 2^lift_d, near 1 / the largest |V scale| so far, so that their products with the scales
  // fill the f16 range (the factor is in l too and cancels)
  int lift_d = 0;
  bool have_d = false;
  for (;;) {
    const int nt = units_of(cur.len), t0 = cur.t, t1 = min(nt, t0 + (u_hi - u));
    const int jh = cur.jt / tiles_h, h0 = (cur.jt - jh * tiles_h) * HT;   // key head, first head of the tile
    const int heads = min(HT, a.group - h0);

#pragma unroll 1
    while (staged < ST && has_tile()) issue();
    // q as operand registers: lane (g, c) of step s holds rows g and g + 8.
    float rs[R];   // what the scores of the lane group's heads are multiplied by
    {
      if constexpr (CT == kCacheF16 || CT == kCacheQ8) {   // the largest |q| of a row into [16, 32)
        float x[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
          x[r] = 0.f;
#pragma unroll
          for (int own = 0; own < kOwn; ++own)
#pragma unroll
            for (int k = 0; k < C::QW; ++k) x[r] = fmaxf(x[r], fabsf(qv[own][r][k]));
          x[r] = fmaxf(x[r], __shfl_xor_sync(0xffffffffu, x[r], 1));
          x[r] = fmaxf(x[r], __shfl_xor_sync(0xffffffffu, x[r], 2));
          if (c == 0) qmax[warp][g + 8 * r] = x[r];
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
          for (int w = 0; w < kAttnWarps; ++w) x[r] = fmaxf(x[r], qmax[w][g + 8 * r]);
          int e = (int)(__float_as_uint(x[r]) >> 23) - 127 - 4;   // x < 2^(e + 5)
          e = max(-100, min(123, e));   // (a row of inf or NaN stays one)
          const float up = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
          for (int own = 0; own < kOwn; ++own)
#pragma unroll
            for (int k = 0; k < C::QW; ++k) qv[own][r][k] *= a.c < 0.f ? -up : up;   // (the factor's sign too)
          rs[r] = fabsf(a.c) * __uint_as_float((uint32_t)(127 + e) << 23);
        }
      } else {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          rs[r] = fabsf(a.c);
#pragma unroll
          for (int own = 0; own < kOwn; ++own)
#pragma unroll
            for (int k = 0; k < C::QW; ++k) qv[own][r][k] = a.c < 0.f ? -qv[own][r][k] : qv[own][r][k];
        }
      }
      uint4* qf = reinterpret_cast<uint4*>(region);
#pragma unroll
      for (int own = 0; own < kOwn; ++own) {
        const int sp = warp + own * kAttnWarps;
        if (sp >= C::SP) break;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int s = 2 * sp + half, i = half * C::QW / 2;
          float (&x)[R][C::QW] = qv[own];
          if constexpr (CT == kCacheF32) {
            uint32_t hi[2][2], lo[2][2];
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const Split v = tf32x2(x[r][i + k]);
                hi[r][k] = v.hi;
                lo[r][k] = v.lo;
              }
            if constexpr (HT == 8) {
              qf[s * 32 + lane] = make_uint4(hi[0][0], lo[0][0], hi[0][1], lo[0][1]);
            } else {
              qf[s * 32 + lane] = make_uint4(hi[0][0], hi[1][0], hi[0][1], hi[1][1]);
              qf[(C::KS + s) * 32 + lane] = make_uint4(lo[0][0], lo[1][0], lo[0][1], lo[1][1]);
            }
          } else if constexpr (HT == 8) {
            uint4 v;
            v.x = plane16<CT>(x[0][i], x[0][i + 1]);
            v.z = plane16<CT>(x[0][i + 2], x[0][i + 3]);
            v.y = plane16<CT>(x[0][i], x[0][i + 1]);
            v.w = plane16<CT>(x[0][i + 2], x[0][i + 3]);
            qf[s * 32 + lane] = v;
            if constexpr (C::QS == 2) {
              v.x = plane16<CT>(x[0][i], x[0][i + 1]);
              v.z = plane16<CT>(x[0][i + 2], x[0][i + 3]);
              reinterpret_cast<uint2*>(qf + C::KS * 32)[s * 32 + lane] = make_uint2(v.x, v.z);
            }
          } else {
#pragma unroll
            for (int p = 0; p < C::QS; ++p) {
              uint4 v;
              v.x = plane16<CT>(x[0][i], x[0][i + 1]);
              v.y = plane16<CT>(x[R - 1][i], x[R - 1][i + 1]);
              v.z = plane16<CT>(x[0][i + 2], x[0][i + 3]);
              v.w = plane16<CT>(x[R - 1][i + 2], x[R - 1][i + 3]);
              qf[(p * C::KS + s) * 32 + lane] = v;
            }
          }
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.f;
      fac[r] = rs[r];
    }
#pragma unroll
    for (int i = 0; i < OT; ++i)
#pragma unroll
      for (int r = 0; r < R; ++r) o[i][r] = make_float2(0.f, 0.f);
    have_d = false;
    lift_d = 0;
    if constexpr (CT == kCacheQ8) {
#pragma unroll
      for (int r = 0; r < R; ++r) l2[r] = make_float2(0.f, 0.f);
    }
    const uint32_t qb = smem_u32(region) + lane * 16, qh = smem_u32(region) + C::KS * 512 + lane * 8;
    auto q_at = [&](int p, int st) {   // register set p of step st
      if (C::kHalf && p == 1) {
        const uint2 v = lds64(qh + st * 256);
        return make_uint4(v.x, 0, v.y, 0);
      }
      return lds128(qb + (p * C::KS + st) * 512);
    };

    for (int t = t0; t < t1; ++t) {
      if ((t * kAttnWarps + warp) * TK >= cur.len) break;
      // this tile's copies, the newer one's still in flight if there is one
      if (staged == 2) cp_wait<1>();
      else cp_wait<0>();
      __syncwarp();
      const uint32_t ks = ring + (used & 1) * C::kStage, vs = ks + C::kOffV;
      const uint64_t ok = valid[warp][used & 1];

      // scores of the tile: lane (g, c) has keys 8 i + 2 c, + 1 of rows g (and g + 8)
      float s[NT][2 * R];
      if constexpr (CT == kCacheQ8) {
        ScalePair<C::NB> ksc[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) ksc[i].load(ks + C::kOffKS + (8 * i + 2 * c) * C::NB * 2);
#pragma unroll
        for (int blk = 0; blk < C::NB; ++blk) {
          uint4 qa[C::QS][2];
#pragma unroll
          for (int p = 0; p < C::QS; ++p)
#pragma unroll
            for (int k = 0; k < 2; ++k) qa[p][k] = q_at(p, 2 * blk + k);
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            const uint2 w =
                lds64(ks + g * C::KP + (((2 * blk + (c >> 1)) ^ C::k_swz(g)) * 16 + (c & 1) * 8) + 8 * i * C::KP);
            const uint32_t w0 = w.x ^ 0x80808080u, w1 = w.y ^ 0x80808080u;
            float d[4];
            const uint32_t b0 = i8pair_f16(w0, 0x4140), b1 = i8pair_f16(w0, 0x4342), b2 = i8pair_f16(w1, 0x4140),
                           b3 = i8pair_f16(w1, 0x4342);
#pragma unroll
            for (int p = 0; p < C::QS; ++p) {
              mma16<CT>(p == 0, d, qa[p][0], b0, b1);
              mma16<CT>(false, d, qa[p][1], b2, b3);
            }
            const float s0 = ksc[i].at(0, blk), s1 = ksc[i].at(1, blk);
            const float2 sc = make_float2(s0, s1);
            float2 x = make_float2(d[0], d[1]);
            const float2 y = make_float2(d[2], d[3]);
            if constexpr (HT == 8) x = add2(x, y);
            x = blk == 0 ? mul2(x, sc) : fma2(x, sc, make_float2(s[i][0], s[i][1]));
            s[i][0] = x.x;
            s[i][1] = x.y;
            if constexpr (HT == 16) {
              const float2 z = blk == 0 ? mul2(y, sc) : fma2(y, sc, make_float2(s[i][2 * R - 2], s[i][2 * R - 1]));
              s[i][2 * R - 2] = z.x;
              s[i][2 * R - 1] = z.y;
            }
          }
        }
      } else {
        float d[NT][C::A][4];
#pragma unroll
        for (int st = 0; st < C::KS; st += 2) {   // one 16-byte read of each key row feeds two steps
          uint4 qa[C::QS][2];
#pragma unroll
          for (int p = 0; p < C::QS; ++p)
#pragma unroll
            for (int k = 0; k < 2; ++k) qa[p][k] = q_at(p, st + k);
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            const uint4 w = lds128(ks + g * C::KP + C::chunk(st / 2, c) * 16 + 8 * i * C::KP);
            if constexpr (CT == kCacheF32) {
              const uint32_t x[4] = {w.x, w.y, w.z, w.w};
              uint32_t hi[4], lo[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const Split v = tf32x2(__uint_as_float(x[k]));
                hi[k] = v.hi;
                lo[k] = v.lo;
              }
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                float (&small)[4] = d[i][C::A == 4 ? 2 + k : 1], (&large)[4] = d[i][C::A == 4 ? k : 0];
                const bool first = st == 0 && (C::A == 4 || k == 0);
                mma8(first, small, qa[0][k], lo[2 * k], lo[2 * k + 1]);
                if constexpr (HT == 16) mma8(false, small, qa[C::QS - 1][k], hi[2 * k], hi[2 * k + 1]);
                mma8(first, large, qa[0][k], hi[2 * k], hi[2 * k + 1]);
              }
            } else {
#pragma unroll
              for (int p = C::QS - 1; p >= 0; --p) {
                mma16<CT>(st == 0 && p == C::QS - 1, d[i][0], qa[p][0], w.x, w.y);
                mma16<CT>(C::A == 2 && st == 0 && p == C::QS - 1, d[i][C::A - 1], qa[p][1], w.z, w.w);
              }
            }
          }
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          float2 x[2];   // rows g, rows g + 8
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            x[h] = make_float2(d[i][0][2 * h], d[i][0][2 * h + 1]);
#pragma unroll
            for (int k = 1; k < C::A; ++k) x[h] = add2(x[h], make_float2(d[i][k][2 * h], d[i][k][2 * h + 1]));
          }
          if constexpr (HT == 8) x[0] = add2(x[0], x[1]);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            s[i][2 * r] = x[r].x;
            s[i][2 * r + 1] = x[r].y;
          }
        }
      }

      // running maximum and weights: m = factor * the largest raw score
      constexpr uint64_t kAll = TK == 64 ? ~0ull : ((1ull << (TK & 63)) - 1);
      const bool masked = (ok & kAll) != kAll;
      // (a Q8_0 block of infinite scale makes a score of -inf where the formula may have NaN: the sum of the weights
      // becomes NaN, which sends the part to plain_part; masked rows are zeros here)
      if constexpr (CT == kCacheQ8) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int r = 0; r < R; ++r)
            l2[r] = fma2(make_float2(s[i][2 * r], s[i][2 * r + 1]), make_float2(0.f, 0.f), l2[r]);
      }
      if (masked) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int k = 0; k < 2 * R; ++k)
            if (!((ok >> (8 * i + 2 * c + (k & 1))) & 1)) s[i][k] = -INFINITY;
      }
      float mx[R];
      bool grew = false;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float x = s[0][2 * r];
#pragma unroll
        for (int i = 0; i < NT; ++i) x = fmaxf(x, fmaxf(s[i][2 * r], s[i][2 * r + 1]));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
        mx[r] = fmaxf(m[r], x * fac[r]);   // (a NaN, or -inf times a factor of 0, leaves m)
        grew |= mx[r] != m[r];
      }
      int new_lift = lift_d;
      ScalePair<C::NB> vsc[CT == kCacheQ8 ? NT : 1];
      if constexpr (CT == kCacheQ8) {
#pragma unroll
        for (int i = 0; i < NT; ++i) vsc[i].load(ks + C::kOffVS + (8 * i + 2 * c) * C::NB * 2);
        // the tile's largest |V scale|, as fp16 bits: a lane looks at a row (two of them at 64 keys)
        uint32_t big = 0;
#pragma unroll
        for (int i = 0; i < C::RPL; ++i) {
          const uint32_t row = ks + C::kOffVS + (lane + 32 * i) * C::NB * 2;
          if constexpr (C::NB == 4) {
            const uint2 w = lds64(row);
            big = max(max(w.x & 0x7fffu, w.x >> 16 & 0x7fffu), max(w.y & 0x7fffu, w.y >> 16 & 0x7fffu));
          } else if constexpr (C::NB == 2) {
            const uint32_t w = lds32(row);
            big = max(w & 0x7fffu, w >> 16 & 0x7fffu);
          } else {
#pragma unroll
            for (int e = 0; e < C::NB; ++e) big = max(big, lds16(row + 2 * e) & 0x7fffu);
          }
        }
        big = __reduce_max_sync(0xffffffffu, big);
        // below 2^(1 - lift) (an infinite scale makes the sums NaN whatever the lift)
        const int lift = 127 - (int)(__float_as_uint(fmaxf(__half2float(__ushort_as_half((uint16_t)big)), 0x1p-24f)) >> 23);
        if (!have_d || lift < lift_d) new_lift = lift;
        grew |= !have_d || new_lift != lift_d;
      }
      if (__any_sync(0xffffffffu, grew)) {
        float shrink[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
          shrink[r] = m[r] == -INFINITY ? 0.f : ex2(m[r] - mx[r]);
          m[r] = mx[r];
          if constexpr (CT == kCacheQ8) shrink[r] *= ex2((float)(new_lift - (have_d ? lift_d : new_lift)));
          if constexpr (CT == kCacheQ8) l2[r] = mul2(l2[r], make_float2(shrink[r], shrink[r]));
          else l[r] *= shrink[r];
        }
        lift_d = new_lift;
        have_d = true;
#pragma unroll
        for (int i = 0; i < OT; ++i)
#pragma unroll
          for (int r = 0; r < R; ++r) o[i][r] = mul2(o[i][r], make_float2(shrink[r], shrink[r]));
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        // 2^(s fac - m + lift), rounded at each of the three steps. The product as the maximum's was: with a fused one
        // the largest key's exponent would be the rounding of m, which passes any range for scores of 2^30. The lift
        // last: lift - m is a multiple of m's last place, so for m of 2^26 the largest weight would be 2^16 instead of
        // 2^14, which f16 cannot hold. (Scalar: the assembler fuses a packed product and sum.)
        const float less = m[r] == -INFINITY ? 0.f : -m[r];
        const float lifted = CT == kCacheQ8 ? kLift + (float)lift_d : kLift;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float x = __fadd_rn(__fmul_rn(s[i][2 * r + k], fac[r]), less);
            if constexpr (CT == kCacheF16 || CT == kCacheQ8) x = __fadd_rn(x, lifted);
            float p = ex2(x);
            if (masked && !((ok >> (8 * i + 2 * c + k)) & 1)) p = 0.f;   // (a factor of 0 makes -inf NaN)
            s[i][2 * r + k] = p;
            if constexpr (CT != kCacheQ8) l[r] += p;
          }
          if constexpr (CT == kCacheQ8) l2[r] = add2(l2[r], make_float2(s[i][2 * r], s[i][2 * r + 1]));
        }
      }

      // sums of weighted values: a tile's products in fresh accumulators, added
      // to the running sums by f32 adds (the tensor core's own sums are cut,
      // not rounded, which would add up over a long history)
      auto gather = [&](int i, const float (&d)[4]) {
        const float2 x = make_float2(d[0], d[1]), y = make_float2(d[2], d[3]);
        if constexpr (HT == 8) {
          o[i][0] = add2(o[i][0], add2(x, y));
        } else {
          o[i][0] = add2(o[i][0], x);
          o[i][R - 1] = add2(o[i][R - 1], y);
        }
      };
      if constexpr (CT == kCacheF32) {
        uint4 ph[NT], pl[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) {   // 8 keys: step k holds key 2 k, step k + 4 key 2 k + 1
          Split v[2 * R];
#pragma unroll
          for (int k = 0; k < 2 * R; ++k) v[k] = tf32x2(s[i][k]);
          if constexpr (HT == 8) {
            ph[i] = make_uint4(v[0].hi, v[0].lo, v[1].hi, v[1].lo);
          } else {
            ph[i] = make_uint4(v[0].hi, v[2 * R - 2].hi, v[1].hi, v[2 * R - 1].hi);
            pl[i] = make_uint4(v[0].lo, v[2 * R - 2].lo, v[1].lo, v[2 * R - 1].lo);
          }
        }
#pragma unroll
        for (int q4 = 0; q4 < DH / 32; ++q4) {   // columns 32 q4 + 4 g .. + 3: one per output tile
          float d[4][4];
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            const uint4 w0 = lds128(vs + 2 * c * C::VP + g * 16 + 8 * i * C::VP + q4 * 128);
            const uint4 w1 = lds128(vs + 2 * c * C::VP + g * 16 + (8 * i + 1) * C::VP + q4 * 128);
            const uint32_t x0[4] = {w0.x, w0.y, w0.z, w0.w}, x1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const Split v0 = tf32x2(__uint_as_float(x0[k])), v1 = tf32x2(__uint_as_float(x1[k]));
              mma8(i == 0, d[k], ph[i], v0.lo, v1.lo);
              if constexpr (HT == 16) mma8(false, d[k], pl[i], v0.hi, v1.hi);
              mma8(false, d[k], ph[i], v0.hi, v1.hi);
            }
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) gather(4 * q4 + k, d[k]);
        }
      } else if constexpr (CT == kCacheQ8) {
#pragma unroll
        for (int blk = 0; blk < C::NB; ++blk) {
          float d[4][4];
#pragma unroll
          for (int i = 0; i < NT; i += 2) {   // 16 keys
            float2 dv[2];   // their scales of this block
#pragma unroll
            for (int k = 0; k < 2; ++k) dv[k] = make_float2(vsc[i + k].at(0, blk), vsc[i + k].at(1, blk));
            uint4 ph, pl;
            if constexpr (HT == 8) {
              float2 x = mul2(make_float2(s[i][0], s[i][1]), dv[0]), y = mul2(make_float2(s[i + 1][0], s[i + 1][1]), dv[1]);
              ph.x = plane_f16(x.x, x.y);
              ph.z = plane_f16(y.x, y.y);
              ph.y = plane_f16(x.x, x.y);
              ph.w = plane_f16(y.x, y.y);
            } else {
              float x[8];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                x[k] = s[i][k] * (k & 1 ? dv[0].y : dv[0].x);
                x[4 + k] = s[i + 1][k] * (k & 1 ? dv[1].y : dv[1].x);
              }
              ph.x = plane_f16(x[0], x[1]);
              ph.y = plane_f16(x[2], x[3]);
              ph.z = plane_f16(x[4], x[5]);
              ph.w = plane_f16(x[6], x[7]);
              pl.x = plane_f16(x[0], x[1]);
              pl.y = plane_f16(x[2], x[3]);
              pl.z = plane_f16(x[4], x[5]);
              pl.w = plane_f16(x[6], x[7]);
            }
            uint32_t w[4];   // columns 32 blk + 4 g .. + 3 of keys 2 c, 2 c + 1, 2 c + 8, 2 c + 9
#pragma unroll
            for (int k = 0; k < 4; ++k)
              w[k] = lds32(vs + 2 * c * C::VP + (((2 * blk + (g >> 2)) ^ C::v_swz(2 * c)) * 16 + (g & 3) * 4) +
                           (8 * (i + (k >> 1)) + (k & 1)) * C::VP) ^
                     0x80808080u;
            const uint32_t p0 = __byte_perm(w[0], w[1], 0x5140), p1 = __byte_perm(w[0], w[1], 0x7362);
            const uint32_t p2 = __byte_perm(w[2], w[3], 0x5140), p3 = __byte_perm(w[2], w[3], 0x7362);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t sel = k & 1 ? 0x4342 : 0x4140;
              const uint32_t b0 = i8pair_f16(k < 2 ? p0 : p1, sel), b1 = i8pair_f16(k < 2 ? p2 : p3, sel);
              if constexpr (HT == 16) mma16<CT>(i == 0, d[k], pl, b0, b1);
              mma16<CT>(HT == 8 && i == 0, d[k], ph, b0, b1);
            }
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) gather(4 * blk + k, d[k]);
        }
      } else {
        constexpr int kP = HT == 8 ? (PL == 3 ? 2 : 1) : PL;   // operand sets
        uint4 pp[NT / 2][kP];
#pragma unroll
        for (int i = 0; i < NT; i += 2) {   // 16 keys
          uint4 (&p)[kP] = pp[i / 2];
          if constexpr (HT == 8) {
            float x0 = s[i][0], x1 = s[i][1], x2 = s[i + 1][0], x3 = s[i + 1][1];
            p[0].x = plane16<CT>(x0, x1);
            p[0].z = plane16<CT>(x2, x3);
            p[0].y = plane16<CT>(x0, x1);
            p[0].w = plane16<CT>(x2, x3);
            if constexpr (kP == 2) {
              p[1].x = plane16<CT>(x0, x1);
              p[1].z = plane16<CT>(x2, x3);
              p[1].y = p[1].w = 0;
            }
          } else {
            float x[8];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              x[k] = s[i][k];
              x[4 + k] = s[i + 1][k];
            }
#pragma unroll
            for (int q = 0; q < kP; ++q) {
              p[q].x = plane16<CT>(x[0], x[1]);
              p[q].y = plane16<CT>(x[2], x[3]);
              p[q].z = plane16<CT>(x[4], x[5]);
              p[q].w = plane16<CT>(x[6], x[7]);
            }
          }
        }
#pragma unroll
        for (int d2 = 0; d2 < OT; d2 += 2) {
          float e0[4], e1[4];
#pragma unroll
          for (int i = 0; i < NT; i += 2) {
            uint32_t b[4];   // keys 0..7 and 8..15 of columns 8 d2 .., then of 8 d2 + 8 ..
            ldmatrix_x4_trans(vs + (lane & 15) * C::VP + (lane >> 4) * 16 + 8 * i * C::VP + d2 * 16, b);
#pragma unroll
            for (int p = kP - 1; p >= 0; --p) {
              mma16<CT>(i == 0 && p == kP - 1, e0, pp[i / 2][p], b[0], b[1]);
              mma16<CT>(i == 0 && p == kP - 1, e1, pp[i / 2][p], b[2], b[3]);
            }
          }
          gather(d2, e0);
          gather(d2 + 1, e1);
        }
      }
      __syncwarp();   // the stage is read
      ++used;
      --staged;
      if (has_tile()) issue();
    }

    // ---- the next history of this CTA: its q is read while this one's sums are joined
    Cursor next = cur;
    int next_first = cur_first;
    u += t1 - t0;
    const bool more = u < u_hi;
    if (more) next_history(next, next_first);
    if (more) load_q(next);

    // ---- the warps' sums joined: weights of a lane group summed
    float2 (&ov)[OT][R] = o;
    if constexpr (CT == kCacheQ8) {   // the same lift in every warp
      const float back = ex2(-(float)lift_d);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        l[r] = (l2[r].x + l2[r].y) * back;
#pragma unroll
        for (int i = 0; i < OT; ++i) ov[i][r] = mul2(ov[i][r], make_float2(back, back));
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    }
    float* buf = reinterpret_cast<float*>(region);
    auto put = [&](float* d) {
      float4* d4 = reinterpret_cast<float4*>(d) + lane;
#pragma unroll
      for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int i = 0; i < OT; i += 2)
          d4[(r * (OT / 2) + i / 2) * 32] = make_float4(ov[i][r].x, ov[i][r].y, ov[i + 1][r].x, ov[i + 1][r].y);
        reinterpret_cast<float2*>(d + OT * 2 * R * 32)[r * 32 + lane] = make_float2(m[r], l[r]);
      }
    };
    auto add = [&](const float* d) {
      const float4* d4 = reinterpret_cast<const float4*>(d) + lane;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float2 ml = reinterpret_cast<const float2*>(d + OT * 2 * R * 32)[r * 32 + lane];
        const float mn = fmaxf(m[r], ml.x);
        // a warp without keys has sums of 0, which any finite factor keeps (and NaN sums stay NaN)
        const float f = m[r] == -INFINITY ? 1.f : ex2(m[r] - mn), e = ml.x == -INFINITY ? 1.f : ex2(ml.x - mn);
        l[r] = l[r] * f + ml.y * e;
        m[r] = mn;
#pragma unroll
        for (int i = 0; i < OT; i += 2) {
          const float4 y = d4[(r * (OT / 2) + i / 2) * 32];
          const float2 e2 = make_float2(e, e), f2 = make_float2(f, f);
          ov[i][r] = fma2(make_float2(y.x, y.y), e2, mul2(ov[i][r], f2));
          ov[i + 1][r] = fma2(make_float2(y.z, y.w), e2, mul2(ov[i + 1][r], f2));
        }
      }
    };
    __syncthreads();   // q is read by every warp
    if constexpr (C::kBufs == 2) {
      if (warp >= 2) put(buf + (warp - 2) * C::kBufFloats);
      __syncthreads();
      if (warp < 2) add(buf + warp * C::kBufFloats);
      __syncthreads();
      if (warp == 1) put(buf);
      __syncthreads();
      if (warp == 0) add(buf);
    } else {
      for (int w = kAttnWarps - 1; w >= 1; --w) {
        if (warp == w) put(buf);
        __syncthreads();
        if (warp == 0) add(buf);
        __syncthreads();
      }
    }
    if (warp == 0) {   // heads whose sums are not finite (a product with 0 is NaN then)
      bool odd[R], any = false;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float2 zero = make_float2(l[r] * 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < OT; ++i) zero = fma2(ov[i][r], make_float2(0.f, 0.f), zero);
        float z = zero.x + zero.y;
        z += __shfl_xor_sync(0xffffffffu, z, 1);
        z += __shfl_xor_sync(0xffffffffu, z, 2);
        odd[r] = z != 0.f;
        any |= odd[r];
      }
      if (__any_sync(0xffffffffu, any)) {
        plain_part<CT, DH, HT, PL>(a, cur.b, cur.jt, t0, t1, buf);
        __syncwarp();
#pragma unroll
        for (int r = 0; r < R; ++r) {
          if (!odd[r]) continue;
          const float2 ml = reinterpret_cast<const float2*>(buf + OT * 2 * R * 32)[r * 32 + lane];
          m[r] = ml.x;
          l[r] = ml.y;
#pragma unroll
          for (int i = 0; i < OT; i += 2) {
            const float4 y = reinterpret_cast<const float4*>(buf)[(r * (OT / 2) + i / 2) * 32 + lane];
            ov[i][r] = make_float2(y.x, y.y);
            ov[i + 1][r] = make_float2(y.z, y.w);
          }
        }
      }
    }

    // The lane's sums of row r as runs of consecutive columns: f(column, values, count).
    auto runs = [&](int r, auto&& f) {
      if constexpr (CT == kCacheF32 || CT == kCacheQ8) {   // tile 4 q + k has column 4 n + k of block q at n
#pragma unroll
        for (int q = 0; q < OT; q += 4) {
          const float v[8] = {ov[q][r].x, ov[q + 1][r].x, ov[q + 2][r].x, ov[q + 3][r].x,
                              ov[q][r].y, ov[q + 1][r].y, ov[q + 2][r].y, ov[q + 3][r].y};
          f(8 * q + 8 * c, v, std::integral_constant<int, 8>{});
        }
      } else {
#pragma unroll
        for (int i = 0; i < OT; ++i) {
          const float v[2] = {ov[i][r].x, ov[i][r].y};
          f(8 * i + 2 * c, v, std::integral_constant<int, 2>{});
        }
      }
    };
    const long long out0 = (long long)cur.b * a.ldo + ((long long)jh * a.group + h0) * DH;
    const long long lse0 = (long long)cur.b * a.n_heads + (long long)jh * a.group + h0;
    const bool whole = t0 == 0 && t1 == nt;
    if (whole) {
      if (warp == 0) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          if (g + 8 * r >= heads) continue;
          const float inv = l[r] == 0.f ? 0.f : 1.f / l[r];
          runs(r, [&](int col, const float* v, auto count) {
            store_rows<decltype(count)::value>(a.out, a.row_type, a.out_vec, out0 + (long long)(g + 8 * r) * DH + col, v,
                                               inv);
          });
          if (a.lse && c == 0)
            a.lse[lse0 + g + 8 * r] = l[r] == 0.f ? -INFINITY : (m[r] + (log2f(l[r]) - kLift)) * 0.693147180559945f;
        }
      }
      __syncthreads();   // the region is read
    } else {
      // the CTAs that hold this history: first .. first + pieces - 1
      const int ub = cur_first + cur.jt * nt, first = cta_of(ub), pieces = cta_of(ub + nt - 1) - first + 1;
      auto slot_of = [&](int cta) { return a.slots + ((long long)cta * 2 + (cta == first)) * (HT * DH + 2 * HT); };
      if (warp == 0) {
        float* d = slot_of(blockIdx.x);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          runs(r, [&](int col, const float* v, auto count) {
            float* to = d + (g + 8 * r) * DH + col;
            if constexpr (decltype(count)::value == 8) {
              __stcg(reinterpret_cast<float4*>(to), make_float4(v[0], v[1], v[2], v[3]));
              __stcg(reinterpret_cast<float4*>(to) + 1, make_float4(v[4], v[5], v[6], v[7]));
            } else {
              __stcg(reinterpret_cast<float2*>(to), make_float2(v[0], v[1]));
            }
          });
          if (c == 0) {
            __stcg(d + HT * DH + g + 8 * r, m[r]);
            __stcg(d + HT * DH + HT + g + 8 * r, l[r]);
          }
        }
      }
      // Added up in order by whoever finishes last: up to kFew pieces at once; more in groups of about the square root
      // of their number, by the CTA that completes a group, then the groups. 55 pieces (one request of 16384 tokens, 32 /
      // 8 heads of 128): 26.2 us in groups, 29.5 at once; 32 pieces (4096): 15.3 and 15.0; 16 pieces: 13.2 and 11.9.
      constexpr int kFew = 32;
      static_assert(kFew <= 32 && kAttnMaxCtas <= 32 * 32, "32 pieces, or groups, at most at a time: a lane to each");
      int group = 1;
      while (group * group < pieces) ++group;
      if (pieces <= kFew) group = pieces;
      int lead = first + (blockIdx.x - first) / group * group, stride = 1, count = min(group, first + pieces - lead);
      unsigned* ticket = a.tickets + lead * 2 + (lead == first);
#pragma unroll 1
      for (;;) {
        __threadfence();   // (this thread's part of the sums)
        __syncthreads();
        if (tid == 0) {
          last_flag = atomicAdd(ticket, 1u) == (unsigned)count - 1;
          if (last_flag) *ticket = 0;   // ready for the next call
        }
        __syncthreads();
        if (!last_flag) break;
        const bool final = group >= pieces || stride > 1;
        __threadfence();
        // HW heads to a warp, a lane for four columns (d_head 128; fewer lanes below), kFly pieces' loads in flight (an
        // L2 read here takes 0.5 us or more, and one after another they were most of the time of a short call)
        constexpr int HW = HT / kAttnWarps, kFly = C::OCC == 3 ? 8 : 4;
        const int col4 = min(lane, DH / 4 - 1);
        // this lane's piece (a lane past the end repeats the last one with weight 0), and the first sums
        const bool on = lane < count;
        const float* d = slot_of(lead + min(lane, count - 1) * stride) + HT * DH + warp;
        float mm[HW], ll[HW], f[HW];
#pragma unroll
        for (int i = 0; i < HW; ++i) {
          mm[i] = __ldcg(d + i * kAttnWarps);
          f[i] = __ldcg(d + HT + i * kAttnWarps);
        }
        float4 x[HW], y[kFly][HW];
        auto read = [&](int k0) {
#pragma unroll
          for (int k = 0; k < kFly; ++k) {
            const float4* src =
                reinterpret_cast<const float4*>(slot_of(lead + min(k0 + k, count - 1) * stride) + warp * DH) + col4;
#pragma unroll
            for (int i = 0; i < HW; ++i) y[k][i] = __ldcg(src + i * kAttnWarps * (DH / 4));
          }
        };
        read(0);
#pragma unroll
        for (int i = 0; i < HW; ++i) {
          const float mp = mm[i];
#pragma unroll
          for (int w = 16; w; w >>= 1) mm[i] = fmaxf(mm[i], __shfl_xor_sync(0xffffffffu, mm[i], w));
          // (a piece without a key, or with NaN scores only, has m -inf: its sums count as they are)
          const float wp = !on ? 0.f : mp == -INFINITY ? 1.f : ex2(mp - mm[i]);
          ll[i] = on ? f[i] * wp : 0.f;
          f[i] = wp;
          x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll 1
        for (int k0 = 0;;) {
#pragma unroll
          for (int k = 0; k < kFly; ++k)
#pragma unroll
            for (int i = 0; i < HW; ++i) {
              const float fk = __shfl_sync(0xffffffffu, f[i], (k0 + k) & 31);
              if (k0 + k >= count) continue;
              x[i].x += fk * y[k][i].x;
              x[i].y += fk * y[k][i].y;
              x[i].z += fk * y[k][i].z;
              x[i].w += fk * y[k][i].w;
            }
          k0 += kFly;
          if (k0 >= count) break;
          read(k0);
        }
#pragma unroll
        for (int i = 0; i < HW; ++i)
#pragma unroll
          for (int w = 16; w; w >>= 1) ll[i] += __shfl_xor_sync(0xffffffffu, ll[i], w);
        if (!final) {   // the group's sums in place of its first piece's (each warp and lane its own part)
          __syncwarp();
          float* to = slot_of(lead);
#pragma unroll
          for (int i = 0; i < HW; ++i) {
            const int h = warp + i * kAttnWarps;
            if (lane < DH / 4) __stcg(reinterpret_cast<float4*>(to + h * DH) + lane, x[i]);
            if (lane == 0) {
              __stcg(to + HT * DH + h, mm[i]);
              __stcg(to + HT * DH + HT + h, ll[i]);
            }
          }
          lead = first;
          stride = group;
          count = (pieces + group - 1) / group;
          ticket = a.tickets + 2 * kAttnMaxCtas + first;
          continue;
        }
#pragma unroll
        for (int i = 0; i < HW; ++i) {
          const int h = warp + i * kAttnWarps;
          if (h >= heads) continue;
          if (lane < DH / 4) {
            const float inv = ll[i] == 0.f ? 0.f : 1.f / ll[i];
            const float v[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
            store_rows<4>(a.out, a.row_type, a.out_vec, out0 + (long long)h * DH + lane * 4, v, inv);
          }
          if (a.lse && lane == 0)
            a.lse[lse0 + h] = ll[i] == 0.f ? -INFINITY : (mm[i] + (log2f(ll[i]) - kLift)) * 0.693147180559945f;
        }
        break;
      }
      __syncthreads();   // the region and the flag are read
    }
    if (!more) break;
    cur = next;
    cur_first = next_first;
  }
  cp_wait<0>();
}

// The kernel's shared memory on the current device.
template <int CT, int DH, int HT, int PL>
int prepare_one() {
  static DeviceOnce setup;
  return setup.ensure([](int) {
    return cudaFuncSetAttribute(paged_attend_kernel<CT, DH, HT, PL>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                Cfg<CT, DH, HT, PL>::kSmem) == cudaSuccess
               ? 0
               : -3;
  });
}

template <int CT, int DH, int HT, int PL>
int launch_one(const PagedAttnArgs& a, cudaStream_t st) {
  using C = Cfg<CT, DH, HT, PL>;
  if (prepare_one<CT, DH, HT, PL>()) return -3;
  const long long most = (long long)a.width * a.kv.page_size;
  const long long units =
      (long long)a.n_req * a.kv.n_kv * ((a.group + HT - 1) / HT) * ((most + C::UK - 1) / C::UK);
  const int grid = (int)std::max<long long>(1, std::min<long long>(C::OCC * 148, units));
  return launch_pdl(paged_attend_kernel<CT, DH, HT, PL>, dim3(grid), dim3(kAttnWarps * 32), C::kSmem, st, a);
}

template <int CT, int PL>
int prepare_type() {
  if (prepare_one<CT, 32, 8, PL>() || prepare_one<CT, 32, 16, PL>() || prepare_one<CT, 64, 8, PL>() ||
      prepare_one<CT, 64, 16, PL>() || prepare_one<CT, 96, 8, PL>() || prepare_one<CT, 96, 16, PL>() ||
      prepare_one<CT, 128, 8, PL>() || prepare_one<CT, 128, 16, PL>())
    return -3;
  return 0;
}

template <int CT, int PL>
int launch_type(const PagedAttnArgs& a, cudaStream_t st) {
  const bool wide = a.group > 8;
  switch (a.kv.dh) {
    case 32: return wide ? launch_one<CT, 32, 16, PL>(a, st) : launch_one<CT, 32, 8, PL>(a, st);
    case 64: return wide ? launch_one<CT, 64, 16, PL>(a, st) : launch_one<CT, 64, 8, PL>(a, st);
    case 96: return wide ? launch_one<CT, 96, 16, PL>(a, st) : launch_one<CT, 96, 8, PL>(a, st);
    default: return wide ? launch_one<CT, 128, 16, PL>(a, st) : launch_one<CT, 128, 8, PL>(a, st);
  }
}

}  // namespace attn

int paged_attend_f32(const PagedAttnArgs& a, cudaStream_t st);
int paged_attend_f16(const PagedAttnArgs& a, cudaStream_t st);
int paged_attend_bf16(const PagedAttnArgs& a, cudaStream_t st);
int paged_attend_q8(const PagedAttnArgs& a, cudaStream_t st);
int paged_prepare_f32();
int paged_prepare_f16();
int paged_prepare_bf16();
int paged_prepare_q8();

}  // namespace tb2
