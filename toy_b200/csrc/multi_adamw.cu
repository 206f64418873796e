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
#include <cmath>

#include "rows.cuh"
#include "runtime.cuh"

namespace tb2 {
namespace {

constexpr int kBlock = 256;        // values that share a scale
constexpr int kMaxTensors = 256;   // tensors a launch

struct Tensors {
  tb2_adamw_tensor t[kMaxTensors];
  int first[kMaxTensors + 1];   // blocks before tensor i
  int n;
};

// e4m3 of x (|x| <= 448), given to 64 bits: rounded once.
__device__ __forceinline__ uint8_t e4m3_of(double x) {
  const double a = fabs(x);
  const int e = a < 0.015625 ? -6 : ilogb(a);
  double q = rint(ldexp(a, 3 - e));   // eighths of the leading bit's weight; at the bottom, multiples of 2^-9
  q = ldexp(q, e - 3);
  return __nv_cvt_float_to_fp8((float)(x < 0 ? -q : q), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float e4m3_to(uint8_t c) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
}

// The power of two of a block whose largest magnitude is top.
__device__ __forceinline__ float block_scale(double top) {
  if (!isfinite(top)) return NAN;
  int e;
  const double f = frexp(top / 448.0, &e);
  return ldexpf(1.f, max(top == 0.0 ? -100 : f == 0.5 ? e - 1 : e, -100));
}

__device__ __forceinline__ double block_max(double v, double* sm) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const double q = __shfl_xor_sync(0xffffffffu, v, o);
    v = q > v || q != q ? q : v;
  }
  __syncthreads();
  if (threadIdx.x % 32 == 0) sm[threadIdx.x / 32] = v;
  __syncthreads();
  for (int w = 0; w < kBlock / 32; ++w) v = sm[w] > v || sm[w] != sm[w] ? sm[w] : v;
  return v;
}

__device__ __forceinline__ float load_value(const void* p, int type, long long i) {
  return type == kTypeF32 ? static_cast<const float*>(p)[i]
       : type == kTypeF16 ? to_f32(static_cast<const __half*>(p)[i])
                          : to_f32(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_value(void* p, int type, long long i, float v) {
  if (type == kTypeF32) static_cast<float*>(p)[i] = v;
  else if (type == kTypeF16) static_cast<__half*>(p)[i] = from_f32<__half>(v);
  else static_cast<__nv_bfloat16*>(p)[i] = from_f32<__nv_bfloat16>(v);
}

// A CTA a block of 256 values.
template <int BITS>
__global__ void __launch_bounds__(kBlock) step_kernel(const __grid_constant__ Tensors ts, int p_type, int g_type,
                                                      int copy_type, const float* hp, const float* factor) {
  griddep_wait();
  __shared__ double sm[kBlock / 32];
  const float a = hp[0], b1 = hp[1], b2 = hp[2], eps = hp[3], wd = hp[4], c1 = hp[5], c2 = sqrtf(hp[6]);
  const float gf = factor ? *factor : 1.f;
  int i = 0;
  while (i + 1 < ts.n && (int)blockIdx.x >= ts.first[i + 1]) ++i;
  const tb2_adamw_tensor& t = ts.t[i];
  const int blk = blockIdx.x - ts.first[i];
  const long long k = (long long)blk * kBlock + threadIdx.x;
  const bool on = k < t.n;
  const double g = on ? (double)load_value(t.g, g_type, k) * gf : 0.0;
  const float p = on ? load_value(t.p, p_type, k) : 0.f;
  double m = 0.0, v = 0.0;
  if (on && BITS == 8) {
    m = e4m3_to(static_cast<uint8_t*>(t.m)[k]) * t.m_scale[blk];
    v = e4m3_to(static_cast<uint8_t*>(t.v)[k]) * t.v_scale[blk];
    v *= v;
  } else if (on) {
    m = static_cast<float*>(t.m)[k];
    v = static_cast<float*>(t.v)[k];
  }
  m = m * b1 + g * (1.0 - b1);
  v = v * b2 + g * g * (1.0 - b2);
  const double r = sqrt(v);
  if (on) {
    const float w = p * (1.f - a * wd) - a * (float)m * c1 / ((float)r * c2 + eps);
    store_value(t.p, p_type, k, w);
    if (t.copy) store_value(t.copy, copy_type, k, p_type == kTypeF32 ? w : load_value(t.p, p_type, k));
  }
  if (BITS == 32) {
    if (on) static_cast<float*>(t.m)[k] = (float)m, static_cast<float*>(t.v)[k] = (float)v;
    return;
  }
  const float sm_ = block_scale(block_max(on ? fabs(m) : 0.0, sm)), sv = block_scale(block_max(on ? r : 0.0, sm));
  if (on) {
    static_cast<uint8_t*>(t.m)[k] = sm_ == sm_ ? e4m3_of(m / sm_) : 0x7f;
    uint8_t q = sv == sv ? e4m3_of(r / sv) : 0x7f;
    static_cast<uint8_t*>(t.v)[k] = q == 0 && r > 0.0 ? 1 : q;
    if (threadIdx.x == 0) t.m_scale[blk] = sm_, t.v_scale[blk] = sv;
  }
}

// out: the values that 8-bit moments stand for (p: m's, copy: v's, f32), or (PUT) the moments from those values
template <bool PUT>
__global__ void __launch_bounds__(kBlock) moments_kernel(const __grid_constant__ Tensors ts) {
  griddep_wait();
  __shared__ double sm[kBlock / 32];
  int i = 0;
  while (i + 1 < ts.n && (int)blockIdx.x >= ts.first[i + 1]) ++i;
  const tb2_adamw_tensor& t = ts.t[i];
  const int blk = blockIdx.x - ts.first[i];
  const long long k = (long long)blk * kBlock + threadIdx.x;
  const bool on = k < t.n;
  uint8_t *mq = static_cast<uint8_t*>(t.m), *vq = static_cast<uint8_t*>(t.v);
  float *mo = static_cast<float*>(t.p), *vo = static_cast<float*>(t.copy);
  if (!PUT) {
    if (!on) return;
    const float r = e4m3_to(vq[k]) * t.v_scale[blk];
    mo[k] = e4m3_to(mq[k]) * t.m_scale[blk];
    vo[k] = r * r;
    return;
  }
  const double m = on ? mo[k] : 0.0, r = on ? sqrt((double)vo[k]) : 0.0;
  const float sm_ = block_scale(block_max(fabs(m), sm)), sv = block_scale(block_max(r, sm));
  if (on) {
    mq[k] = sm_ == sm_ ? e4m3_of(m / sm_) : 0x7f;
    uint8_t q = sv == sv ? e4m3_of(r / sv) : 0x7f;
    vq[k] = q == 0 && r > 0.0 ? 1 : q;
    if (threadIdx.x == 0) t.m_scale[blk] = sm_, t.v_scale[blk] = sv;
  }
}

bool tensor_ok(const tb2_adamw_tensor& t, int p_type, int g_type, int copy_type, int bits) {
  if (t.n < 0 || t.n > (1LL << 38)) return false;
  if (t.n == 0) return true;
  if (!t.p || !t.g || !t.m || !t.v || (t.copy && !aligned(t.copy, type_bytes(copy_type)))) return false;
  if (!aligned(t.p, type_bytes(p_type)) || !aligned(t.g, type_bytes(g_type))) return false;
  if (bits == 32) return all_aligned(4, {t.m, t.v});
  return t.m_scale && t.v_scale && all_aligned(4, {t.m_scale, t.v_scale});
}

// The tensors in groups of what a launch takes, empty ones left out.
template <class F>
int in_groups(const tb2_adamw_tensor* t, int n, F&& launch) {
  Tensors g;
  for (int i = 0; i < n;) {
    g.n = 0;
    long long blocks = 0;
    for (; i < n && g.n < kMaxTensors; ++i) {
      if (t[i].n == 0) continue;
      const long long b = (t[i].n + kBlock - 1) / kBlock;
      if (blocks + b > 0x7fffffffLL) break;
      g.first[g.n] = (int)blocks;
      g.t[g.n++] = t[i];
      blocks += b;
    }
    g.first[g.n] = (int)blocks;
    if (g.n)
      if (int rc = launch(g, (int)blocks)) return rc;
  }
  return 0;
}

}  // namespace

int multi_adamw_prepare() {
  return load_kernel(step_kernel<8>) || load_kernel(step_kernel<32>) || load_kernel(moments_kernel<true>) ||
                 load_kernel(moments_kernel<false>)
             ? -3
             : 0;
}

}  // namespace tb2

extern "C" {

int tb2_adamw_multi(const tb2_adamw_multi_args* a, void* stream) {
  using namespace tb2;
  if (!a || a->n_tensors < 0 || (a->n_tensors && !a->tensors) || (a->state_bits != 8 && a->state_bits != 32)) return -1;
  if (!row_type_ok(a->p_type) || !row_type_ok(a->g_type) || !row_type_ok(a->copy_type)) return -1;
  if (!a->hp || !all_aligned(4, {a->hp, a->grad_scale})) return -1;
  for (int i = 0; i < a->n_tensors; ++i)
    if (!tensor_ok(a->tensors[i], a->p_type, a->g_type, a->copy_type, a->state_bits)) return -1;
  return in_groups(a->tensors, a->n_tensors, [&](const Tensors& g, int blocks) {
    return launch_pdl(a->state_bits == 8 ? step_kernel<8> : step_kernel<32>, dim3(blocks), dim3(kBlock), 0,
                      static_cast<cudaStream_t>(stream), g, a->p_type, a->g_type, a->copy_type, a->hp, a->grad_scale);
  });
}

int tb2_adamw_moments(const tb2_adamw_tensor* tensors, int n_tensors, int put, void* stream) {
  using namespace tb2;
  if (n_tensors < 0 || (n_tensors && !tensors)) return -1;
  for (int i = 0; i < n_tensors; ++i) {
    const tb2_adamw_tensor& t = tensors[i];
    if (t.n < 0 || t.n > (1LL << 38)) return -1;
    if (t.n && (!t.p || !t.copy || !t.m || !t.v || !t.m_scale || !t.v_scale ||
                !all_aligned(4, {t.p, t.copy, t.m_scale, t.v_scale})))
      return -1;
  }
  return in_groups(tensors, n_tensors, [&](const Tensors& g, int blocks) {
    return launch_pdl(put ? moments_kernel<true> : moments_kernel<false>, dim3(blocks), dim3(kBlock), 0,
                      static_cast<cudaStream_t>(stream), g);
  });
}

}  // extern "C"
