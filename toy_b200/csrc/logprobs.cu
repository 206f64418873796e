// Log probabilities of given tokens, entropy and the most likely alternatives
// of each row of logits, and the gradient back to the logits.
//
// With z = a x (a the scale), m = max z, s = sum exp(z - m):
//   ln p_j = (z_j - m) - ln s,   H = ln s - sum exp(z - m) (z - m) / s.
#include <cmath>

#include "rows.cuh"
#include "runtime.cuh"

namespace tb2 {
namespace {

constexpr int kThreads = 256, kMaxTop = 32;

struct ScoreArgs {
  const void* x;
  long long ld;
  const long long* tokens;
  float *logprob, *stats, *entropy, *top_lp;
  long long* top_ids;
  int* err;
  float scale;
  int n, V, top;
};

// Values in the order of (x, lower index first) as whole numbers: NaN above everything, -0 equal to 0.
__device__ __forceinline__ unsigned long long top_key(float x, int j) {
  x += 0.0f;
  unsigned b = __float_as_uint(x);
  b = x != x ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
  return (unsigned long long)b << 32 | (unsigned)(0x7fffffff - j);
}

template <class F>
__device__ float block_reduce(float v, F&& f, float* sm) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if (threadIdx.x % 32 == 0) sm[threadIdx.x / 32] = v;
  __syncthreads();
  v = sm[0];
  for (int w = 1; w < kThreads / 32; ++w) v = f(v, sm[w]);
  return v;
}

template <class T>
__global__ void __launch_bounds__(kThreads) score_kernel(ScoreArgs a) {
  griddep_wait();
  __shared__ float sm[kThreads / 32];
  __shared__ unsigned long long best[kThreads / 32];
  const int V = a.V;
  for (long long r = blockIdx.x; r < a.n; r += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + r * a.ld;
    float m = -INFINITY;
    for (int j = threadIdx.x; j < V; j += kThreads) {
      const float z = to_f32(x[j]) * a.scale;
      m = z > m || z != z ? z : m;
    }
    m = block_reduce(m, [](float p, float q) { return p != p || p > q ? p : q; }, sm);
    const float ref = m == -INFINITY ? 0.f : m;
    float s = 0.f, u = 0.f;
    for (int j = threadIdx.x; j < V; j += kThreads) {
      const float t = to_f32(x[j]) * a.scale - ref, e = expf(t);
      s += e;
      u += e * (t < -1000.f ? -1000.f : t);
    }
    auto add = [](float p, float q) { return p + q; };
    s = block_reduce(s, add, sm);
    u = block_reduce(u, add, sm);
    const float ln = logf(s);
    if (threadIdx.x == 0) {
      a.stats[2 * r] = ref;
      a.stats[2 * r + 1] = ln;
      const long long t = a.tokens[r];
      float lp = 0.f;
      if (t >= V) {
        atomicExch(a.err, (int)kErrToken);
        lp = NAN;
      } else if (t >= 0) {
        lp = s > 0.f || s != s ? (to_f32(x[t]) * a.scale - ref) - ln : -INFINITY;
      }
      a.logprob[r] = lp;
      if (a.entropy) a.entropy[r] = s == 0.f ? 0.f : ln - u / s;
    }
    unsigned long long last = ~0ull;
    for (int k = 0; k < a.top; ++k) {
      unsigned long long b = 0;
      for (int j = threadIdx.x; j < V; j += kThreads) {
        const unsigned long long key = top_key(to_f32(x[j]), j);
        if (key < last && key > b) b = key;
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) {
        const unsigned long long q = __shfl_xor_sync(0xffffffffu, b, o);
        b = q > b ? q : b;
      }
      __syncthreads();
      if (threadIdx.x % 32 == 0) best[threadIdx.x / 32] = b;
      __syncthreads();
      for (int w = 0; w < kThreads / 32; ++w) b = best[w] > b ? best[w] : b;
      last = b;
      if (threadIdx.x == 0) {
        const int j = 0x7fffffff - (int)(unsigned)b;
        a.top_ids[r * a.top + k] = j;
        a.top_lp[r * a.top + k] = s == 0.f ? -INFINITY : (to_f32(x[j]) * a.scale - ref) - ln;
      }
    }
    __syncthreads();
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
  int n, V, top;
};

template <class T>
__global__ void __launch_bounds__(kThreads) score_grad_kernel(GradArgs a) {
  griddep_wait();
  __shared__ float x_at[kMaxTop + 1], g_at[kMaxTop + 1];
  __shared__ int at[kMaxTop + 1];
  const int V = a.V, tid = threadIdx.x;
  for (long long r = blockIdx.x; r < a.n; r += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + r * a.ld;
    T* d = static_cast<T*>(a.d) + r * a.ldd;
    __syncthreads();
    // the words with a gradient of their own: the token, then the alternatives
    if (tid <= a.top) {
      const long long j = tid == 0 ? a.tokens[r] : a.top_ids[r * a.top + tid - 1];
      float g = tid == 0 ? (a.g_lp ? a.g_lp[r] : 0.f) : a.g_top[r * a.top + tid - 1];
      const bool ok = j >= 0 && j < V && a.stats[2 * r + 1] != -INFINITY;   // (a row without a word has no gradient)
      if (j >= V || (j < 0 && tid)) atomicExch(a.err, (int)kErrToken);
      at[tid] = ok ? (int)j : -1;
      g_at[tid] = ok ? g : 0.f;
      x_at[tid] = ok ? to_f32(x[j]) : 0.f;
    }
    __syncthreads();
    float g = 0.f;
    for (int k = 0; k <= a.top; ++k) g += g_at[k];
    const float m = a.stats[2 * r], ln = a.stats[2 * r + 1];
    const float gh = a.g_h ? a.g_h[r] : 0.f, h = a.g_h ? a.entropy[r] : 0.f;
    auto base = [&](float xv) {
      const float t = (xv * a.scale - m) - ln;
      const float p = ln == -INFINITY ? 0.f : expf(t);
      return -p * (g + gh * ((t < -1000.f ? -1000.f : t) + h));
    };
    for (int j = tid; j < V; j += kThreads) d[j] = from_f32<T>(base(to_f32(x[j])) * a.scale);
    __syncthreads();
    if (tid <= a.top && at[tid] >= 0) {
      float v = 0.f;
      for (int k = 0; k <= a.top; ++k)
        if (at[k] == at[tid]) v += g_at[k];
      d[at[tid]] = from_f32<T>((base(x_at[tid]) + v) * a.scale);
    }
  }
}

bool rows_ok(long long ld, int V, const void* p, int type) {
  return p && ld >= V && aligned(p, type_bytes(type));
}

template <class T>
int prepare_type() {
  return load_kernel(score_kernel<T>) || load_kernel(score_grad_kernel<T>) ? -3 : 0;
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
  if (!rows_ok(a->ld, a->vocab, a->logits, a->row_type) || !(a->scale > 0.f) || !std::isfinite(a->scale)) return -1;
  if (!a->tokens || !a->logprob || !a->stats || a->top < 0 || a->top > kMaxTop || a->top > a->vocab) return -1;
  if (a->top && (!a->top_ids || !a->top_logprobs)) return -1;
  if (!all_aligned(8, {a->tokens, a->stats, a->top_ids}) || !all_aligned(4, {a->logprob, a->entropy, a->top_logprobs}))
    return -1;
  int* err = device_error_word();
  if (!err) return -3;
  ScoreArgs k = {a->logits, a->ld, a->tokens, a->logprob, a->stats, a->entropy, a->top_logprobs, a->top_ids, err,
                 a->scale, a->n_rows, a->vocab, a->top};
  return by_row_type(a->row_type, [&](auto t) {
    return launch_pdl(score_kernel<decltype(t)>, dim3(a->n_rows), dim3(kThreads), 0, static_cast<cudaStream_t>(stream),
                      k);
  });
}

int tb2_logprobs_grad(const tb2_logprobs_grad_args* a, void* stream) {
  using namespace tb2;
  if (!a || a->n_rows < 0 || a->vocab < 1 || !row_type_ok(a->row_type)) return -1;
  if (a->n_rows == 0) return 0;
  if (!rows_ok(a->ld, a->vocab, a->logits, a->row_type) || !(a->scale > 0.f) || !std::isfinite(a->scale)) return -1;
  if (!rows_ok(a->ldd, a->vocab, a->d_logits, a->row_type)) return -1;
  if (!a->tokens || !a->stats || a->top < 0 || a->top > kMaxTop || a->top > a->vocab) return -1;
  if (a->top && (!a->top_ids || !a->g_top)) return -1;
  if (a->g_entropy && !a->entropy) return -1;
  if (!all_aligned(8, {a->tokens, a->stats, a->top_ids}) ||
      !all_aligned(4, {a->entropy, a->g_logprob, a->g_entropy, a->g_top}))
    return -1;
  int* err = device_error_word();
  if (!err) return -3;
  GradArgs k = {a->logits, a->ld, a->tokens, a->stats, a->entropy, a->g_logprob, a->g_entropy, a->g_top, a->top_ids,
                a->d_logits, a->ldd, err, a->scale, a->n_rows, a->vocab, a->top};
  return by_row_type(a->row_type, [&](auto t) {
    return launch_pdl(score_grad_kernel<decltype(t)>, dim3(a->n_rows), dim3(kThreads), 0,
                      static_cast<cudaStream_t>(stream), k);
  });
}

}  // extern "C"
