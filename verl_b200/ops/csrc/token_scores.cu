// Scores of rows of logits: log-probs of given tokens, entropy, log-sum-exp, the most likely tokens; and the gradient of log-probs and entropy.
//
// With z = x / temperature and m the largest z so far, a row is read once for
//   s = sum e^(z - m),  w = sum e^(z - m) (z - m):   lse = m + log s,  H = log s - w / s
// and the gradient of sum_j g_j logprob_j + h H is
//   dL/dx_v = 1/T (sum_j g_j [v = id_j] - p_v (sum_j g_j + h (log p_v + H))).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "rollout_ops.h"

namespace vb {

constexpr int TS_THREADS = 256;

struct Stat {
  float m, s, w;  // largest z, sum e^(z - m), sum e^(z - m) (z - m)
};
__device__ __forceinline__ Stat join(Stat a, Stat b) {
  if (!(b.s == b.s)) return b;
  if (!(a.s == a.s)) return a;
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) return {m, 0.f, 0.f};
  const float da = a.m - m, db = b.m - m, ea = expf(da), eb = expf(db);
  const float wa = ea > 0.f ? ea * (a.w + a.s * da) : 0.f, wb = eb > 0.f ? eb * (b.w + b.s * db) : 0.f;
  return {m, a.s * ea + b.s * eb, wa + wb};
}

// Order of the values as whole numbers: NaN above everything, -0 with +0.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

template <typename T>
__global__ void __launch_bounds__(TS_THREADS)
token_scores_simple_kernel(const VbScores p) {
  const long long t = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + t * p.ldx;
  __shared__ Stat red[TS_THREADS];
  __shared__ unsigned long long best[TS_THREADS];
  Stat a{-INFINITY, 0.f, 0.f};
  for (int v = threadIdx.x; v < p.V; v += TS_THREADS) {
    const float z = static_cast<float>(x[v]) * p.inv_temp;
    a = join(a, Stat{z, z - z == 0.f || z == -INFINITY ? 1.f : NAN, 0.f});
  }
  red[threadIdx.x] = a;
  __syncthreads();
  for (int o = TS_THREADS / 2; o > 0; o >>= 1) {
    if (threadIdx.x < o) red[threadIdx.x] = join(red[threadIdx.x], red[threadIdx.x + o]);
    __syncthreads();
  }
  a = red[0];
  const float lse = a.m == -INFINITY && a.s == a.s ? -INFINITY : a.m + logf(a.s);
  const auto logprob = [&](float z) { return lse == -INFINITY ? -INFINITY : z - lse; };
  if (threadIdx.x == 0) {
    p.lse[t] = lse;
    p.entropy[t] = lse == -INFINITY ? 0.f : logf(a.s) - a.w / a.s;
  }
  for (int j = threadIdx.x; j < p.K; j += TS_THREADS) {
    const long long id = p.ids[t * p.K + j];
    p.logprob[t * p.K + j] = id >= 0 && id < p.V ? logprob(static_cast<float>(x[id]) * p.inv_temp) : 0.f;
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < p.top; ++k) {  // the largest (value, lowest place) below the last one
    unsigned long long b = 0;
    for (int v = threadIdx.x; v < p.V; v += TS_THREADS) {
      const unsigned long long key = (static_cast<unsigned long long>(order_key(static_cast<float>(x[v]))) << 32) | (0xffffffffu - v);
      if (key < last && key > b) b = key;
    }
    __syncthreads();
    best[threadIdx.x] = b;
    __syncthreads();
    for (int o = TS_THREADS / 2; o > 0; o >>= 1) {
      if (threadIdx.x < o) best[threadIdx.x] = max(best[threadIdx.x], best[threadIdx.x + o]);
      __syncthreads();
    }
    last = best[0];
    if (threadIdx.x == 0) {
      const uint32_t v = 0xffffffffu - static_cast<uint32_t>(last);
      p.top_ids[t * p.top + k] = v;
      p.top_lp[t * p.top + k] = logprob(static_cast<float>(x[v]) * p.inv_temp);
    }
    __syncthreads();
  }
}

template <typename T>
__global__ void __launch_bounds__(TS_THREADS)
token_scores_bwd_simple_kernel(const VbScores p, const float* g_lp, const float* g_ent, T* dx, long long lddx, int columns) {
  const long long t = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + t * p.ldx;
  T* d = dx + t * lddx;
  const float lse = p.lse[t], H = p.entropy[t], h = g_ent != nullptr ? g_ent[t] : 0.f;
  float g = 0.f;
  for (int j = 0; j < p.K; ++j) {
    const long long id = p.ids[t * p.K + j];
    if (id >= 0 && id < p.V) g += g_lp[t * p.K + j];
  }
  const auto slope = [&](int v, float extra) {
    const float lp = static_cast<float>(x[v]) * p.inv_temp - lse;
    if (lse == -INFINITY) return 0.f;
    const float pv = expf(lp);
    return p.inv_temp * (extra - (pv == 0.f ? 0.f : pv * (g + h * (lp + H))));
  };
  for (int v = threadIdx.x; v < columns; v += TS_THREADS) {
    float extra = 0.f;
    for (int j = 0; j < p.K; ++j)
      if (p.ids[t * p.K + j] == v) extra += g_lp[t * p.K + j];
    d[v] = static_cast<T>(v < p.V ? slope(v, extra) : 0.f);
  }
}

}  // namespace vb

using namespace vb;

extern "C" int vb_token_scores(const VbScores* a, cudaStream_t s) {
  if (a->T == 0) return 0;
  if (a->type == 0) token_scores_simple_kernel<__nv_bfloat16><<<a->T, TS_THREADS, 0, s>>>(*a);
  else if (a->type == 1) token_scores_simple_kernel<__half><<<a->T, TS_THREADS, 0, s>>>(*a);
  else token_scores_simple_kernel<float><<<a->T, TS_THREADS, 0, s>>>(*a);
  verl_count_launches(1);
  return static_cast<int>(cudaGetLastError());
}

extern "C" int vb_token_scores_bwd(const VbScores* a, const float* g_lp, const float* g_ent, void* dx, long long lddx, int columns, cudaStream_t s) {
  if (a->T == 0 || columns == 0) return 0;
  if (a->type == 0) token_scores_bwd_simple_kernel<<<a->T, TS_THREADS, 0, s>>>(*a, g_lp, g_ent, static_cast<__nv_bfloat16*>(dx), lddx, columns);
  else if (a->type == 1) token_scores_bwd_simple_kernel<<<a->T, TS_THREADS, 0, s>>>(*a, g_lp, g_ent, static_cast<__half*>(dx), lddx, columns);
  else token_scores_bwd_simple_kernel<<<a->T, TS_THREADS, 0, s>>>(*a, g_lp, g_ent, static_cast<float*>(dx), lddx, columns);
  verl_count_launches(1);
  return static_cast<int>(cudaGetLastError());
}
