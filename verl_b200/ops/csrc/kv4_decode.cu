// Attention of one query token per sequence over the 4-bit cache (layout: kv4_common.cuh).
#include <math.h>

#include "kv4_common.cuh"
#include "rollout_ops.h"

namespace vb {

constexpr int KD_MAXG = 16;

template <int HD, typename T>
__global__ void __launch_bounds__(128)
kv4_decode_simple_kernel(const VbKv4Decode p) {
  constexpr int CH = HD / 32;
  const int kvh = blockIdx.x, b = blockIdx.y, G = p.nh / p.nkv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int len = static_cast<int>(min(static_cast<long long>(max(p.ctx[b], 0)), static_cast<long long>(p.width) * p.block_size));
  __shared__ float qs[KD_MAXG][HD];
  __shared__ float os[4][HD], ms[4], ls[4];
  for (int i = threadIdx.x; i < G * HD; i += 128)
    qs[i / HD][i % HD] = static_cast<float>(static_cast<const T*>(p.q)[b * p.ldq + static_cast<long long>(kvh * G) * HD + i]);
  __syncthreads();
  for (int g = 0; g < G; ++g) {
    float m = -INFINITY, l = 0.f, o[CH] = {};
    for (int t = warp; t < len; t += 4) {
      const int blk = p.table[b * p.ldt + t / p.block_size], off = t % p.block_size;
      if (blk < 0 || blk >= p.num_blocks) continue;
      const uint8_t* page = p.pages + (static_cast<long long>(blk) * p.nkv + kvh) * kv4_page_bytes(p.block_size, HD);
      float x[2][CH];
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          const int d = lane * CH + c;
          const uint8_t byte = page[kv4_codes_at(p.block_size, HD, w) + off * (HD / 2) + d / 2];
          const __half2 par = *reinterpret_cast<const __half2*>(page + kv4_params_at(p.block_size, HD, w) + (off * (HD / KV4_GROUP) + d / KV4_GROUP) * 4);
          x[w][c] = fmaf(static_cast<float>(d & 1 ? byte >> 4 : byte & 15), __low2float(par), __high2float(par));
        }
      float s = 0.f;
#pragma unroll
      for (int c = 0; c < CH; ++c) s += x[0][c] * qs[g][lane * CH + c];
#pragma unroll
      for (int k = 16; k > 0; k >>= 1) s += __shfl_xor_sync(0xffffffffu, s, k);
      s *= p.scale;
      const float mn = fmaxf(m, s), e = expf(s - mn), a = expf(m - mn);
      l = l * a + e;
      m = mn;
#pragma unroll
      for (int c = 0; c < CH; ++c) o[c] = o[c] * a + e * x[1][c];
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) os[warp][lane * CH + c] = o[c];
    if (lane == 0) { ms[warp] = m; ls[warp] = l; }
    __syncthreads();
    if (threadIdx.x < HD) {
      const float M = fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3]));
      float L = 0.f, acc = 0.f;
      for (int w = 0; w < 4; ++w) {
        const float f = ls[w] > 0.f || ls[w] != ls[w] ? expf(ms[w] - M) : 0.f;
        L += ls[w] * f;
        acc += os[w][threadIdx.x] * f;
      }
      static_cast<T*>(p.out)[(static_cast<long long>(b) * p.nh + kvh * G + g) * HD + threadIdx.x] = static_cast<T>(L == 0.f ? 0.f : acc / L);
    }
    __syncthreads();
  }
}

}  // namespace vb

using namespace vb;

extern "C" long long vb_kv4_decode_scratch(int B, int nh, int nkv, int hd) { return 0; }
extern "C" int vb_kv4_status() { return 0; }

extern "C" int vb_kv4_decode(const VbKv4Decode* a, cudaStream_t s) {
  const int G = a->nh / a->nkv;
  if (a->B == 0) return 0;
  if ((a->hd != 64 && a->hd != 128) || G * a->nkv != a->nh || G > KD_MAXG || a->B > 65535) return -2;
  const dim3 grid(a->nkv, a->B);
  if (a->hd == 128) {
    if (a->type == 0) kv4_decode_simple_kernel<128, __nv_bfloat16><<<grid, 128, 0, s>>>(*a);
    else kv4_decode_simple_kernel<128, __half><<<grid, 128, 0, s>>>(*a);
  } else {
    if (a->type == 0) kv4_decode_simple_kernel<64, __nv_bfloat16><<<grid, 128, 0, s>>>(*a);
    else kv4_decode_simple_kernel<64, __half><<<grid, 128, 0, s>>>(*a);
  }
  verl_count_launches(1);
  return static_cast<int>(cudaGetLastError());
}
