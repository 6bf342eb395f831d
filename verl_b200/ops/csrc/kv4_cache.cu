// Append to and gathering from the 4-bit cache (layout: kv4_common.cuh).
//
// A group of 32 channels of one head of one token is quantised between its least and its largest value:
//   least = f16(min), scale = f16((max - min) / 15), q = clamp(rint((x - least) / scale), 0, 15), 0 where the scale is 0.
// Every step is one correctly rounded fp32 operation, so that the codes are those of the same formula anywhere. Values beyond
// +- 7600 are taken as that: scales stay below 1024, on which the attention counts. A NaN makes the parameters of its group NaN, so that what
// is read back is NaN, as from a 16-bit cache.
//
// Both kernels move bytes: 8 channels a thread (16 bytes of input, 4 of codes), four threads a group, the group's extremes by two shuffles.
#include "kv4_common.cuh"
#include "rollout_ops.h"

namespace vb {

// minimum and maximum that keep a NaN, unlike fminf and fmaxf
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <typename T2>
__global__ void __launch_bounds__(256)
kv4_append_kernel(const T2* __restrict__ k, const T2* __restrict__ v, long long ldk, long long ldv, const long long* __restrict__ slots,
                  uint8_t* __restrict__ pages, long long items, int nkv, int hd, int bs, long long num_slots) {
  const int per = hd >> 3;  // threads of a head
  const long long item = blockIdx.x * 256LL + threadIdx.x;
  const bool in = item < items;
  const long long i = in ? item : items - 1;  // whole warps take part in the shuffles
  const int c = static_cast<int>(i % per);
  const long long th = i / per;
  const int h = static_cast<int>(th % nkv);
  const long long tv = th / nkv;
  const int value = static_cast<int>(tv & 1);
  const long long t = tv >> 1;
  const long long slot = slots[t];
  const T2* src = (value ? v + t * ldv / 2 : k + t * ldk / 2) + (h * hd + c * 8) / 2;
  const uint4 raw = *reinterpret_cast<const uint4*>(src);
  const T2* r2 = reinterpret_cast<const T2*>(&raw);
  float x[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = kv4_pair(r2[j]);
    x[2 * j] = f.x;
    x[2 * j + 1] = f.y;
  }
  float lo = KV4_LIMIT, hi = -KV4_LIMIT;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    x[j] = min_nan(max_nan(x[j], -KV4_LIMIT), KV4_LIMIT);
    lo = min_nan(lo, x[j]);
    hi = max_nan(hi, x[j]);
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  const __half scale = __float2half_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.f)), least = __float2half_rn(lo);
  const float s = __half2float(scale), m = __half2float(least);
  uint32_t codes = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float q = s > 0.f ? rintf(__fdiv_rn(__fsub_rn(x[j], m), s)) : 0.f;
    codes |= static_cast<uint32_t>(fminf(fmaxf(q, 0.f), 15.f)) << (4 * j);
  }
  if (!in || slot < 0 || slot >= num_slots) return;
  const int off = static_cast<int>(slot % bs);
  uint8_t* page = pages + (slot / bs * nkv + h) * kv4_page_bytes(bs, hd);
  *reinterpret_cast<uint32_t*>(page + kv4_codes_at(bs, hd, value) + off * (hd / 2) + c * 4) = codes;
  if ((c & 3) == 0)
    *reinterpret_cast<__half2*>(page + kv4_params_at(bs, hd, value) + (off * (hd / KV4_GROUP) + (c >> 2)) * 4) = __halves2half2(scale, least);
}

template <typename T2>
__global__ void __launch_bounds__(256)
kv4_gather_kernel(const uint8_t* __restrict__ pages, const long long* __restrict__ slots, T2* __restrict__ k, T2* __restrict__ v, long long items,
                  int nkv, int hd, int bs, long long num_slots) {
  const int per = hd >> 3;
  const long long i = blockIdx.x * 256LL + threadIdx.x;
  if (i >= items) return;
  const int c = static_cast<int>(i % per);
  const long long th = i / per;
  const int h = static_cast<int>(th % nkv);
  const long long tv = th / nkv;
  const int value = static_cast<int>(tv & 1);
  const long long t = tv >> 1, slot = slots[t];
  uint4 out = make_uint4(0u, 0u, 0u, 0u);
  if (slot >= 0 && slot < num_slots) {
    const int off = static_cast<int>(slot % bs);
    const uint8_t* page = pages + (slot / bs * nkv + h) * kv4_page_bytes(bs, hd);
    const uint32_t codes = *reinterpret_cast<const uint32_t*>(page + kv4_codes_at(bs, hd, value) + off * (hd / 2) + c * 4);
    const __half2 par = *reinterpret_cast<const __half2*>(page + kv4_params_at(bs, hd, value) + (off * (hd / KV4_GROUP) + (c >> 2)) * 4);
    const float s = __low2float(par), m = __high2float(par);
    T2* o2 = reinterpret_cast<T2*>(&out);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      o2[j] = kv4_pack<T2>(fmaf(static_cast<float>((codes >> (8 * j)) & 15u), s, m), fmaf(static_cast<float>((codes >> (8 * j + 4)) & 15u), s, m));
  }
  *reinterpret_cast<uint4*>((value ? v : k) + ((t * nkv + h) * hd + c * 8) / 2) = out;
}

}  // namespace vb

using namespace vb;

// Rows of k and v start on 16-byte boundaries (ldk, ldv elements apart), heads are hd apart, hd a multiple of 32.
extern "C" int vb_kv4_append(int type, const void* k, const void* v, long long ldk, long long ldv, const long long* slots, void* pages, int T, int nkv,
                             int hd, int block_size, long long num_slots, cudaStream_t s) {
  if (hd % KV4_GROUP || ldk % 8 || ldv % 8) return -2;
  const long long items = 2LL * T * nkv * (hd >> 3), blocks = (items + 255) / 256;
  if (items == 0) return 0;
  if (blocks > 0x7fffffffLL) return -3;
  if (type == 0)
    kv4_append_kernel<<<static_cast<int>(blocks), 256, 0, s>>>(static_cast<const __nv_bfloat162*>(k), static_cast<const __nv_bfloat162*>(v), ldk, ldv, slots,
                                                              static_cast<uint8_t*>(pages), items, nkv, hd, block_size, num_slots);
  else
    kv4_append_kernel<<<static_cast<int>(blocks), 256, 0, s>>>(static_cast<const __half2*>(k), static_cast<const __half2*>(v), ldk, ldv, slots,
                                                              static_cast<uint8_t*>(pages), items, nkv, hd, block_size, num_slots);
  return static_cast<int>(cudaGetLastError());
}

extern "C" int vb_kv4_gather(int type, const void* pages, const long long* slots, void* k, void* v, int T, int nkv, int hd, int block_size,
                             long long num_slots, cudaStream_t s) {
  if (hd % KV4_GROUP) return -2;
  const long long items = 2LL * T * nkv * (hd >> 3), blocks = (items + 255) / 256;
  if (items == 0) return 0;
  if (blocks > 0x7fffffffLL) return -3;
  if (type == 0)
    kv4_gather_kernel<<<static_cast<int>(blocks), 256, 0, s>>>(static_cast<const uint8_t*>(pages), slots, static_cast<__nv_bfloat162*>(k),
                                                              static_cast<__nv_bfloat162*>(v), items, nkv, hd, block_size, num_slots);
  else
    kv4_gather_kernel<<<static_cast<int>(blocks), 256, 0, s>>>(static_cast<const uint8_t*>(pages), slots, static_cast<__half2*>(k),
                                                              static_cast<__half2*>(v), items, nkv, hd, block_size, num_slots);
  return static_cast<int>(cudaGetLastError());
}
