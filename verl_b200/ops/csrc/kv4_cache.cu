// Append to and gathering from the 4-bit cache (layout: kv4_common.cuh).
//
// A group of 32 channels of one head of one token is quantised between its least and its largest value:
//   least = f16(min), scale = f16((max - min) / 15), q = clamp(rint((x - least) / scale), 0, 15), 0 where the scale is 0.
// Every step is one correctly rounded fp32 operation, so that the codes are those of the same formula anywhere. Values beyond
// +- 7600 are taken as that: scales stay below 1024, on which the attention counts. A NaN makes the parameters of its group NaN, so that what
// is read back is NaN, as from a 16-bit cache.
//
// Both kernels move bytes: 8 channels of a token a thread (16 bytes of input, 4 of codes), four threads a group, the group's extremes by two shuffles.
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

// clamp(rint(d / s), 0, 15), 0 where s is not positive. The quotient is wanted as if it were rounded once and then to a whole number: d times the
// reciprocal is off by at most two fp32 steps (below 2^-19 where the result can matter), so that only quotients that near to a half are divided.
__device__ __forceinline__ uint32_t level(float d, float s) {
  const float q = d * __frcp_rn(s), r = rintf(q);
  const float whole = fabsf(fabsf(q - r) - 0.5f) < 1e-5f ? rintf(__fdiv_rn(d, s)) : r;
  return s > 0.f ? static_cast<uint32_t>(fminf(fmaxf(whole, 0.f), 15.f)) : 0u;
}

// A thread's place among the 2 nkv hd / 8 pieces of a token (keys or values, head, 8 channels): the same for all tokens that it meets, so that the
// divisions are made once. Tokens of a block are `step` apart for a thread; UNR of them are on their way at a time.
constexpr int KC_THREADS = 256, KC_UNR = 4;
struct Piece {
  int value, head, c, first, step;
  bool on;
  __device__ __forceinline__ Piece(int nkv, int hd) {
    const int per = hd >> 3, pieces = 2 * nkv * per;
    const int rows = max(1, KC_THREADS / pieces), e = pieces <= KC_THREADS ? threadIdx.x % pieces : blockIdx.y * KC_THREADS + threadIdx.x;
    const int row = pieces <= KC_THREADS ? threadIdx.x / pieces : 0;
    on = row < rows && e < pieces;
    const int at = on ? e : (e & 3);  // whole quads are on or off: any piece of the same place in its quad
    value = at / (nkv * per);
    head = at / per % nkv;
    c = at % per;
    step = rows;
    first = blockIdx.x * rows * KC_UNR + min(row, rows - 1);
  }
};

template <typename T2>
__global__ void __launch_bounds__(KC_THREADS)
kv4_append_kernel(const T2* __restrict__ k, const T2* __restrict__ v, long long ldk, long long ldv, const long long* __restrict__ slots,
                  uint8_t* __restrict__ pages, int T, int nkv, int hd, int bs, long long num_slots) {
  const Piece p(nkv, hd);
  const T2* src = (p.value ? v : k) + (p.head * hd + p.c * 8) / 2;
  const long long ld = (p.value ? ldv : ldk) / 2;
  const long long page_bytes = kv4_page_bytes(bs, hd);
  uint8_t* codes_at = pages + p.head * page_bytes + kv4_codes_at(bs, hd, p.value) + p.c * 4;
  uint8_t* params_at = pages + p.head * page_bytes + kv4_params_at(bs, hd, p.value) + (p.c >> 2) * 4;
  uint4 raw[KC_UNR];
  long long slot[KC_UNR];
#pragma unroll
  for (int u = 0; u < KC_UNR; ++u) {
    const int t = p.first + u * p.step;
    slot[u] = -1;
    raw[u] = make_uint4(0u, 0u, 0u, 0u);
    if (t < T && p.on) {
      slot[u] = slots[t];
      raw[u] = *reinterpret_cast<const uint4*>(src + t * ld);
    }
  }
#pragma unroll
  for (int u = 0; u < KC_UNR; ++u) {
    const T2* r2 = reinterpret_cast<const T2*>(&raw[u]);
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
    for (int j = 0; j < 8; ++j) codes |= level(__fsub_rn(x[j], m), s) << (4 * j);
    if (slot[u] < 0 || slot[u] >= num_slots) continue;
    const int blk = static_cast<int>(slot[u]) / bs, off = static_cast<int>(slot[u]) - blk * bs;
    const long long page = static_cast<long long>(blk) * nkv * page_bytes;
    *reinterpret_cast<uint32_t*>(codes_at + page + off * (hd / 2)) = codes;
    if ((p.c & 3) == 0) *reinterpret_cast<__half2*>(params_at + page + off * (hd / KV4_GROUP) * 4) = __halves2half2(scale, least);
  }
}

template <typename T2>
__global__ void __launch_bounds__(KC_THREADS)
kv4_gather_kernel(const uint8_t* __restrict__ pages, const long long* __restrict__ slots, T2* __restrict__ k, T2* __restrict__ v, int T, int nkv, int hd,
                  int bs, long long num_slots) {
  const Piece p(nkv, hd);
  if (!p.on) return;
  const long long page_bytes = kv4_page_bytes(bs, hd);
  const uint8_t* codes_at = pages + p.head * page_bytes + kv4_codes_at(bs, hd, p.value) + p.c * 4;
  const uint8_t* params_at = pages + p.head * page_bytes + kv4_params_at(bs, hd, p.value) + (p.c >> 2) * 4;
  T2* dst = (p.value ? v : k) + (p.head * hd + p.c * 8) / 2;
  uint32_t codes[KC_UNR], par[KC_UNR];
#pragma unroll
  for (int u = 0; u < KC_UNR; ++u) {
    const int t = p.first + u * p.step;
    const long long slot = t < T ? slots[t] : -1;
    codes[u] = par[u] = 0u;  // zeros for a token without a slot
    if (slot >= 0 && slot < num_slots) {
      const int blk = static_cast<int>(slot) / bs, off = static_cast<int>(slot) - blk * bs;
      const long long page = static_cast<long long>(blk) * nkv * page_bytes;
      codes[u] = *reinterpret_cast<const uint32_t*>(codes_at + page + off * (hd / 2));
      par[u] = *reinterpret_cast<const uint32_t*>(params_at + page + off * (hd / KV4_GROUP) * 4);
    }
  }
#pragma unroll
  for (int u = 0; u < KC_UNR; ++u) {
    const int t = p.first + u * p.step;
    if (t >= T) break;
    const __half2 sm = *reinterpret_cast<const __half2*>(&par[u]);
    const float s = __low2float(sm), m = __high2float(sm);
    uint4 out;
    T2* o2 = reinterpret_cast<T2*>(&out);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      o2[j] = kv4_pack<T2>(fmaf(static_cast<float>((codes[u] >> (8 * j)) & 15u), s, m), fmaf(static_cast<float>((codes[u] >> (8 * j + 4)) & 15u), s, m));
    *reinterpret_cast<uint4*>(dst + static_cast<long long>(t) * nkv * hd / 2) = out;
  }
}

static dim3 kc_grid(int T, int nkv, int hd) {
  const int pieces = 2 * nkv * (hd >> 3), rows = max(1, KC_THREADS / pieces);
  return dim3((T + rows * KC_UNR - 1) / (rows * KC_UNR), pieces <= KC_THREADS ? 1 : (pieces + KC_THREADS - 1) / KC_THREADS);
}

}  // namespace vb

using namespace vb;

// Rows of k and v start on 16-byte boundaries (ldk, ldv elements apart), heads are hd apart, hd a multiple of 32.
extern "C" int vb_kv4_append(int type, const void* k, const void* v, long long ldk, long long ldv, const long long* slots, void* pages, int T, int nkv,
                             int hd, int block_size, long long num_slots, cudaStream_t s) {
  if (hd % KV4_GROUP || ldk % 8 || ldv % 8 || num_slots > 0x7fffffffLL) return -2;
  if (T == 0 || nkv == 0) return 0;
  const dim3 grid = kc_grid(T, nkv, hd);
  uint8_t* out = static_cast<uint8_t*>(pages);
  if (type == 0)
    kv4_append_kernel<<<grid, KC_THREADS, 0, s>>>(static_cast<const __nv_bfloat162*>(k), static_cast<const __nv_bfloat162*>(v), ldk, ldv, slots, out, T, nkv, hd,
                                                 block_size, num_slots);
  else
    kv4_append_kernel<<<grid, KC_THREADS, 0, s>>>(static_cast<const __half2*>(k), static_cast<const __half2*>(v), ldk, ldv, slots, out, T, nkv, hd, block_size,
                                                 num_slots);
  return static_cast<int>(cudaGetLastError());
}

extern "C" int vb_kv4_gather(int type, const void* pages, const long long* slots, void* k, void* v, int T, int nkv, int hd, int block_size,
                             long long num_slots, cudaStream_t s) {
  if (hd % KV4_GROUP || num_slots > 0x7fffffffLL) return -2;
  if (T == 0 || nkv == 0) return 0;
  const dim3 grid = kc_grid(T, nkv, hd);
  const uint8_t* in = static_cast<const uint8_t*>(pages);
  if (type == 0)
    kv4_gather_kernel<<<grid, KC_THREADS, 0, s>>>(in, slots, static_cast<__nv_bfloat162*>(k), static_cast<__nv_bfloat162*>(v), T, nkv, hd, block_size, num_slots);
  else
    kv4_gather_kernel<<<grid, KC_THREADS, 0, s>>>(in, slots, static_cast<__half2*>(k), static_cast<__half2*>(v), T, nkv, hd, block_size, num_slots);
  return static_cast<int>(cudaGetLastError());
}
