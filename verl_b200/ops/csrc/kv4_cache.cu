// Append to and gathering from the 4-bit cache (layout: kv4_common.cuh).
//
// A group of 32 channels of one head of one token is quantised between its least and its largest value:
//   least = f16(min), scale = f16((max - min) / 15), q = clamp(rint((x - least) / scale), 0, 15), 0 where the scale is 0.
// Every step is one correctly rounded fp32 operation, so that the codes are those of the same formula anywhere. Values beyond
// +- 7600 are taken as that: scales stay below 1024, on which the attention counts. A NaN makes the parameters of its group NaN, so that what
// is read back is NaN, as from a 16-bit cache.
//
// Both kernels move bytes: 8 channels of a token a thread (16 bytes of input, 4 of codes), four threads a group, the group's extremes by two shuffles.
// 16384 tokens of 8 heads of 128 channels: append 39 us for 88 MB (2.3 TB/s), gather 23 us for 88 MB (3.8 TB/s), both bound by the instructions
// that they issue (about 200 and 110 for the 8 channels of a thread, a slot's address and a group's parameters among them; 0.74 and 0.66 a cycle and
// scheduler). With a block for every few tokens append took 53 us and gather 30: each thread works out its place by divisions. A decode step's few tokens
// cost a launch, 6 us.
#include "kv4_common.cuh"
#include "rollout_ops.h"

namespace vb {

int num_sms();

// minimum and maximum that keep a NaN, unlike fminf and fmaxf; of three values as well
__device__ __forceinline__ float min_nan(float a, float b, float c) {
  float r;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
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

// The eight codes clamp(rint((x - m) / s), 0, 15) of a thread, four bits each; 0 where s is not positive. The quotient is wanted as if it were rounded
// once and then to a whole number. A fifteenth of it, u, from the approximate reciprocal, is at most five fp32 roundings off and is held in
// [0, 1] by the multiplication itself, so that 15 u is off by less than 15 * 2^-21.6 = 5e-6: only where one comes within 1e-5 of a half all eight
// are divided. Adding 1.5 * 2^23 rounds to a whole number, halves to the even one. Four codes are put together as a number below 2^16 behind 2^23.
__device__ __forceinline__ uint32_t kv4_codes(const float (&x)[8], float s, float m) {
  constexpr float ROUND = 12582912.f, WHOLE = 8388608.f;
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
  inv = __fmul_rn(inv, 1.f / 15.f);
  float four[2] = {WHOLE, WHOLE};
  bool near = false;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float u = __saturatef(__fmul_rn(__fsub_rn(x[j], m), inv)), q = __fsub_rn(__fmaf_rn(u, 15.f, ROUND), ROUND);
    near |= fabsf(__fmaf_rn(u, 15.f, -q)) > 0.5f - 1e-5f;
    four[j / 4] = __fmaf_rn(q, static_cast<float>(1 << (4 * (j % 4))), four[j / 4]);
  }
  if (near) {
    four[0] = four[1] = WHOLE;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float q = __fsub_rn(__fadd_rn(fminf(fmaxf(__fdiv_rn(__fsub_rn(x[j], m), s), 0.f), 15.f), ROUND), ROUND);
      four[j / 4] = __fmaf_rn(q, static_cast<float>(1 << (4 * (j % 4))), four[j / 4]);
    }
  }
  return s > 0.f ? __byte_perm(__float_as_uint(four[0]), __float_as_uint(four[1]), 0x5410) : 0u;
}

// A thread's place among the 2 nkv hd / 8 pieces of a token (keys or values, head, 8 channels): the same for all tokens that it meets, so that the
// divisions are made once. Tokens of a block are `step` apart for a thread, KC_UNR of them are on their way at a time, `turns` times.
constexpr int KC_THREADS = 256, KC_UNR = 4;
struct Piece {
  int value, head, c, first, step, row;
  bool on;
  __device__ __forceinline__ Piece(int nkv, int hd, int turns) {
    const int per = hd >> 3, pieces = 2 * nkv * per;
    const int rows = max(1, KC_THREADS / pieces), e = pieces <= KC_THREADS ? threadIdx.x % pieces : blockIdx.y * KC_THREADS + threadIdx.x;
    const int mine = pieces <= KC_THREADS ? threadIdx.x / pieces : 0;
    on = mine < rows && e < pieces;
    row = min(mine, rows - 1);
    const int at = on ? e : (e & 3);  // whole quads are on or off: any piece of the same place in its quad
    value = at / (nkv * per);
    head = at / per % nkv;
    c = at % per;
    step = rows;
    first = blockIdx.x * rows * KC_UNR * turns + row;
  }
};

template <typename T2>
__global__ void __launch_bounds__(KC_THREADS)
kv4_append_kernel(const T2* __restrict__ k, const T2* __restrict__ v, long long ldk, long long ldv, const long long* __restrict__ slots,
                  uint8_t* __restrict__ pages, int T, int nkv, int hd, int bs, int shift, long long num_slots, int turns) {
  const Piece p(nkv, hd, turns);
  const T2* src = (p.value ? v : k) + (p.head * hd + p.c * 8) / 2;
  const long long ld = (p.value ? ldv : ldk) / 2;
  const long long block_bytes = nkv * kv4_page_bytes(bs, hd);
  uint8_t* codes_at = pages + p.head * kv4_page_bytes(bs, hd) + kv4_codes_at(bs, hd, p.value) + p.c * 4;
  uint8_t* params_at = pages + p.head * kv4_page_bytes(bs, hd) + kv4_params_at(bs, hd, p.value) + (p.c >> 2) * 4;
  for (int turn = 0; turn < turns; ++turn) {
    const int t0 = p.first + turn * KC_UNR * p.step;
    if (t0 - p.row >= T) break;  // the same for the whole block: its threads take part in the shuffles
    uint4 raw[KC_UNR];
    long long slot[KC_UNR];
#pragma unroll
    for (int u = 0; u < KC_UNR; ++u) {
      const int t = t0 + u * p.step;
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
      float lo = min_nan(min_nan(x[0], x[1], x[2]), min_nan(x[3], x[4], x[5]), min_nan(x[6], x[7]));
      float hi = max_nan(max_nan(x[0], x[1], x[2]), max_nan(x[3], x[4], x[5]), max_nan(x[6], x[7]));
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      }
      lo = min_nan(max_nan(lo, -KV4_LIMIT), KV4_LIMIT);  // values beyond the limit end in the first or the last code
      hi = min_nan(max_nan(hi, -KV4_LIMIT), KV4_LIMIT);
      const __half scale = __float2half_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.f)), least = __float2half_rn(lo);
      const uint32_t codes = kv4_codes(x, __half2float(scale), __half2float(least));
      if (slot[u] < 0 || slot[u] >= num_slots) continue;
      const int at = static_cast<int>(slot[u]), blk = shift >= 0 ? at >> shift : at / bs, off = at - blk * bs;
      const long long block = blk * block_bytes;
      *reinterpret_cast<uint32_t*>(codes_at + block + off * (hd / 2)) = codes;
      if ((p.c & 3) == 0) *reinterpret_cast<__half2*>(params_at + block + off * (hd / KV4_GROUP) * 4) = __halves2half2(scale, least);
    }
  }
}

template <typename T2>
__global__ void __launch_bounds__(KC_THREADS)
kv4_gather_kernel(const uint8_t* __restrict__ pages, const long long* __restrict__ slots, T2* __restrict__ k, T2* __restrict__ v, int T, int nkv, int hd,
                  int bs, int shift, long long num_slots, int turns) {
  const Piece p(nkv, hd, turns);
  if (!p.on) return;
  const long long block_bytes = nkv * kv4_page_bytes(bs, hd);
  const uint8_t* codes_at = pages + p.head * kv4_page_bytes(bs, hd) + kv4_codes_at(bs, hd, p.value) + p.c * 4;
  const uint8_t* params_at = pages + p.head * kv4_page_bytes(bs, hd) + kv4_params_at(bs, hd, p.value) + (p.c >> 2) * 4;
  T2* dst = (p.value ? v : k) + (p.head * hd + p.c * 8) / 2;
  const long long ld = static_cast<long long>(nkv) * hd / 2;
  for (int turn = 0; turn < turns; ++turn) {
    const int t0 = p.first + turn * KC_UNR * p.step;
    if (t0 >= T) return;
    uint32_t codes[KC_UNR], par[KC_UNR];
#pragma unroll
    for (int u = 0; u < KC_UNR; ++u) {
      const int t = t0 + u * p.step;
      const long long slot = t < T ? slots[t] : -1;
      codes[u] = par[u] = 0u;  // zeros for a token without a slot
      if (slot >= 0 && slot < num_slots) {
        const int at = static_cast<int>(slot), blk = shift >= 0 ? at >> shift : at / bs, off = at - blk * bs;
        const long long block = blk * block_bytes;
        codes[u] = *reinterpret_cast<const uint32_t*>(codes_at + block + off * (hd / 2));
        par[u] = *reinterpret_cast<const uint32_t*>(params_at + block + off * (hd / KV4_GROUP) * 4);
      }
    }
#pragma unroll
    for (int u = 0; u < KC_UNR; ++u) {
      const int t = t0 + u * p.step;
      if (t >= T) return;
      const __half2 sm = *reinterpret_cast<const __half2*>(&par[u]);
      const float s = __low2float(sm), m = __high2float(sm);
      uint4 out;
      T2* o2 = reinterpret_cast<T2*>(&out);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        o2[j] = kv4_pack<T2>(fmaf(static_cast<float>((codes[u] >> (8 * j)) & 15u), s, m), fmaf(static_cast<float>((codes[u] >> (8 * j + 4)) & 15u), s, m));
      *reinterpret_cast<uint4*>(dst + t * ld) = out;
    }
  }
}

struct KcLaunch {
  dim3 grid;
  int turns, shift;
  KcLaunch(int T, int nkv, int hd, int bs) {
    const int pieces = 2 * nkv * (hd >> 3), rows = max(1, KC_THREADS / pieces) * KC_UNR, across = pieces <= KC_THREADS ? 1 : (pieces + KC_THREADS - 1) / KC_THREADS;
    const long long blocks = (static_cast<long long>(T) + rows - 1) / rows;
    turns = static_cast<int>(min(8LL, max(1LL, blocks * across / (8LL * num_sms()))));  // more than a wave: fewer blocks, which divide less
    grid = dim3(static_cast<unsigned>((blocks + turns - 1) / turns), across);
    shift = (bs & (bs - 1)) == 0 ? __builtin_ctz(static_cast<unsigned>(bs)) : -1;
  }
};

}  // namespace vb

using namespace vb;

// Rows of k and v start on 16-byte boundaries (ldk, ldv elements apart), heads are hd apart, hd a multiple of 32.
extern "C" int vb_kv4_append(int type, const void* k, const void* v, long long ldk, long long ldv, const long long* slots, void* pages, int T, int nkv,
                             int hd, int block_size, long long num_slots, cudaStream_t s) {
  if (hd % KV4_GROUP || ldk % 8 || ldv % 8 || num_slots > 0x7fffffffLL) return -2;
  if (T == 0 || nkv == 0) return 0;
  const KcLaunch l(T, nkv, hd, block_size);
  uint8_t* out = static_cast<uint8_t*>(pages);
  if (type == 0)
    kv4_append_kernel<<<l.grid, KC_THREADS, 0, s>>>(static_cast<const __nv_bfloat162*>(k), static_cast<const __nv_bfloat162*>(v), ldk, ldv, slots, out, T, nkv, hd,
                                                 block_size, l.shift, num_slots, l.turns);
  else
    kv4_append_kernel<<<l.grid, KC_THREADS, 0, s>>>(static_cast<const __half2*>(k), static_cast<const __half2*>(v), ldk, ldv, slots, out, T, nkv, hd, block_size,
                                                 l.shift, num_slots, l.turns);
  return static_cast<int>(cudaGetLastError());
}

extern "C" int vb_kv4_gather(int type, const void* pages, const long long* slots, void* k, void* v, int T, int nkv, int hd, int block_size,
                             long long num_slots, cudaStream_t s) {
  if (hd % KV4_GROUP || num_slots > 0x7fffffffLL) return -2;
  if (T == 0 || nkv == 0) return 0;
  const KcLaunch l(T, nkv, hd, block_size);
  const uint8_t* in = static_cast<const uint8_t*>(pages);
  if (type == 0)
    kv4_gather_kernel<<<l.grid, KC_THREADS, 0, s>>>(in, slots, static_cast<__nv_bfloat162*>(k), static_cast<__nv_bfloat162*>(v), T, nkv, hd, block_size, l.shift,
                                                 num_slots, l.turns);
  else
    kv4_gather_kernel<<<l.grid, KC_THREADS, 0, s>>>(in, slots, static_cast<__half2*>(k), static_cast<__half2*>(v), T, nkv, hd, block_size, l.shift,
                                                 num_slots, l.turns);
  return static_cast<int>(cudaGetLastError());
}
