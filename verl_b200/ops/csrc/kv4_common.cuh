// Layout of the 4-bit cache. A page holds `block` tokens of one KV head as one run of bytes:
//   codes of the keys   [block][hd / 2]        channel 2 j of a token in the low half of byte j, channel 2 j + 1 in the high half
//   codes of the values [block][hd / 2]
//   parameters of the keys   [block][hd / 32]  (scale, least) in fp16 for each group of 32 channels
//   parameters of the values [block][hd / 32]
// and a code q stands for q * scale + least. The pages of a block follow one another by head: [blocks][heads][page]. A tile of 64 tokens of
// one head is thus a few contiguous runs (one, for blocks of 64), which a bulk copy fetches without a tensor map; 0.625 bytes an element.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace vb {

constexpr int KV4_GROUP = 32;
constexpr float KV4_LIMIT = 7600.f;  // largest magnitude that is kept: scales are at most 15200 / 15

__host__ __device__ constexpr long long kv4_page_bytes(int block, int hd) { return static_cast<long long>(block) * hd + block * hd / 4; }
__host__ __device__ constexpr int kv4_codes_at(int block, int hd, int value) { return value ? block * hd / 2 : 0; }
__host__ __device__ constexpr int kv4_params_at(int block, int hd, int value) { return block * hd + (value ? block * hd / 8 : 0); }

__device__ __forceinline__ float2 kv4_pair(__nv_bfloat162 v) { return __bfloat1622float2(v); }
__device__ __forceinline__ float2 kv4_pair(__half2 v) { return __half22float2(v); }
template <typename T2> __device__ __forceinline__ T2 kv4_pack(float a, float b);
template <> __device__ __forceinline__ __nv_bfloat162 kv4_pack<__nv_bfloat162>(float a, float b) { return __floats2bfloat162_rn(a, b); }
template <> __device__ __forceinline__ __half2 kv4_pack<__half2>(float a, float b) { return __floats2half2_rn(a, b); }

}  // namespace vb
