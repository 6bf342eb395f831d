// C launchers of the page bookkeeping, the 4-bit cache and the scores of logits.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

extern "C" {
void verl_count_launches(long long n);  // bindings.cpp
// page_maps.cu
int vb_decode_slot_map(const int* table, long long ldt, int width, const int* pos, const int* ctx, const bool* active, int S, int block_size,
                       long long* slots, int* ctx_out, int* plan, cudaStream_t s);
int vb_extend_block_tables(int* table, long long ldt, int S, int width, const int* rows, const int* have, const int* lengths, int B, const int* pool,
                           int pool_size, int block_size, int* used, cudaStream_t s);
int vb_build_slot_map(const int* table, long long ldt, int S, int width, const int* rows, const int* starts, const int* ends, int B, int block_size,
                      int total, int* cu, int* positions, long long* slots, cudaStream_t s);
// kv4_cache.cu: type 0 = bf16, 1 = fp16
int vb_kv4_append(int type, const void* k, const void* v, long long ldk, long long ldv, const long long* slots, void* pages, int T, int nkv, int hd,
                  int block_size, long long num_slots, cudaStream_t s);
int vb_kv4_gather(int type, const void* pages, const long long* slots, void* k, void* v, int T, int nkv, int hd, int block_size,
                  long long num_slots, cudaStream_t s);
// kv4_decode.cu
struct VbKv4Decode {
  const void* q; long long ldq;        // [B, nh, hd], rows ldq apart
  const uint8_t* pages; int num_blocks, block_size;
  const int* table; int width; long long ldt;
  const int* ctx; const int* plan;     // plan null: one is written to plan_ws
  int* plan_ws;
  void* out;                           // [B, nh, hd] contiguous
  float* part;                         // scratch of vb_kv4_decode_scratch() floats
  int B, nh, nkv, hd, type;
  float scale;
};
long long vb_kv4_decode_scratch(int B, int nh, int nkv, int hd);
int vb_kv4_decode(const VbKv4Decode* a, cudaStream_t s);
// token_scores.cu: type 0 = bf16, 1 = fp16, 2 = fp32
struct VbScores {
  const void* x; long long ldx; int type; int T, V;    // V: columns that count
  float inv_temp;
  const long long* ids; int K;                         // [T, K]
  int top;
  float* logprob; float* entropy; float* lse;
  long long* top_ids; float* top_lp;                   // [T, top]
  float* stat;                                         // [T, 4], what the gradient wants of a row; forward: may be null
};
int vb_token_scores(const VbScores* a, cudaStream_t s);
int vb_token_scores_bwd(const VbScores* a, const float* g_lp, const float* g_ent, void* dx, long long lddx, int columns, cudaStream_t s);
}
