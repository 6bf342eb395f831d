// Page bookkeeping of the rollout engine on the device: block tables grown from a list of free pages, the cache slots and positions of the
// tokens of a prefill batch, and the slots, contexts and attention plan of a decode step, all from the lengths of the requests.
//
// need_i = ceil(length_i / block), new_i = max(need_i - have_i, 0), and sequence i takes pool[sum of new_j over j < i ...]; token t of a packed
// batch belongs to the sequence i with cu_i <= t < cu_{i+1} and lies at position starts_i + t - cu_i. Both are exclusive sums over the batch,
// which every block of a launch takes for itself (a batch is mostly some hundred sequences, read from L2): one launch, no block waits
// for another. Slots of more than 8192 sequences take a launch more, for the sums. Nothing out of range is read or written whatever the tensors hold: a token whose row, position or page is none gets slot -1.
#include <cuda_runtime.h>
#include <stdint.h>

#include "rollout_ops.h"

namespace vb {

constexpr int PM_THREADS = 1024;

// Sums of counts, and sums of which no more than `most` is wanted or held: two of those fit 32 bits without a sign.
struct Sum {
  __device__ __forceinline__ int operator()(int a, int b) const { return a + b; }
};
struct SumUpTo {
  int most;
  __device__ __forceinline__ int operator()(int a, int b) const {
    return static_cast<int>(min(static_cast<unsigned>(a) + static_cast<unsigned>(b), static_cast<unsigned>(most)));
  }
};

// inclusive sum over the block; `red` holds 32 ints. Every thread also gets the block's total.
template <typename Add = Sum>
__device__ __forceinline__ int pm_scan(int v, int* red, int& total, const Add& add = Add()) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v = add(v, u);
  }
  __syncthreads();
  if (lane == 31) red[warp] = v;
  __syncthreads();
  int w = lane < nw ? red[lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w = add(w, u);
  }
  total = __shfl_sync(0xffffffffu, w, 31);
  const int before = __shfl_sync(0xffffffffu, w, max(warp - 1, 0));
  return add(v, warp > 0 ? before : 0);
}

// One block over all slots. The plan counts the 64-token pieces of the contexts in front of every sequence: what the attention over the
// 4-bit cache deals to its CTAs.
__global__ void __launch_bounds__(PM_THREADS)
decode_slot_map_kernel(const int* __restrict__ table, long long ldt, int width, const int* __restrict__ pos, const int* __restrict__ ctx,
                       const bool* __restrict__ active, int S, int bs, long long* __restrict__ slots, int* __restrict__ ctx_out,
                       int* __restrict__ plan) {
  __shared__ int red[32];
  int carry = 0;
  if (threadIdx.x == 0) plan[0] = 0;
  for (int base = 0; base < S; base += blockDim.x) {
    const int s = base + threadIdx.x;
    int n = 0;
    if (s < S) {
      const bool on = active[s];
      const int p = pos[s], c = on ? max(ctx[s], 0) : 0;
      long long slot = -1;
      if (on && p >= 0 && p / bs < width) {
        const int blk = table[s * ldt + p / bs];
        if (blk >= 0) slot = static_cast<long long>(blk) * bs + p % bs;
      }
      slots[s] = slot;
      ctx_out[s] = c;
      const int seen = static_cast<int>(min(static_cast<long long>(c), static_cast<long long>(width) * bs));
      n = seen / 64 + (seen % 64 != 0);
    }
    int total;
    const int inc = pm_scan(n, red, total);
    if (s < S) plan[s + 1] = carry + inc;
    carry += total;
  }
}

// A warp per row, 32 rows a block; every block sums the whole batch (for the verdict) and what stands in front of its rows.
__global__ void __launch_bounds__(PM_THREADS)
extend_block_tables_kernel(int* __restrict__ table, long long ldt, int S, int width, const int* __restrict__ rows, const int* __restrict__ have,
                           const int* __restrict__ lengths, int B, const int* __restrict__ pool, int pool_size, int bs, int* __restrict__ used) {
  __shared__ int red[32], off[32], fresh[32];
  __shared__ int bad;
  if (threadIdx.x == 0) bad = 0;
  __syncthreads();
  const int first = blockIdx.x * 32;
  long long all = 0;
  for (int base = 0; base < B; base += blockDim.x) {
    const int i = base + threadIdx.x;
    int n = 0;
    if (i < B) {
      const int len = max(lengths[i], 0), need = len / bs + (len % bs != 0);
      n = max(need - have[i], 0);
      if (rows[i] < 0 || rows[i] >= S || have[i] < 0 || have[i] > width || need > width) { bad = 1; n = 0; }
    }
    int total;
    const int inc = pm_scan(n, red, total);
    if (i >= first && i < first + 32) {   // sums fit an int where the verdict lets the rows be written: pool_size does
      off[i - first] = static_cast<int>(all) + inc - n;
      fresh[i - first] = n;
    }
    all += total;
  }
  __syncthreads();
  const bool fits = !bad && all <= pool_size;
  if (blockIdx.x == 0 && threadIdx.x == 0) used[0] = fits ? static_cast<int>(all) : -1;
  const int w = threadIdx.x >> 5, i = first + w;
  if (!fits || i >= B) return;
  int* row = table + rows[i] * ldt + have[i];
  for (int j = threadIdx.x & 31; j < fresh[w]; j += 32) row[j] = pool[off[w] + j];
}

constexpr int SM_THREADS = 256;
constexpr int SM_TOKENS = 4;  // consecutive tokens of a thread: 16 and 32 bytes of output
constexpr int SM_OWN_SUMS = 8192;  // sequences whose sums fit the shared memory that every launch has
constexpr int SM_TURNS = 4;   // times that a block goes on: its sums over the batch are made once for 4096 tokens
// 512 sequences of 2.3 million tokens: 13 us for 28 MB (2.1 TB/s; 4.5 us at the copy rate) in 568 blocks. A block's time is a chain: two sums over the
// batch, the search for its sequences, row and start, page, stores. Look-ups token by token, of which a warp nearly always needs some, took 17 us.

// cu[i + 1]: the tokens up to and with sequence i, no more than `total` of them.
__device__ __forceinline__ void sum_lengths(int* cu, const int* __restrict__ starts, const int* __restrict__ ends, int B, int total, int* red) {
  const SumUpTo add{total};
  int carry = 0;
  if (threadIdx.x == 0) cu[0] = 0;
  for (int base = 0; base < B; base += blockDim.x) {
    const int i = base + threadIdx.x, from = i < B ? max(starts[i], 0) : 0, to = i < B ? ends[i] : 0;
    int sum;
    const int inc = pm_scan(to > from ? min(to - from, total) : 0, red, sum, add);
    if (i < B) cu[i + 1] = add(carry, inc);
    carry = add(carry, sum);
  }
}

// For more sequences than a block's shared memory holds the sums of: they are taken once, by one block, and then read from memory.
__global__ void __launch_bounds__(PM_THREADS)
sum_lengths_kernel(const int* __restrict__ starts, const int* __restrict__ ends, int B, int total, int* __restrict__ cu) {
  __shared__ int red[32];
  sum_lengths(cu, starts, ends, B, total, red);
}

template <bool SUMMED>  // cu_out holds the sums already
__global__ void __launch_bounds__(SM_THREADS)
build_slot_map_kernel(const int* __restrict__ table, long long ldt, int S, int width, const int* __restrict__ rows, const int* __restrict__ starts,
                      const int* __restrict__ ends, int B, int bs, int shift, int total, int* cu_out, int* __restrict__ positions,
                      long long* __restrict__ slots) {
  extern __shared__ int own_cu[];  // [B + 1]
  __shared__ int red[32];
  const int* cu = SUMMED ? cu_out : own_cu;
  if constexpr (!SUMMED) {
    sum_lengths(own_cu, starts, ends, B, total, red);
    __syncthreads();
    if (blockIdx.x == 0)
      for (int i = threadIdx.x; i <= B; i += blockDim.x) cu_out[i] = own_cu[i];
  }
  const int end = cu[B];
  // Four tokens of one sequence are on one page or two: those of all turns are looked up together. A warp's tokens always meet the end of a page.
  int t0[SM_TURNS], p0[SM_TURNS], lo[SM_TURNS], row[SM_TURNS], blk[SM_TURNS], next[SM_TURNS];
#pragma unroll
  for (int turn = 0; turn < SM_TURNS; ++turn) {
    t0[turn] = ((blockIdx.x * SM_TURNS + turn) * SM_THREADS + threadIdx.x) * SM_TOKENS;
    int i = 0, hi = B;  // the sequence of t0: the last i with cu[i] <= t0, as far as there is one
    if (t0[turn] < end)
      while (hi - i > 1) {
        const int mid = (i + hi) >> 1;
        if (cu[mid] <= t0[turn]) i = mid; else hi = mid;
      }
    lo[turn] = i;
    p0[turn] = row[turn] = -1;
    if (t0[turn] < end) {
      p0[turn] = max(starts[i], 0) + t0[turn] - cu[i];
      row[turn] = rows[i];
    }
  }
#pragma unroll
  for (int turn = 0; turn < SM_TURNS; ++turn) {
    const int p = p0[turn], r = row[turn], j = shift >= 0 ? p >> shift : p / bs, k = j + (p - j * bs + SM_TOKENS > bs);
    const bool there = p >= 0 && r >= 0 && r < S;
    blk[turn] = there && j < width ? table[r * ldt + j] : -1;
    next[turn] = there && k < width ? table[r * ldt + k] : -1;
  }
#pragma unroll
  for (int turn = 0; turn < SM_TURNS; ++turn) {
    if (t0[turn] >= total) return;
    int at[SM_TOKENS];
    long long slot[SM_TOKENS];
    const int p = p0[turn], off = shift >= 0 ? p & (bs - 1) : p % bs;
    if (p >= 0 && t0[turn] + SM_TOKENS <= cu[lo[turn] + 1] && bs >= SM_TOKENS) {
      const long long first = static_cast<long long>(blk[turn]) * bs + off, second = (static_cast<long long>(next[turn]) - 1) * bs + off;
#pragma unroll
      for (int u = 0; u < SM_TOKENS; ++u) {
        const bool same = off + u < bs;
        at[u] = p + u;
        slot[u] = (same ? blk[turn] : next[turn]) >= 0 ? (same ? first : second) + u : -1;
      }
    } else {
      int i = lo[turn];
#pragma unroll
      for (int u = 0; u < SM_TOKENS; ++u) {
        const int t = t0[turn] + u;
        at[u] = 0;
        slot[u] = -1;
        if (t >= end) continue;
        while (cu[i + 1] <= t) ++i;
        const int q = max(starts[i], 0) + t - cu[i], j = shift >= 0 ? q >> shift : q / bs, r = rows[i];
        at[u] = q;
        if (q < 0 || r < 0 || r >= S || j >= width) continue;
        const int page = table[r * ldt + j];
        if (page >= 0) slot[u] = static_cast<long long>(page) * bs + (q - j * bs);
      }
    }
    if (t0[turn] + SM_TOKENS <= total) {
      *reinterpret_cast<int4*>(positions + t0[turn]) = make_int4(at[0], at[1], at[2], at[3]);
      *reinterpret_cast<longlong2*>(slots + t0[turn]) = make_longlong2(slot[0], slot[1]);
      *reinterpret_cast<longlong2*>(slots + t0[turn] + 2) = make_longlong2(slot[2], slot[3]);
    } else {
#pragma unroll
      for (int u = 0; u < SM_TOKENS; ++u)
        if (t0[turn] + u < total) {
          positions[t0[turn] + u] = at[u];
          slots[t0[turn] + u] = slot[u];
        }
    }
  }
}

}  // namespace vb

using namespace vb;

extern "C" int vb_decode_slot_map(const int* table, long long ldt, int width, const int* pos, const int* ctx, const bool* active, int S, int block_size,
                                  long long* slots, int* ctx_out, int* plan, cudaStream_t s) {
  const int threads = S >= PM_THREADS ? PM_THREADS : max(32, (S + 31) / 32 * 32);
  decode_slot_map_kernel<<<1, threads, 0, s>>>(table, ldt, width, pos, ctx, active, S, block_size, slots, ctx_out, plan);
  return static_cast<int>(cudaGetLastError());
}

extern "C" int vb_extend_block_tables(int* table, long long ldt, int S, int width, const int* rows, const int* have, const int* lengths, int B,
                                      const int* pool, int pool_size, int block_size, int* used, cudaStream_t s) {
  extend_block_tables_kernel<<<(B + 31) / 32, PM_THREADS, 0, s>>>(table, ldt, S, width, rows, have, lengths, B, pool, pool_size, block_size, used);
  return static_cast<int>(cudaGetLastError());
}

extern "C" int vb_build_slot_map(const int* table, long long ldt, int S, int width, const int* rows, const int* starts, const int* ends, int B,
                                 int block_size, int total, int* cu, int* positions, long long* slots, cudaStream_t s) {
  const int per = SM_THREADS * SM_TOKENS * SM_TURNS, shift = (block_size & (block_size - 1)) == 0 ? __builtin_ctz(static_cast<unsigned>(block_size)) : -1;
  if (total > 0x7fffffff - per) return -2;  // places of the last block are counted in 31 bits
  const int blocks = total > 0 ? (total + per - 1) / per : 1;
  if (B <= SM_OWN_SUMS) {
    build_slot_map_kernel<false><<<blocks, SM_THREADS, (B + 1) * sizeof(int), s>>>(table, ldt, S, width, rows, starts, ends, B, block_size, shift, total, cu,
                                                                                  positions, slots);
  } else {
    verl_count_launches(1);
    sum_lengths_kernel<<<1, PM_THREADS, 0, s>>>(starts, ends, B, total, cu);
    build_slot_map_kernel<true><<<blocks, SM_THREADS, 0, s>>>(table, ldt, S, width, rows, starts, ends, B, block_size, shift, total, cu, positions, slots);
  }
  return static_cast<int>(cudaGetLastError());
}
