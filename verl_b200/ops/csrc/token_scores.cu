// Scores of rows of logits: log-probs of given tokens, entropy, log-sum-exp, the most likely tokens; and the gradient of log-probs and entropy.
//
// With y = x log2(e) / temperature and a reference M near the largest y, a row is read once for
//   s = sum 2^(y - M),  w = sum 2^(y - M) (y - M):   lse = ln2 (M + log2 s),  H = ln2 (log2 s - w / s)
// four instructions and one exponential a value. A thread keeps a reference of its own, the largest of its first values, which moves only when the sum
// is 2^16 above it.
//
// The most likely tokens come with the same pass: every thread also keeps the largest value that it met, and the k-th largest of those of a
// block is a bound that at least k values of the row reach. The largest value of each group of 32 (16 of 32 bits) stays in shared memory, and
// only groups that reach the bound are looked at again (hardly more than k, from L2); what reaches it there is again hardly more than k
// values, which are ranked by counting. Where over 768 values reach it (few different values, or a mask that leaves fewer than k), the row is
// gone over again for what is above the bound and for the first values that equal it; rows with NaN or +inf are searched k times over.
//
// Blocks stay for many rows. One warp of a block brings the rows into a ring of shared memory by bulk copies, so that the next row is on its way
// while the block ranks the last one. Where rows are few, a row belongs to a cluster of up to 8 blocks, which exchange their sums, bounds and
// candidates through distributed shared memory. The gradient needs no exchange:
//   dL/dx_v = 1/T (sum_j g_j [v = id_j] - p_v (sum_j g_j + h (log p_v + H)))
// is one more pass, 2^y (a + b y) a value, with the given tokens' columns written again behind it. It takes log p from the reference and the
// logarithm of the sum that the forward pass left, not from their sum, the log-sum-exp.
//
// Measured, rows of 152064: 2048 of bf16 without alternatives 104 us (6.0 TB/s, 0.93 of the copy rate), with 64 of them 135 us, with 128 161 us; the same in
// fp32 221 us with 64 (0.87); their gradient, which reads once and writes once, 209 us in bf16 (0.92). One row of 151936: 12 us. What bounds the bf16
// forward is HBM beside its exponentials (70 us at the 16 a cycle that an SM has), and with alternatives the end of a row (15000 cycles of 75000:
// the bound 2300, the groups 2300, their values from memory 6600, ranks 4200), a chain that an SM's three other blocks do not cover: blocks that
// start a part of a row apart take as long. 256 threads and four blocks an SM: with fewer blocks less covers that end, with more the registers do not
// hold a vector's work. 24 slots, because a row of 152064 has 19 stages; the keys of larger groups bring more values to look at. Stages of 16 KB: with
// 8 KB, and as many bytes on their way or more, 137 us where they take 115, for what a stage costs beside its values.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "rollout_ops.h"
#include "tcgen05_common.cuh"

namespace vb {

namespace cg = cooperative_groups;
int num_sms();

constexpr int TS_THREADS = 256;    // that compute
constexpr int TS_BLOCKS = 4;       // blocks of an SM
constexpr int TS_BATCH = 4;        // 16-byte vectors of a thread in flight (gradient)
constexpr int TS_STAGES = 2;
constexpr int TS_PER = 4;                      // 16-byte vectors of a thread in a stage
constexpr int TS_CHUNK = TS_PER * TS_THREADS;  // vectors of a stage: 16 KB
constexpr int TS_CANDIDATES = 768;
constexpr int TS_SLOTS = 24;       // groups of a thread that are told apart: stages of the row, modulo this
constexpr float TS_LOG2E = 1.4426950408889634f, TS_LN2 = 0.6931471805599453f;
// Exponents of 2 that a thread's sum, and so any of its terms, stays below: a term 2^d is off by the rounding of d, half a step of 2^-20 at 16.
constexpr float TS_ABOVE = 16.f;
constexpr float TS_FLOOR = -200.f;  // exponents below this are zeros: keeps 0 * inf out of the sums

__device__ __forceinline__ float ts_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two fp32 numbers in one instruction, each rounded as alone
__device__ __forceinline__ unsigned long long ts_two(float a, float b) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 ts_of(unsigned long long v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
__device__ __forceinline__ unsigned long long ts_fma(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ unsigned long long ts_add(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ int g_ts_status[4];

// barrier of the threads that compute
__device__ __forceinline__ void ts_sync() { asm volatile("bar.sync 1, %0;" ::"n"(TS_THREADS) : "memory"); }
__device__ __forceinline__ int ts_count(bool p) {
  int n;
  asm volatile("{\n.reg .pred q;\nsetp.ne.u32 q, %1, 0;\nbarrier.cta.red.popc.aligned.u32 %0, 1, %2, q;\n}\n" : "=r"(n) : "r"(static_cast<uint32_t>(p)), "n"(TS_THREADS) : "memory");
  return n;
}
__device__ __forceinline__ float ts_max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 16 bytes of a row as floats
template <typename T> struct Lane;
template <> struct Lane<float> {
  static constexpr int N = 4, LOW = 16;  // values in 16 bytes, low bits of their keys that the bound leaves out (zero, or of little use)
  static __device__ __forceinline__ uint4 none() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
  static __device__ __forceinline__ void open(const uint4& v, float (&f)[N]) {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ uint4 close(const float (&f)[N]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};
// The larger of two pairs of 16-bit floats, by their bits: right where either is not negative, and negative (by its sign bit) where neither is.
__device__ __forceinline__ uint32_t pair_max(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.s16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t pair_max(const uint4& v) { return pair_max(pair_max(v.x, v.y), pair_max(v.z, v.w)); }

template <> struct Lane<__nv_bfloat16> {
  static constexpr int N = 8, LOW = 16;
  static __device__ __forceinline__ uint4 none() { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
  static __device__ __forceinline__ void open(const uint4& v, float (&f)[N]) {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(u[i] << 16);
      f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 close(const float (&f)[N]) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u[i]) : "f"(f[2 * i + 1]), "f"(f[2 * i]));
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
};
template <> struct Lane<__half> {
  static constexpr int N = 8, LOW = 13;
  static __device__ __forceinline__ uint4 none() { return make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u); }
  static __device__ __forceinline__ void open(const uint4& v, float (&f)[N]) {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      f[2 * i] = a.x;
      f[2 * i + 1] = a.y;
    }
  }
  static __device__ __forceinline__ uint4 close(const float (&f)[N]) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(u[i]) : "f"(f[2 * i + 1]), "f"(f[2 * i]));
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
};

// A row cut for 16-byte accesses: `head` values up to the first boundary, `vecs` vectors, the rest.
template <typename T>
struct Row {
  const T* x;
  int V, head, vecs;
  __device__ __forceinline__ Row(const T* row, int n) : x(row), V(n) {
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15) / static_cast<int>(sizeof(T));
    head = min(off == 0 ? 0 : Lane<T>::N - off, n);
    vecs = (n - head) / Lane<T>::N;
  }
  __device__ __forceinline__ const uint4* vec() const { return reinterpret_cast<const uint4*>(x + head); }
  __device__ __forceinline__ int loose() const { return V - vecs * Lane<T>::N; }                            // values outside the vectors
  __device__ __forceinline__ int loose_at(int i) const { return i < head ? i : i + vecs * Lane<T>::N; }
};

// Order of the values as whole numbers: NaN above everything, -0 with +0.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

struct Stat {
  float m, s, w;  // reference, sum 2^(y - m), sum 2^(y - m) (y - m)
  __device__ __forceinline__ void move(float to) {
    const float d = m - to, f = ts_exp2(fmaxf(d, -1e4f));
    w = f * (w + s * fmaxf(d, -1e4f));
    s *= f;
    m = to;
  }
  // a value f with y = f c, by the one rounding of f c - m that its log-prob has, so that a value that the sum consists of has a log-prob of 0
  __device__ __forceinline__ void add(float f, float c) {
    const float d = ts_max_nan(fmaf(f, c, -m), TS_FLOOR), e = ts_exp2(d);
    s += e;
    w = fmaf(e, d, w);
  }
};

// The sums of all threads of a block, in every thread. `red` holds 3 x 16 floats.
__device__ __forceinline__ Stat block_stat(Stat a, float* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float m = a.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  a.move(m);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
    a.w += __shfl_xor_sync(0xffffffffu, a.w, o);
  }
  ts_sync();
  if (lane == 0) { red[warp] = a.m; red[16 + warp] = a.s; red[32 + warp] = a.w; }
  ts_sync();
  constexpr int W = TS_THREADS / 32;
  Stat b{red[lane % W], red[16 + lane % W], red[32 + lane % W]};
  m = b.m;
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  b.move(m);
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) {
    b.s += __shfl_xor_sync(0xffffffffu, b.s, o);
    b.w += __shfl_xor_sync(0xffffffffu, b.w, o);
  }
  return b;
}

__device__ __forceinline__ unsigned long long block_max(unsigned long long v, unsigned long long* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  ts_sync();
  if (lane == 0) red[warp] = v;
  ts_sync();
  v = lane < TS_THREADS / 32 ? red[lane] : 0ull;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// What log2 p = y - m - log2 s takes of a row: the reference, and log2 s as a whole number and the logarithm of what is left, in [1, 2). Neither is
// added to the reference, which would round off digits of p by the size of the logits (log-sum-exp 9e4: p off by 4e-3); and for the value that s
// consists of, y - m and the whole number are close and their difference exact: 1 - p is off by at most 2e-6, in rows of 32000 by 4e-7.
struct Norm {
  float m, whole, part;
  static __device__ __forceinline__ Norm of(const Stat& a) {
    const int e = static_cast<int>(__float_as_uint(a.s) >> 23) - 127;  // s is a normal number: at least one term of it is
    return {a.m, static_cast<float>(e), log2f(__uint_as_float((__float_as_uint(a.s) & 0x007fffffu) | 0x3f800000u))};
  }
  __device__ __forceinline__ float log2_s() const { return whole + part; }
  __device__ __forceinline__ float log2_p(float f, float c) const { return fmaf(f, c, -m) - whole - part; }
};

// Log-prob of value f. A value near the type's lowest is its own log-prob: log2(e) times it is not finite.
__device__ __forceinline__ float scaled_logprob(float f, float inv_temp, const Norm& n) {
  const float y = n.log2_p(f, inv_temp * TS_LOG2E);
  return y == -INFINITY ? f * inv_temp : TS_LN2 * y;
}

// Largest z = x / temperature and sum e^(z - m), sum e^(z - m) (z - m) of any row, by one block: for a row whose largest value is NaN or +inf
// the sums are NaN, for one of nothing but -inf m is -inf.
template <typename T>
__device__ Stat any_stat(const T* x, int V, float inv_temp, float* red) {
  float m = -INFINITY;
  for (int v = threadIdx.x; v < V; v += TS_THREADS) m = ts_max_nan(m, static_cast<float>(x[v]) * inv_temp);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = ts_max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  ts_sync();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  ts_sync();
  for (int i = 0; i < TS_THREADS / 32; ++i) m = ts_max_nan(m, red[i]);
  Stat a{0.f, 0.f, 0.f};
  if (m > -INFINITY || m != m)
    for (int v = threadIdx.x; v < V; v += TS_THREADS) {
      const float d = static_cast<float>(x[v]) * inv_temp - m, e = expf(d);
      a.s += e;
      if (e > 0.f) a.w = fmaf(e, d, a.w);
      if (e != e) a.w = e;
    }
  a = block_stat(a, red);
  a.m = m;
  return a;
}

// A place for each of the n things of this thread, warp by warp: the counter goes up once for all 32 threads, which all take part.
template <typename F>
__device__ __forceinline__ int warp_places(int n, const F& count) {
  const int lane = threadIdx.x & 31;
  int upto = n;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int before = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += before;
  }
  int base = 0;
  if (lane == 31 && upto > 0) base = count(upto);
  return __shfl_sync(0xffffffffu, base, 31) + upto - n;
}

struct Shared {
  float red[48];
  Stat stat;               // of this block's part of the row
  uint32_t bound;          // at least top values of the part have this key or a larger one (0: the part has fewer threads with values)
  int groups, found;
  unsigned long long wide[16];
  uint16_t group[TS_CANDIDATES];           // slot * TS_THREADS + thread of the groups that reach the bound
  uint16_t top[TS_SLOTS][TS_THREADS];      // upper halves of the keys of the groups' largest values
  unsigned long long list[TS_CANDIDATES];  // (key, place backwards)
};

template <typename T>
__device__ void scores_any(const VbScores& p, long long t, const T* x, Shared& sh) {
  const Stat a = any_stat(x, p.V, p.inv_temp, sh.red);
  const float ls = logf(a.s), none = -INFINITY;
  const bool empty = a.m == -INFINITY;
  const auto logprob = [&](float v) { return empty ? none : v * p.inv_temp - a.m - ls; };
  if (threadIdx.x == 0) {
    p.lse[t] = empty ? none : a.m + ls;
    p.entropy[t] = empty ? 0.f : ls - a.w / a.s;
    if (p.stat != nullptr) reinterpret_cast<float4*>(p.stat)[t] = make_float4(NAN, 0.f, 0.f, 0.f);  // the gradient reads the row again
  }
  for (int j = threadIdx.x; j < p.K; j += TS_THREADS) {
    const long long id = p.ids[t * p.K + j];
    p.logprob[t * p.K + j] = id >= 0 && id < p.V ? logprob(static_cast<float>(x[id])) : 0.f;
  }
}

// The largest (value, lowest place) below the last one, `top` times over.
template <typename T, typename F>
__device__ void top_any(const VbScores& p, long long t, const T* x, Shared& sh, const F& logprob) {
  unsigned long long last = ~0ull;
  for (int k = 0; k < p.top; ++k) {
    unsigned long long b = 0;
    for (int v = threadIdx.x; v < p.V; v += TS_THREADS) {
      const unsigned long long key = (static_cast<unsigned long long>(order_key(static_cast<float>(x[v]))) << 32) | (0xffffffffu - v);
      if (key < last && key > b) b = key;
    }
    last = block_max(b, sh.wide);
    if (threadIdx.x == 0) {
      const uint32_t v = 0xffffffffu - static_cast<uint32_t>(last);
      p.top_ids[t * p.top + k] = v;
      p.top_lp[t * p.top + k] = logprob(static_cast<float>(x[v]));
    }
  }
}

// Writes the tokens of the list, which holds `found` values, at their ranks: four lanes a candidate count the larger ones.
template <typename F>
__device__ void write_ranked(const VbScores& p, long long t, const Shared& sh, int found, const F& logprob) {
  for (int i0 = 0; i0 < found; i0 += TS_THREADS / 4) {
    const int i = i0 + (threadIdx.x >> 2), quarter = threadIdx.x & 3;
    if ((i & ~7) >= found) break;  // the warp's eight
    const unsigned long long key = sh.list[min(i, found - 1)];
    int rank = 0;
#pragma unroll 4
    for (int j = quarter; j < found; j += 4) rank += sh.list[j] > key;
    rank += __shfl_xor_sync(0xffffffffu, rank, 1);
    rank += __shfl_xor_sync(0xffffffffu, rank, 2);
    if (i >= found || quarter != 0 || rank >= p.top) continue;
    const long long at = t * p.top + rank;
    p.top_ids[at] = 0xffffffffu - static_cast<uint32_t>(key);
    p.top_lp[at] = logprob(key_value(static_cast<uint32_t>(key >> 32)));
  }
}

// The most likely tokens of a row without NaN in three passes of one block: the `top`-th largest of the threads' largest values, what is above
// it, and as many of the first values that equal it as are missing. False where over TS_CANDIDATES values are above it.
template <typename T, typename F>
__device__ bool top_ties(const VbScores& p, long long t, const T* x, Shared& sh, const F& logprob) {
  float most = -INFINITY;
  for (int v = threadIdx.x; v < p.V; v += TS_THREADS) most = fmaxf(most, static_cast<float>(x[v]));
  const uint32_t mine = static_cast<int>(threadIdx.x) < p.V ? order_key(most) : 0u;
  uint32_t bound = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t want = bound | (1u << bit);
    if (ts_count(mine >= want) >= min(p.top, TS_THREADS)) bound = want;
  }
  const float limit = bound <= order_key(-INFINITY) ? -INFINITY : key_value(bound);
  if (threadIdx.x == 0) sh.found = 0;
  ts_sync();
  for (int v = threadIdx.x; v < p.V; v += TS_THREADS) {
    const float f = static_cast<float>(x[v]);
    if (f > limit) {
      const int k = atomicAdd(&sh.found, 1);
      if (k < TS_CANDIDATES) sh.list[k] = (static_cast<unsigned long long>(order_key(f)) << 32) | (0xffffffffu - v);
    }
  }
  ts_sync();
  int found = sh.found;
  if (found > TS_CANDIDATES) return false;
  constexpr int EACH = 8;  // consecutive values of a thread
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int v0 = 0; v0 < p.V && found < p.top; v0 += TS_THREADS * EACH) {
    const int v = v0 + threadIdx.x * EACH;
    uint32_t equal = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i)
      if (v + i < p.V && static_cast<float>(x[v + i]) == limit) equal |= 1u << i;
    int before = __popc(equal);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int n = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += n;
    }
    ts_sync();
    if (lane == 31) sh.red[warp] = static_cast<float>(before);  // whole numbers below 2^24
    ts_sync();
    int all = 0;
    for (int w = 0; w < TS_THREADS / 32; ++w) {
      const int n = static_cast<int>(sh.red[w]);
      if (w < warp) before += n;
      all += n;
    }
    before -= __popc(equal);
    for (uint32_t e = equal; e != 0 && found + before < p.top; e &= e - 1, ++before)
      sh.list[found + before] = (static_cast<unsigned long long>(order_key(limit)) << 32) | (0xffffffffu - (v + __ffs(e) - 1));
    found = min(found + all, p.top);
  }
  ts_sync();
  write_ranked(p, t, sh, found, logprob);
  return true;
}

template <typename T>
__device__ __forceinline__ void bulk_row(void* dst, const T* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes),
               "r"(smem_u32(bar))
               : "memory");
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(TS_THREADS + 32, TS_BLOCKS)
token_scores_kernel(const VbScores p, int* status) {
  using L = Lane<T>;
  extern __shared__ __align__(16) uint4 ring[];  // TS_STAGES x TS_CHUNK
  __shared__ Shared sh;
  __shared__ uint64_t full[TS_STAGES], empty[TS_STAGES];
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = static_cast<int>(cluster.num_blocks()), part = static_cast<int>(cluster.block_rank());
  const int t0 = blockIdx.x / parts, dt = gridDim.x / parts;  // rows of this cluster: with several parts, one
  const float c = p.inv_temp * TS_LOG2E;
  if (threadIdx.x == 0) {
    for (int i = 0; i < TS_STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], TS_THREADS / 32);
    }
    mbar_fence_init();
  }
  __syncthreads();

  if (threadIdx.x >= TS_THREADS) {
    // ---- the warp that loads
    if (threadIdx.x == TS_THREADS) {
      bool ok = true;
      long long k = 0;
      for (int t = t0; t < p.T && ok; t += dt) {
        const Row<T> row(static_cast<const T*>(p.x) + t * p.ldx, p.V);
        const int per = (row.vecs + parts - 1) / parts, v0 = min(row.vecs, part * per), n = min(row.vecs, v0 + per) - v0;
        for (int v = 0; v < n && ok; v += TS_CHUNK, ++k) {
          const int s = static_cast<int>(k % TS_STAGES);
          if (k >= TS_STAGES) ok = mbar_wait(&empty[s], static_cast<uint32_t>((k / TS_STAGES - 1) & 1));
          if (!ok) break;
          const uint32_t bytes = min(TS_CHUNK, n - v) * 16;
          mbar_expect_tx(&full[s], bytes);
          bulk_row(ring + s * TS_CHUNK, row.vec() + v0 + v, bytes, &full[s]);
        }
      }
      if (!ok) atomicExch(status, ST_TIMEOUT_PRODUCER);
      for (long long i = max(k - TS_STAGES, 0LL); i < k; ++i) mbar_wait(&full[i % TS_STAGES], static_cast<uint32_t>((i / TS_STAGES) & 1));  // no copy outlives the block
    }
    return;
  }

  bool ok = true;
  int stage = 0;
  uint32_t round = 0;
  for (int t = t0; t < p.T; t += dt) {
    const T* x = static_cast<const T*>(p.x) + t * p.ldx;
    const Row<T> row(x, p.V);
    const int per = (row.vecs + parts - 1) / parts, v0 = min(row.vecs, part * per), n = min(row.vecs, v0 + per) - v0;
    const uint4* vec = row.vec() + v0;
    if (threadIdx.x == 0) sh.groups = sh.found = 0;
    // the value of this thread's given token, on its way during the pass
    const long long id0 = part == 0 && static_cast<int>(threadIdx.x) < p.K ? p.ids[static_cast<long long>(t) * p.K + threadIdx.x] : -1;
    const T given = x[id0 >= 0 && id0 < p.V ? id0 : 0];

    // ---- the pass
    Stat a{-1e30f, 0.f, 0.f};
    float most = -INFINITY;
    for (int v = 0, slot = 0; v < n; v += TS_CHUNK, ++slot) {
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&full[stage], round & 1));
      const uint4* at = ring + stage * TS_CHUNK + threadIdx.x;
      const int left = n - v - static_cast<int>(threadIdx.x);
      const auto largest = [&]() {  // of this thread's values in the stage, NaN left aside
        float big = -INFINITY;
#pragma unroll
        for (int u = 0; u < TS_PER; ++u) {
          float f[L::N];
          L::open(left > u * TS_THREADS ? at[u * TS_THREADS] : L::none(), f);
#pragma unroll
          for (int i = 0; i < L::N; i += 2) big = fmaxf(big, fmaxf(f[i], f[i + 1]));
        }
        return big;
      };
      if (slot == 0) {
        const float big = largest();
        if (big * c > a.m) a.move(big * c);
      }
      unsigned long long s2 = ts_two(a.s, 0.f), w2 = ts_two(a.w, 0.f);
      const unsigned long long c2 = ts_two(c, c), m2 = ts_two(-a.m, -a.m);
      uint32_t pairs = 0x80008000u;
      float big = -INFINITY;
#pragma unroll
      for (int u = 0; u < TS_PER; ++u) {
        if (left <= u * TS_THREADS) break;
        const uint4 v = at[u * TS_THREADS];
        float f[L::N];
        L::open(v, f);
        if constexpr (TOP && sizeof(T) == 2) pairs = pair_max(pairs, pair_max(v));
#pragma unroll
        for (int i = 0; i < L::N; i += 2) {
          if constexpr (TOP && sizeof(T) == 4) big = fmaxf(big, fmaxf(f[i], f[i + 1]));
          const unsigned long long d2 = ts_fma(ts_two(f[i], f[i + 1]), c2, m2);
          const float2 d = ts_of(d2);
          const unsigned long long e2 = ts_two(ts_exp2(d.x), ts_exp2(d.y));
          s2 = ts_add(s2, e2);
          w2 = ts_fma(e2, d2, w2);
        }
      }
      const float2 s = ts_of(s2), w = ts_of(w2);
      if (s.x + s.y < 0x1p16f && w.x + w.y == w.x + w.y) {
        a.s = s.x + s.y;
        a.w = w.x + w.y;
      } else {  // too far above the reference, or 0 * -inf got into the sums: again, with a floor under the exponents
        const float up = fmaxf(largest() * c, a.s > 0.f ? a.m + log2f(a.s) : -INFINITY);
        if (up > a.m + 0.5f * TS_ABOVE) a.move(up);
#pragma unroll 1
        for (int u = 0; u < TS_PER; ++u) {
          if (left <= u * TS_THREADS) break;
          float f[L::N];
          L::open(at[u * TS_THREADS], f);
#pragma unroll
          for (int i = 0; i < L::N; ++i) a.add(f[i], c);
        }
      }
      if constexpr (TOP) {
        if constexpr (sizeof(T) == 2) {
          pairs = pair_max(pairs, pairs >> 16 | 0x80000000u) & 0xffffu;
          big = pairs < 0x8000u ? static_cast<float>(*reinterpret_cast<const T*>(&pairs)) : largest();  // nothing that is not negative
        }
        most = fmaxf(most, big);
        uint16_t* keep = &sh.top[slot % TS_SLOTS][threadIdx.x];
        const uint16_t key = static_cast<uint16_t>(order_key(big) >> 16);
        *keep = slot < TS_SLOTS ? key : max(*keep, key);
      }
      __syncwarp();
      if ((threadIdx.x & 31) == 0) mbar_arrive(&empty[stage]);
      if (++stage == TS_STAGES) {
        stage = 0;
        ++round;
      }
    }
    const bool has_loose = part == 0 && static_cast<int>(threadIdx.x) < row.loose();
    const int loose_at = has_loose ? row.loose_at(threadIdx.x) : 0;
    const float loose = has_loose ? static_cast<float>(x[loose_at]) : -INFINITY;
    const bool any = has_loose || static_cast<int>(threadIdx.x) < n;
    if (has_loose) {
      most = fmaxf(most, loose);
      if (loose * c > a.m + TS_ABOVE) a.move(loose * c);
      a.add(loose, c);
    }
    a = block_stat(a, sh.red);

    // ---- the bound: bit by bit, the largest key that `top` threads' largest values reach (100 cycles a bit; by one warp with eight keys a lane, 170)
    uint32_t bound = 0;
    const uint32_t mine = any ? order_key(most) : 0u;
    if constexpr (TOP)
      for (int bit = 31; bit >= L::LOW; --bit) {
        const uint32_t want = bound | (1u << bit);
        if (ts_count(mine >= want) >= p.top) bound = want;
      }
    if (parts > 1) {
      if (threadIdx.x == 0) {
        sh.stat = a;
        sh.bound = bound;
      }
      cluster.sync();
      a = *cluster.map_shared_rank(&sh.stat, 0);
      float m = a.m;
      for (int i = 1; i < parts; ++i) m = fmaxf(m, cluster.map_shared_rank(&sh, i)->stat.m);
      a.move(m);
      for (int i = 1; i < parts; ++i) {
        Stat o = cluster.map_shared_rank(&sh, i)->stat;
        o.move(m);
        a.s += o.s;
        a.w += o.w;
      }
      for (int i = 0; i < parts; ++i) bound = max(bound, cluster.map_shared_rank(&sh, i)->bound);
    }
    const bool odd = !(a.s > 0.f && a.s < INFINITY && fabsf(a.m) < 1e30f);  // NaN, +inf, or nothing that the reference can be compared with

    // ---- what reaches the bound, into the first block's list
    Shared* first = parts > 1 ? cluster.map_shared_rank(&sh, 0) : &sh;
    if (TOP && !odd) {
      const float limit = bound <= order_key(-INFINITY) ? -INFINITY : key_value(bound);
      const int chunks = (n + TS_CHUNK - 1) / TS_CHUNK, low = static_cast<int>(bound >> 16);
      uint32_t hits = 0;
      if (mine >= bound)
#pragma unroll 8
        for (int slot = 0; slot < min(chunks, TS_SLOTS); ++slot) hits |= static_cast<uint32_t>(sh.top[slot][threadIdx.x] >= low) << slot;
      int k = warp_places(__popc(hits), [&](int n) { return atomicAdd(&sh.groups, n); });
      for (; hits != 0; hits &= hits - 1, ++k)
        if (k < TS_CANDIDATES) sh.group[k] = static_cast<uint16_t>((__ffs(hits) - 1) * TS_THREADS + threadIdx.x);
      ts_sync();
      const int groups = min(sh.groups, TS_CANDIDATES), turns = (chunks + TS_SLOTS - 1) / TS_SLOTS, items = groups * TS_PER * turns;
      if (sh.groups > TS_CANDIDATES && threadIdx.x == 0) atomicAdd(&first->found, TS_CANDIDATES + 1);  // too many: the slow path
      const auto found = [&](int n) { return parts > 1 ? atomicAdd(&first->found, n) : atomicAdd(&sh.found, n); };
      const auto put = [&](float f, int at, int k) {
        if (k < TS_CANDIDATES) first->list[k] = (static_cast<unsigned long long>(order_key(f)) << 32) | (0xffffffffu - at);
      };
      // item i: vector i % TS_PER of group i / TS_PER, and for rows of more stages than slots the same place some stages on
      for (int i0 = static_cast<int>(threadIdx.x) & ~31; i0 < items; i0 += 2 * TS_THREADS) {
        uint4 raw[2];
        int at[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int i = i0 + (threadIdx.x & 31) + u * TS_THREADS, turn = turns == 1 ? 0 : i / (groups * TS_PER), k = i - turn * groups * TS_PER;
          const int g = i < items ? sh.group[k / TS_PER] : 0;
          at[u] = i < items ? ((turn * TS_SLOTS + g / TS_THREADS) * TS_PER + k % TS_PER) * TS_THREADS + g % TS_THREADS : n;
          raw[u] = at[u] < n ? __ldg(vec + at[u]) : L::none();
        }
        uint32_t reach = 0;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float f[L::N];
          L::open(raw[u], f);
#pragma unroll
          for (int j = 0; j < L::N; ++j)
            if (f[j] >= limit && at[u] < n) reach |= 1u << (u * L::N + j);
        }
        int k = warp_places(__popc(reach), found);
        if (reach != 0)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float f[L::N];
            L::open(raw[u], f);
#pragma unroll
            for (int j = 0; j < L::N; ++j)
              if (reach >> (u * L::N + j) & 1u) put(f[j], row.head + (v0 + at[u]) * L::N + j, k++);
          }
      }
      if (row.loose() > 0) {
        const bool reaches = has_loose && loose >= limit;
        k = warp_places(reaches, found);
        if (reaches) put(loose, loose_at, k);
      }
    }
    if (parts > 1) cluster.sync(); else ts_sync();
    if (part != 0) return;

    if (odd) {
      scores_any(p, t, x, sh);
      ts_sync();
      if (p.top > 0) {
        const Stat b = any_stat(x, p.V, p.inv_temp, sh.red);
        const float bls = logf(b.s);
        const auto logprob = [&](float f) { return b.m == -INFINITY ? -INFINITY : f * p.inv_temp - b.m - bls; };
        const bool wild = !(b.s >= 0.f) || b.m == INFINITY;  // NaN or +inf in it
        if (wild || !top_ties(p, t, x, sh, logprob)) top_any(p, t, x, sh, logprob);
      }
      ts_sync();
      continue;
    }
    const Norm norm = Norm::of(a);
    const auto logprob = [&](float f) { return scaled_logprob(f, p.inv_temp, norm); };
    if (threadIdx.x == 0) {
      p.lse[t] = TS_LN2 * (a.m + norm.log2_s());
      p.entropy[t] = TS_LN2 * (norm.log2_s() - a.w / a.s);
      if (!TOP && p.stat != nullptr) reinterpret_cast<float4*>(p.stat)[t] = make_float4(norm.m, norm.whole, norm.part, 0.f);
    }
    for (int j = threadIdx.x; j < p.K; j += TS_THREADS) {
      const long long at = static_cast<long long>(t) * p.K + j, id = j < TS_THREADS ? id0 : p.ids[at];
      const bool there = id >= 0 && id < p.V;
      p.logprob[at] = there ? logprob(static_cast<float>(j < TS_THREADS ? given : x[id])) : 0.f;
    }
    if (p.top > 0) {
      const int found = sh.found;
      if (found >= p.top && found <= TS_CANDIDATES)
        write_ranked(p, t, sh, found, logprob);
      else if (!top_ties(p, t, x, sh, logprob))
        top_any(p, t, x, sh, logprob);
    }
    ts_sync();  // the next row starts with an empty list
  }
  if (!ok && (threadIdx.x & 31) == 0) atomicExch(status, ST_TIMEOUT_EPILOGUE);
}

// ---- gradient: blockIdx.x is the row, blockIdx.y one of gridDim.y parts of its columns
template <typename T>
__global__ void __launch_bounds__(TS_THREADS, TS_BLOCKS)
token_scores_bwd_kernel(const VbScores p, const float* __restrict__ g_lp, const float* __restrict__ g_ent, T* __restrict__ dx, long long lddx, int columns) {
  using L = Lane<T>;
  __shared__ Shared sh;
  const long long t = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + t * p.ldx;
  T* d = dx + t * lddx;
  const float lse = p.lse[t], H = p.entropy[t], h = g_ent != nullptr ? g_ent[t] : 0.f;
  const long long* ids = p.ids + t * p.K;
  const float* gl = g_lp + t * p.K;
  Stat gs{0.f, 0.f, 0.f};
  for (int j = threadIdx.x; j < p.K; j += TS_THREADS)
    if (ids[j] >= 0 && ids[j] < p.V) gs.s += gl[j];
  const float g = block_stat(gs, sh.red).s;
  // log2 p from the row's reference and sum as the forward pass had them: the log-sum-exp alone has lost log s in its own rounding
  const float4 kept = reinterpret_cast<const float4*>(p.stat)[t];
  const Norm norm{kept.x, kept.y, kept.z};
  const float c = p.inv_temp * TS_LOG2E;
  float m = 0.f, ls = 0.f;
  const bool apart = norm.m != norm.m;  // a row that has no such reference: both again, and the differences before they are scaled
  if (apart) {
    const Stat b = any_stat(x, p.V, p.inv_temp, sh.red);
    m = b.m;
    ls = logf(b.s) * TS_LOG2E;
  }
  const bool empty = lse == -INFINITY;
  const float a0 = -p.inv_temp * (g + h * H), a1 = -p.inv_temp * h * TS_LN2;
  const auto log2_p = [&](float f) { return ts_max_nan(apart ? (f * p.inv_temp - m) * TS_LOG2E - ls : norm.log2_p(f, c), TS_FLOOR); };
  const auto slope = [&](float f) {
    const float y = log2_p(f);
    return empty ? 0.f : ts_exp2(y) * fmaf(a1, y, a0);
  };
  // vectors where the row and its gradient lie alike
  const Row<T> row(x, p.V);
  const bool alike = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(d)) & 15) == 0;
  const int head = alike ? row.head : 0, vecs = alike ? row.vecs : 0;
  const int per = (vecs + gridDim.y - 1) / gridDim.y, v0 = min(vecs, static_cast<int>(blockIdx.y) * per), v1 = min(vecs, v0 + per);
  const uint4* from = reinterpret_cast<const uint4*>(x + head);
  uint4* to = reinterpret_cast<uint4*>(d + head);
  for (int v = v0 + threadIdx.x; v < v1; v += TS_THREADS * TS_BATCH) {
    uint4 raw[TS_BATCH];
#pragma unroll
    for (int u = 0; u < TS_BATCH; ++u) raw[u] = v + u * TS_THREADS < v1 ? __ldg(from + v + u * TS_THREADS) : L::none();
#pragma unroll
    for (int u = 0; u < TS_BATCH; ++u) {
      float f[L::N];
      L::open(raw[u], f);
#pragma unroll
      for (int i = 0; i < L::N; ++i) f[i] = slope(f[i]);
      if (v + u * TS_THREADS < v1) to[v + u * TS_THREADS] = L::close(f);
    }
  }
  // the columns outside the vectors, and those that do not count: the last part's
  const int behind = head + vecs * L::N;
  if (blockIdx.y == gridDim.y - 1) {
    for (int v = threadIdx.x; v < head; v += TS_THREADS) d[v] = static_cast<T>(slope(static_cast<float>(x[v])));
    for (int v = behind + threadIdx.x; v < columns; v += TS_THREADS) d[v] = static_cast<T>(v < p.V ? slope(static_cast<float>(x[v])) : 0.f);
  }
  ts_sync();
  // the given tokens: a token's first place in the list gathers all its gradients, in their order
  for (int j = threadIdx.x; j < p.K; j += TS_THREADS) {
    const long long id = ids[j];
    if (id < 0 || id >= p.V) continue;
    const int in_vec = id >= head && id < behind ? (static_cast<int>(id) - head) / L::N : -1;
    if (in_vec >= 0 ? in_vec < v0 || in_vec >= v1 : blockIdx.y != gridDim.y - 1) continue;
    float sum = 0.f;
    bool earlier = false;
    for (int i = 0; i < p.K; ++i)
      if (ids[i] == id) {
        earlier |= i < j;
        sum += gl[i];
      }
    if (earlier || empty) continue;
    const float f = static_cast<float>(x[id]), y = log2_p(f);
    // sum - p (g + h (log p + H)), and where p is above a half as (sum - g) + g (1 - p) - p h (log p + H): a token that is all but certain has a small
    // difference, not two large terms
    d[id] = static_cast<T>(y < -1.f ? fmaf(p.inv_temp, sum, slope(f)) : p.inv_temp * (sum - g - g * expm1f(TS_LN2 * y) - ts_exp2(y) * h * fmaf(TS_LN2, y, H)));
  }
}

template <typename T>
static cudaError_t ts_forward(const VbScores& a, cudaStream_t s) {
  // A row to several blocks while there are at most three to an SM then (64 rows of 128256 in 32 bits: 17 us in 256 blocks, 19 us in 512; 100 rows of
  // 152064: 19 us in 400, 23 us in 100), with at least 1024 vectors for each. With more rows than the card holds blocks, blocks that stay.
  int parts = 1;
  while (parts < 8 && 2LL * parts * a.T <= 3 * num_sms() && a.V / Lane<T>::N >= 2048 * parts) parts *= 2;
  constexpr int smem = TS_STAGES * TS_CHUNK * 16;
  auto kern = a.top > 0 ? token_scores_kernel<T, true> : token_scores_kernel<T, false>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  int* status = nullptr;
  if (e == cudaSuccess) e = cudaGetSymbolAddress(reinterpret_cast<void**>(&status), g_ts_status);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(parts > 1 ? a.T * parts : min(a.T, TS_BLOCKS * num_sms()));
  cfg.blockDim = dim3(TS_THREADS + 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, a, status);
}

template <typename T>
static cudaError_t ts_backward(const VbScores& a, const float* g_lp, const float* g_ent, void* dx, long long lddx, int columns, cudaStream_t s) {
  int parts = 1;
  while (parts < 32 && 2LL * parts * a.T <= TS_BLOCKS * num_sms() && a.V / Lane<T>::N >= 2048 * parts) parts *= 2;
  token_scores_bwd_kernel<T><<<dim3(a.T, parts), TS_THREADS, 0, s>>>(a, g_lp, g_ent, static_cast<T*>(dx), lddx, columns);
  return cudaGetLastError();
}

}  // namespace vb

using namespace vb;

extern "C" int vb_token_scores_status() {
  int h[4] = {0, 0, 0, 0};
  if (cudaMemcpyFromSymbol(h, g_ts_status, sizeof(h)) != cudaSuccess) return -1;
  if (h[0] != 0) {
    int z[4] = {0, 0, 0, 0};
    cudaMemcpyToSymbol(g_ts_status, z, sizeof(z));
  }
  return h[0];
}

extern "C" int vb_token_scores(const VbScores* a, cudaStream_t s) {
  if (a->T == 0) return 0;
  verl_count_launches(1);
  return static_cast<int>(a->type == 0 ? ts_forward<__nv_bfloat16>(*a, s) : a->type == 1 ? ts_forward<__half>(*a, s) : ts_forward<float>(*a, s));
}

extern "C" int vb_token_scores_bwd(const VbScores* a, const float* g_lp, const float* g_ent, void* dx, long long lddx, int columns, cudaStream_t s) {
  if (a->T == 0 || columns == 0) return 0;
  verl_count_launches(1);
  return static_cast<int>(a->type == 0   ? ts_backward<__nv_bfloat16>(*a, g_lp, g_ent, dx, lddx, columns, s)
                          : a->type == 1 ? ts_backward<__half>(*a, g_lp, g_ent, dx, lddx, columns, s)
                                         : ts_backward<float>(*a, g_lp, g_ent, dx, lddx, columns, s));
}
