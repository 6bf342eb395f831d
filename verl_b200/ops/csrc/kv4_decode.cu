// Attention of one query token per sequence over the 4-bit cache (layout: kv4_common.cuh): one pass over the codes, running maximum and sum.
//
// Work: contexts are cut into pieces of 64 tokens; the pieces of all (sequence, KV head) pairs, laid end to end, are dealt to the CTAs of one
// wave in equal runs, whatever the lengths are (the plan holds the pieces in front of every sequence). A CTA that starts or ends inside a
// (sequence, head) leaves its sums in a slot of its own, and a second small launch, started early by programmatic dependence, joins them
// by their maxima, in the order of the runs: no atomics, the same bits every time.
//
// A CTA: one warp brings pieces into a ring of shared memory by bulk copies (a piece is at most 16 contiguous runs; four for blocks of 64 and
// more), several pieces and the next segment's queries ahead; four warps own 16 of a piece's 64 tokens each and meet at the end of a segment.
//   S^T[16 tokens, 8 heads] = K[16, hd] Q^T        keys are the A operand of m16n8k16: a thread's share of a token's row is one contiguous run
//   O^T[hd, 8 heads]       += V^T[hd, 16] P^T      values are the A operand as well; P^T is S^T's accumulator through movmatrix
// so that with up to 8 heads to a KV head a matrix instruction takes 256 cache elements (query heads as the 16 rows would take 128).
// A code becomes a number without a conversion: (w & 0x000f000f) | 0x6400.. is 1024 + q in fp16, (w & 0x00f000f0) | 0x5400.. is 64 + q; one
// subtraction (exact) and one multiply-add with the group's scale and least value, in pairs: 1.6 instructions an element. That rounds a value
// to fp16 once; queries are scaled by a power of two per head so that fp16 holds them exactly, and weights are e^(s - max) <= 1 in fp16.
#include <math.h>

#include "kv4_common.cuh"
#include "rollout_ops.h"
#include "tcgen05_common.cuh"

namespace vb {

int num_sms();

constexpr int KD_PIECE = 64;
constexpr int KD_WARPS = 4;                      // warps that compute
constexpr int KD_THREADS = (KD_WARPS + 1) * 32;
constexpr int KD_STAGES = 4;
constexpr int KD_MIN_PIECES = 4;                 // shortest run of a CTA

__device__ int g_kv4_status[4];

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes),
               "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix_t(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t h2_bits(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }
__device__ __forceinline__ __half2 h2_of(uint32_t v) { return *reinterpret_cast<__half2*>(&v); }
// pairs 0 / 1 of the four that a word of codes holds: its nibbles (0, 4) and (1, 5); the other two after a shift by 8
__device__ __forceinline__ uint32_t codes_even(uint32_t w, __half2 s, __half2 m) {
  uint32_t x;
  asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(x) : "r"(w));
  return h2_bits(__hfma2(__hadd2(h2_of(x), h2_of(0xe400e400u)), s, m));  // - 1024
}
__device__ __forceinline__ uint32_t codes_odd(uint32_t w, __half2 s, __half2 m) {
  uint32_t x;
  asm("lop3.b32 %0, %1, 0x00f000f0, 0x54005400, 0xea;" : "=r"(x) : "r"(w));
  return h2_bits(__hfma2(__hadd2(h2_of(x), h2_of(0xd400d400u)), s, m));  // - 64
}

template <int HD, int NT>
struct KDSmem {
  static constexpr int CODES = KD_PIECE * HD / 2;             // of keys, or of values
  static constexpr int PARAMS = KD_PIECE * (HD / KV4_GROUP) * 4;
  static constexpr int OFF_PK = 2 * CODES;
  static constexpr int OFF_Q = 2 * CODES + 2 * PARAMS;
  static constexpr int STAGE = OFF_Q + NT * 8 * HD * 2;       // a multiple of 128 bytes
  static constexpr int MROW = HD + 4;                         // a head's sums and (maximum, sum of weights)
  static constexpr int OFF_MERGE = KD_STAGES * STAGE;
  static constexpr int OFF_BAR = OFF_MERGE + KD_WARPS * NT * 8 * MROW * 4;
  static constexpr int TOTAL = OFF_BAR + KD_STAGES * (8 + 8 + 4) + 128;
};

// The sequence that piece u (over all heads) belongs to: the last one with plan[b] * nkv <= u. The whole warp searches, 32 places a round.
__device__ __forceinline__ int kd_locate(const int* plan, int B, int nkv, long long u) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = B;
  while (n > 1) {
    const int step = (n + 31) / 32, at = lo + lane * step;
    const bool le = lane * step < n && static_cast<long long>(plan[at]) * nkv <= u;
    const uint32_t mask = __ballot_sync(0xffffffffu, le);
    const int k = mask == 0 ? 0 : 31 - __clz(mask);
    lo += k * step;
    n = min(step, n - k * step);
  }
  return lo;
}

struct KDRun {
  long long first, end;  // this CTA's pieces
};
__device__ __forceinline__ long long kd_total(const VbKv4Decode& p) {
  const long long most = static_cast<long long>(p.B) * ((static_cast<long long>(p.width) * p.block_size + KD_PIECE - 1) / KD_PIECE);
  return min(max(static_cast<long long>(p.plan[p.B]), 0LL), most) * p.nkv;
}
__device__ __forceinline__ long long kd_per(long long total, int ctas) { return max(static_cast<long long>(KD_MIN_PIECES), (total + ctas - 1) / ctas); }
__device__ __forceinline__ long long kd_len(const VbKv4Decode& p, int b) {
  return min(static_cast<long long>(max(p.ctx[b], 0)), static_cast<long long>(p.width) * p.block_size);
}

// One (sequence, head) of a run.
struct KDSegment {
  int b, kvh;
  long long base, n;  // its first piece and how many it has, in the numbering over everything
  __device__ __forceinline__ void find(const VbKv4Decode& p, int b_, long long u) {
    b = b_;
    while (b + 1 < p.B && static_cast<long long>(p.plan[b + 1]) * p.nkv <= u) ++b;
    const long long at = static_cast<long long>(p.plan[b]) * p.nkv;
    n = max(static_cast<long long>(p.plan[b + 1]) - p.plan[b], 1LL);
    kvh = static_cast<int>(min(max((u - at) / n, 0LL), static_cast<long long>(p.nkv - 1)));
    base = at + kvh * n;
  }
};

template <int HD, int NT, typename T>
__global__ void __launch_bounds__(KD_THREADS, NT == 1 ? 3 : 2)
kv4_decode_kernel(const VbKv4Decode p, int* status) {
  using L = KDSmem<HD, NT>;
  constexpr int HEADS = NT * 8, CPR = HD / 4, VPR = HD / 8, KW = CPR / 8, VW = VPR / 8;  // channels of a thread's run, and words of them
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* empty = full + KD_STAGES;
  uint32_t* absent = reinterpret_cast<uint32_t*>(empty + KD_STAGES);  // per stage: the pages of its piece that do not exist
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = p.nh / p.nkv, bs = p.block_size;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const long long total = kd_total(p), per = kd_per(total, gridDim.x);
  const long long u0 = blockIdx.x * per, u1 = min(total, u0 + per);
  if (u0 >= u1) return;
  if (threadIdx.x == 0) {
    for (int s = 0; s < KD_STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], KD_WARPS);
    }
    mbar_fence_init();
  }
  __syncthreads();

  if (warp == KD_WARPS) {
    // ---- the warp that loads: 4 lanes per page of a piece (keys' codes, values' codes, keys' parameters, values' parameters)
    const int pages = bs < KD_PIECE ? KD_PIECE / bs : 1, lanes = 4 * pages, batch = 32 / lanes;
    const int page = (lane % lanes) >> 2, what = lane & 3, tokens = min(bs, KD_PIECE);
    const uint32_t bytes = what < 2 ? tokens * HD / 2 : tokens * (HD / KV4_GROUP) * 4;
    const int dst_off = (what < 2 ? what * L::CODES : L::OFF_PK + (what - 2) * L::PARAMS) + page * bytes;
    const int src_off = what < 2 ? kv4_codes_at(bs, HD, what) : kv4_params_at(bs, HD, what - 2);
    KDSegment g;
    g.b = kd_locate(p.plan, p.B, p.nkv, u0);
    bool ok = true;
    long long done = 0;
    for (long long u = u0; u < u1 && ok; u += batch) {
      const long long mine = min(u + lane / lanes, u1 - 1);
      g.find(p, g.b, mine);
      const long long piece = max(mine - g.base, 0LL);
      const long long tok = piece * KD_PIECE + page * bs;  // first token of this lane's page (of its 64, for larger blocks)
      const bool inside = tok < kd_len(p, g.b);            // pages behind the context are not looked up
      int blk = -1;
      if (inside) blk = p.table[g.b * p.ldt + tok / bs];
      const bool there = blk >= 0 && blk < p.num_blocks;
      const uint8_t* src = p.pages + (static_cast<long long>(max(blk, 0)) * p.nkv + g.kvh) * kv4_page_bytes(bs, HD) + src_off +
                           static_cast<int>(tok % bs) * (what < 2 ? HD / 2 : (HD / KV4_GROUP) * 4);
      const bool first = mine == u0 || piece == 0;
      const uint32_t copies = __ballot_sync(0xffffffffu, there && what == 0), lost = __ballot_sync(0xffffffffu, inside && !there && what == 0);
      for (int i = 0; i < batch && u + i < u1; ++i) {
        const long long k = u + i - u0;
        const int s = static_cast<int>(k % KD_STAGES);
        if (k >= KD_STAGES) ok = __all_sync(0xffffffffu, mbar_wait(&empty[s], static_cast<uint32_t>((k / KD_STAGES - 1) & 1)));
        if (!ok) break;
        uint8_t* stage = smem + s * L::STAGE;
        if (lane == i * lanes) {
          const uint32_t group = lanes == 32 ? 0xffffffffu : ((1u << lanes) - 1) << lane;
          uint32_t gone = 0;
          for (int j = 0; j < pages; ++j) gone |= ((lost >> (lane + 4 * j)) & 1u) << j;
          absent[s] = gone;
          mbar_expect_tx(&full[s], __popc(copies & group) * tokens * (HD + HD / 4) + (first ? G * HD * 2 : 0));
          if (first) bulk_load(stage + L::OFF_Q, static_cast<const T*>(p.q) + g.b * p.ldq + static_cast<long long>(g.kvh) * G * HD, G * HD * 2, &full[s]);
        }
        __syncwarp();
        if (lane / lanes == i && there) bulk_load(stage + dst_off, src, bytes, &full[s]);
        done = k + 1;
      }
      g.b = __shfl_sync(0xffffffffu, g.b, min(batch, static_cast<int>(min(u1 - u, 32LL))) * lanes - 1);
    }
    if (!ok && lane == 0) atomicExch(status, ST_TIMEOUT_PRODUCER);
    // no copy is in flight when the CTA ends, not even where a wait ran out
    for (long long k = max(done - KD_STAGES, 0LL); k < done; ++k) mbar_wait(&full[k % KD_STAGES], static_cast<uint32_t>((k / KD_STAGES) & 1));
    return;
  }

  // ---- the warps that compute
  const int r = lane >> 2, c = lane & 3;
  const int krow = (r & 1) * 4 + (r >> 1);  // row r of S^T is this token of the first 8, row r + 8 the same of the others: a thread's
                                            // share of V^T (rows 2c, 2c + 1, 2c + 8, 2c + 9) is then tokens c, c + 4, c + 8, c + 12
  float* merge = reinterpret_cast<float*>(smem + L::OFF_MERGE);
  uint32_t qf[NT][KW][4];                   // a word's four pairs of channels (0, 4), (1, 5), (2, 6), (3, 7)
  float o[NT][HD / 16][4], m[NT][2], l[NT][2], sc[NT][2];
  KDSegment g;
  long long len = 0, seg_end = u0, seg_first = u0;
  g.b = kd_locate(p.plan, p.B, p.nkv, u0);
  bool ok = true;
  for (long long u = u0; u < u1; ++u) {
    const long long k = u - u0;
    const int s = static_cast<int>(k % KD_STAGES);
    const uint8_t* stage = smem + s * L::STAGE;
    const bool fresh = u == seg_end;
    if (fresh) {
      g.find(p, g.b, u);
      seg_first = u;
      seg_end = min(u1, max(g.base + g.n, u + 1));
      len = kd_len(p, g.b);
    }
    if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&full[s], static_cast<uint32_t>((k / KD_STAGES) & 1)));  // else: no more work, the barriers only
    if (fresh) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int head = t * 8 + r;
        const T* q = reinterpret_cast<const T*>(stage + L::OFF_Q) + head * HD + c * CPR;
        float x[CPR], big = 0.f;
#pragma unroll
        for (int j = 0; j < CPR; ++j) {
          x[j] = head < G ? static_cast<float>(q[j]) : 0.f;
          big = fmaxf(big, fabsf(x[j]));
        }
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
        // largest value into [2^14, 2^15): fp16 then holds all 11 bits of what is at least 2^-28 of it
        const int e = max(static_cast<int>(__float_as_uint(big) >> 23) - 127, -100);
        const float f = __uint_as_float(static_cast<uint32_t>(14 - e + 127) << 23);
#pragma unroll
        for (int w = 0; w < KW; ++w)
#pragma unroll
          for (int j = 0; j < 4; ++j) qf[t][w][j] = h2_bits(__floats2half2_rn(x[w * 8 + j] * f, x[w * 8 + j + 4] * f));
        const float back = p.scale * 1.4426950408889634f * __uint_as_float(static_cast<uint32_t>(e - 14 + 127) << 23);
        sc[t][0] = __shfl_sync(0xffffffffu, back, 8 * c);
        sc[t][1] = __shfl_sync(0xffffffffu, back, 8 * c + 4);
        m[t][0] = m[t][1] = -INFINITY;
        l[t][0] = l[t][1] = 0.f;
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) o[t][i][0] = o[t][i][1] = o[t][i][2] = o[t][i][3] = 0.f;
      }
    }
    const long long left = len - (u - g.base) * KD_PIECE - warp * 16;  // tokens of this warp's 16 that count
    uint32_t gone = absent[s];
    if (bs < KD_PIECE) gone >>= warp * 16 / bs;
    if (ok && left > 0 && !(gone & 1u)) {
      const int t0 = warp * 16;
      const uint8_t* kc = stage + (t0 + krow) * (HD / 2) + c * (CPR / 2);
      const uint8_t* kp = stage + L::OFF_PK + ((t0 + krow) * (HD / KV4_GROUP) + c * CPR / KV4_GROUP) * 4;
      uint32_t wk[2][KW];
      __half2 ks[2], km[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if constexpr (KW == 4) {
          const uint4 v = *reinterpret_cast<const uint4*>(kc + h * 8 * (HD / 2));
          wk[h][0] = v.x; wk[h][1] = v.y; wk[h][2] = v.z; wk[h][3] = v.w;
        } else {
          const uint2 v = *reinterpret_cast<const uint2*>(kc + h * 8 * (HD / 2));
          wk[h][0] = v.x; wk[h][1] = v.y;
        }
        const __half2 par = *reinterpret_cast<const __half2*>(kp + h * 8 * (HD / KV4_GROUP) * 4);
        ks[h] = __low2half2(par);
        km[h] = __high2half2(par);
      }
      float st[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t) st[t][0] = st[t][1] = st[t][2] = st[t][3] = 0.f;
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        const uint32_t a = wk[0][w], b = wk[1][w], a8 = a >> 8, b8 = b >> 8;
        const uint32_t a0 = codes_even(a, ks[0], km[0]), a1 = codes_even(b, ks[1], km[1]), a2 = codes_odd(a, ks[0], km[0]), a3 = codes_odd(b, ks[1], km[1]);
        const uint32_t b0 = codes_even(a8, ks[0], km[0]), b1 = codes_even(b8, ks[1], km[1]), b2 = codes_odd(a8, ks[0], km[0]),
                       b3 = codes_odd(b8, ks[1], km[1]);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          mma_f16_16816(st[t], a0, a1, a2, a3, qf[t][w][0], qf[t][w][1]);
          mma_f16_16816(st[t], b0, b1, b2, b3, qf[t][w][2], qf[t][w][3]);
        }
      }
      // values: this thread's run of channels of four tokens
      const uint8_t* vc = stage + L::CODES + (t0 + c) * (HD / 2) + r * (VPR / 2);
      const uint8_t* vp = stage + L::OFF_PK + L::PARAMS + ((t0 + c) * (HD / KV4_GROUP) + r * VPR / KV4_GROUP) * 4;
      uint32_t wv[4][VW], pv[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (VW == 2) {
          const uint2 v = *reinterpret_cast<const uint2*>(vc + j * 4 * (HD / 2));
          wv[j][0] = v.x; wv[j][1] = v.y;
        } else {
          wv[j][0] = *reinterpret_cast<const uint32_t*>(vc + j * 4 * (HD / 2));
        }
        pv[j] = *reinterpret_cast<const uint32_t*>(vp + j * 4 * (HD / KV4_GROUP) * 4);
      }
      if (left < 16) {  // what lies behind the context may be anything: no score (below), and values of zero
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c + 4 * j >= left) pv[j] = 0u;
      }
      uint32_t pb[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float alpha[2], e[4];
        bool grew = false;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          st[t][h] *= sc[t][h];
          st[t][2 + h] *= sc[t][h];
          if (left < 16) {
            if (krow >= left) st[t][h] = -INFINITY;
            if (krow + 8 >= left) st[t][2 + h] = -INFINITY;
          }
          float mx = fmaxf(st[t][h], st[t][2 + h]);
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          const float mn = fmaxf(m[t][h], mx);
          grew |= mn > m[t][h];
          alpha[h] = m[t][h] == -INFINITY ? 0.f : fast_exp2(m[t][h] - mn);
          const float mu = mn == -INFINITY ? 0.f : mn;
          e[h] = fast_exp2(st[t][h] - mu);
          e[2 + h] = fast_exp2(st[t][2 + h] - mu);
          l[t][h] = l[t][h] * alpha[h] + (e[h] + e[2 + h]);
          m[t][h] = mn;
        }
        pb[t][0] = movmatrix_t(h2_bits(__floats2half2_rn(e[0], e[1])));
        pb[t][1] = movmatrix_t(h2_bits(__floats2half2_rn(e[2], e[3])));
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
          for (int i = 0; i < HD / 16; ++i) {
            o[t][i][0] *= alpha[0]; o[t][i][1] *= alpha[1];
            o[t][i][2] *= alpha[0]; o[t][i][3] *= alpha[1];
          }
        }
      }
      const __half2 s01 = h2_of(__byte_perm(pv[0], pv[1], 0x5410)), m01 = h2_of(__byte_perm(pv[0], pv[1], 0x7632));
      const __half2 s23 = h2_of(__byte_perm(pv[2], pv[3], 0x5410)), m23 = h2_of(__byte_perm(pv[2], pv[3], 0x7632));
#pragma unroll
      for (int w = 0; w < VW; ++w)
#pragma unroll
        for (int half = 0; half < 2; ++half) {  // channels 0..3 and 4..7 of the word: a pair of tokens side by side
          const uint32_t sel = half == 0 ? 0x5410 : 0x7632;
          const uint32_t x = __byte_perm(wv[0][w], wv[1][w], sel), y = __byte_perm(wv[2][w], wv[3][w], sel), x8 = x >> 8, y8 = y >> 8;
          const uint32_t a0 = codes_even(x, s01, m01), a1 = codes_odd(x, s01, m01), a2 = codes_even(y, s23, m23), a3 = codes_odd(y, s23, m23);
          const uint32_t b0 = codes_even(x8, s01, m01), b1 = codes_odd(x8, s01, m01), b2 = codes_even(y8, s23, m23), b3 = codes_odd(y8, s23, m23);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            mma_f16_16816(o[t][w * 4 + half * 2], a0, a1, a2, a3, pb[t][0], pb[t][1]);
            mma_f16_16816(o[t][w * 4 + half * 2 + 1], b0, b1, b2, b3, pb[t][0], pb[t][1]);
          }
        }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[s]);
    if (u + 1 < seg_end) continue;

    // ---- end of a segment: the four warps' sums meet. O^T[channel r VPR + 2 i (+ 1), head]
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float sum = l[t][h];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        float* row = merge + (warp * HEADS + t * 8 + 2 * c + h) * L::MROW;
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) *reinterpret_cast<float2*>(row + r * VPR + 2 * i) = make_float2(o[t][i][h], o[t][i][2 + h]);
        if (r == 0) {
          row[HD] = m[t][h];
          row[HD + 1] = sum;
        }
      }
    asm volatile("bar.sync 1, %0;" ::"n"(KD_WARPS * 32) : "memory");
    const bool whole = seg_first == g.base && seg_end == g.base + g.n;
    float* part = p.part + (2LL * blockIdx.x + (seg_first == u0 ? 0 : 1)) * G * (HD + 2);
    for (int i = threadIdx.x; i < G * HD; i += KD_WARPS * 32) {
      const int head = i / HD, d = i % HD;
      const float* row = merge + head * L::MROW;
      float M = -INFINITY, sum = 0.f, acc = 0.f;
#pragma unroll
      for (int w = 0; w < KD_WARPS; ++w) M = fmaxf(M, row[w * HEADS * L::MROW + HD]);
#pragma unroll
      for (int w = 0; w < KD_WARPS; ++w) {
        const float* rw = row + w * HEADS * L::MROW;
        const float f = rw[HD] == -INFINITY ? 0.f : fast_exp2(rw[HD] - M);
        sum += rw[HD + 1] * f;
        acc += rw[d] * f;
      }
      if (whole) {
        static_cast<T*>(p.out)[(static_cast<long long>(g.b) * p.nh + g.kvh * G + head) * HD + d] = static_cast<T>(sum == 0.f ? 0.f : acc / sum);
      } else {
        part[head * (HD + 2) + d] = acc;
        if (d == 0) {
          part[head * (HD + 2) + HD] = M;
          part[head * (HD + 2) + HD + 1] = sum;
        }
      }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(KD_WARPS * 32) : "memory");
  }
  if (!ok && lane == 0) atomicExch(status, ST_TIMEOUT_EPILOGUE);
}

// Joins the runs of every (sequence, head) that more than one CTA worked on, and writes zeros for contexts of no tokens.
template <int HD, typename T>
__global__ void __launch_bounds__(HD)
kv4_join_kernel(const VbKv4Decode p, int ctas) {
  __shared__ float red[HD / 32];
  __shared__ float wgt[HD];
  const int b = blockIdx.y, h = blockIdx.x, G = p.nh / p.nkv, kvh = h / G, head = h % G;
  const long long total = kd_total(p), per = kd_per(total, ctas);
  const long long n = static_cast<long long>(p.plan[b + 1]) - p.plan[b];
  T* out = static_cast<T*>(p.out) + (static_cast<long long>(b) * p.nh + h) * HD + threadIdx.x;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the runs' sums, and what came before them
  if (n <= 0 || kd_len(p, b) == 0) {
    *out = static_cast<T>(0.f);
    return;
  }
  const long long base = static_cast<long long>(p.plan[b]) * p.nkv + kvh * n;
  const long long i0 = base / per, i1 = min((base + n - 1) / per, static_cast<long long>(ctas - 1));
  if (i0 >= i1) return;
  const auto slot = [&](long long i) { return p.part + ((2 * i + (i * per >= base ? 0 : 1)) * G + head) * (HD + 2); };
  float M = -INFINITY;
  for (long long i = i0 + threadIdx.x; i <= i1; i += HD) M = fmaxf(M, slot(i)[HD]);
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, k));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = M;
  __syncthreads();
  M = red[0];
#pragma unroll
  for (int w = 1; w < HD / 32; ++w) M = fmaxf(M, red[w]);
  float acc = 0.f, sum = 0.f;
  for (long long at = i0; at <= i1; at += HD) {
    const int k = static_cast<int>(min(static_cast<long long>(HD), i1 - at + 1));
    __syncthreads();
    if (threadIdx.x < k) {
      const float mi = slot(at + threadIdx.x)[HD];
      wgt[threadIdx.x] = mi == -INFINITY ? 0.f : fast_exp2(mi - M);
    }
    __syncthreads();
#pragma unroll 8
    for (int i = 0; i < k; ++i) {
      const float* s = slot(at + i);
      acc += wgt[i] * s[threadIdx.x];
      sum += wgt[i] * s[HD + 1];
    }
  }
  *out = static_cast<T>(sum == 0.f ? 0.f : acc / sum);
}

// Pieces in front of every sequence, for calls without a plan.
__global__ void __launch_bounds__(1024)
kv4_plan_kernel(const VbKv4Decode p) {
  __shared__ int red[32];
  int carry = 0;
  if (threadIdx.x == 0) p.plan_ws[0] = 0;
  for (int base = 0; base < p.B; base += 1024) {
    const int b = base + threadIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int v = b < p.B ? static_cast<int>((kd_len(p, b) + KD_PIECE - 1) / KD_PIECE) : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += x;
    }
    __syncthreads();
    if (lane == 31) red[warp] = v;
    __syncthreads();
    int w = red[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += x;
    }
    const int before = __shfl_sync(0xffffffffu, w, max(warp - 1, 0));
    if (b < p.B) p.plan_ws[b + 1] = carry + v + (warp > 0 ? before : 0);
    carry += __shfl_sync(0xffffffffu, w, 31);
  }
}

template <int HD, int NT, typename T>
static cudaError_t kd_launch(const VbKv4Decode& p, int* status, cudaStream_t s) {
  auto kern = kv4_decode_kernel<HD, NT, T>;
  constexpr int smem = KDSmem<HD, NT>::TOTAL;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  const int ctas = num_sms() * (NT == 1 ? 3 : 2);
  kern<<<ctas, KD_THREADS, smem, s>>>(p, status);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(p.nh, p.B);
  cfg.blockDim = dim3(HD);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv4_join_kernel<HD, T>, p, ctas);
}

template <typename T>
static cudaError_t kd_dispatch(const VbKv4Decode& p, int* status, cudaStream_t s) {
  const bool wide = p.nh / p.nkv > 8;
  if (p.hd == 128) return wide ? kd_launch<128, 2, T>(p, status, s) : kd_launch<128, 1, T>(p, status, s);
  return wide ? kd_launch<64, 2, T>(p, status, s) : kd_launch<64, 1, T>(p, status, s);
}

}  // namespace vb

using namespace vb;

extern "C" long long vb_kv4_decode_scratch(int B, int nh, int nkv, int hd) {
  const int G = nh / nkv;
  return 2LL * num_sms() * (G <= 8 ? 3 : 2) * G * (hd + 2);
}

extern "C" int vb_kv4_status() {
  int h[4] = {0, 0, 0, 0};
  if (cudaMemcpyFromSymbol(h, g_kv4_status, sizeof(h)) != cudaSuccess) return -1;
  if (h[0] != 0) {
    int z[4] = {0, 0, 0, 0};
    cudaMemcpyToSymbol(g_kv4_status, z, sizeof(z));
  }
  return h[0];
}

extern "C" int vb_kv4_decode(const VbKv4Decode* a, cudaStream_t s) {
  if (a->B == 0) return 0;
  if ((a->hd != 64 && a->hd != 128) || a->nh % a->nkv || a->nh / a->nkv > 16 || a->B > 65535) return -2;
  VbKv4Decode p = *a;
  int* status = nullptr;
  cudaError_t e = cudaGetSymbolAddress(reinterpret_cast<void**>(&status), g_kv4_status);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (p.plan == nullptr) {
    kv4_plan_kernel<<<1, 1024, 0, s>>>(p);
    e = cudaGetLastError();
    if (e != cudaSuccess) return static_cast<int>(e);
    p.plan = p.plan_ws;
    verl_count_launches(1);
  }
  verl_count_launches(2);
  e = p.type == 0 ? kd_dispatch<__nv_bfloat16>(p, status, s) : kd_dispatch<__half>(p, status, s);
  return static_cast<int>(e);
}
