// Attention of one query token per sequence over the 4-bit cache (layout: kv4_common.cuh): one pass over the codes, running maximum and sum.
//
// Work: contexts are cut into pieces of 64 tokens; the pieces of all (sequence, KV head) pairs, laid end to end, are dealt to the CTAs of one
// wave in equal runs, whatever the lengths are (the plan holds the pieces in front of every sequence). A CTA that starts or ends inside a
// (sequence, head) leaves its sums in a slot of its own, and a second small launch, started early by programmatic dependence, joins them
// by their maxima, in the order of the runs: no atomics, the same bits every time.
//
// A CTA: one warp brings pieces into a ring of shared memory by bulk copies (a piece is at most 16 contiguous runs; four for blocks of 64 and
// more); four warps take one piece after the other, each by itself, and meet at the end of a segment.
//   S^T[64 tokens, 8 heads] = K[64, hd] Q^T        keys are the A operand of m16n8k16: a thread's share of a token's row is one contiguous run
//   O^T[hd, 8 heads]       += V^T[hd, 64] P^T      values are the A operand as well; P^T is S^T's accumulator through movmatrix
// so that with up to 8 heads to a KV head a matrix instruction takes 256 cache elements (query heads as the 16 rows would take 128).
//
// A code becomes a number without a conversion: (w & 0x000f000f) | 0x5400.. is 64 + q / 16 in fp16 and (w & 0x00f000f0) | 0x4400.. is 4 + q / 16, so
// that one multiply-add, x s - 64 s, gives a pair of q s / 16, each rounded once (64 s is exact; it is finite because the append keeps s below 1024).
// The least values m of the groups go through the matrix unit apart from the codes:
//   S gains m (sum of q over the thread's channels), one more k step of an instruction that has m twice against that sum's two fp16 halves;
//   O gains sum_t p_t m_t, the same for all channels of a thread: one accumulator more, added at the end.
// 1.2 instructions an element. Queries are scaled by a power of two per head so that fp16 holds them exactly; weights are e^(s - max) <= 1 in fp16.
#include <math.h>

#include "kv4_common.cuh"
#include "rollout_ops.h"
#include "tcgen05_common.cuh"

namespace vb {

int num_sms();

constexpr int KD_PIECE = 64;
constexpr int KD_WARPS = 4;                      // warps that compute
constexpr int KD_THREADS = (KD_WARPS + 1) * 32;
constexpr int KD_STAGES = 2 * KD_WARPS;           // a stage belongs to one warp: its barrier's phases are then met one by one
constexpr int KD_CTAS = 2;                       // CTAs of an SM
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
// Factors of a pair of codes: their scales, and what 64 and 4 become under them.
struct Scales {
  __half2 s, n64, n4;
  __device__ __forceinline__ explicit Scales(__half2 v) : s(v), n64(__hmul2(v, __float2half2_rn(-64.f))), n4(__hmul2(v, __float2half2_rn(-4.f))) {}
};
// q s / 16 for pairs 0 / 1 of the four that a word of codes holds: its nibbles (0, 4) and (1, 5); the other two after a shift by 8
__device__ __forceinline__ uint32_t codes_even(uint32_t w, const Scales& f) {
  uint32_t x;
  asm("lop3.b32 %0, %1, 0x000f000f, 0x54005400, 0xea;" : "=r"(x) : "r"(w));
  return h2_bits(__hfma2(h2_of(x), f.s, f.n64));
}
__device__ __forceinline__ uint32_t codes_odd(uint32_t w, const Scales& f) {
  uint32_t x;
  asm("lop3.b32 %0, %1, 0x00f000f0, 0x44004400, 0xea;" : "=r"(x) : "r"(w));
  return h2_bits(__hfma2(h2_of(x), f.s, f.n4));
}

template <int HD, int NT>
struct KDSmem {
  static constexpr int CODES = KD_PIECE * HD / 2;             // of keys, or of values
  static constexpr int PARAMS = KD_PIECE * (HD / KV4_GROUP) * 4;
  static constexpr int OFF_PK = 2 * CODES;
  static constexpr int STAGE = 2 * CODES + 2 * PARAMS;        // a multiple of 128 bytes
  static constexpr int MROW = HD + 4;                         // a head's sums and (maximum, sum of weights)
  static constexpr int OFF_MERGE = KD_STAGES * STAGE;
  static constexpr int OFF_BAR = OFF_MERGE + KD_WARPS * 8 * MROW * 4;
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
__global__ void __launch_bounds__(KD_THREADS, KD_CTAS)
kv4_decode_kernel(const VbKv4Decode p, int* status) {
  using L = KDSmem<HD, NT>;
  constexpr int STEP = NT == 1 ? 4 : 2;  // 16-token tiles between two looks at the maximum: what the registers hold
  constexpr int CPR = HD / 4, VPR = HD / 8, KW = CPR / 8, VW = VPR / 8;  // channels of a thread's run, and words of them
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
      mbar_init(&empty[s], 1);
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
          mbar_expect_tx(&full[s], __popc(copies & group) * tokens * (HD + HD / 4));
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
  const int krow = (r & 1) * 4 + (r >> 1);  // row r of S^T is this token of the first 8 of 16, row r + 8 the same of the others: a thread's
                                            // share of V^T (rows 2c, 2c + 1, 2c + 8, 2c + 9) is then tokens c, c + 4, c + 8, c + 12
  float* merge = reinterpret_cast<float*>(smem + L::OFF_MERGE);
  int at = warp, stage_at = warp, round = 0;  // this warp's next piece, its stage (stages s, s + 4 .. are warp s's) and how often it was here
  KDSegment g;
  g.b = kd_locate(p.plan, p.B, p.nkv, u0);
  bool ok = true;
  for (long long seg = u0; seg < u1;) {
    g.find(p, g.b, seg);
    const long long seg_end = min(u1, max(g.base + g.n, seg + 1));
    const int stop = static_cast<int>(seg_end - u0);
    const long long len = kd_len(p, g.b), ahead = (u0 - g.base) * KD_PIECE;  // token of piece i: ahead + 64 i
    uint32_t qf[NT][KW][4], qs[NT];  // a word's four pairs of channels (0, 4), (1, 5), (2, 6), (3, 7); the run's sum / 16 in two halves
    float o[NT][HD / 16][4], z[NT][4], m[NT][2], l[NT][2], sc[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int head = t * 8 + r;
      float x[CPR], big = 0.f, sum = 0.f;
      if (head < G) {
        const uint4* q = reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + g.b * p.ldq + (static_cast<long long>(g.kvh) * G + head) * HD + c * CPR);
#pragma unroll
        for (int j = 0; j < CPR / 8; ++j) {
          const uint4 v = q[j];
          const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
          for (int i = 0; i < 8; ++i) x[j * 8 + i] = static_cast<float>(e[i]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < CPR; ++j) x[j] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < CPR; ++j) big = fmaxf(big, fabsf(x[j]));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
      // largest value into [2^10, 2^11): fp16 then holds all 11 bits of what is at least 2^-24 of it, and the sum of 32 channels
      const int e = max(static_cast<int>(__float_as_uint(big) >> 23) - 127, -100);
      const float f = __uint_as_float(static_cast<uint32_t>(10 - e + 127) << 23);
#pragma unroll
      for (int j = 0; j < CPR; ++j) {
        x[j] *= f;
        sum += x[j] * 0.0625f;
      }
#pragma unroll
      for (int w = 0; w < KW; ++w)
#pragma unroll
        for (int j = 0; j < 4; ++j) qf[t][w][j] = h2_bits(__floats2half2_rn(x[w * 8 + j], x[w * 8 + j + 4]));
      const float hi = __half2float(__float2half_rn(sum));
      qs[t] = h2_bits(__floats2half2_rn(hi, sum - hi));
      const float back = p.scale * (16.f * 1.4426950408889634f) * __uint_as_float(static_cast<uint32_t>(e - 10 + 127) << 23);
      sc[t][0] = __shfl_sync(0xffffffffu, back, 8 * c);
      sc[t][1] = __shfl_sync(0xffffffffu, back, 8 * c + 4);
      m[t][0] = m[t][1] = -INFINITY;
      l[t][0] = l[t][1] = 0.f;
      z[t][0] = z[t][1] = z[t][2] = z[t][3] = 0.f;
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) o[t][i][0] = o[t][i][1] = o[t][i][2] = o[t][i][3] = 0.f;
    }
    for (; at < stop; at += KD_WARPS) {
      const uint8_t* stage = smem + stage_at * L::STAGE;
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&full[stage_at], round & 1));  // else: no more work, the barriers only
      const uint32_t gone = absent[stage_at];
      const int left = static_cast<int>(min(len - (ahead + static_cast<long long>(at) * KD_PIECE), static_cast<long long>(KD_PIECE)));  // tokens that count
#pragma unroll 1
      for (int i0 = 0; ok && i0 < left; i0 += STEP * 16) {
        const bool ragged = left < i0 + STEP * 16 || gone != 0;
        // does token i of the step count?
        const auto counts = [&](int i) { return i0 + i < left && !((gone >> (bs < KD_PIECE ? (i0 + i) / bs : 0)) & 1u); };
        const uint8_t* kc = stage + (i0 + krow) * (HD / 2) + c * (CPR / 2);
        const uint8_t* kp = stage + L::OFF_PK + ((i0 + krow) * (HD / KV4_GROUP) + c * CPR / KV4_GROUP) * 4;
        float st[NT][STEP][4];
#pragma unroll
        for (int i = 0; i < STEP; ++i) {
          uint32_t wk[2][KW];
          __half2 par[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint8_t* at_k = kc + (i * 16 + h * 8) * (HD / 2);
            if constexpr (KW == 4) {
              const uint4 v = *reinterpret_cast<const uint4*>(at_k);
              wk[h][0] = v.x; wk[h][1] = v.y; wk[h][2] = v.z; wk[h][3] = v.w;
            } else {
              const uint2 v = *reinterpret_cast<const uint2*>(at_k);
              wk[h][0] = v.x; wk[h][1] = v.y;
            }
            par[h] = *reinterpret_cast<const __half2*>(kp + (i * 16 + h * 8) * (HD / KV4_GROUP) * 4);
          }
          const Scales f0(__low2half2(par[0])), f1(__low2half2(par[1]));
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            st[t][i][0] = st[t][i][1] = st[t][i][2] = st[t][i][3] = 0.f;
            mma_f16_16816(st[t][i], h2_bits(__high2half2(par[0])), h2_bits(__high2half2(par[1])), 0u, 0u, qs[t], 0u);
          }
#pragma unroll
          for (int w = 0; w < KW; ++w) {
            const uint32_t a = wk[0][w], b = wk[1][w], a8 = a >> 8, b8 = b >> 8;
            const uint32_t a0 = codes_even(a, f0), a1 = codes_even(b, f1), a2 = codes_odd(a, f0), a3 = codes_odd(b, f1);
            const uint32_t b0 = codes_even(a8, f0), b1 = codes_even(b8, f1), b2 = codes_odd(a8, f0), b3 = codes_odd(b8, f1);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              mma_f16_16816(st[t][i], a0, a1, a2, a3, qf[t][w][0], qf[t][w][1]);
              mma_f16_16816(st[t][i], b0, b1, b2, b3, qf[t][w][2], qf[t][w][3]);
            }
          }
        }
        uint32_t pb[NT][STEP][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          float alpha[2];
          bool grew = false;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < STEP; ++i) {
              st[t][i][h] *= sc[t][h];
              st[t][i][2 + h] *= sc[t][h];
            }
            if (ragged) {  // what does not count may be anything
#pragma unroll
              for (int i = 0; i < STEP; ++i) {
                if (!counts(i * 16 + krow)) st[t][i][h] = -INFINITY;
                if (!counts(i * 16 + krow + 8)) st[t][i][2 + h] = -INFINITY;
              }
            }
            float mx = m[t][h];
#pragma unroll
            for (int i = 0; i < STEP; ++i) mx = fmaxf(mx, fmaxf(st[t][i][h], st[t][i][2 + h]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            grew |= mx > m[t][h];
            alpha[h] = m[t][h] == -INFINITY ? 0.f : fast_exp2(m[t][h] - mx);
            m[t][h] = mx;
            const float mu = mx == -INFINITY ? 0.f : mx;
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < STEP; ++i) {
              st[t][i][h] = fast_exp2(st[t][i][h] - mu);
              st[t][i][2 + h] = fast_exp2(st[t][i][2 + h] - mu);
              sum += st[t][i][h] + st[t][i][2 + h];
            }
            l[t][h] = l[t][h] * alpha[h] + sum;
          }
#pragma unroll
          for (int i = 0; i < STEP; ++i) {
            pb[t][i][0] = movmatrix_t(h2_bits(__floats2half2_rn(st[t][i][0], st[t][i][1])));
            pb[t][i][1] = movmatrix_t(h2_bits(__floats2half2_rn(st[t][i][2], st[t][i][3])));
          }
          if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
            for (int i = 0; i < HD / 16; ++i) {
              o[t][i][0] *= alpha[0]; o[t][i][1] *= alpha[1];
              o[t][i][2] *= alpha[0]; o[t][i][3] *= alpha[1];
            }
            z[t][0] *= alpha[0]; z[t][1] *= alpha[1];
          }
        }
        // values: this thread's run of channels of four tokens at a time
        const uint8_t* vc = stage + L::CODES + (i0 + c) * (HD / 2) + r * (VPR / 2);
        const uint8_t* vp = stage + L::OFF_PK + L::PARAMS + ((i0 + c) * (HD / KV4_GROUP) + r * VPR / KV4_GROUP) * 4;
#pragma unroll
        for (int i = 0; i < STEP; ++i) {
          uint32_t wv[4][VW], pv[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint8_t* at_v = vc + (i * 16 + j * 4) * (HD / 2);
            if constexpr (VW == 2) {
              const uint2 v = *reinterpret_cast<const uint2*>(at_v);
              wv[j][0] = v.x; wv[j][1] = v.y;
            } else {
              wv[j][0] = *reinterpret_cast<const uint32_t*>(at_v);
            }
            pv[j] = *reinterpret_cast<const uint32_t*>(vp + (i * 16 + j * 4) * (HD / KV4_GROUP) * 4);
          }
          if (ragged) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (!counts(i * 16 + j * 4 + c)) pv[j] = 0u;  // values of zero
          }
          const Scales f01(h2_of(__byte_perm(pv[0], pv[1], 0x5410))), f23(h2_of(__byte_perm(pv[2], pv[3], 0x5410)));
          const uint32_t m01 = __byte_perm(pv[0], pv[1], 0x7632), m23 = __byte_perm(pv[2], pv[3], 0x7632);
#pragma unroll
          for (int t = 0; t < NT; ++t) mma_f16_16816(z[t], m01, 0u, m23, 0u, pb[t][i][0], pb[t][i][1]);
#pragma unroll
          for (int w = 0; w < VW; ++w)
#pragma unroll
            for (int half = 0; half < 2; ++half) {  // channels 0..3 and 4..7 of the word: a pair of tokens side by side
              const uint32_t sel = half == 0 ? 0x5410 : 0x7632;
              const uint32_t x = __byte_perm(wv[0][w], wv[1][w], sel), y = __byte_perm(wv[2][w], wv[3][w], sel), x8 = x >> 8, y8 = y >> 8;
              const uint32_t a0 = codes_even(x, f01), a1 = codes_odd(x, f01), a2 = codes_even(y, f23), a3 = codes_odd(y, f23);
              const uint32_t b0 = codes_even(x8, f01), b1 = codes_odd(x8, f01), b2 = codes_even(y8, f23), b3 = codes_odd(y8, f23);
#pragma unroll
              for (int t = 0; t < NT; ++t) {
                mma_f16_16816(o[t][w * 4 + half * 2], a0, a1, a2, a3, pb[t][i][0], pb[t][i][1]);
                mma_f16_16816(o[t][w * 4 + half * 2 + 1], b0, b1, b2, b3, pb[t][i][0], pb[t][i][1]);
              }
            }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[stage_at]);
      stage_at += KD_WARPS;
      if (stage_at >= KD_STAGES) {
        stage_at -= KD_STAGES;
        ++round;
      }
    }

    // ---- end of a segment: the four warps' sums meet, 8 heads at a time. O^T[channel r VPR + 2 i (+ 1), head] = 16 o + z
    const bool whole = seg == g.base && seg_end == g.base + g.n;
    float* part = p.part + (2LL * blockIdx.x + (seg == u0 ? 0 : 1)) * G * (HD + 2);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float sum = l[t][h];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        float* row = merge + (warp * 8 + 2 * c + h) * L::MROW;
#pragma unroll
        for (int i = 0; i < HD / 16; ++i)
          *reinterpret_cast<float2*>(row + r * VPR + 2 * i) = make_float2(fmaf(16.f, o[t][i][h], z[t][h]), fmaf(16.f, o[t][i][2 + h], z[t][h]));
        if (r == 0) {
          row[HD] = m[t][h];
          row[HD + 1] = sum;
        }
      }
      asm volatile("bar.sync 1, %0;" ::"n"(KD_WARPS * 32) : "memory");
      for (int i = threadIdx.x; i < min(G - t * 8, 8) * HD; i += KD_WARPS * 32) {
        const int d = i % HD, head = t * 8 + i / HD;
        const float* row = merge + (i / HD) * L::MROW;
        float M = -INFINITY, sum = 0.f, acc = 0.f;
#pragma unroll
        for (int w = 0; w < KD_WARPS; ++w) M = fmaxf(M, row[w * 8 * L::MROW + HD]);
#pragma unroll
        for (int w = 0; w < KD_WARPS; ++w) {
          const float* rw = row + w * 8 * L::MROW;
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
    seg = seg_end;
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
  const int ctas = num_sms() * KD_CTAS;
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
  return 2LL * num_sms() * KD_CTAS * G * (hd + 2);
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
