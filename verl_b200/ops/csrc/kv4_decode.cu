// Attention of one query token per sequence over the 4-bit cache (layout: kv4_common.cuh): one pass over the codes, running maximum and sum.
//
// Work: contexts are cut into pieces of 64 tokens; the pieces of all (sequence, KV head) pairs, laid end to end, are dealt to the warps of one
// wave in equal runs, whatever the lengths are (the plan holds the pieces in front of every sequence). A warp that starts or ends inside a
// (sequence, head) leaves its sums in a slot of its own, and a second small launch, started early by programmatic dependence, joins them
// by their maxima, in the order of the runs: no atomics, the same bits every time.
//
// No warp waits for another. Each has room for the keys and the values of one piece, which it fills by bulk copies (a half is at most 8
// contiguous runs, two for blocks of 64 and more): the next keys while it works on values, the next values while it works on keys.
//   S^T[64 tokens, 8 heads] = K[64, hd] Q^T        keys are the A operand of m16n8k16: a thread's share of a token's row is one contiguous run
//   O^T[hd, 8 heads]       += V^T[hd, 64] P^T      values are the A operand as well; P^T is S^T's accumulator through movmatrix
// so that with up to 8 heads to a KV head a matrix instruction takes 256 cache elements (query heads as the 16 rows would take 128).
//
// Codes become numbers without a conversion, two bytes at a time: a byte that holds codes (a, b) under the exponent of 64 is 64 + b + a / 16 in
// fp16, and 64 + a / 16 with b masked off, so that one multiply-add, x s - 64 s, gives a pair of (b + a / 16) s or of a s / 16, each rounded
// once (64 s is exact; it is finite because the append keeps s below 1024). b is not taken apart from a:
//   q_a a + q_b b = q_b (b + a / 16) + (16 q_a - q_b) a / 16        for keys, where the queries are brought into that form once a segment
//   sum p b       = sum p (b + a / 16) - sum p a / 16               for values, once at the end
// The least values m of the groups go through the matrix unit apart from the codes:
//   S gains m (sum of q over the thread's channels), one more k step of an instruction that has m twice against that sum's two fp16 halves;
//   O gains sum_t p_t m_t, the same for all channels of a thread: one accumulator more, added at the end.
// 1.1 instructions an element. Queries are scaled by a power of two per head, into fp16's range; weights are 2^(s - reference) <= 2^14 in fp16.
// These roundings to 11 bits (6e-4 of the output's norm in all) are below those of a bf16 output (1.7e-3); what one channel adds to a score is off by up
// to 2^-11 of itself, and the token's weight with it (a score of 14 from one channel: 7e-3). For fp16 (2.1e-4 by its own rounding) there are
// none: codes apart from each other, scales in two parts of at most seven bits, under which codes are exact, weights in two halves; values count from
// code 8, because the sum of codes and that of least values would each be hundreds of times their difference over a long context, and matrix
// instructions add up by cutting off. That takes two and three matrix instructions for one, and 1.75 times the time where instructions count.
//
// 320 sequences of 28 heads over 4 KV heads of 128 channels, 2560 tokens on average: 119 us for 525 MB with the join (0.68 of the copy rate; fp16 207),
// 4 of them for the reference that follows the scores. Neither HBM (57 %) nor the schedulers (0.51 instructions a cycle) are full: three warps to a
// scheduler, each of which goes through keys, softmax and values one behind the other, do not cover what they wait for. One sequence of 131072 tokens,
// 8 KV heads: 50 us for 168 MB (fp16 74), 8 of them the join's. Four of 160 tokens: 12 us, two launches.
#include <math.h>

#include <type_traits>

#include "kv4_common.cuh"
#include "rollout_ops.h"
#include "tcgen05_common.cuh"

namespace vb {

int num_sms();

constexpr int KD_PIECE = 64;                     // tokens that the plan counts in
constexpr int KD_WARPS = 4;
constexpr int KD_THREADS = KD_WARPS * 32;
constexpr int KD_TILES = KD_PIECE / 16;
// CTAs of an SM: three leave 168 registers a thread (four of 128: 129 us where three take 127); 16 heads of 128 channels need more (three: 68 us,
// with spills, where two take 59)
__host__ __device__ constexpr int kd_ctas(int hd, int nt) { return hd == 128 && nt == 2 ? 2 : 3; }
constexpr int KD_MIN_PIECES = 1;                 // shortest run of a warp
// The reference of a head's weights lies 2^8 below the largest score of the piece that set it: weights of up to 2^14 are as exact in fp16 as those of
// 1, and smaller ones keep 11 bits down to 2^-14. It is set again by a piece with a score 2^14 above it, and by one that has none above 2^-4: behind a
// token that outweighs all others, as the first one of a sequence often does, the others would be left with no bits, and where that token's
// value is small they are what the output consists of (a token of weight 0.9997 before 65536 others: bf16 and fp16 outputs off by 2e-2 with a reference
// that only rises). The sums may then grow to 2^60, which fp32 holds. Weights below 2^-32 of the largest one of their own piece are lost.
constexpr float KD_BELOW = 8.f, KD_HIGH = 14.f, KD_LOW = -4.f;
constexpr int KD_ROOM = 60;
constexpr int KD_FOLD = 64;                      // pieces after which a warp's sums of products go to shared memory

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
__device__ __forceinline__ void mma_f16_16816_from_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
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
// fp16 pairs as the 32 bits that they are
__device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
// Factors of a pair of codes: their scales, and what -64 becomes under them.
struct Scales {
  uint32_t s, n;
  __device__ __forceinline__ explicit Scales(uint32_t v) : s(v), n(mul2(v, 0xd400d400u)) {}
};
// The four pairs of a word w of codes 0 .. 7: (0, 4) / 16, (1, 5) + (0, 4) / 16, (2, 6) / 16, (3, 7) + (2, 6) / 16, times their scales.
// `magic` is 0x54005400 in a register: an instruction takes one constant.
__device__ __forceinline__ void kd_numbers(uint32_t (&x)[4], uint32_t w, const Scales& f, uint32_t magic) {
  const uint32_t high = __byte_perm(w, magic, 0x7351);  // bytes 1 and 3, each under the exponent
  asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xea;" : "=r"(x[0]) : "r"(w), "r"(magic));
  asm("lop3.b32 %0, %1, 0x00ff00ff, %2, 0xea;" : "=r"(x[1]) : "r"(w), "r"(magic));
  x[0] = fma2(x[0], f.s, f.n);
  x[1] = fma2(x[1], f.s, f.n);
  x[2] = fma2(high & 0xff0fff0fu, f.s, f.n);
  x[3] = fma2(high, f.s, f.n);
}

// For fp16 outputs, all of it exact: the codes apart from each other, and the scale in two parts of at most seven bits, under which a code is a
// number of at most eleven.
struct FineScales {
  Scales hi, lo;
  static __device__ __forceinline__ uint32_t rest(uint32_t v) {
    uint32_t d;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(v), "r"(v & 0xfff0fff0u));
    return d;
  }
  __device__ __forceinline__ explicit FineScales(uint32_t v) : hi(v & 0xfff0fff0u), lo(rest(v)) {}
};
__device__ __forceinline__ uint32_t add2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t minus2(uint32_t a) { return a ^ 0x80008000u; }
// The pairs (0, 4), (1, 5), (2, 6), (3, 7) of a word, x[0..3] times the first part of their scales and x[4..7] times the second. EIGHT: codes - 8, as
// products that a long sum does not take away from each other again.
template <bool EIGHT = false>
__device__ __forceinline__ void kd_numbers(uint32_t (&x)[8], uint32_t w, const FineScales& f, uint32_t magic) {
  const uint32_t up = w << 4;
  uint32_t c[4];
  asm("lop3.b32 %0, %1, 0x00f000f0, %2, 0xea;" : "=r"(c[0]) : "r"(up), "r"(magic));
  asm("lop3.b32 %0, %1, 0x00f000f0, %2, 0xea;" : "=r"(c[1]) : "r"(w), "r"(magic));
  c[2] = __byte_perm(up, magic, 0x7351) & 0xfff0fff0u;
  c[3] = __byte_perm(w, magic, 0x7351) & 0xfff0fff0u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (EIGHT) {
      c[i] = add2(c[i], 0xd480d480u);  // -72; times it the scale could be infinite
      x[i] = mul2(c[i], f.hi.s);
      x[4 + i] = mul2(c[i], f.lo.s);
    } else {
      x[i] = fma2(c[i], f.hi.s, f.hi.n);
      x[4 + i] = fma2(c[i], f.lo.s, f.lo.n);
    }
  }
}
template <bool EIGHT>
__device__ __forceinline__ void kd_numbers(uint32_t (&x)[4], uint32_t w, const Scales& f, uint32_t magic) {
  kd_numbers(x, w, f, magic);
}
// Least values with 8 scales added, as a rounded sum and what it leaves, which is exact
__device__ __forceinline__ void kd_least(uint32_t& m, uint32_t& rest, uint32_t scales) {
  const uint32_t e = mul2(scales, 0x48004800u), sum = add2(m, e), part = add2(sum, minus2(m));
  rest = add2(add2(m, minus2(add2(sum, minus2(part)))), add2(e, minus2(part)));
  m = sum;
}
// What is left of two numbers behind their fp16 roundings
__device__ __forceinline__ uint32_t pack2_rest(float lo, float hi, uint32_t rounded) {
  const __half2 h = *reinterpret_cast<const __half2*>(&rounded);
  return pack2(lo - __low2float(h), hi - __high2float(h));
}

template <int HD, int NT, bool FOLD>
struct KDSmem {
  static constexpr int CODES = KD_PIECE * HD / 2;             // of keys, or of values
  static constexpr int PARAMS = KD_PIECE * (HD / KV4_GROUP) * 4;
  static constexpr int OFF_PK = 2 * CODES;
  static constexpr int STAGE = 2 * CODES + 2 * PARAMS;        // of a warp, a multiple of 128 bytes
  static constexpr int SUMS = NT * (HD / 16 + 2) * 512;       // of a warp: four numbers a thread and sum, and the references that they are under
  static constexpr int OFF_SUMS = KD_WARPS * STAGE;
  static constexpr int OFF_BAR = OFF_SUMS + (FOLD ? KD_WARPS * SUMS : 0);
  static constexpr int TOTAL = OFF_BAR + KD_WARPS * 2 * 8;
};

// The sequence that piece u (over all heads) belongs to: the last one with plan[b] * nkv <= u. The whole warp searches, 32 places a round.
__device__ __forceinline__ int kd_locate(const int* plan, int B, int nkv, int u) {
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

// Pieces of everything and of a run. The launcher sees that pieces, and tokens of a table row, are counted in 31 bits.
__device__ __forceinline__ int kd_total(const VbKv4Decode& p) {
  return min(max(p.plan[p.B], 0), p.B * ((p.width * p.block_size + KD_PIECE - 1) / KD_PIECE)) * p.nkv;
}
__device__ __forceinline__ int kd_per(int total, int runs) { return max(KD_MIN_PIECES, (total + runs - 1) / runs); }
__device__ __forceinline__ int kd_len(const VbKv4Decode& p, int b) { return min(max(p.ctx[b], 0), p.width * p.block_size); }

// One (sequence, head).
struct KDSegment {
  int b, kvh, base, end, len;  // its pieces in the numbering over everything, its tokens
  __device__ __forceinline__ void find(const VbKv4Decode& p, int u) {
    while (b + 1 < p.B && p.plan[b + 1] * p.nkv <= u) ++b;
    const int at = p.plan[b] * p.nkv, n = max(p.plan[b + 1] - p.plan[b], 1);
    kvh = min(max(u - at, 0) / n, p.nkv - 1);
    base = at + kvh * n;
    end = max(base + n, u + 1);
    len = kd_len(p, b);
  }
};

// as mbar_wait, asleep up to 2 us at a time
__device__ __forceinline__ bool kd_try_wait(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 2000;\nselp.u32 %0, 1, 0, p;\n}\n"
               : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool kd_wait(uint64_t* full, uint32_t parity) {
  const uint32_t bar = smem_u32(full);
  if (kd_try_wait(bar, parity)) return true;
  const uint64_t t0 = global_timer_ns();
  while (!kd_try_wait(bar, parity))
    if (global_timer_ns() - t0 > VB_WAIT_LIMIT_NS) return false;
  return true;
}

template <int HD, int NT, bool FOLD, typename T>
__global__ void __launch_bounds__(KD_THREADS, kd_ctas(HD, NT))
kv4_decode_kernel(const VbKv4Decode p, int block_shift, int* status) {
  using L = KDSmem<HD, NT, FOLD>;
  constexpr bool FINE = std::is_same<T, __half>::value;  // numbers, queries and weights without a rounding that an output of 11 bits would show
  using Sc = std::conditional_t<FINE, FineScales, Scales>;
  constexpr int PARTS = FINE ? 2 : 1;
  constexpr int CPR = HD / 4, VPR = HD / 8, KW = CPR / 8, VW = VPR / 8;  // channels of a thread's run, and words of them
  extern __shared__ __align__(16) uint8_t smem[];  // 16 bytes are what bulk copies ask for
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = p.nh / p.nkv, bs = p.block_size;
  uint8_t* stage = smem + warp * L::STAGE;
  float4* sums = reinterpret_cast<float4*>(smem + L::OFF_SUMS + warp * L::SUMS) + lane;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR) + warp * 2;  // keys are there, values are there
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int run = blockIdx.x * KD_WARPS + warp, total = kd_total(p), per = kd_per(total, gridDim.x * KD_WARPS);
  if (static_cast<long long>(run) * per >= total) return;
  const int u0 = run * per, u1 = min(total - u0, per) + u0;  // this warp's pieces
  if (lane == 0) {
    mbar_init(&full[0], 1);
    mbar_init(&full[1], 1);
    mbar_fence_init();
  }
  __syncwarp();

  // ---- loading. Lanes 16 j .. 16 j + 15 look up and fetch the j-th of the warp's next two pieces: four lanes a page (keys' codes, values'
  // codes, keys' parameters, values' parameters), one, two or four pages a piece
  const int tokens = min(bs, KD_PIECE), page = (lane >> 2) & 3, what = lane & 3;
  const uint32_t row = what < 2 ? HD / 2 : (HD / KV4_GROUP) * 4, bytes = tokens * row;
  const int dst_off = (what < 2 ? what * L::CODES : L::OFF_PK + (what - 2) * L::PARAMS) + page * bytes;
  const int src_off = what < 2 ? kv4_codes_at(bs, HD, what) : kv4_params_at(bs, HD, what - 2);
  KDSegment ahead;  // of the piece that this lane looks up
  ahead.b = kd_locate(p.plan, p.B, p.nkv, u0);
  KDSegment g;
  g.b = ahead.b;
  g.end = u0;
  ahead.end = u0;
  const uint8_t* src = nullptr;  // what this lane fetches (null: nothing)
  bool missing = false;          // of a page that does not exist
  const auto look = [&](int u) {  // piece u is the first of the two; the answer is used half a piece later
    u += lane >> 4;
    src = nullptr;
    missing = false;
    if (u >= u1 || page * tokens >= KD_PIECE) return;
    if (u >= ahead.end) ahead.find(p, u);
    const int tok = (u - ahead.base) * KD_PIECE + page * tokens;
    if (tok < 0 || tok >= ahead.len) return;
    const int blk = p.table[ahead.b * p.ldt + (tok >> block_shift)];
    missing = blk < 0 || blk >= p.num_blocks;
    if (!missing)
      src = p.pages + (static_cast<long long>(blk) * p.nkv + ahead.kvh) * kv4_page_bytes(bs, HD) + src_off + (tok & (bs - 1)) * row;
  };
  uint32_t there = 0, gone = 0;  // lanes that fetch, and that miss a page
  const auto look_all = [&](int u) {
    look(u);
    there = __ballot_sync(0xffffffffu, src != nullptr);
    gone = __ballot_sync(0xffffffffu, missing);
  };
  const auto load = [&](int j, int value) {  // keys or values of the j-th of the two; returns the pages of it that do not exist (bits 0, 4, 8, 12)
    const uint32_t codes = 0x1111u << (16 * j + value);  // the lanes of its codes
    if (lane == 0) mbar_expect_tx(&full[value], __popc(there & codes) * tokens * (HD / 2 + HD / 8));
    __syncwarp();
    if ((lane >> 4) == j && (what & 1) == value && src != nullptr) bulk_load(stage + dst_off, src, bytes, &full[value]);
    return (gone >> (16 * j + value)) & 0x1111u;
  };
  uint32_t lost = 0, lost_next = 0;
  look_all(u0);
  lost_next = load(0, 0);
  load(0, 1);
  int looked = 1;  // the next of the two

  // ---- computing
  const int r = lane >> 2, c = lane & 3;
  const int krow = (r & 1) * 4 + (r >> 1);  // row r of S^T is this token of the first 8 of 16, row r + 8 the same of the others: a thread's
                                            // share of V^T (rows 2c, 2c + 1, 2c + 8, 2c + 9) is then tokens c, c + 4, c + 8, c + 12
  uint32_t magic;
  asm volatile("mov.b32 %0, 0x54005400;" : "=r"(magic));
  uint32_t round = 0;  // pieces that were here
  bool ok = true;
  for (int u = u0; u < u1;) {
    const int seg = u;
    g.find(p, seg);
    const int seg_end = min(u1, g.end);
    uint32_t qf[NT][KW][4], qs[NT];  // per word of 8 channels: 16 q - q' and q' for (0, 4), (1, 5), (2, 6), (3, 7); the run's sum in two halves
    float o[NT][HD / 16][4], z[NT][4], m[NT][2], l[NT][2], sc[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int head = t * 8 + r;
      float x[CPR], big = 0.f, sum = 0.f;
      if (head < G) {
        const uint4* q = reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + g.b * p.ldq + (g.kvh * G + head) * HD + c * CPR);
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
      // largest magnitude into [2^9, 2^10): fp16 then holds all 11 bits of what is at least 2^-23 of it, 16 q - q', and the sum of 32 channels
      const int e = max(static_cast<int>(__float_as_uint(big) >> 23) - 127, -100);
      const float f = copysignf(__uint_as_float(static_cast<uint32_t>(9 - e + 127) << 23), p.scale);
#pragma unroll
      for (int j = 0; j < CPR; ++j) {
        x[j] *= f;
        sum += x[j];
      }
#pragma unroll
      for (int w = 0; w < KW; ++w)
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          if constexpr (FINE)
            qf[t][w][j] = pack2(x[w * 8 + j], x[w * 8 + j + 4]);
          else
            qf[t][w][j] = pack2(fmaf(16.f, x[w * 8 + j], -x[w * 8 + j + 1]), fmaf(16.f, x[w * 8 + j + 4], -x[w * 8 + j + 5]));
          qf[t][w][j + 1] = pack2(x[w * 8 + j + 1], x[w * 8 + j + 5]);
        }
      const float hi = __half2float(__float2half_rn(sum));
      qs[t] = pack2(hi, sum - hi);
      // not zero, so that -inf stays what it is under it
      const float back = fmaxf(fabsf(p.scale) * 1.4426950408889634f * __uint_as_float(static_cast<uint32_t>(e - 9 + 127) << 23), 1e-37f);
      sc[t][0] = __shfl_sync(0xffffffffu, back, 8 * c);
      sc[t][1] = __shfl_sync(0xffffffffu, back, 8 * c + 4);
      m[t][0] = m[t][1] = -INFINITY;
      l[t][0] = l[t][1] = 0.f;
      z[t][0] = z[t][1] = z[t][2] = z[t][3] = 0.f;
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) o[t][i][0] = o[t][i][1] = o[t][i][2] = o[t][i][3] = 0.f;
    }
    // Matrix instructions add up by cutting off, always towards zero: over thousands of tokens that is far more than what is left where values of either
    // sign cancel (131072 tokens a warp: outputs off by 1.6e-2 of their norm in bf16 and 2.8e-3 in fp16 beside their own rounding). So sums of KD_FOLD
    // pieces are added up here, rounded to nearest: 3.6e-4 and 5e-6 (of 32: 2.5e-4, 3e-6). Every thread has a place of its own in shared memory. `keep`: what is there is taken
    // along; `back`: it comes back into the registers.
    const auto fold = [&](bool keep, bool back) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float4* at = sums + t * (HD / 16 + 2) * 32;
        float f[2] = {0.f, 0.f};
        if (keep) {
          const float4 old = at[(HD / 16 + 1) * 32];
          f[0] = old.x == m[t][0] ? 1.f : fast_exp2(old.x - m[t][0]);
          f[1] = old.y == m[t][1] ? 1.f : fast_exp2(old.y - m[t][1]);
        }
#pragma unroll
        for (int i = 0; i <= HD / 16; ++i) {
          float (&a)[4] = i < HD / 16 ? o[t][i < HD / 16 ? i : 0] : z[t];
          if (keep) {
            const float4 old = at[i * 32];
            a[0] = fmaf(old.x, f[0], a[0]);
            a[1] = fmaf(old.y, f[1], a[1]);
            a[2] = fmaf(old.z, f[0], a[2]);
            a[3] = fmaf(old.w, f[1], a[3]);
          }
          if (!back) {
            at[i * 32] = make_float4(a[0], a[1], a[2], a[3]);
            a[0] = a[1] = a[2] = a[3] = 0.f;
          }
        }
        if (!back) at[(HD / 16 + 1) * 32] = make_float4(m[t][0], m[t][1], 0.f, 0.f);
      }
    };
    for (; u < seg_end; ++u, ++round) {
      const int next = u + 1, done = u - seg;
      if (FOLD && done > 0 && done % KD_FOLD == 0) fold(done > KD_FOLD, false);
      if (looked == 2) {
        looked = 0;
        if (next < u1) look_all(next);
      }
      lost = lost_next;
      if (ok) {
        ok = __all_sync(0xffffffffu, kd_wait(&full[0], round & 1));
        if (!ok) kd_wait(&full[1], round & 1);  // no more work; what is in flight gets another while to land
      }
      const int left = min(g.len - (u - g.base) * KD_PIECE, KD_PIECE);  // tokens that count
      const bool work = ok && left > 0, ragged = left < KD_PIECE || lost != 0;
      // does token i of the piece count?
      const auto counts = [&](int i) { return i < left && !((lost >> (4 * (i / tokens))) & 1u); };
      uint32_t pb[PARTS][NT][KD_TILES][2];
      if (work) {
        const uint8_t* kc = stage + krow * (HD / 2) + c * (CPR / 2);
        const uint8_t* kp = stage + L::OFF_PK + (krow * (HD / KV4_GROUP) + c * CPR / KV4_GROUP) * 4;
        float st[NT][KD_TILES][4];
#pragma unroll
        for (int i = 0; i < KD_TILES; ++i) {
          uint32_t wk[2][KW];
          uint32_t par[2];
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
            par[h] = *reinterpret_cast<const uint32_t*>(kp + (i * 16 + h * 8) * (HD / KV4_GROUP) * 4);
          }
          const Sc f0(__byte_perm(par[0], 0u, 0x1010)), f1(__byte_perm(par[1], 0u, 0x1010));
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            mma_f16_16816_from_zero(st[t][i], __byte_perm(par[0], 0u, 0x3232), __byte_perm(par[1], 0u, 0x3232), 0u, 0u, qs[t], 0u);
          }
#pragma unroll
          for (int w = 0; w < KW; ++w) {
            uint32_t a[4 * PARTS], b[4 * PARTS];
            kd_numbers(a, wk[0][w], f0, magic);
            kd_numbers(b, wk[1][w], f1, magic);
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int k = 0; k < 4 * PARTS; k += 2) mma_f16_16816(st[t][i], a[k], b[k], a[k + 1], b[k + 1], qf[t][w][k & 3], qf[t][w][(k & 3) + 1]);
          }
        }
        __syncwarp();
        if (next < u1) lost_next = load(looked, 0);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          float top[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (ragged) {  // what does not count may be anything
#pragma unroll
              for (int i = 0; i < KD_TILES; ++i) {
                if (!counts(i * 16 + krow)) st[t][i][h] = -INFINITY;
                if (!counts(i * 16 + krow + 8)) st[t][i][2 + h] = -INFINITY;
              }
            }
            top[h] = fmaxf(st[t][0][h], st[t][0][2 + h]);
#pragma unroll
            for (int i = 1; i < KD_TILES; ++i) top[h] = fmaxf(top[h], fmaxf(st[t][i][h], st[t][i][2 + h]));
            top[h] *= sc[t][h];  // the factor is not negative: its sign is the query's
          }
          const uint32_t column = 0x11111111u << c;  // the lanes of this thread's heads
          // distances, which are exact where they are small, however large the scores are
          const uint32_t near0 = __ballot_sync(0xffffffffu, top[0] - m[t][0] >= KD_LOW), near1 = __ballot_sync(0xffffffffu, top[1] - m[t][1] >= KD_LOW);
          const bool high = top[0] - m[t][0] > KD_HIGH || top[1] - m[t][1] > KD_HIGH, low = (near0 & column) == 0u || (near1 & column) == 0u;
          if (__any_sync(0xffffffffu, high || low)) {
            float alpha[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float mx = top[h], big = l[t][h], to = m[t][h];
#pragma unroll
              for (int step = 4; step < 32; step *= 2) {
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, step));
                big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, step));
              }
              const int room = KD_ROOM + 127 - static_cast<int>(__float_as_uint(big) >> 23);
              const float below = mx - (mx - KD_BELOW) <= KD_HIGH ? mx - KD_BELOW : mx;  // the score itself where steps are larger
              if (mx - to > KD_HIGH)
                to = below;
              else if (mx - to < KD_LOW && mx > -INFINITY && room > 0)
                to = fmaxf(below, to - static_cast<float>(room));
              alpha[h] = to == m[t][h] ? 1.f : fast_exp2(m[t][h] - to);
              m[t][h] = to;
              l[t][h] *= alpha[h];
              z[t][h] *= alpha[h];
              z[t][2 + h] *= alpha[h];
            }
#pragma unroll
            for (int i = 0; i < HD / 16; ++i) {
              o[t][i][0] *= alpha[0]; o[t][i][1] *= alpha[1];
              o[t][i][2] *= alpha[0]; o[t][i][3] *= alpha[1];
            }
          }
          // Scores of 2^22 and more are rounded as the reference was: half a step of theirs is no exponent of 2 any more
          const bool far = __any_sync(0xffffffffu, fmaxf(fabsf(m[t][0]), fabsf(m[t][1])) >= 0x1p22f);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float mu = m[t][h] == -INFINITY ? 0.f : m[t][h];
            float by = sc[t][h];
            if (far) {
#pragma unroll
              for (int i = 0; i < KD_TILES; ++i) {
                st[t][i][h] = __fmul_rn(st[t][i][h], by);
                st[t][i][2 + h] = __fmul_rn(st[t][i][2 + h], by);
              }
              by = 1.f;
            }
            float sum = 0.f;  // of the piece first: beside a sum that is far larger its parts would be lost
#pragma unroll
            for (int i = 0; i < KD_TILES; ++i) {
              st[t][i][h] = fast_exp2(fmaf(st[t][i][h], by, -mu));
              st[t][i][2 + h] = fast_exp2(fmaf(st[t][i][2 + h], by, -mu));
              sum += st[t][i][h] + st[t][i][2 + h];
            }
            l[t][h] += sum;
          }
#pragma unroll
          for (int i = 0; i < KD_TILES; ++i) {
            const uint32_t w0 = pack2(st[t][i][0], st[t][i][1]), w1 = pack2(st[t][i][2], st[t][i][3]);
            pb[0][t][i][0] = movmatrix_t(w0);
            pb[0][t][i][1] = movmatrix_t(w1);
            if constexpr (FINE) {
              pb[1][t][i][0] = movmatrix_t(pack2_rest(st[t][i][0], st[t][i][1], w0));
              pb[1][t][i][1] = movmatrix_t(pack2_rest(st[t][i][2], st[t][i][3], w1));
            }
          }
        }
      } else if (ok && next < u1) {
        lost_next = load(looked, 0);
      }
      if (ok) {
        ok = __all_sync(0xffffffffu, kd_wait(&full[1], round & 1));
        if (!ok && next < u1) kd_wait(&full[0], (round + 1) & 1);
      }
      if (ok && left > 0) {
        // values: this thread's run of channels of four tokens at a time
        const uint8_t* vc = stage + L::CODES + c * (HD / 2) + r * (VPR / 2);
        const uint8_t* vp = stage + L::OFF_PK + L::PARAMS + (c * (HD / KV4_GROUP) + r * VPR / KV4_GROUP) * 4;
#pragma unroll
        for (int i = 0; i < KD_TILES; ++i) {
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
          const Sc f01(__byte_perm(pv[0], pv[1], 0x5410)), f23(__byte_perm(pv[2], pv[3], 0x5410));
          uint32_t m01 = __byte_perm(pv[0], pv[1], 0x7632), m23 = __byte_perm(pv[2], pv[3], 0x7632), r01 = 0u, r23 = 0u;
          if constexpr (FINE) {
            kd_least(m01, r01, __byte_perm(pv[0], pv[1], 0x5410));
            kd_least(m23, r23, __byte_perm(pv[2], pv[3], 0x5410));
          }
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int k = 0; k < PARTS; ++k) mma_f16_16816(z[t], m01, r01, m23, r23, pb[k][t][i][0], pb[k][t][i][1]);
#pragma unroll
          for (int w = 0; w < VW; ++w)
#pragma unroll
            for (int half = 0; half < 2; ++half) {  // channels 0..3 and 4..7 of the word: a pair of tokens side by side
              const uint32_t sel = half == 0 ? 0x5410 : 0x7632;
              uint32_t x[4 * PARTS], y[4 * PARTS];
              kd_numbers<FINE>(x, __byte_perm(wv[0][w], wv[1][w], sel), f01, magic);
              kd_numbers<FINE>(y, __byte_perm(wv[2][w], wv[3][w], sel), f23, magic);
#pragma unroll
              for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                  float (&to)[4] = o[t][w * 4 + half * 2 + k];
                  mma_f16_16816(to, x[2 * k], x[2 * k + 1], y[2 * k], y[2 * k + 1], pb[0][t][i][0], pb[0][t][i][1]);
                  if constexpr (FINE) {
                    mma_f16_16816(to, x[4 + 2 * k], x[5 + 2 * k], y[4 + 2 * k], y[5 + 2 * k], pb[0][t][i][0], pb[0][t][i][1]);
                    mma_f16_16816(to, x[2 * k], x[2 * k + 1], y[2 * k], y[2 * k + 1], pb[1][t][i][0], pb[1][t][i][1]);
                  }
                }
            }
        }
      }
      __syncwarp();
      if (ok && next < u1) load(looked, 1);
      ++looked;
    }

    if (FOLD && seg_end - seg > KD_FOLD) fold(true, true);
    // ---- end of a segment. O^T[channel r VPR + 2 i, head] = 16 o + z, and the channel behind it o' - o + z
    const bool whole = seg == g.base && seg_end == g.end;
    float* part = p.part + (2LL * run + (seg == u0 ? 0 : 1)) * G * (HD + 4);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float sum = l[t][h];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        const int head = t * 8 + 2 * c + h;
        if (head >= G) continue;
        float x[VPR];
        const float least = FINE ? z[t][h] + z[t][2 + h] : z[t][h];
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) {
          x[2 * i] = fmaf(FINE ? 1.f : 16.f, o[t][i][h], least);
          x[2 * i + 1] = o[t][i][2 + h] - (FINE ? 0.f : o[t][i][h]) + least;
        }
        if (whole) {
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
          T* out = static_cast<T*>(p.out) + (static_cast<long long>(g.b) * p.nh + g.kvh * G + head) * HD + r * VPR;
#pragma unroll
          for (int i = 0; i < VPR; i += 8) {
            uint4 v;
            T* e = reinterpret_cast<T*>(&v);
#pragma unroll
            for (int j = 0; j < 8; ++j) e[j] = static_cast<T>(x[i + j] * inv);
            *reinterpret_cast<uint4*>(out + i) = v;
          }
        } else {
          float* to = part + head * (HD + 4);
#pragma unroll
          for (int i = 0; i < VPR; i += 4) *reinterpret_cast<float4*>(to + r * VPR + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
          if (r == 0) *reinterpret_cast<float2*>(to + HD) = make_float2(m[t][h], sum);
        }
      }
  }
  if (!ok && lane == 0) atomicExch(status, ST_TIMEOUT_EPILOGUE);
}

// Joins the runs of every (sequence, head) that more than one warp worked on, and writes zeros for contexts of no tokens. A block takes
// `heads` query heads of a (sequence, KV head), eight channels a thread; what threads are left share the runs and meet in shared memory.
struct KDSum {
  float m, s, x[8];
  __device__ __forceinline__ void add(float mo, float so, const float (&v)[8]) {
    const float M = fmaxf(m, mo), mu = M == -INFINITY ? 0.f : M, fa = fast_exp2(m - mu), fb = fast_exp2(mo - mu);
    m = M;
    s = s * fa + so * fb;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = x[i] * fa + v[i] * fb;
  }
};

template <int HD, typename T>
__global__ void __launch_bounds__(512)
kv4_join_kernel(const VbKv4Decode p, int runs, int heads) {
  extern __shared__ __align__(16) KDSum sums[];  // one a thread
  const int b = blockIdx.y, h0 = blockIdx.x * heads, G = p.nh / p.nkv, kvh = h0 / G, g0 = h0 % G;
  const int total = kd_total(p), per = kd_per(total, runs), n = p.plan[b + 1] - p.plan[b], len = kd_len(p, b);
  T* out = static_cast<T*>(p.out) + (static_cast<long long>(b) * p.nh + h0) * HD;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the runs' sums, and what came before them
  const auto store = [&](int at, const float (&v)[8], float f) {
    uint4 o;
    T* e = reinterpret_cast<T*>(&o);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = static_cast<T>(v[i] * f);
    *reinterpret_cast<uint4*>(out + at * 8) = o;
  };
  const int lanes = heads * HD / 8, groups = max(1, static_cast<int>(blockDim.x) / lanes), group = threadIdx.x / lanes;
  KDSum a{-INFINITY, 0.f, {}};
  if (n <= 0 || len == 0) {
    for (int at = threadIdx.x; at < lanes; at += blockDim.x) store(at, a.x, 0.f);
    return;
  }
  const int base = p.plan[b] * p.nkv + kvh * n, i0 = max(base, 0) / per, i1 = min((base + n - 1) / per, runs - 1);
  if (i0 >= i1) return;
  for (int at0 = 0; at0 < lanes; at0 += blockDim.x) {  // more than once for more channels than threads, with one group then
    const int at = at0 + static_cast<int>(threadIdx.x) - (groups > 1 ? group * lanes : 0), head = at / (HD / 8), d = at % (HD / 8) * 8;
    a = KDSum{-INFINITY, 0.f, {}};
    if (group < groups && at < lanes) {
#pragma unroll 2
      for (int i = i0 + (groups > 1 ? group : 0); i <= i1; i += groups) {
        const float* s = p.part + ((2LL * i + (i * per >= base ? 0 : 1)) * G + g0 + head) * (HD + 4);
        const float2 ms = *reinterpret_cast<const float2*>(s + HD);
        const float4 lo = *reinterpret_cast<const float4*>(s + d), hi = *reinterpret_cast<const float4*>(s + d + 4);
        const float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
        a.add(ms.x, ms.y, v);
      }
    }
    const int used = min(groups, i1 - i0 + 1);
    for (int k = 1; k < used; k *= 2) {  // group g takes over group g + k's sums
      if (group < used) sums[threadIdx.x] = a;
      __syncthreads();
      if (group % (2 * k) == 0 && group + k < used) {
        const KDSum o = sums[threadIdx.x + k * lanes];
        a.add(o.m, o.s, o.x);
      }
      __syncthreads();
    }
    if (at < lanes && (groups == 1 || group == 0)) store(at, a.x, a.s == 0.f ? 0.f : 1.f / a.s);
  }
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

template <int HD, int NT, bool FOLD, typename T>
static cudaError_t kd_launch(const VbKv4Decode& p, int* status, cudaStream_t s) {
  auto kern = kv4_decode_kernel<HD, NT, FOLD, T>;
  constexpr int smem = KDSmem<HD, NT, FOLD>::TOTAL;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  const int ctas = num_sms() * kd_ctas(HD, NT);
  kern<<<ctas, KD_THREADS, smem, s>>>(p, __builtin_ctz(static_cast<unsigned>(p.block_size)), status);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  // A block per (sequence, KV head), or where each has many runs (few sequences with long contexts) one per query head with threads that share
  // the runs: one sequence of 131072 tokens (222 runs a head) 24 us and 8 us; 320 sequences (2 runs a head) 8.4 us.
  const int runs = ctas * KD_WARPS, many = runs / (p.B * p.nkv) >= 16, heads = many ? 1 : p.nh / p.nkv, threads = many ? 512 : 128;
  cfg.gridDim = dim3(p.nh / heads, p.B);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = threads * sizeof(KDSum);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv4_join_kernel<HD, T>, p, runs, heads);
}

// The kernel without folding where no warp can have more than KD_FOLD pieces of a (sequence, head), which the size of the table says: 320 sequences of
// up to 4096 tokens take 119 us (fp16 207), and 125 (213) with the other one, which folds nothing there either but has other registers.
template <int HD, int NT, typename T>
static cudaError_t kd_fold(const VbKv4Decode& p, int* status, cudaStream_t s) {
  const long long most = (static_cast<long long>(p.width) * p.block_size + KD_PIECE - 1) / KD_PIECE, runs = num_sms() * kd_ctas(HD, NT) * KD_WARPS;
  const long long run = (most * p.B * p.nkv + runs - 1) / runs;
  return min(most, run) > KD_FOLD ? kd_launch<HD, NT, true, T>(p, status, s) : kd_launch<HD, NT, false, T>(p, status, s);
}

template <typename T>
static cudaError_t kd_dispatch(const VbKv4Decode& p, int* status, cudaStream_t s) {
  const bool wide = p.nh / p.nkv > 8;
  if (p.hd == 128) return wide ? kd_fold<128, 2, T>(p, status, s) : kd_fold<128, 1, T>(p, status, s);
  return wide ? kd_fold<64, 2, T>(p, status, s) : kd_fold<64, 1, T>(p, status, s);
}

}  // namespace vb

using namespace vb;

extern "C" long long vb_kv4_decode_scratch(int B, int nh, int nkv, int hd) {
  const int G = nh / nkv;
  return 2LL * num_sms() * kd_ctas(hd, G <= 8 ? 1 : 2) * KD_WARPS * G * (hd + 4);
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
  if ((a->hd != 64 && a->hd != 128) || a->nh % a->nkv || a->nh / a->nkv > 16 || a->B > 65535 || (a->block_size & (a->block_size - 1)) || a->block_size < 16) return -2;
  const long long tokens = static_cast<long long>(a->width) * a->block_size;
  if (tokens > 1LL << 30 || (tokens + KD_PIECE - 1) / KD_PIECE * a->B * a->nkv > 0x3fffffffLL) return -4;  // counted in 31 bits
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
