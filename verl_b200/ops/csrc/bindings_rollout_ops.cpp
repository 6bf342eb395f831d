// torch.ops.verl_b200.* bindings of the page bookkeeping, the 4-bit cache and the scores of logits.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <algorithm>
#include <tuple>

#include "rollout_ops.h"

namespace {

using at::Tensor;
using OptTensor = c10::optional<at::Tensor>;

inline cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }
inline long long* lptr(const Tensor& t) { return reinterpret_cast<long long*>(t.data_ptr<int64_t>()); }
#define CHECK_RC(rc, what) TORCH_CHECK((rc) == 0, what " failed with code ", (rc))

// What the host form refuses with a ValueError is refused alike here; what only a GPU cannot take (a type, another device) is a RuntimeError.

// A vector of n whole numbers on the device of `like`.
void check_vec(const Tensor& t, at::ScalarType type, int64_t n, const Tensor& like, const char* what) {
  TORCH_CHECK_VALUE(t.scalar_type() == type && t.dim() == 1 && t.size(0) == n, what, ": expected a ", type, " vector of ", n, ", got ", t.scalar_type(), " ",
                    t.sizes());
  TORCH_CHECK(t.device() == like.device() && t.is_contiguous(), what, ": expected a contiguous vector on ", like.device(), ", got one on ", t.device());
}
int64_t length(const Tensor& t) { return t.dim() == 1 ? t.size(0) : -1; }
void check_table(const Tensor& t, const char* what) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.dim() == 2, what, ": block_table must be an int32 matrix [rows, blocks], got ", t.scalar_type(), " ", t.sizes());
  TORCH_CHECK(t.is_cuda() && (t.stride(1) == 1 || t.size(1) <= 1) && t.size(0) <= INT_MAX && t.size(1) <= INT_MAX, what,
              ": block_table must be a CUDA matrix with contiguous rows");
}
int type_of(const Tensor& t, bool f32, const char* what) {
  TORCH_CHECK_VALUE(at::isFloatingType(t.scalar_type()), what, ": expected floating numbers, got ", t.scalar_type());
  TORCH_CHECK(t.is_cuda(), what, ": expected a CUDA tensor");
  if (t.scalar_type() == at::kBFloat16) return 0;
  if (t.scalar_type() == at::kHalf) return 1;
  TORCH_CHECK(f32 && t.scalar_type() == at::kFloat, what, f32 ? ": expected bf16, fp16 or fp32" : ": expected bf16 or fp16", ", got ", t.scalar_type());
  return 2;
}

std::tuple<Tensor, Tensor, Tensor> decode_slot_map(const Tensor& table, const Tensor& pos, const Tensor& ctx, const Tensor& active, int64_t bs) {
  check_table(table, "decode_slot_map");
  const int64_t S = table.size(0);
  TORCH_CHECK(S <= (1 << 30), "decode_slot_map: at most 2^30 rows, got ", S);
  check_vec(pos, at::kInt, S, table, "decode_slot_map: pos");
  check_vec(ctx, at::kInt, S, table, "decode_slot_map: ctx");
  check_vec(active, at::kBool, S, table, "decode_slot_map: active");
  TORCH_CHECK(bs > 0 && bs <= (1 << 20), "decode_slot_map: block_size");
  const c10::cuda::CUDAGuard guard(table.device());
  Tensor slots = at::empty({S}, table.options().dtype(at::kLong)), ctx_out = at::empty({S}, table.options()), plan = at::empty({S + 1}, table.options());
  verl_count_launches(1);
  CHECK_RC(vb_decode_slot_map(table.data_ptr<int>(), table.stride(0), (int)table.size(1), pos.data_ptr<int>(), ctx.data_ptr<int>(),
                              active.data_ptr<bool>(), (int)S, (int)bs, lptr(slots), ctx_out.data_ptr<int>(), plan.data_ptr<int>(), cur_stream()),
           "vb_decode_slot_map");
  return {slots, ctx_out, plan};
}

Tensor extend_block_tables_(Tensor table, const Tensor& rows, const Tensor& have, const Tensor& lengths, const Tensor& pool, int64_t bs) {
  check_table(table, "extend_block_tables_");
  const int64_t B = length(rows);
  check_vec(rows, at::kInt, B, table, "extend_block_tables_: rows");
  check_vec(have, at::kInt, B, table, "extend_block_tables_: have");
  check_vec(lengths, at::kInt, B, table, "extend_block_tables_: lengths");
  check_vec(pool, at::kInt, length(pool), table, "extend_block_tables_: pool");
  TORCH_CHECK(bs > 0 && bs <= (1 << 20) && table.size(1) <= (1 << 20) && B <= (1 << 20) && pool.size(0) <= INT_MAX,
              "extend_block_tables_: at most 2^20 rows of at most 2^20 blocks");
  const c10::cuda::CUDAGuard guard(table.device());
  Tensor used = at::empty({1}, table.options());
  if (B == 0) return used.zero_();
  verl_count_launches(1);
  CHECK_RC(vb_extend_block_tables(table.data_ptr<int>(), table.stride(0), (int)table.size(0), (int)table.size(1), rows.data_ptr<int>(),
                                  have.data_ptr<int>(), lengths.data_ptr<int>(), (int)B, pool.data_ptr<int>(), (int)pool.size(0), (int)bs,
                                  used.data_ptr<int>(), cur_stream()),
           "vb_extend_block_tables");
  return used;
}

std::tuple<Tensor, Tensor, Tensor> build_slot_map(const Tensor& table, const Tensor& rows, const Tensor& starts, const Tensor& ends, int64_t bs,
                                                  int64_t total) {
  check_table(table, "build_slot_map");
  const int64_t B = length(rows);
  check_vec(rows, at::kInt, B, table, "build_slot_map: rows");
  check_vec(starts, at::kInt, B, table, "build_slot_map: starts");
  check_vec(ends, at::kInt, B, table, "build_slot_map: ends");
  TORCH_CHECK(bs > 0 && bs <= (1 << 20), "build_slot_map: block_size");
  TORCH_CHECK_VALUE(total >= 0, "build_slot_map: total must not be negative, got ", total);
  TORCH_CHECK(total <= (1LL << 31) - (1 << 13) && B <= (1 << 30), "build_slot_map: fewer than 2^31 - 2^13 tokens of at most 2^30 sequences, got ", total, " of ", B);
  const c10::cuda::CUDAGuard guard(table.device());
  Tensor cu = at::empty({B + 1}, table.options()), positions = at::empty({total}, table.options()),
         slots = at::empty({total}, table.options().dtype(at::kLong));
  verl_count_launches(1);
  CHECK_RC(vb_build_slot_map(table.data_ptr<int>(), table.stride(0), (int)table.size(0), (int)table.size(1), rows.data_ptr<int>(),
                             starts.data_ptr<int>(), ends.data_ptr<int>(), (int)B, (int)bs, (int)total, cu.data_ptr<int>(),
                             positions.data_ptr<int>(), lptr(slots), cur_stream()),
           "vb_build_slot_map");
  return {cu, positions, slots};
}

// Block size of a 4-bit pool [blocks, heads, bytes of a page] for heads of hd channels.
int64_t kv4_block(const Tensor& pages, int64_t hd, const char* what) {
  TORCH_CHECK_VALUE(pages.scalar_type() == at::kByte && pages.dim() == 3 && pages.is_contiguous(), what,
                    ": pages must be a contiguous uint8 tensor [blocks, kv_heads, page bytes], got ", pages.scalar_type(), " ", pages.sizes());
  TORCH_CHECK_VALUE(hd > 0 && hd % 32 == 0 && hd <= 1024, what, ": heads of a multiple of 32 channels, at most 1024, got ", hd);
  const int64_t bs = pages.size(2) * 4 / (5 * hd);
  TORCH_CHECK_VALUE(bs > 0 && bs * hd * 5 == pages.size(2) * 4 && bs % 16 == 0 && bs <= 1024, what, ": pages of ", pages.size(2),
                    " bytes hold no multiple of 16 tokens, at most 1024, of a head of ", hd);
  TORCH_CHECK(pages.is_cuda() && reinterpret_cast<uintptr_t>(pages.data_ptr()) % 16 == 0 && pages.size(0) * bs <= INT_MAX, what,
              ": pages must lie on a CUDA device and hold fewer than 2^31 tokens");
  return bs;
}

void kv4_append_(const Tensor& k, const Tensor& v, const Tensor& slots, Tensor pages) {
  TORCH_CHECK_VALUE(v.scalar_type() == k.scalar_type() && k.dim() == 3 && v.sizes() == k.sizes(),
                    "kv4_append_: k and v must be [tokens, heads, channels] of one floating type, got ", k.scalar_type(), " ", k.sizes(), ", ", v.scalar_type(), " ",
                    v.sizes());
  const int type = type_of(k, false, "kv4_append_");
  const int64_t T = k.size(0), nkv = k.size(1), hd = k.size(2);
  const int64_t bs = kv4_block(pages, hd, "kv4_append_");
  TORCH_CHECK_VALUE(pages.size(1) == nkv, "kv4_append_: the pool holds ", pages.size(1), " heads, k has ", nkv);
  TORCH_CHECK(v.device() == k.device() && pages.device() == k.device(), "kv4_append_: k, v and the pages on one device");
  TORCH_CHECK(T <= (1 << 30), "kv4_append_: at most 2^30 tokens, got ", T);
  check_vec(slots, at::kLong, T, k, "kv4_append_: slots");
  if (T == 0 || nkv == 0 || pages.size(0) == 0) return;
  for (const Tensor* t : {&k, &v})
    TORCH_CHECK(t->stride(2) == 1 && (nkv == 1 || t->stride(1) == hd) && (T == 1 || t->stride(0) % 8 == 0) &&
                reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0, "kv4_append_: heads of a token side by side, tokens on 16-byte boundaries");
  const c10::cuda::CUDAGuard guard(k.device());
  verl_count_launches(1);
  CHECK_RC(vb_kv4_append(type, k.data_ptr(), v.data_ptr(), T == 1 ? 0 : k.stride(0), T == 1 ? 0 : v.stride(0), lptr(slots), pages.data_ptr(), (int)T,
                         (int)nkv, (int)hd, (int)bs, pages.size(0) * bs, cur_stream()),
           "vb_kv4_append");
}

std::tuple<Tensor, Tensor> kv4_gather(const Tensor& pages, const Tensor& slots, int64_t hd, at::ScalarType dtype) {
  const int64_t bs = kv4_block(pages, hd, "kv4_gather"), T = length(slots), nkv = pages.size(1);
  TORCH_CHECK(dtype == at::kBFloat16 || dtype == at::kHalf, "kv4_gather: bf16 or fp16");
  TORCH_CHECK(T <= (1 << 30), "kv4_gather: at most 2^30 tokens, got ", T);
  check_vec(slots, at::kLong, T, pages, "kv4_gather: slots");
  const c10::cuda::CUDAGuard guard(pages.device());
  Tensor k = at::empty({T, nkv, hd}, pages.options().dtype(dtype)), v = at::empty_like(k);
  if (T == 0 || nkv == 0) return {k, v};
  verl_count_launches(1);
  CHECK_RC(vb_kv4_gather(dtype == at::kHalf, pages.data_ptr(), lptr(slots), k.data_ptr(), v.data_ptr(), (int)T, (int)nkv, (int)hd, (int)bs,
                         pages.size(0) * bs, cur_stream()),
           "vb_kv4_gather");
  return {k, v};
}

Tensor paged_decode_kv4(const Tensor& q, const Tensor& pages, const Tensor& table, const Tensor& ctx, const OptTensor& plan, double scale) {
  VbKv4Decode a{};
  TORCH_CHECK_VALUE(q.dim() == 3, "paged_decode_attention_kv4: q must be [sequences, heads, channels], got ", q.sizes());
  a.type = type_of(q, false, "paged_decode_attention_kv4");
  const int64_t B = q.size(0), nh = q.size(1), hd = q.size(2), bs = kv4_block(pages, hd, "paged_decode_attention_kv4"), nkv = pages.size(1);
  check_table(table, "paged_decode_attention_kv4");
  TORCH_CHECK_VALUE(nkv > 0 && nh > 0 && nh % nkv == 0 && table.size(0) == B, "paged_decode_attention_kv4: ", B, " sequences of ", nh, " heads against tables of ",
                    table.size(0), " rows and ", nkv, " KV heads");
  check_vec(ctx, at::kInt, B, q, "paged_decode_attention_kv4: ctx_len");
  if (plan.has_value()) check_vec(*plan, at::kInt, B + 1, q, "paged_decode_attention_kv4: plan");
  TORCH_CHECK(pages.device() == q.device() && table.device() == q.device(), "paged_decode_attention_kv4: tensors on several devices");
  TORCH_CHECK((hd == 64 || hd == 128) && nh / nkv <= 16, "paged_decode_attention_kv4: heads of 64 or 128 channels, at most 16 to a KV head, got ", nh, " / ", nkv,
              " of ", hd);
  TORCH_CHECK((bs & (bs - 1)) == 0 && bs <= 256, "paged_decode_attention_kv4: blocks of 16, 32, 64, 128 or 256 tokens, got ", bs);
  TORCH_CHECK(B <= 65535, "paged_decode_attention_kv4: at most 65535 sequences, got ", B);
  TORCH_CHECK(table.size(1) * bs <= (1LL << 30) && (table.size(1) * bs + 63) / 64 * B * nkv <= (1LL << 30) - 1, "paged_decode_attention_kv4: a table of ", B, " x ",
              table.size(1), " blocks of ", bs, " is more than the kernel counts in 30 bits");
  const c10::cuda::CUDAGuard guard(q.device());
  Tensor out = at::empty({B, nh, hd}, q.options());
  if (B == 0) return out;
  if (pages.size(0) == 0 || table.size(1) == 0) return out.zero_();
  TORCH_CHECK(q.stride(2) == 1 && q.stride(1) == hd && (B == 1 || q.stride(0) % 8 == 0) && reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0,
              "paged_decode_attention_kv4: heads of a sequence side by side, sequences on 16-byte boundaries");
  a.q = q.data_ptr(); a.ldq = B == 1 ? 0 : q.stride(0);
  a.pages = pages.data_ptr<uint8_t>(); a.num_blocks = (int)pages.size(0); a.block_size = (int)bs;
  a.table = table.data_ptr<int>(); a.width = (int)table.size(1); a.ldt = table.stride(0);
  a.ctx = ctx.data_ptr<int>(); a.out = out.data_ptr();
  a.B = (int)B; a.nh = (int)nh; a.nkv = (int)nkv; a.hd = (int)hd; a.scale = (float)scale;
  Tensor made, part;
  if (plan.has_value()) {
    a.plan = plan->data_ptr<int>();
  } else {
    made = at::empty({B + 1}, ctx.options());
    a.plan_ws = made.data_ptr<int>();
  }
  const long long n = vb_kv4_decode_scratch(a.B, a.nh, a.nkv, a.hd);
  if (n > 0) {
    part = at::empty({n}, q.options().dtype(at::kFloat));
    a.part = part.data_ptr<float>();
  }
  CHECK_RC(vb_kv4_decode(&a, cur_stream()), "vb_kv4_decode");
  return out;
}

// Logits with contiguous rows, and what the kernels are told about them. `valid` 0: all columns.
VbScores scores_of(const Tensor& x, const Tensor& ids, double temperature, int64_t valid, const char* what) {
  VbScores a{};
  TORCH_CHECK_VALUE(x.dim() == 2 && x.size(1) > 0, what, ": logits must be [rows, vocabulary], got ", x.sizes());
  TORCH_CHECK_VALUE(ids.scalar_type() == at::kLong && (ids.dim() == 1 || ids.dim() == 2) && ids.size(0) == x.size(0), what, ": ids must be int64 [", x.size(0),
                    "] or [", x.size(0), ", n], got ", ids.scalar_type(), " ", ids.sizes());
  TORCH_CHECK_VALUE(ids.dim() == 1 || ids.size(1) <= 4096, what, ": at most 4096 given tokens a row, got ", ids.size(1));
  TORCH_CHECK_VALUE(temperature > 0, what, ": temperature must be positive, got ", temperature);
  TORCH_CHECK_VALUE(valid >= 0 && valid <= x.size(1), what, ": valid_vocab must lie in 0 .. ", x.size(1), ", got ", valid);
  a.type = type_of(x, true, what);
  TORCH_CHECK((x.stride(1) == 1 || x.size(1) == 1) && ids.device() == x.device() && ids.is_contiguous(), what,
              ": logits and ids on one device, with contiguous rows");
  a.x = x.data_ptr(); a.ldx = x.size(0) <= 1 ? 0 : x.stride(0); a.T = (int)x.size(0); a.V = (int)(valid ? valid : x.size(1));
  a.inv_temp = (float)(1.0 / temperature);
  a.ids = lptr(ids); a.K = ids.dim() == 1 ? 1 : (int)ids.size(1);
  return a;
}
// Rows with contiguous columns. Rows and columns are counted in 31 bits, by steps of up to some thousand.
Tensor by_rows(const Tensor& x) {
  TORCH_CHECK(x.dim() != 2 || std::max(x.size(0), x.size(1)) <= (1LL << 31) - (1 << 14), "logits of ", x.sizes(), ": at most 2^31 - 2^14 rows and columns");
  return x.dim() == 2 && x.stride(1) != 1 && x.size(1) > 1 ? x.contiguous() : x;
}

// `stat`, where the gradient is to follow: [rows, 4] fp32, what it wants of the rows.
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> scores(const Tensor& logits, const Tensor& given, int64_t top, double temperature, int64_t valid, float* stat) {
  const Tensor x = by_rows(logits), ids = given.contiguous();
  VbScores a = scores_of(x, ids, temperature, valid, "token_scores");
  TORCH_CHECK_VALUE(top >= 0 && top <= std::min(128, a.V), "token_scores: top_k must lie in 0 .. ", std::min(128, a.V), ", got ", top);
  const c10::cuda::CUDAGuard guard(x.device());
  const auto f32 = x.options().dtype(at::kFloat);
  Tensor lp = at::empty(ids.sizes(), f32), ent = at::empty({x.size(0)}, f32), lse = at::empty({x.size(0)}, f32);
  Tensor top_ids = at::empty({x.size(0), top}, ids.options()), top_lp = at::empty({x.size(0), top}, f32);
  a.top = (int)top;
  a.logprob = lp.data_ptr<float>(); a.entropy = ent.data_ptr<float>(); a.lse = lse.data_ptr<float>();
  a.top_ids = lptr(top_ids); a.top_lp = top_lp.data_ptr<float>();
  a.stat = stat;
  CHECK_RC(vb_token_scores(&a, cur_stream()), "vb_token_scores");
  return {lp, ent, lse, top_ids, top_lp};
}
Tensor stat_of(const Tensor& logits) { return at::empty({logits.dim() == 2 ? logits.size(0) : 0, 4}, logits.options().dtype(at::kFloat)); }

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> token_scores(const Tensor& logits, const Tensor& given, int64_t top, double temperature, int64_t valid) {
  return scores(logits, given, top, temperature, valid, nullptr);
}

// `kept`: the rows' stat as the forward pass left it, or nothing: the rows are gone over once more for it.
Tensor scores_bwd(const Tensor& logits, const Tensor& given, const Tensor& lse, const Tensor& ent, const Tensor& kept, const Tensor& g_lp, const OptTensor& g_ent,
                  double temperature, int64_t valid) {
  const Tensor x = by_rows(logits), ids = given.contiguous();
  VbScores a = scores_of(x, ids, temperature, valid, "token_scores_bwd");
  const int64_t T = x.size(0);
  check_vec(lse, at::kFloat, T, x, "token_scores_bwd: lse");
  check_vec(ent, at::kFloat, T, x, "token_scores_bwd: entropy");
  TORCH_CHECK_VALUE(g_lp.scalar_type() == at::kFloat && g_lp.sizes() == ids.sizes(), "token_scores_bwd: g_logprob must be fp32, of the shape of ids");
  TORCH_CHECK(g_lp.device() == x.device() && g_lp.is_contiguous(), "token_scores_bwd: g_logprob must be contiguous and on the device of the logits");
  if (g_ent.has_value()) check_vec(*g_ent, at::kFloat, T, x, "token_scores_bwd: g_entropy");
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor stat = kept;
  if (!stat.defined()) {
    stat = stat_of(x);
    scores(x, at::empty({T, 0}, ids.options()), 0, temperature, valid, stat.data_ptr<float>());
  }
  Tensor dx = at::empty({T, x.size(1)}, x.options());
  a.stat = stat.data_ptr<float>();
  a.lse = lse.data_ptr<float>(); a.entropy = ent.data_ptr<float>();
  CHECK_RC(vb_token_scores_bwd(&a, g_lp.data_ptr<float>(), g_ent.has_value() ? g_ent->data_ptr<float>() : nullptr, dx.data_ptr(), dx.stride(0),
                               (int)x.size(1), cur_stream()),
           "vb_token_scores_bwd");
  return dx;
}
Tensor token_scores_bwd(const Tensor& logits, const Tensor& given, const Tensor& lse, const Tensor& ent, const Tensor& g_lp, const OptTensor& g_ent,
                        double temperature, int64_t valid, const OptTensor& stat) {
  if (stat.has_value())
    TORCH_CHECK(stat->scalar_type() == at::kFloat && stat->dim() == 2 && stat->size(0) == logits.size(0) && stat->size(1) == 4 && stat->is_contiguous() &&
                stat->device() == logits.device() && reinterpret_cast<uintptr_t>(stat->data_ptr()) % 16 == 0,
                "token_scores_bwd: stat must be what token_scores_kept returned for these logits");
  return scores_bwd(logits, given, lse, ent, stat.has_value() ? *stat : Tensor(), g_lp, g_ent, temperature, valid);
}

// Log-probs, entropy and log-sum-exp with what their gradient wants, for an autograd function that is written elsewhere.
std::tuple<Tensor, Tensor, Tensor, Tensor> token_scores_kept(const Tensor& logits, const Tensor& given, double temperature, int64_t valid) {
  TORCH_CHECK(logits.is_cuda(), "token_scores_kept: expected a CUDA tensor");
  const Tensor stat = stat_of(logits);
  auto [lp, ent, lse, top, top_lp] = scores(logits, given, 0, temperature, valid, stat.data_ptr<float>());
  return {lp, ent, lse, stat};
}

// Log-probs and entropy with their gradient. In C++, because a function written in Python costs more on the host than the kernels of most
// batches on the device: 146 us a step where this takes 68 (of which about 45 are any graph's).
struct TokenLogprobs : public torch::autograd::Function<TokenLogprobs> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& ids, double temperature, int64_t valid) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor stat = stat_of(x);
    auto [lp, ent, lse, top, top_lp] = scores(x, ids, 0, temperature, valid, x.is_cuda() ? stat.data_ptr<float>() : nullptr);
    ctx->save_for_backward({x, ids, lse, ent, stat});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["valid"] = valid;
    ctx->set_materialize_grads(false);
    return {lp, ent};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list g) {
    Tensor none, dx;
    if (g[0].defined() || g[1].defined()) {
      const bool again = at::GradMode::is_enabled();
      const auto saved = ctx->get_saved_variables();
      {
        at::NoGradGuard guard;
        const Tensor g_lp = g[0].defined() ? g[0].contiguous() : at::zeros(saved[1].sizes(), saved[2].options());
        OptTensor g_ent;
        if (g[1].defined()) g_ent = g[1].contiguous();
        dx = scores_bwd(saved[0].detach(), saved[1], saved[2], saved[3].detach(), saved[4], g_lp, g_ent, ctx->saved_data["temperature"].toDouble(), ctx->saved_data["valid"].toInt());
      }
      if (again)  // a graph of the gradient is asked for: an error where it is used
        dx = std::make_shared<torch::autograd::DelayedError>("token_logprobs can be differentiated once", 2)->apply({dx, saved[0]})[0];
    }
    return {dx, none, none, none};
  }
};

std::tuple<Tensor, Tensor> token_logprobs(const Tensor& logits, const Tensor& given, double temperature, int64_t valid) {
  TORCH_CHECK_NOT_IMPLEMENTED(!logits._fw_grad(0).defined(), "token_logprobs: logits with a tangent (forward-mode derivatives)");
  const Tensor x = by_rows(logits), ids = given.contiguous();
  if (at::GradMode::is_enabled() && x.requires_grad()) {
    auto out = TokenLogprobs::apply(x, ids, temperature, valid);
    return {out[0], out[1]};
  }
  auto out = token_scores(x, ids, 0, temperature, valid);
  return {std::get<0>(out), std::get<1>(out)};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(verl_b200, m) {
  m.def("decode_slot_map", &decode_slot_map);
  m.def("extend_block_tables_", &extend_block_tables_);
  m.def("build_slot_map", &build_slot_map);
  m.def("kv4_append_", &kv4_append_);
  m.def("kv4_gather", &kv4_gather);
  m.def("paged_decode_kv4", &paged_decode_kv4);
  m.def("token_scores", &token_scores);
  m.def("token_scores_bwd", &token_scores_bwd);
  m.def("token_scores_kept", &token_scores_kept);
  m.def("token_logprobs", &token_logprobs);
}
