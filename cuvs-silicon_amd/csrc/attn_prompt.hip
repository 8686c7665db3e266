// Plans and calls of attention over packed sequences (attn_prompt.hpp has the kernels).
#include <algorithm>

#include "attn_prompt.hpp"

namespace cvs {
namespace attn {

void check_view(const cvs_heads* x, const char* what) {
  const std::string w(what);
  if (!x) fail(CVS_ERR_INVALID_ARGUMENT, "null " + w);
  if (x->type != CVS_FP16 && x->type != CVS_BF16) fail(CVS_ERR_UNSUPPORTED, w + " must be fp16 or bf16");
  if (x->tokens < 0 || x->heads < 1) fail(CVS_ERR_INVALID_ARGUMENT, w + " must have heads and no negative size");
  if (x->head_dim < 8 || x->head_dim % 8 != 0 || x->head_dim > kMaxDim)
    fail(CVS_ERR_UNSUPPORTED, w + ": head_dim must be a multiple of 8 from 8 to " + std::to_string(kMaxDim));
  if (x->tokens > 0 && !x->data) fail(CVS_ERR_INVALID_ARGUMENT, "null data of " + w);
  // The kernels read and write 16 bytes at a time and count rows within 31 bits of bytes.
  const int64_t most = int64_t(1) << 23;
  if (x->token_stride < 0 || x->head_stride < 0 || (x->tokens > 1 && x->token_stride > most))
    fail(CVS_ERR_UNSUPPORTED, w + ": strides must be non-negative, the tokens' at most 2^23 elements");
  if (reinterpret_cast<uintptr_t>(x->data) % 16 != 0 || (x->tokens > 1 && x->token_stride % 8 != 0) ||
      (x->heads > 1 && x->head_stride % 8 != 0))
    fail(CVS_ERR_UNSUPPORTED, w + ": data must be 16-byte aligned, strides multiples of 8 elements");
}

void check_rows_apart(const cvs_heads* x, const char* what, int64_t layers, int64_t layer_stride) {
  if (x->tokens == 0) return;
  // From the axis of the smallest stride on, each has to step over all that the ones before it span.
  std::pair<int64_t, int64_t> axes[3] = {{x->token_stride, x->tokens}, {x->head_stride, x->heads}, {layer_stride, layers}};
  std::sort(axes, axes + 3);
  __int128 span = x->head_dim;
  for (const auto& [stride, count] : axes) {
    if (count == 1) continue;
    if (stride < span) fail(CVS_ERR_INVALID_ARGUMENT, std::string(what) + ": rows of an output must not overlap");
    span += __int128(stride) * (count - 1);
  }
}

float scale_log2(float scale, int dim) {
  if (!(scale >= 0.f) || std::isinf(scale))
    fail(CVS_ERR_INVALID_ARGUMENT, "scale must be finite and positive, or 0 for 1 / sqrt(head_dim)");
  if (scale > 2e38f) fail(CVS_ERR_UNSUPPORTED, "scale must be at most 2e38");  // log2(e) times it is a number of 32 bits
  return (scale == 0.f ? 1.f / std::sqrt(float(dim)) : scale) * kLog2e;
}

ScoreArgs score_args(const cvs_scores* scores, float scale, int dim) {
  ScoreArgs a{};
  a.c = scale_log2(scale, dim);
  if (!scores) return a;
  if (!(scores->cap >= 0.f) || std::isinf(scores->cap))
    fail(CVS_ERR_INVALID_ARGUMENT, "cap must be finite and positive, or 0 for none");
  if (reinterpret_cast<uintptr_t>(scores->slopes) % 4 != 0)
    fail(CVS_ERR_UNSUPPORTED, "slopes must be aligned to 4 bytes");
  a.slopes = scores->slopes;
  if (scores->cap == 0.f) return a;
  // u = ratio * s.  A cap that is larger still would be applied where a product's square has left the range of fp32, and
  // be off by its own last places there, far more than the score.
  const double ratio = double(a.c) / (double(scores->cap) * double(kLog2e)), y = ratio * ratio;
  if (scores->cap < 1e-30f || scores->cap > 1e38f || ratio < 1e-18)
    fail(CVS_ERR_UNSUPPORTED, "cap must be from 1e-30 to 1e38 and at most 1e18 times the scale");
  a.cap = scores->cap * kLog2e;
  a.twice = float(std::min(2.0 * ratio * double(kLog2e), 1e38));
  // P's coefficients are c ratio^2, ratio^4 and ratio^6 times these.  All have to be normal numbers of fp32: of a cap far
  // above the scale (from 9e5 times it on, for a scale of 1/8) the last ones would be rounded to few bits or to 0.  Then a
  // P of fewer terms, tanh's series, goes up to a |u| where the first term that it leaves out is below 2^-21, and larger
  // scores are the exponential's.  Of a scale so far above the cap that a coefficient is infinite, all are.
  struct Terms {
    double largest_u, of[3];
  };
  constexpr Terms kinds[] = {{0.5, {-3.332826464e-01, 1.320671470e-01, -4.478946771e-02}},
                             {0.125, {-1.0 / 3.0, 2.0 / 15.0, 0.0}},     // less 17/315 u^6
                             {0.03125, {-1.0 / 3.0, 0.0, 0.0}},          // 2/15 u^4
                             {0.0009765625, {0.0, 0.0, 0.0}}};           // u^2 / 3
  for (const Terms& k : kinds) {
    double power = double(a.c);
    bool all = true;
    for (int i = 0; i < 3; ++i) {
      power *= y;
      a.a[i] = float(k.of[i] * power);
      all &= k.of[i] == 0.0 || std::isnormal(a.a[i]) || std::isinf(a.a[i]);
    }
    a.largest_y = float(k.largest_u * k.largest_u / y);
    if (all) break;
  }
  if (ratio > 1e4 || std::isinf(a.a[2])) {
    a.a[0] = a.a[1] = a.a[2] = 0.f;
    a.largest_y = -1.f;
  }
  a.apart = a.cap >= 16777216.f;
  return a;
}

}  // namespace attn
}  // namespace cvs

using namespace cvs;
using namespace cvs::attn;

struct cvs_prompt_plan {
  cvs_context* ctx = nullptr;
  int64_t q_tokens = 0, k_tokens = 0;
  int heads = 0, kv_heads = 0, causal = 0;
  int64_t items = 0;
  DeviceBuffer blob;
  mutable bool captured = false;  // the blob is the context's to keep
};

namespace {

int make_plan(cvs_context* ctx, const int64_t* q_lengths, const int64_t* k_lengths, const int64_t* prefixes, int64_t n,
              int heads, int kv_heads, int causal, cvs_prompt_plan** out_plan) {
  return guarded([&] {
    bind(ctx);
    if (!out_plan) fail(CVS_ERR_INVALID_ARGUMENT, "null out_plan");
    *out_plan = nullptr;
    if (n < 0 || (n > 0 && !q_lengths)) fail(CVS_ERR_INVALID_ARGUMENT, "null lengths or negative count");
    if (heads < 1 || kv_heads < 1 || heads % kv_heads != 0)
      fail(CVS_ERR_INVALID_ARGUMENT, "heads must be a positive multiple of kv_heads");
    const int group = heads / kv_heads;
    int64_t tq = 0, tk = 0;
    std::vector<PromptItem> items;
    std::vector<int64_t> cost;
    for (int64_t i = 0; i < n; ++i) {
      const int64_t ql = q_lengths[i], kl = k_lengths ? k_lengths[i] : ql, prefix = prefixes ? prefixes[i] : 0;
      if (ql < 0 || kl < 0) fail(CVS_ERR_INVALID_ARGUMENT, "negative length");
      if (prefix < 0 || prefix > kl) fail(CVS_ERR_INVALID_ARGUMENT, "a prefix must lie within its sequence's keys");
      constexpr int64_t most = kv::PageBook::kMaxTokens;
      if (ql > most - tq || kl > most - tk || ql > most / group)
        fail(CVS_ERR_UNSUPPORTED, "token and row counts must fit 31 bits");
      for (int64_t row = 0; row < ql * group; row += kRows) {
        items.push_back({int32_t(tq), int32_t(ql), int32_t(tk), int32_t(kl), int32_t(row), int32_t(prefix)});
        const int64_t last = (std::min(row + kRows, ql * group) - 1) / group;
        cost.push_back(causal ? std::max(prefix, std::min(kl, last + 1 + kl - ql)) : kl);
      }
      tq += ql;
      tk += kl;
    }
    if (int64_t(items.size()) * kv_heads > kMaxBlocks) fail(CVS_ERR_UNSUPPORTED, "too many rows");
    // Longest first, so that the last workgroups to start are short ones.
    std::vector<int64_t> order(items.size());
    for (size_t i = 0; i < order.size(); ++i) order[i] = int64_t(i);
    std::stable_sort(order.begin(), order.end(), [&](int64_t x, int64_t y) { return cost[size_t(x)] > cost[size_t(y)]; });
    std::vector<PromptItem> sorted(items.size());
    for (size_t i = 0; i < order.size(); ++i) sorted[i] = items[size_t(order[i])];
    auto plan = std::make_unique<cvs_prompt_plan>();
    plan->ctx = ctx;
    plan->q_tokens = tq;
    plan->k_tokens = tk;
    plan->heads = heads;
    plan->kv_heads = kv_heads;
    plan->causal = causal != 0;
    plan->items = int64_t(items.size());
    if (!sorted.empty()) {
      need_no_capture(ctx, "plans cannot be made");
      const size_t bytes = sorted.size() * sizeof(PromptItem);
      plan->blob = take_blob(ctx->plan_blobs, ctx->live_prompt_plans, bytes);
      try {
        upload(ctx, plan->blob.ptr, sorted.data(), bytes);
      } catch (...) {
        ctx->plan_blobs.push_back(plan->blob);
        throw;
      }
    }
    ++ctx->live_prompt_plans;
    ++ctx->live_children;
    *out_plan = plan.release();
  });
}

}  // namespace

extern "C" {

int cvs_prompt_plan_create(cvs_context* ctx, const int64_t* q_lengths, const int64_t* k_lengths, int64_t n, int heads,
                           int kv_heads, int causal, cvs_prompt_plan** out_plan) {
  return make_plan(ctx, q_lengths, k_lengths, nullptr, n, heads, kv_heads, causal, out_plan);
}

int cvs_prompt_plan_create_prefix(cvs_context* ctx, const int64_t* q_lengths, const int64_t* k_lengths,
                                  const int64_t* prefixes, int64_t n, int heads, int kv_heads,
                                  cvs_prompt_plan** out_plan) {
  return make_plan(ctx, q_lengths, k_lengths, prefixes, n, heads, kv_heads, 1, out_plan);
}

int cvs_prompt_plan_destroy(cvs_prompt_plan* plan) {
  return guarded([&] {
    if (!plan) return;
    // Later plans use the memory on the same stream, after whatever still reads it.
    if (plan->blob.ptr && !plan->captured) plan->ctx->plan_blobs.push_back(plan->blob);
    --plan->ctx->live_prompt_plans;
    --plan->ctx->live_children;
    delete plan;
  });
}

int cvs_prompt_attention_async(cvs_context* ctx, const cvs_prompt_plan* plan, const cvs_heads* q, const cvs_heads* k,
                               const cvs_heads* v, const cvs_heads* out, float* lse, float scale) {
  return cvs_prompt_attention_scored_async(ctx, plan, q, k, v, out, lse, scale, nullptr);
}

int cvs_prompt_attention_scored_async(cvs_context* ctx, const cvs_prompt_plan* plan, const cvs_heads* q,
                                      const cvs_heads* k, const cvs_heads* v, const cvs_heads* out, float* lse,
                                      float scale, const cvs_scores* scores) {
  return guarded([&] {
    bind(ctx);
    if (!plan) fail(CVS_ERR_INVALID_ARGUMENT, "null plan");
    if (plan->ctx != ctx) fail(CVS_ERR_INVALID_ARGUMENT, "the plan belongs to another context");
    check_view(q, "q");
    check_view(k, "k");
    check_view(v, "v");
    check_view(out, "out");
    if (q->tokens != plan->q_tokens || out->tokens != plan->q_tokens)
      fail(CVS_ERR_INVALID_ARGUMENT, "q and out must have the plan's " + std::to_string(plan->q_tokens) + " tokens");
    if (k->tokens != plan->k_tokens || v->tokens != plan->k_tokens)
      fail(CVS_ERR_INVALID_ARGUMENT, "k and v must have the plan's " + std::to_string(plan->k_tokens) + " tokens");
    if (q->heads != plan->heads || out->heads != plan->heads || k->heads != plan->kv_heads ||
        v->heads != plan->kv_heads)
      fail(CVS_ERR_INVALID_ARGUMENT, "head counts differ from the plan's");
    if (q->head_dim != k->head_dim || q->head_dim != v->head_dim || q->head_dim != out->head_dim)
      fail(CVS_ERR_INVALID_ARGUMENT, "q, k, v and out must have one head_dim");
    if (q->type != k->type || q->type != v->type || q->type != out->type)
      fail(CVS_ERR_INVALID_ARGUMENT, "q, k, v and out must have one type");
    check_rows_apart(out, "out");
    const ScoreArgs sc = score_args(scores, scale, q->head_dim);
    if (plan->items == 0) return;
    if (!plan->captured && capturing(ctx)) {
      ctx->kept.push_back(plan->blob);
      plan->captured = true;
    }
    const PromptArgs a{view_of(q), view_of(k), view_of(v), view_of(out), lse,
                       plan->blob.as<PromptItem>(), plan->q_tokens, plan->kv_heads,
                       plan->heads / plan->kv_heads, q->head_dim, plan->causal, sc};
    const int64_t blocks = plan->items * plan->kv_heads;
    if (sc.cap > 0.f || sc.slopes) launch_prompt_scored(ctx, a, blocks, q->type);
    else if (q->type == CVS_BF16) launch_prompt<true, PlainScores>(ctx, a, blocks);
    else launch_prompt<false, PlainScores>(ctx, a, blocks);
  });
}

}  // extern "C"
