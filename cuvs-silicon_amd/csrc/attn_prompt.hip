// Attention over packed sequences of different lengths: every token's query
// against the keys of its own sequence, causal or not, with query heads that
// share key/value heads in groups.
//
//   out_i = sum_j 2^(c q_i.k_j - m) v_j / sum_j 2^(c q_i.k_j - m),
//   c = scale log2(e), m the row's largest c q_i.k_j, over the keys j that i sees.
//
// A workgroup of 4 waves holds 128 query rows of one sequence and kv head, 32
// a wave; the rows are (token, head of the group) pairs, token by token, so
// that heads which share keys share the tile's reads and a short sequence
// fills its tiles.  It runs through the keys once, 64 at a time: keys and
// values go straight to LDS (buffer_load ... lds), double-buffered, while the
// tile before is multiplied.
//
// LDS holds rows as they are in memory, in 16-byte pieces, with the piece
// order of each row permuted so that both products read without bank
// conflicts: the keys' A operand is 16 bytes of 32 different rows (ds_read_b128),
// the values' A operand (V^T) 4 keys of one column through the transposing
// read (ds_read_b64_tr_b16).  The permutation costs nothing: each lane of a
// load picks the piece that belongs at its place.
//
// Why 128 rows and 64 keys: a wave's 32 rows make each LDS operand worth one
// 32 x 32 product, two workgroups of 64 KiB (heads of 128) fit a compute unit,
// and the values' accumulators (64 registers), the queries (32) and two half
// tiles in flight leave two waves a SIMD their 256 registers.  Heads of 64 and
// 96 run four and three workgroups.
//
// Bounds: long prompts with heads of 128 the matrix cores (busy 61% of the
// cycles, the vector unit 52%: 12,000 causal tokens, 32/8 heads, bf16, in
// 1.03 ms = 1.14 PFLOP/s, 0.80 of the vendor's plain product).  Prompts with
// smaller heads no one unit: 64 passages of 40 to 512 tokens, 12 heads of 64,
// take 45 us with the vector unit busy 51% of the cycles (193 instructions a
// 64-key step, 32 exponentials among them), the matrix cores 27%, the waves 27%
// of their time waiting, and 146 MB fetched for 88 MB of inputs: row blocks
// that share keys run on different XCDs, each with an L2 of its own.  Short
// prompts each workgroup's first loads.
#include <algorithm>

#include "attn_common.hpp"

namespace cvs {
namespace attn {
namespace {

constexpr int kRows = 128;  // query rows of a workgroup
constexpr int kKeys = 64;   // keys of a step

struct PromptItem {
  int32_t q0, q_len;  // the sequence's tokens in q
  int32_t k0, k_len;  // and in k, v
  int32_t row0;       // first of the item's rows (token * group + head of the group)
};

struct PromptArgs {
  View q, k, v, out;
  float* lse;
  const PromptItem* items;
  int64_t q_tokens;  // lse rows are heads of q_tokens
  int kv_heads, group, dim, causal;
  float c;
};

// How the pieces of LDS row r are swapped (piece p stands at place p ^ swap)
// so that the 64 4-byte banks are read evenly.  Rows of 192 bytes begin 48
// banks apart, so 4 rows cover all banks and every 4th row is swapped within
// groups of 4 pieces; rows of 128 and 256 bytes begin at the same banks.
template <int P>
__device__ CVS_INLINE int swap_k(int r) {  // a read takes one piece of 16 rows
  return P == 12 ? (r >> 2) & 3 : P == 8 ? (r >> 1) & 7 : r & 15;
}
template <int P>
__device__ CVS_INLINE int swap_v(int r) {  // a read takes 4 pieces of 4 rows
  return P == 12 ? 0 : P == 8 ? 4 * ((r >> 1) & 1) : 4 * (r & 3);
}

// A kv head of one sequence, for attend_tiles.
template <int NB>
struct PromptSource {
  static constexpr int P = 4 * NB;  // 16-byte pieces of a row in LDS
  static constexpr int kPitch = 16 * P;
  static constexpr int kLoads = kKeys * P / 256;  // of a wave, keys or values
  static constexpr int kBuf = kKeys * kPitch;
  static constexpr uint32_t kNowhere = 0x80000000u;

  char *lds_k, *lds_v;
  int to_k, to_v;  // LDS addresses of the wave's share
  const char *base_k, *base_v;
  int64_t step_k, step_v;
  int k_len, first;  // first: of the lane's places in a buffer
  uint32_t off_k[kLoads], off_v[kLoads];
  int k_even, k_odd, v_first;

  __device__ CVS_INLINE PromptSource(const PromptArgs& a, const PromptItem& it, int g, int wave, char* sk, char* sv) {
    const int lane = __lane_id(), col = lane & 31, half = lane >> 5;
    lds_k = sk;
    lds_v = sv;
    to_k = lds_addr(sk) + wave * kLoads * 1024;
    to_v = lds_addr(sv) + wave * kLoads * 1024;
    base_k = a.k.p + 2 * (it.k0 * a.k.token + g * a.k.head);
    base_v = a.v.p + 2 * (it.k0 * a.v.token + g * a.v.head);
    step_k = kKeys * a.k.token * 2;
    step_v = kKeys * a.v.token * 2;
    k_len = it.k_len;
    // LDS place n = 64 i + lane of a wave's share is row n / P, place n % P.  Out of range reads zeros: pieces past the
    // head's end, and rows past the sequence's end in its last tile.
    first = wave * kLoads * 64 + lane;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int n = first + i * 64, r = n / P, p = n % P;
      const int pk = p ^ swap_k<P>(r), pv = p ^ swap_v<P>(r);
      off_k[i] = 8 * pk < a.dim ? r * uint32_t(2 * a.k.token) + 16 * pk : kNowhere;
      off_v[i] = 8 * pv < a.dim ? r * uint32_t(2 * a.v.token) + 16 * pv : kNowhere;
      asm("" : "+v"(off_k[i]), "+v"(off_v[i]));  // kept, not computed again for every tile
    }
    // Operand addresses within a buffer: of the keys' pieces 2 i + half (i even and odd: the piece order is swapped
    // within groups of four, or by more where rows are 128 or 256 bytes), of 4 keys of a column group.
    const int sw = swap_k<P>(col), li = lane & 15, vkey = 4 * half + (li >> 2);
    k_even = col * kPitch + 16 * (half ^ sw);
    k_odd = col * kPitch + 16 * ((2 + half) ^ sw);
    v_first = vkey * kPitch + 8 * (li & 1) + 16 * ((2 * ((lane >> 4) & 1) + ((li & 3) >> 1)) ^ swap_v<P>(vkey));
  }
  __device__ CVS_INLINE void load(const char* base, int64_t step, int to, const uint32_t (&off)[kLoads], int t) {
    const rsrc4 rs = make_rsrc(base + t * step, 0x7fffffff);
    const int left = k_len - t * kKeys;
    to += (t & 1) * kBuf;
    if (left >= kKeys) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) lds_dma<16, false>(rs, to + i * 1024, off[i], 0);
    } else {
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
        lds_dma<16, false>(rs, to + i * 1024, (first + i * 64) / P < left ? off[i] : kNowhere, 0);
    }
  }
  __device__ CVS_INLINE void load_keys(int t) { load(base_k, step_k, to_k, off_k, t); }
  __device__ CVS_INLINE void load_values(int t) { load(base_v, step_v, to_v, off_v, t); }
  __device__ CVS_INLINE u32x4 keys(int t, int h, int i) {
    const int at = P == 12 ? (i & 1 ? k_odd : k_even) + 64 * (i / 2) : k_even ^ 32 * i;
    return *reinterpret_cast<const u32x4*>(lds_k + (t & 1) * kBuf + h * 32 * kPitch + at);
  }
  __device__ CVS_INLINE u32x4 values(int t, int h, int b, int k) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
    typedef __attribute__((address_space(3))) s16x4* lds_ptr;
    char* const from = lds_v + (t & 1) * kBuf + (32 * h + 16 * k) * kPitch + (P == 12 ? v_first + 64 * b : v_first ^ 64 * b);
    const auto x = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)from));
    const auto y = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(from + 8 * kPitch)));
    return u32x4{x[0], x[1], y[0], y[1]};
  }
  __device__ CVS_INLINE u32x4 hide(u32x4 v, int, int, int) { return v; }  // past the sequence's end are zeros
};

template <bool kBf, int NB, int KS>
__global__ __launch_bounds__(256, NB == 4 ? 2 : NB == 3 ? 3 : 4) void prompt_attn_kernel(const PromptArgs a) {
  typedef PromptSource<NB> Source;
  __shared__ __align__(16) char s_k[2 * Source::kBuf];
  __shared__ __align__(16) char s_v[2 * Source::kBuf];

  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = blockIdx.x % a.kv_heads;
  const PromptItem it = a.items[blockIdx.x / a.kv_heads];

  // The lane's row; past the last row, the last one's again (not stored).
  const int rows = it.q_len * a.group;
  const int row = it.row0 + 32 * wave + col;
  const bool there = row < rows;
  const int rc = there ? row : rows - 1;
  const int tok = rc / a.group, head = g * a.group + rc % a.group;
  auto limit_of = [&](int t) CVS_INLINE {
    return a.causal ? max(0, min(it.k_len, it.k_len + (t + 1 - it.q_len))) : it.k_len;
  };
  const int limit = limit_of(tok);
  // Limits grow with the row, so the first and last row bound the workgroup's.
  const int wg_min = limit_of(it.row0 / a.group), wg_max = limit_of((min(it.row0 + kRows, rows) - 1) / a.group);

  Source src(a, it, g, wave, s_k, s_v);
  u32x4 q[KS];
  load_row<KS>(a.q.p + 2 * ((it.q0 + tok) * a.q.token + head * a.q.head), a.dim, q);
  const char* const base_v = src.base_v;
  RowState<NB> st;
  st.init();
  bool bad = false;
  // Keys between the first row's limit and the sequence's end: not only where limits differ, as the rows of a block may
  // all be one token's (128 and more heads on a kv head).
  attend_tiles<kBf, NB, KS>(st, q, src, (wg_max + kKeys - 1) / kKeys, wg_min / kKeys, wg_min < it.k_len, limit, a.c, bad);
  if (it.row0 + 32 * wave >= rows) return;
  const float l = both_sum(st.l);
  // A row that sees no key gives zeros; one whose keys' weights are all 0 (or NaN) gives what the formula does.
  const float inv = limit > 0 ? 1.f / l : 0.f;
  uint16_t* const out = reinterpret_cast<uint16_t*>(a.out.p) + (it.q0 + tok) * a.out.token + head * a.out.head;
  store_row<kBf, NB>(st, inv, out, a.dim, there);
  if (bad)
    add_nonfinite<kBf>(
        first_cleaned(wg_min, wg_max), there && l == l ? limit : 0, a.dim,
        [&](int j, int d) CVS_INLINE { return reinterpret_cast<const uint16_t*>(base_v)[j * a.v.token + d]; },
        [&](int d, float x) CVS_INLINE {
          x += to_float<kBf>(out[d]);
          out[d] = uint16_t(pack2<kBf>(x, x));
        });
  if (a.lse && there && half == 0)
    a.lse[int64_t(head) * a.q_tokens + it.q0 + tok] = limit > 0 ? (st.m + __builtin_amdgcn_logf(l)) * kLn2 : -INFINITY;
}

template <bool kBf>
void launch(cvs_context* ctx, const PromptArgs& a, int64_t blocks) {
  const TimerSpan ts = timer_span(ctx, "prompt_attention");
  auto go = [&](auto kernel) {
    hipExtLaunchKernelGGL(kernel, dim3(unsigned(blocks)), dim3(256), 0, ctx->stream, ts.start, ts.stop, 0, a);
  };
  // Blocks of 32 columns for the values, steps of 16 for the scores: heads of 72 and 80, 104 and 112 go without a step
  // that would multiply zeros.
  if (a.dim <= 64) go(prompt_attn_kernel<kBf, 2, 4>);
  else if (a.dim <= 80) go(prompt_attn_kernel<kBf, 3, 5>);
  else if (a.dim <= 96) go(prompt_attn_kernel<kBf, 3, 6>);
  else if (a.dim <= 112) go(prompt_attn_kernel<kBf, 4, 7>);
  else go(prompt_attn_kernel<kBf, 4, 8>);
  after_launch("prompt_attn_kernel");
}

}  // namespace

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
  return (scale == 0.f ? 1.f / std::sqrt(float(dim)) : scale) * kLog2e;
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

extern "C" {

int cvs_prompt_plan_create(cvs_context* ctx, const int64_t* q_lengths, const int64_t* k_lengths, int64_t n, int heads,
                           int kv_heads, int causal, cvs_prompt_plan** out_plan) {
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
      const int64_t ql = q_lengths[i], kl = k_lengths ? k_lengths[i] : ql;
      if (ql < 0 || kl < 0) fail(CVS_ERR_INVALID_ARGUMENT, "negative length");
      constexpr int64_t most = kv::PageBook::kMaxTokens;
      if (ql > most - tq || kl > most - tk || ql > most / group)
        fail(CVS_ERR_UNSUPPORTED, "token and row counts must fit 31 bits");
      for (int64_t row = 0; row < ql * group; row += kRows) {
        items.push_back({int32_t(tq), int32_t(ql), int32_t(tk), int32_t(kl), int32_t(row)});
        const int64_t last = (std::min(row + kRows, ql * group) - 1) / group;
        cost.push_back(causal ? std::max<int64_t>(0, std::min(kl, last + 1 + kl - ql)) : kl);
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
    const float c = scale_log2(scale, q->head_dim);
    if (plan->items == 0) return;
    if (!plan->captured && capturing(ctx)) {
      ctx->kept.push_back(plan->blob);
      plan->captured = true;
    }
    const PromptArgs a{view_of(q), view_of(k), view_of(v), view_of(out), lse,
                       plan->blob.as<PromptItem>(), plan->q_tokens, plan->kv_heads,
                       plan->heads / plan->kv_heads, q->head_dim, plan->causal, c};
    if (q->type == CVS_BF16) launch<true>(ctx, a, plan->items * plan->kv_heads);
    else launch<false>(ctx, a, plan->items * plan->kv_heads);
  });
}

}  // extern "C"
