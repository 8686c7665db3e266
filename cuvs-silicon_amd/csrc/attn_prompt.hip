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
#include <algorithm>
#include <type_traits>

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

template <bool kBf, int NB>
__global__ __launch_bounds__(256, NB == 4 ? 2 : NB == 3 ? 3 : 4) void prompt_attn_kernel(const PromptArgs a) {
  constexpr int P = 4 * NB;                 // 16-byte pieces of a row in LDS
  constexpr int kPitch = 16 * P;
  constexpr int kLoads = kKeys * P / 256;   // loads of a wave, keys or values
  constexpr int kBuf = kKeys * kPitch;
  __shared__ __align__(16) char s_k[2][kBuf];
  __shared__ __align__(16) char s_v[2][kBuf];

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
    return a.causal ? max(0, min(it.k_len, t + 1 + it.k_len - it.q_len)) : it.k_len;
  };
  const int limit = limit_of(tok);
  const bool busy = it.row0 + 32 * wave < rows;
  // Limits grow with the row, so the first and last row bound the workgroup's.
  const int wg_min = limit_of(it.row0 / a.group), wg_max = limit_of((min(it.row0 + kRows, rows) - 1) / a.group);

  u32x4 q[2 * NB];
  {
    const char* src = a.q.p + 2 * ((it.q0 + tok) * a.q.token + head * a.q.head);
#pragma unroll
    for (int s = 0; s < 2 * NB; ++s)
      q[s] = 16 * s + 8 * half < a.dim ? *reinterpret_cast<const u32x4*>(src + 32 * s + 16 * half) : u32x4{};
  }

  // Loads: LDS place n = 64 i + lane of a wave's share is row n / P, place n % P.  Out of range reads zeros: pieces
  // past the head's end, and rows past the sequence's end in its last tile.
  constexpr uint32_t kNowhere = 0x80000000u;
  uint32_t off_k[kLoads], off_v[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int n = (wave * kLoads + i) * 64 + lane, r = n / P, p = n % P;
    const int pk = p ^ swap_k<P>(r), pv = p ^ swap_v<P>(r);
    off_k[i] = 8 * pk < a.dim ? uint32_t(r * a.k.token * 2 + 16 * pk) : kNowhere;
    off_v[i] = 8 * pv < a.dim ? uint32_t(r * a.v.token * 2 + 16 * pv) : kNowhere;
    asm("" : "+v"(off_k[i]), "+v"(off_v[i]));  // kept, not computed again for every tile
  }
  const char* const base_k = a.k.p + 2 * (it.k0 * a.k.token + g * a.k.head);
  const char* const base_v = a.v.p + 2 * (it.k0 * a.v.token + g * a.v.head);
  const int64_t step_k = kKeys * a.k.token * 2, step_v = kKeys * a.v.token * 2;
  const int lds_k = lds_addr(s_k[0]) + wave * kLoads * 1024, lds_v = lds_addr(s_v[0]) + wave * kLoads * 1024;
  auto load_tile = [&](const char* base, int64_t step, int lds, const uint32_t(&off)[kLoads], int t) CVS_INLINE {
    const rsrc4 rs = make_rsrc(base + t * step, 0x7fffffff);
    const int left = it.k_len - t * kKeys;
    lds += (t & 1) * kBuf;
    if (left >= kKeys) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) lds_dma<16, false>(rs, lds + i * 1024, off[i], 0);
    } else {
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
        lds_dma<16, false>(rs, lds + i * 1024, ((wave * kLoads + i) * 64 + lane) / P < left ? off[i] : kNowhere, 0);
    }
  };

  // Operand addresses within a buffer: of the keys' pieces 2 i + half (i even and odd: the piece order is swapped
  // within groups of four, or by more where rows are 128 or 256 bytes), of 4 keys of a column group.
  const int sw = swap_k<P>(col), li = lane & 15, vkey = 4 * half + (li >> 2);
  const int k_even = col * kPitch + 16 * (half ^ sw), k_odd = col * kPitch + 16 * ((2 + half) ^ sw);
  auto key_at = [&](int i) CVS_INLINE { return P == 12 ? (i & 1 ? k_odd : k_even) + 64 * (i / 2) : k_even ^ 32 * i; };
  const int v_first = vkey * kPitch + 8 * (li & 1) +
                      16 * ((2 * ((lane >> 4) & 1) + ((li & 3) >> 1)) ^ swap_v<P>(vkey));
  auto value_at = [&](int b) CVS_INLINE { return P == 12 ? v_first + 64 * b : v_first ^ 64 * b; };

  RowState<NB> st;
  st.init();
  uint32_t bad = 0;
  f32x16 s[2];   // scores of a tile's two halves
  u32x4 p[2][2];  // and their probabilities
  auto scores = [&](int t, int h) CVS_INLINE {
    const char* const at = s_k[0] + (t & 1) * kBuf + h * 32 * kPitch;
    f32x16 x{};
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) x = mfma<kBf>(*reinterpret_cast<const u32x4*>(at + key_at(i)), q[i], x);
    return x;
  };
  auto add_values = [&](int t, int h, auto masked) CVS_INLINE {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
    typedef __attribute__((address_space(3))) s16x4* lds_ptr;
    char* const at = s_v[0] + (t & 1) * kBuf + h * 32 * kPitch;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        char* const from = at + value_at(b) + k * 16 * kPitch;
        const auto x = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)from));
        const auto y =
            __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(from + 8 * kPitch)));
        u32x4 v{x[0], x[1], y[0], y[1]};
        if constexpr (masked) v = clean<kBf>(v, bad);
        st.o[b] = mfma<kBf>(v, p[h][k], st.o[b]);
      }
  };
  auto mask = [&](int t, int h) CVS_INLINE {
    const int seen = limit - t * kKeys - 32 * h - 4 * half;
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if (8 * (r / 4) + r % 4 >= seen) s[h][r] = -INFINITY;
  };
  auto probabilities = [&](int h) CVS_INLINE {
    exponentials(s[h], st, a.c);
#pragma unroll
    for (int k = 0; k < 2; ++k) p[h][k] = prob_operand<kBf>(s[h], k);
  };

  // Half tiles in a pipeline of three: the products of one with the values and of the next with the keys run while
  // the one between goes through its exponentials.  In the middle of tile t everyone is done with its keys and with
  // the values before it; what was asked for one tile ago, the next keys and its values, has to be there.
  const int tiles = (wg_max + kKeys - 1) / kKeys, open_tiles = wg_min / kKeys;  // no row is masked in the open ones
  auto step = [&](int t, auto masked) CVS_INLINE {
    if (t > 0) add_values(t - 1, 1, masked);
    if constexpr (masked) mask(t, 0);
    raise_max(s[0], st, a.c);
    s[1] = scores(t, 1);
    probabilities(0);
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    __syncthreads();
    if (t + 2 < tiles) load_tile(base_k, step_k, lds_k, off_k, t + 2);
    if (t + 1 < tiles) load_tile(base_v, step_v, lds_v, off_v, t + 1);
    add_values(t, 0, masked);
    if constexpr (masked) mask(t, 1);
    raise_max(s[1], st, a.c);
    s[0] = scores(t + 1, 0);  // past the last tile: of whatever is there, and not used
    probabilities(1);
  };
  if (tiles > 0) {
    load_tile(base_k, step_k, lds_k, off_k, 0);
    load_tile(base_v, step_v, lds_v, off_v, 0);
    if (tiles > 1) load_tile(base_k, step_k, lds_k, off_k, 1);
    __builtin_amdgcn_s_waitcnt(0x0F70);
    __syncthreads();
    s[0] = scores(0, 0);
    int t = 0;
    for (; t < open_tiles; ++t) step(t, std::false_type{});
    for (; t < tiles; ++t) step(t, std::true_type{});
    add_values(tiles - 1, 1, std::true_type{});
  }
  if (!busy) return;
  const float l = both_sum(st.l);
  // A row that sees no key gives zeros; one whose keys' weights are all 0 (or NaN) gives what the formula does.
  const float inv = limit > 0 ? 1.f / l : 0.f;
  uint16_t* const out = reinterpret_cast<uint16_t*>(a.out.p) + (it.q0 + tok) * a.out.token + head * a.out.head;
  store_row<kBf, NB>(st, inv, out, a.dim, there);
  if (__ballot(bad != 0))
    store_nonfinite<kBf>(
        0, there && l == l ? limit : 0, a.dim,
        [&](int j, int d) CVS_INLINE { return reinterpret_cast<const uint16_t*>(base_v)[j * a.v.token + d]; },
        [&](int d, float x) CVS_INLINE { out[d] = uint16_t(pack2<kBf>(x, x)); });
  if (a.lse && there && half == 0)
    a.lse[int64_t(head) * a.q_tokens + it.q0 + tok] = limit > 0 ? (st.m + __builtin_amdgcn_logf(l)) * kLn2 : -INFINITY;
}

template <bool kBf>
void launch(cvs_context* ctx, const PromptArgs& a, int64_t blocks) {
  const TimerSpan ts = timer_span(ctx, "prompt_attention");
  auto go = [&](auto kernel) {
    hipExtLaunchKernelGGL(kernel, dim3(unsigned(blocks)), dim3(256), 0, ctx->stream, ts.start, ts.stop, 0, a);
  };
  if (a.dim <= 64) go(prompt_attn_kernel<kBf, 2>);
  else if (a.dim <= 96) go(prompt_attn_kernel<kBf, 3>);
  else go(prompt_attn_kernel<kBf, 4>);
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
  if (x->token_stride < 0 || x->head_stride < 0 || x->token_stride > most)
    fail(CVS_ERR_UNSUPPORTED, w + ": strides must be non-negative, the tokens' at most 2^23 elements");
  if (reinterpret_cast<uintptr_t>(x->data) % 16 != 0 || (x->tokens > 1 && x->token_stride % 8 != 0) ||
      (x->heads > 1 && x->head_stride % 8 != 0))
    fail(CVS_ERR_UNSUPPORTED, w + ": data must be 16-byte aligned, strides multiples of 8 elements");
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
  void* dev = nullptr;
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
      if (tq + ql > kv::PageBook::kMaxTokens || tk + kl > kv::PageBook::kMaxTokens || ql * group > kv::PageBook::kMaxTokens)
        fail(CVS_ERR_UNSUPPORTED, "token and row counts must fit 31 bits");
      for (int64_t row = 0; row < ql * group; row += kRows) {
        items.push_back({int32_t(tq), int32_t(ql), int32_t(tk), int32_t(kl), int32_t(row)});
        const int64_t last = (std::min(row + kRows, ql * group) - 1) / group;
        cost.push_back(causal ? std::max<int64_t>(0, std::min(kl, last + 1 + kl - ql)) : kl);
      }
      tq += ql;
      tk += kl;
    }
    if (int64_t(items.size()) * kv_heads > (int64_t(1) << 31) - 1) fail(CVS_ERR_UNSUPPORTED, "too many rows");
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
      const size_t bytes = sorted.size() * sizeof(PromptItem);
      CVS_HIP(hipMalloc(&plan->dev, bytes));
      try {
        upload(ctx, plan->dev, sorted.data(), bytes);
      } catch (...) {
        (void)hipFree(plan->dev);
        throw;
      }
    }
    ++ctx->live_children;
    *out_plan = plan.release();
  });
}

int cvs_prompt_plan_destroy(cvs_prompt_plan* plan) {
  return guarded([&] {
    if (!plan) return;
    bind(plan->ctx);
    (void)hipStreamSynchronize(plan->ctx->stream);
    if (plan->dev) (void)hipFree(plan->dev);
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
    const float c = scale_log2(scale, q->head_dim);
    if (plan->items == 0) return;
    const PromptArgs a{view_of(q), view_of(k), view_of(v), view_of(out), lse,
                       static_cast<const PromptItem*>(plan->dev), plan->q_tokens, plan->kv_heads,
                       plan->heads / plan->kv_heads, q->head_dim, plan->causal, c};
    if (q->type == CVS_BF16) launch<true>(ctx, a, plan->items * plan->kv_heads);
    else launch<false>(ctx, a, plan->items * plan->kv_heads);
  });
}

}  // extern "C"
