// A step's new tokens on their way into the paged cache: keys normed and
// rotated by their positions, values as they are, and the queries beside them
// normed and rotated, in one launch.
//
// A workgroup takes one tile of up to 32 tokens: a wave for each of up to 4 kv
// heads; or, by all of its waves, query heads of some of the tokens.  Its
// threads first make the factors of these tokens, a pair of channels each, for
// all heads (rotary.hpp).  A wave's keys are normed and rotated as rows of
// pieces on their way to LDS, where they change places, in the factors' room;
// values go straight from their rows to the pool (kv_tiles.hpp).  All of a
// wave's loads of keys and values are under way before the factors are made.
//
// Bounds: prompts the memory (24 of up to 2,000 tokens, 20/4 heads of 80, bf16,
// normed: 38 us, 5.0 TB/s read and write, inputs in the last-level cache), steps a
// chain of loads, factors and two barriers (a token of each of 64 sequences, 32/8
// heads of 128, normed: 7.6 us; of one, 16/4 heads of 64: 5.2 us).  Workgroups of
// tiles without a new token end at once: in pages of 4,096 the 64 sequences take
// 26.5 us.
#include <algorithm>
#include <cstring>

#include "rotary.hpp"

namespace cvs {
namespace attn {
namespace {

struct AppendArgs {
  char* pool;  // of the layer
  int64_t page_bytes, head_bytes;
  const Span* spans;  // null: inline
  View k, v, q, q_out;
  Norm k_norm, q_norm;
  const int64_t* positions;  // null: the tokens' places in their sequences
  Turning turning;
  int n_spans, page_tiles, by_tile;
  int kv_heads, kv_groups;         // workgroups of a tile's kv heads
  int q_parts;                     // of its query tokens,
  int q_heads, q_chunk, q_chunks;  // and of their heads
  uint32_t q_magic, q_last_magic;  // of a chunk's heads, and of the last one's
  int kv_blocks;
  int at_rows;  // in LDS, of kChannels' rows
};

template <bool kBf, int NB, Pairs kPairs, bool kNorm>
__global__ __launch_bounds__(256) void append_kernel(const AppendArgs a, const Spans inl) {
  constexpr int P = 4 * NB, kLanes = NB > 2 ? 16 : P;
  constexpr int kRows = 64 / kLanes, kSteps = 32 / kRows;  // tokens of a wave's step
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool queries = int(blockIdx.x) >= a.kv_blocks;
  const int block = queries ? blockIdx.x - a.kv_blocks : blockIdx.x, each = queries ? a.q_parts * a.q_chunks : a.kv_groups;
  int part = block % each;
  const int n = block / each;
  const int at = a.by_tile ? n % a.n_spans : n / a.page_tiles, tile = a.by_tile ? n / a.n_spans : n % a.page_tiles;
  const Span sp = a.spans ? a.spans[at] : inl.s[at];
  int lo = max(sp.begin() - 32 * tile, 0), hi = min(sp.end() - 32 * tile, 32);
  if (lo >= hi) return;
  if (queries && a.q_parts > 1) {
    const int of = part / a.q_chunks, all = hi - lo, from = lo;
    part -= of * a.q_chunks;
    lo = from + all * of / a.q_parts;
    hi = from + all * (of + 1) / a.q_parts;
    if (lo == hi) return;
  }
  const int64_t row = int64_t(sp.row0) + 32 * tile - sp.begin();  // of the tile's token 0

  const HeadLane<kLanes> l(a.turning.dim, a.turning.half);
  // The factors, and, when all waves are through with them, the keys that change places: each wave its own.
  float* const s_own = reinterpret_cast<float*>(lds) - lo * l.dim;
  float* const s_other = s_own + 32 * l.dim;
  u32x4* const s_keys = reinterpret_cast<u32x4*>(lds) + wave * 32 * P;
  u32x4* const s_rows = reinterpret_cast<u32x4*>(lds + a.at_rows) + threadIdx.x;
  auto before = [&]() CVS_INLINE {
    const int64_t first = int64_t(sp.index) * (32 * a.page_tiles) + 32 * tile;
    make_turning<kBf, kPairs>(a.turning, queries ? a.q_norm : a.k_norm, lo, hi, s_own, s_other, [&](int t) CVS_INLINE {
      return a.positions ? a.positions[row + t] : first + t;
    });
    __syncthreads();
  };

  if (queries) {
    const int h0 = part * a.q_chunk, nh = min(a.q_chunk, a.q_heads - h0);
    auto first = [&](const View& v) CVS_INLINE {
      return RowView{v.p + 2 * ((row + lo) * v.token + h0 * v.head), uint32_t(2 * v.token), uint32_t(2 * v.head)};
    };
    const Rows rows{(hi - lo) * nh, nh, nh == a.q_chunk ? a.q_magic : a.q_last_magic, first(a.q), first(a.q_out),
                    s_own + lo * l.dim, s_other + lo * l.dim, a.q_norm.weight != nullptr, a.q_norm.eps};
    ready_rows<kBf, kLanes, kPairs, kNorm>(l, rows, s_rows, before);
    return;
  }

  // The workgroups' shares of heads are even; a wave too many does the last head's again, and stores nothing.
  const int g0 = a.kv_heads * part / a.kv_groups, g1 = a.kv_heads * (part + 1) / a.kv_groups;
  const int g = min(g0 + wave, g1 - 1);
  const bool spare = g0 + wave >= g1;
  char* const kt = a.pool + sp.page * a.page_bytes + g * a.head_bytes + int64_t(tile) * 4096 * NB;
  const char* const ks = a.k.p + 2 * (row * a.k.token + g * a.k.head);
  const char* const vs = a.v.p + 2 * (row * a.v.token + g * a.v.head);
  TileValues<NB> values(kt + 2048 * NB, lo, hi);
  u32x4 x[kSteps];
#pragma unroll
  for (int i = 0; i < kSteps; ++i)
    x[i] = *reinterpret_cast<const u32x4*>(ks + 2 * (values.held(kRows * i + lane / kLanes) * a.k.token + 8 * l.piece));
  values.load(vs, a.v.token, l.pieces);
  before();
  if (!spare) values.store(l.pieces);
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    if (kRows * i + kRows <= lo || kRows * i >= hi) continue;  // none of the step's tokens is the call's
    const int t = values.held(kRows * i + lane / kLanes);
    x[i] = ready<kBf, kLanes, kPairs, kNorm>(x[i], l, s_own + t * l.dim, s_other + t * l.dim, a.k_norm.weight != nullptr,
                                             a.k_norm.eps, s_rows);
    row_done(x[i]);
  }
  __syncthreads();  // everyone has read the factors
  if (spare) return;
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int t = kRows * i + lane / kLanes;
    if (l.in < P) s_keys[staged<NB>(t, l.in)] = l.in < l.pieces ? x[i] : u32x4{};
  }
  wave_lds_ready();
  store_keys<NB>(s_keys, kt, lo, hi);
}

template <bool kBf, int NB>
void launch(cvs_context* ctx, const AppendArgs& args, const Spans& inl, Pairs pairs, bool norm, unsigned blocks,
            int waves) {
  AppendArgs a = args;
  a.at_rows = std::max(waves * 512 * 4 * NB, 2 * 32 * 4 * a.turning.dim);
  const size_t lds = size_t(a.at_rows) + (pairs == kChannels ? size_t(waves) * 1024 : 0);
  const TimerSpan ts = timer_span(ctx, "kv_append");
  auto go = [&](auto kernel) {
    hipExtLaunchKernelGGL(kernel, dim3(blocks), dim3(unsigned(64 * waves)), lds, ctx->stream, ts.start, ts.stop, 0, a, inl);
  };
  switch (pairs) {
    case kNeighbours: norm ? go(append_kernel<kBf, NB, kNeighbours, true>) : go(append_kernel<kBf, NB, kNeighbours, false>); break;
    case kPieces: norm ? go(append_kernel<kBf, NB, kPieces, true>) : go(append_kernel<kBf, NB, kPieces, false>); break;
    default: norm ? go(append_kernel<kBf, NB, kChannels, true>) : go(append_kernel<kBf, NB, kChannels, false>); break;
  }
  after_launch("append_kernel");
}

template <bool kBf>
void launch(cvs_context* ctx, const AppendArgs& a, const Spans& inl, Pairs pairs, bool norm, unsigned blocks, int waves) {
  switch ((a.turning.dim + 31) / 32) {
    case 1: launch<kBf, 1>(ctx, a, inl, pairs, norm, blocks, waves); break;
    case 2: launch<kBf, 2>(ctx, a, inl, pairs, norm, blocks, waves); break;
    case 3: launch<kBf, 3>(ctx, a, inl, pairs, norm, blocks, waves); break;
    default: launch<kBf, 4>(ctx, a, inl, pairs, norm, blocks, waves); break;
  }
}

}  // namespace
}  // namespace attn
}  // namespace cvs

using namespace cvs;
using namespace cvs::attn;

extern "C" int cvs_kv_append_async(cvs_kv_cache* cache, cvs_kv_plan* plan, int layer, const cvs_rotary* rotary,
                                   const int64_t* positions, const cvs_heads* k, const cvs_head_norm* k_norm,
                                   const cvs_heads* v, const cvs_heads* q, const cvs_heads* q_out,
                                   const cvs_head_norm* q_norm) {
  return guarded([&] {
    if (!cache) fail(CVS_ERR_INVALID_ARGUMENT, "null cache");
    if (!plan) fail(CVS_ERR_INVALID_ARGUMENT, "null plan");
    if (plan->cache != cache) fail(CVS_ERR_INVALID_ARGUMENT, "the plan belongs to another cache");
    cvs_context* const ctx = cache->ctx;
    bind(ctx);
    check_move(plan, layer, 1, k, v, true);
    if (rotary) check_rotary(rotary, ctx, cache->dim);
    if (positions && !rotary) fail(CVS_ERR_INVALID_ARGUMENT, "positions without a rotary");
    check_positions(positions);
    AppendArgs a{};
    a.k_norm = norm_of(k_norm, cache->type, "k");
    if (q) {
      for (const cvs_heads* x : {q, q_out}) {
        const char* const what = x == q ? "q" : "q_out";
        check_view(x, what);
        if (x->tokens != plan->tokens)
          fail(CVS_ERR_INVALID_ARGUMENT,
               std::string(what) + " must have the plan's " + std::to_string(plan->tokens) + " tokens");
        if (x->head_dim != cache->dim || x->type != cache->type)
          fail(CVS_ERR_INVALID_ARGUMENT, std::string(what) + " must have the cache's head_dim and type");
        if (x->heads != q->heads) fail(CVS_ERR_INVALID_ARGUMENT, "q_out must have the heads of q");
        if (plan->heads > 0 && x->heads != plan->heads)
          fail(CVS_ERR_INVALID_ARGUMENT, std::string(what) + " must have the plan's heads");
        if (x->heads > 65535) fail(CVS_ERR_UNSUPPORTED, "too many heads");
      }
      check_rows_apart(q_out, "q_out");
      a.q_norm = norm_of(q_norm, cache->type, "q");
    } else if (q_out || q_norm) {
      fail(CVS_ERR_INVALID_ARGUMENT, "an output or a norm of q without q");
    }
    if (plan->spans.empty()) return;
    captured_call(plan);
    a.pool = cache->pool + layer * cache->layer_bytes;
    a.page_bytes = cache->page_bytes;
    a.head_bytes = cache->head_bytes;
    a.k = view_of(k);
    a.v = view_of(v);
    if (rotary) {
      captured_rotary(rotary);
      a.positions = positions;
      a.turning.turns = rotary->turns.as<uint64_t>();
      a.turning.magnitude = rotary->magnitude;
      a.turning.half = rotary->dims / 2;
    }
    a.n_spans = int(plan->spans.size());
    a.page_tiles = int(cache->book->page_tokens() / 32);
    a.by_tile = spans_by_tile(plan);
    a.turning.dim = cache->dim;
    a.kv_heads = cache->kv_heads;
    a.kv_groups = (cache->kv_heads + 3) / 4;
    int waves = (cache->kv_heads + a.kv_groups - 1) / a.kv_groups;
    const int64_t tiles = int64_t(a.n_spans) * a.page_tiles;
    int64_t blocks = tiles * a.kv_groups;
    if (blocks <= kMaxBlocks) a.kv_blocks = int(blocks);
    if (q) {
      a.q = view_of(q);
      a.q_out = view_of(q_out);
      a.q_heads = q->heads;
      // A tile's queries by workgroups of some of its tokens and all heads, about 32 KB of them (tiles whole: 24 prompts of
      // up to 2,000 tokens, 32/8 heads of 128, normed, take 134 us instead of 123), or, where that leaves compute units
      // without one, of fewer heads, down to 16 rows each.  Counted by all tiles of the spans' pages: in large pages that
      // new tokens fill little of, a workgroup gets more (300 tokens of a prompt in pages of 64 take 9.3 us, of 4,096 15.0).
      const int64_t fill = std::max<int64_t>(1, plan->tokens / tiles), filled = (plan->tokens + fill - 1) / fill;
      a.q_parts = int(std::clamp<int64_t>(q->heads * fill * cache->dim / 16384, 1, fill));
      const int64_t fit = std::clamp<int64_t>(2 * ctx->compute_units / (filled * a.q_parts), 1,
                                              (q->heads * fill / a.q_parts + 15) / 16);
      a.q_chunk = int(std::min<int64_t>((q->heads + fit - 1) / fit, 1024));
      if (!rows_near(a.q, a.q_chunk) || !rows_near(a.q_out, a.q_chunk)) a.q_chunk = 1;
      a.q_chunks = (q->heads + a.q_chunk - 1) / a.q_chunk;
      // A wave for each 16 rows, however few the kv heads are: with one of those, the prompts above take 84 us, and 150
      // with one wave.
      waves = int(std::clamp<int64_t>((a.q_chunk * fill / a.q_parts + 15) / 16, waves, 4));
      a.q_magic = magic_of(a.q_chunk);
      a.q_last_magic = magic_of(q->heads - (a.q_chunks - 1) * a.q_chunk);
      blocks += tiles * a.q_parts * a.q_chunks;
    }
    if (blocks > kMaxBlocks) fail(CVS_ERR_UNSUPPORTED, "too many tokens");
    Spans inl;
    const bool small = plan->spans.size() <= size_t(kInlineSpans);
    if (small) std::memcpy(inl.s, plan->spans.data(), plan->spans.size() * sizeof(Span));
    else a.spans = reinterpret_cast<const Span*>(plan->blob.as<char>() + plan->at_spans);
    const bool norm = a.k_norm.weight || a.q_norm.weight;
    if (cache->type == CVS_BF16) launch<true>(ctx, a, inl, pairs_of(rotary), norm, unsigned(blocks), waves);
    else launch<false>(ctx, a, inl, pairs_of(rotary), norm, unsigned(blocks), waves);
  });
}
