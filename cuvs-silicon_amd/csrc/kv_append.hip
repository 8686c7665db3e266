// A step's new tokens on their way into the paged cache: keys normed and
// rotated by their positions, values as they are, and the queries beside them
// normed and rotated, in one launch.
//
// A workgroup takes one tile of up to 32 tokens: a wave for each of up to 4 kv
// heads, or some query heads by all of them.  Its threads first make the
// cosines and sines of the tile's tokens, one each, for all heads.  A wave's
// keys are normed and rotated as rows of pieces (rotary.hpp) on their way to
// LDS, where they change places; values go straight from their rows to the
// pool (kv_tiles.hpp).  All of a wave's loads are under way before the cosines
// are made.
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
  const uint64_t* turns;
  float magnitude;
  int n_spans, page_tiles, by_tile, dim, dims;
  int kv_heads, kv_groups;             // workgroups of a tile's kv heads
  int q_heads, q_chunk, q_chunks;      // and of its query heads
  int kv_blocks;
};

template <bool kBf, int NB, Pairs kPairs, bool kNorm>
__global__ __launch_bounds__(256) void append_kernel(const AppendArgs a, const Spans inl) {
  constexpr int P = 4 * NB, kLanes = NB > 2 ? 16 : P;
  constexpr int kRows = 64 / kLanes, kSteps = 32 / kRows;  // tokens of a wave's step
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const bool queries = int(blockIdx.x) >= a.kv_blocks;
  const int block = queries ? blockIdx.x - a.kv_blocks : blockIdx.x, each = queries ? a.q_chunks : a.kv_groups;
  const int part = block % each, n = block / each;
  const int at = a.by_tile ? n % a.n_spans : n / a.page_tiles, tile = a.by_tile ? n / a.n_spans : n % a.page_tiles;
  const Span sp = a.spans ? a.spans[at] : inl.s[at];
  const int lo = max(sp.begin() - 32 * tile, 0), hi = min(sp.end() - 32 * tile, 32);
  if (lo >= hi) return;
  const int64_t row = int64_t(sp.row0) + 32 * tile - sp.begin();  // of the tile's token 0

  const HeadLane<kLanes> l(a.dim, a.dims);
  const int pitch = (l.half + 3) & ~3;
  u32x4* const s_keys = reinterpret_cast<u32x4*>(lds) + wave * 32 * P;  // the wave's
  float* const s_w = reinterpret_cast<float*>(lds + waves * 512 * P);
  float* const s_cos = s_w + (kNorm ? kMaxDim : 0);
  float* const s_sin = s_cos + 32 * pitch;
  auto before = [&]() CVS_INLINE {
    const int64_t first = int64_t(sp.index) * (32 * a.page_tiles) + 32 * tile;
    for (int i = threadIdx.x; i < (hi - lo) * l.half; i += blockDim.x) {
      const int t = lo + i / l.half, p = i % l.half;
      const int64_t position = a.positions ? a.positions[row + t] : first + t;
      const float2 cs = cos_sin(a.turns[p] * uint64_t(position));
      s_cos[t * pitch + p] = a.magnitude * cs.x;
      s_sin[t * pitch + p] = a.magnitude * cs.y;
    }
    if constexpr (kNorm) load_weight<kBf>(s_w, queries ? a.q_norm : a.k_norm, a.dim);
    __syncthreads();
  };

  if (queries) {
    const int h0 = part * a.q_chunk, nh = min(a.q_chunk, a.q_heads - h0);
    const bool normed = kNorm && a.q_norm.weight;
    auto place = [&](int r) CVS_INLINE {
      const int t = lo + r / nh, h = h0 + r % nh;
      return HeadRow{a.q.p + 2 * ((row + t) * a.q.token + h * a.q.head),
                     a.q_out.p + 2 * ((row + t) * a.q_out.token + h * a.q_out.head), s_cos + t * pitch,
                     s_sin + t * pitch, normed ? s_w : nullptr, a.q_norm.eps};
    };
    ready_rows<kBf, kLanes, kPairs, kNorm>(l, (hi - lo) * nh, s_keys + lane, place, before);
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
  if (spare) return;
  values.store(l.pieces);
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    if (kRows * i + kRows <= lo || kRows * i >= hi) continue;  // none of the step's tokens is the call's
    const int t = kRows * i + lane / kLanes, tc = values.held(t);
    x[i] = ready<kBf, kLanes, kPairs, kNorm>(x[i], l, s_cos + tc * pitch, s_sin + tc * pitch,
                                             kNorm && a.k_norm.weight ? s_w : nullptr, a.k_norm.eps, s_keys + lane);
  }
  // Staged behind all of them, whose raw rows may have passed through the same places.
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int t = kRows * i + lane / kLanes;
    if (l.in < P) s_keys[staged<NB>(t, l.in)] = l.in < l.pieces ? x[i] : u32x4{};
  }
  wave_lds_ready();
  store_keys<NB>(s_keys, kt, lo, hi);
}

template <bool kBf, int NB>
void launch(cvs_context* ctx, const AppendArgs& a, const Spans& inl, Pairs pairs, bool norm, unsigned blocks, int waves) {
  const size_t pitch = size_t((a.dims / 2 + 3) / 4 * 4);
  const size_t lds = size_t(waves) * 512 * 4 * NB + (norm ? kMaxDim * 4 : 0) + 2 * 32 * pitch * 4;
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
  switch ((a.dim + 31) / 32) {
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
        if (x->heads > 65536) fail(CVS_ERR_UNSUPPORTED, "too many heads");
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
      a.turns = rotary->turns.as<uint64_t>();
      a.magnitude = rotary->magnitude;
      a.dims = rotary->dims;
    }
    a.n_spans = int(plan->spans.size());
    a.page_tiles = int(cache->book->page_tokens() / 32);
    a.by_tile = spans_by_tile(plan);
    a.dim = cache->dim;
    a.kv_heads = cache->kv_heads;
    a.kv_groups = (cache->kv_heads + 3) / 4;
    const int waves = (cache->kv_heads + a.kv_groups - 1) / a.kv_groups;
    const int64_t tiles = int64_t(a.n_spans) * a.page_tiles;
    int64_t blocks = tiles * a.kv_groups;
    if (blocks <= kMaxBlocks) a.kv_blocks = int(blocks);
    if (q) {
      a.q = view_of(q);
      a.q_out = view_of(q_out);
      a.q_heads = q->heads;
      // About 128 rows a workgroup.
      const int64_t fill = std::max<int64_t>(1, plan->tokens / tiles);
      a.q_chunk = int(std::min<int64_t>(q->heads, std::max<int64_t>(1, 128 / fill)));
      a.q_chunks = (q->heads + a.q_chunk - 1) / a.q_chunk;
      blocks += tiles * a.q_chunks;
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
