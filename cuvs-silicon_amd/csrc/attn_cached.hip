// Plans and calls of attention over a paged cache (attn_cached.hpp has the
// kernels), and the joining of rows' parts.
#include <algorithm>
#include <cstring>

#include "attn_cached.hpp"

namespace cvs {
namespace attn {
namespace {

constexpr int kJoin = 4;        // parts of a row that a lane reads at a time

// The parts that a run gives the rows of its sequences: part p of row r has
// slot slot0 + p * rows + r.  parent: the run that its pages follow, or -1.
struct Parts {
  int32_t slot0, rows, count, parent;
};

struct JoinArgs {
  const Parts* parts;      // run by run
  const int32_t* runs;     // per token, the last of its sequence's
  const int32_t* q_rows;
  const float* part_o;
  const float2* part_ml;
  int64_t slots, rows;     // rows: tokens * heads
  View out;
  float* lse;
  int64_t q_tokens;
  int heads, group, dim;
};

// One wave a (token, head) row, in one pass over the row's parts with a
// running maximum.  A lane takes 4 columns; 8 NB lanes have a part, and the
// wave's groups of so many take the parts in turn and join at the end.  Bound
// by latency: 5.0 us for 8 sequences' 256 rows over 100,003 shared tokens, 4.7
// to 6.0 in other batches.
template <bool kBf, int NB>
__global__ __launch_bounds__(256) void join_parts_kernel(const JoinArgs a) {
  constexpr int kLanes = 8 * NB, kGroups = 64 / kLanes;
  const int64_t i = int64_t(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (i >= a.rows) return;
  const int lane = threadIdx.x & 63, in = lane % kLanes;
  const int group = min(lane / kLanes, kGroups - 1);  // lanes past the last group repeat it and are not looked at
  const int tok = int(i / a.heads), head = int(i % a.heads);
  const int64_t base = int64_t(head / a.group) * a.slots + tok * a.group + head % a.group;
  int r = word(a.runs, tok);
  const int64_t q_row = word(a.q_rows, tok);
  float m = -INFINITY, l = 0.f;
  float4 o{0.f, 0.f, 0.f, 0.f};
  while (r >= 0) {
    const Parts run = words(a.parts, r);
    r = run.parent;
    const int64_t first = base + run.slot0;
    for (int p = group; p < run.count; p += kGroups * kJoin) {
      float2 ml[kJoin];
      float4 x[kJoin];
#pragma unroll
      for (int k = 0; k < kJoin; ++k) {  // past the last part, that one again, and taken out below
        const int64_t at = first + int64_t(min(p + k * kGroups, run.count - 1)) * run.rows;
        ml[k] = a.part_ml[at];
        x[k] = *reinterpret_cast<const float4*>(a.part_o + at * (32 * NB) + 4 * in);
      }
      float top = m;
#pragma unroll
      for (int k = 0; k < kJoin; ++k) {
        if (p + k * kGroups >= run.count) {
          ml[k].x = -INFINITY;
          x[k] = float4{0.f, 0.f, 0.f, 0.f};  // no weight times infinity would be no number
        }
        top = fmaxf(top, ml[k].x);
      }
      const float from = top == -INFINITY ? 0.f : top;
      const float keep = __builtin_amdgcn_exp2f(m - from);
      l *= keep;
      o.x *= keep;
      o.y *= keep;
      o.z *= keep;
      o.w *= keep;
#pragma unroll
      for (int k = 0; k < kJoin; ++k) {
        // A part of no weight has nothing the row sees, or what has underflowed beside the rest.
        const float w = __builtin_amdgcn_exp2f(ml[k].x - from);
        l += w * ml[k].y;
        o.x += w * x[k].x;
        o.y += w * x[k].y;
        o.z += w * x[k].z;
        o.w += w * x[k].w;
      }
      m = top;
    }
  }
  float top = m;
#pragma unroll
  for (int k = 0; k < kGroups; ++k) top = fmaxf(top, __shfl(m, k * kLanes + in));
  const float w = __builtin_amdgcn_exp2f(m - (top == -INFINITY ? 0.f : top));
  // In the order of the groups.
  float sum[5] = {0.f, 0.f, 0.f, 0.f, 0.f};
  const float mine[5] = {w * l, w * o.x, w * o.y, w * o.z, w * o.w};
#pragma unroll
  for (int k = 0; k < kGroups; ++k)
#pragma unroll
    for (int c = 0; c < 5; ++c) sum[c] += __shfl(mine[c], k * kLanes + in);
  const float inv = 1.f / sum[0];
  if (lane < kLanes && 4 * in < a.dim)
    *reinterpret_cast<uint2*>(a.out.p + 2 * (q_row * a.out.token + head * a.out.head + 4 * in)) =
        uint2{pack2<kBf>(sum[1] * inv, sum[2] * inv), pack2<kBf>(sum[3] * inv, sum[4] * inv)};
  if (a.lse && lane == 0) a.lse[int64_t(head) * a.q_tokens + q_row] = (top + __builtin_amdgcn_logf(sum[0])) * kLn2;
}

template <bool kBf>
void launch_join(cvs_context* ctx, const JoinArgs& a, int nb) {
  const TimerSpan ts = timer_span(ctx, "kv_join");
  auto go = [&](auto kernel) {
    hipExtLaunchKernelGGL(kernel, dim3(unsigned((a.rows + 3) / 4)), dim3(256), 0, ctx->stream, ts.start, ts.stop, 0, a);
  };
  switch (nb) {
    case 1: go(join_parts_kernel<kBf, 1>); break;
    case 2: go(join_parts_kernel<kBf, 2>); break;
    case 3: go(join_parts_kernel<kBf, 3>); break;
    default: go(join_parts_kernel<kBf, 4>); break;
  }
  after_launch("join_parts_kernel");
}

template <typename T>
size_t append(std::vector<char>& blob, const std::vector<T>& v) {
  const size_t at = (blob.size() + 15) / 16 * 16;
  blob.resize(at + v.size() * sizeof(T));
  if (!v.empty()) std::memcpy(blob.data() + at, v.data(), v.size() * sizeof(T));
  return at;
}

}  // namespace

void plan_attention(cvs_kv_plan* plan, const int64_t* lengths, const int64_t* tokens, std::vector<char>& blob) {
  cvs_kv_cache* const c = plan->cache;
  kv::PageBook& book = *c->book;
  const int64_t pt = book.page_tokens();
  const int group = plan->heads / c->kv_heads;
  // The sequences with queries, and where their rows are in q.
  std::vector<const int32_t*> lists;
  std::vector<int64_t> counts, from, first_row;
  int64_t q_row = 0;
  for (size_t i = 0; i < plan->seqs.size(); ++i) {
    if (tokens[i] > 0) {
      lists.push_back(book.at(plan->seqs[i]).pages.data());
      counts.push_back(book.pages_for(lengths[i]));
      from.push_back(int64_t(i));
      first_row.push_back(q_row);
    }
    q_row += tokens[i];
  }
  if (lists.empty()) return;
  if (plan->tokens * group > kv::PageBook::kMaxTokens) fail(CVS_ERR_UNSUPPORTED, "query rows must fit 31 bits");
  // A small batch is worked on sequence by sequence, whatever its sequences share: in one kernel, as none is long enough
  // to be split (kFewTiles), where a shared run would need the second one to join it with what is behind it.  9
  // sequences of 364 + 8 tokens: 7.7 us, and 8.5 + 4.3 shared; 22 of 142 + 7: 7.4 and 8.8 + 5.2.  The bytes bound what
  // is read again and again.
  constexpr int64_t kFewTiles = 32, kManyTiles = 16, kOverhead = 4, kSmallBytes = int64_t(32) << 20;
  const size_t n = lists.size();
  int64_t longest_list = 0, sum_tiles = 0;
  for (size_t i = 0; i < n; ++i) {
    const int64_t tiles = (lengths[from[i]] + kTile - 1) / kTile;
    longest_list = std::max(longest_list, tiles);
    sum_tiles += tiles;
  }
  const bool small = longest_list <= kFewTiles && int64_t(n) * c->kv_heads <= 2 * c->ctx->compute_units &&
                     sum_tiles * kTile * c->kv_heads * 128 * c->nb <= kSmallBytes;
  std::vector<int64_t> order(n);
  std::vector<kv::SharedRun> shared;
  if (small)
    for (size_t i = 0; i < n; ++i) {
      order[i] = int64_t(i);
      shared.push_back({0, counts[i], int64_t(i), int64_t(i) + 1, int64_t(i)});
    }
  else
    shared = kv::shared_runs(lists, counts, order);

  std::vector<int32_t> limits, q_rows;
  std::vector<int64_t> tok0(n + 1, 0);
  for (size_t p = 0; p < n; ++p) {
    const int64_t s = order[p], len = lengths[from[size_t(s)]], new_tokens = tokens[from[size_t(s)]];
    for (int64_t j = 0; j < new_tokens; ++j) {
      limits.push_back(int32_t(len - new_tokens + j + 1));
      q_rows.push_back(int32_t(first_row[size_t(s)] + j));
    }
    tok0[p + 1] = tok0[p] + new_tokens;
  }

  // Rows of a run go in blocks of up to 128, a block's tiles in equal segments, one a workgroup.  Splitting a block
  // costs a second kernel and, for each segment, what a workgroup does before its first tile and after its last (about
  // kOverhead tiles), so blocks are not split into segments of fewer tiles than these: one short sequence of 25 tiles
  // takes 7.3 us whole and 8.8 in parts of 8, 32 questions of 5 tokens over 126 tiles 25.2 us in parts of 16, 31.6 in
  // parts of 32 and 29.0 in parts of 8.
  std::vector<int64_t> run_tiles(shared.size()), run_rows(shared.size());
  int64_t longest = 1;
  for (size_t r = 0; r < shared.size(); ++r) {
    const kv::SharedRun& s = shared[r];
    int64_t most = 0;
    for (int64_t p = s.lo; p < s.hi; ++p) most = std::max(most, lengths[from[size_t(order[size_t(p)])]]);
    run_tiles[r] = (std::min((s.first + s.count) * pt, most) - s.first * pt + kTile - 1) / kTile;
    run_rows[r] = (tok0[size_t(s.hi)] - tok0[size_t(s.lo)]) * group;
    longest = std::max(longest, run_tiles[r]);
  }
  // Where no run lies behind another and all are at most half longer than that, nothing is split and nothing joined: one
  // sequence of 1,025 tokens 10.6 us, and 8.4 + 4.1 in two parts; 7 of 500 with 21 new tokens 16.0, and 15.1 + 5.6.
  bool whole = true;
  for (size_t r = 0; r < shared.size(); ++r)
    whole = whole && shared[r].first == 0 && 2 * run_tiles[r] <= 3 * (run_rows[r] > kTile ? kManyTiles : kFewTiles);
  // Segments of at most `share` tiles.
  auto parts_of = [&](size_t r, int64_t share) {
    if (whole) return int64_t(1);
    const int64_t least = run_rows[r] > kTile ? kManyTiles : kFewTiles;
    return (run_tiles[r] + std::max(share, least) - 1) / std::max(share, least);
  };
  auto segments_at = [&](int64_t share) {
    int64_t sum = 0;
    for (size_t r = 0; r < shared.size(); ++r) sum += parts_of(r, share) * ((run_rows[r] + kBlock - 1) / kBlock);
    return sum;
  };
  // Two workgroups a compute unit run at a time: the smallest share that fits one such round, or two or three.
  int64_t share = longest, cost = INT64_MAX;
  for (int64_t rounds = 1; rounds <= 3; ++rounds) {
    const int64_t fit = std::max<int64_t>(1, rounds * 2 * c->ctx->compute_units / c->kv_heads);
    int64_t lo = 1, hi = longest;
    while (lo < hi) {
      const int64_t mid = (lo + hi) / 2;
      if (segments_at(mid) <= fit) hi = mid;
      else lo = mid + 1;
    }
    int64_t most = 0;  // tiles of the largest segment
    for (size_t r = 0; r < shared.size(); ++r) {
      const int64_t parts = parts_of(r, lo);
      most = std::max(most, (run_tiles[r] + parts - 1) / parts);
    }
    if (rounds * (most + kOverhead) < cost) {
      share = lo;
      cost = rounds * (most + kOverhead);
    }
  }

  std::vector<Segment> segments;
  std::vector<Parts> parts(shared.size());
  std::vector<int32_t> pages, last_runs, cur(n, -1);
  int64_t slots = 0;
  bool one_part = true;
  for (size_t r = 0; r < shared.size(); ++r) {
    const kv::SharedRun& s = shared[r];
    const int64_t t0 = tok0[size_t(s.lo)], count = parts_of(r, share), rows = run_rows[r];
    const int32_t parent = cur[size_t(s.lo)];
    for (int64_t p = s.lo; p < s.hi; ++p) cur[size_t(p)] = int32_t(r);
    if (parent >= 0 || count > 1) one_part = false;
    if (slots + rows * count > kv::PageBook::kMaxTokens) fail(CVS_ERR_UNSUPPORTED, "too many partial results");
    parts[r] = {int32_t(slots - t0 * group), int32_t(rows), int32_t(count), parent};
    const int32_t page_first = int32_t(pages.size());
    const int32_t* const list = lists[size_t(s.member)];
    pages.insert(pages.end(), list + s.first, list + s.first + s.count);
    const int64_t each = (run_tiles[r] + count - 1) / count;
    for (int64_t part = 0; part < count; ++part)
      for (int64_t row = 0; row < rows; row += kBlock) {
        const int64_t in = std::min<int64_t>(kBlock, rows - row), tile = part * each;
        int32_t lo = INT32_MAX, hi = 0;
        for (int64_t t = t0 + row / group; t <= t0 + (row + in - 1) / group; ++t) {
          lo = std::min(lo, limits[size_t(t)]);
          hi = std::max(hi, limits[size_t(t)]);
        }
        // Not the tiles that none of the block's rows sees; a segment that has no others still writes its (empty) part.
        const int64_t seen = std::min(run_tiles[r], (hi - s.first * pt + kTile - 1) / kTile);
        segments.push_back({page_first, int32_t(tile), int32_t(std::clamp<int64_t>(seen - tile, 0, each)),
                            int32_t(s.first * pt), int32_t(t0 * group + row), int32_t(in),
                            int32_t(slots + part * rows + row), lo, hi});
      }
    slots += rows * count;
  }
  // The longest first, so that the last workgroups to start are short ones.
  std::stable_sort(segments.begin(), segments.end(),
                   [](const Segment& x, const Segment& y) { return x.tiles > y.tiles; });
  if (int64_t(segments.size()) * c->kv_heads > kMaxBlocks || (!one_part && plan->tokens * plan->heads > kMaxBlocks * 4))
    fail(CVS_ERR_UNSUPPORTED, "too many query rows");
  for (size_t p = 0; p < n; ++p) last_runs.insert(last_runs.end(), size_t(tok0[p + 1] - tok0[p]), cur[p]);
  plan->workgroups = int(segments.size());
  plan->slots = one_part ? 0 : slots;
  plan->at_segments = append(blob, segments);
  plan->at_pages = append(blob, pages);
  plan->at_limits = append(blob, limits);
  plan->at_rows = append(blob, q_rows);
  if (one_part) return;
  plan->at_runs = append(blob, last_runs);
  plan->at_parts = append(blob, parts);
}

}  // namespace attn
}  // namespace cvs

using namespace cvs;
using namespace cvs::attn;

extern "C" int cvs_kv_attention_async(cvs_kv_cache* cache, cvs_kv_plan* plan, int layer, const cvs_heads* q,
                                      const cvs_heads* out, float* lse, float scale) {
  return cvs_kv_attention_scored_async(cache, plan, layer, q, out, lse, scale, nullptr);
}

extern "C" int cvs_kv_attention_scored_async(cvs_kv_cache* cache, cvs_kv_plan* plan, int layer, const cvs_heads* q,
                                             const cvs_heads* out, float* lse, float scale,
                                             const cvs_scores* scores) {
  return guarded([&] {
    if (!cache) fail(CVS_ERR_INVALID_ARGUMENT, "null cache");
    if (!plan) fail(CVS_ERR_INVALID_ARGUMENT, "null plan");
    if (plan->cache != cache) fail(CVS_ERR_INVALID_ARGUMENT, "the plan belongs to another cache");
    cvs_context* const ctx = cache->ctx;
    bind(ctx);
    check_plan(plan);
    if (plan->heads == 0) fail(CVS_ERR_INVALID_ARGUMENT, "the plan was made without query heads");
    if (layer < 0 || layer >= cache->layers)
      fail(CVS_ERR_INVALID_ARGUMENT, "layer outside the cache's " + std::to_string(cache->layers));
    for (const cvs_heads* x : {q, out}) {
      const char* const what = x == q ? "q" : "out";
      check_view(x, what);
      if (x->tokens != plan->tokens)
        fail(CVS_ERR_INVALID_ARGUMENT,
             std::string(what) + " must have the plan's " + std::to_string(plan->tokens) + " tokens");
      if (x->heads != plan->heads) fail(CVS_ERR_INVALID_ARGUMENT, std::string(what) + " must have the plan's heads");
      if (x->head_dim != cache->dim || x->type != cache->type)
        fail(CVS_ERR_INVALID_ARGUMENT, std::string(what) + " must have the cache's head_dim and type");
    }
    check_rows_apart(out, "out");
    const ScoreArgs sc = score_args(scores, scale, cache->dim);
    if (plan->workgroups == 0) return;
    const char* const blob = plan->blob.as<char>();
    const int group = plan->heads / cache->kv_heads;
    float* part_o = nullptr;
    float2* part_ml = nullptr;
    const size_t slots = size_t(plan->slots) * size_t(cache->kv_heads), width = size_t(32 * cache->nb);
    const bool captured = captured_call(plan);
    if (slots) {
      const size_t bytes = slots * (width * sizeof(float) + sizeof(float2));
      if (bytes > ctx->ws_attn.bytes) {
        if (captured)
          fail(CVS_ERR_INVALID_ARGUMENT, "a call's memory cannot be made while the context's stream is being captured "
                                         "into a graph: make the call once before");
        if (ctx->ws_attn_captured) {
          ctx->kept.push_back(ctx->ws_attn);
          ctx->ws_attn = DeviceBuffer();
          ctx->ws_attn_captured = false;
        }
      }
      ctx->ws_attn.reserve(bytes);
      ctx->ws_attn_captured |= captured;
      part_o = ctx->ws_attn.as<float>();
      part_ml = reinterpret_cast<float2*>(part_o + slots * width);
    }
    int shift = 0;
    while ((kTile << shift) < cache->book->page_tokens()) ++shift;
    const CachedArgs a{cache->pool + layer * cache->layer_bytes, cache->page_bytes, cache->head_bytes, shift,
                       reinterpret_cast<const Segment*>(blob + plan->at_segments),
                       reinterpret_cast<const int32_t*>(blob + plan->at_pages),
                       reinterpret_cast<const int32_t*>(blob + plan->at_limits),
                       reinterpret_cast<const int32_t*>(blob + plan->at_rows), view_of(q), view_of(out), lse,
                       plan->tokens, cache->kv_heads, group, cache->dim, part_o, part_ml, plan->slots, sc};
    const int64_t blocks = int64_t(plan->workgroups) * cache->kv_heads;
    const bool is_bf = cache->type == CVS_BF16;
    if (sc.cap > 0.f || sc.slopes) launch_cached_scored(ctx, a, cache->nb, blocks, cache->type);
    else if (is_bf) launch_cached<true, PlainScores>(ctx, a, cache->nb, blocks);
    else launch_cached<false, PlainScores>(ctx, a, cache->nb, blocks);
    if (!slots) return;
    const JoinArgs j{reinterpret_cast<const Parts*>(blob + plan->at_parts),
                     reinterpret_cast<const int32_t*>(blob + plan->at_runs),
                     reinterpret_cast<const int32_t*>(blob + plan->at_rows), part_o, part_ml, plan->slots,
                     plan->tokens * plan->heads, view_of(out), lse, plan->tokens, plan->heads, group, cache->dim};
    if (is_bf) launch_join<true>(ctx, j, cache->nb);
    else launch_join<false>(ctx, j, cache->nb);
  });
}
