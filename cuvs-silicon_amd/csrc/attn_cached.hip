// Attention of a batch's newest tokens over a paged cache, with what the
// sequences share read once for all of them.
//
// The plan lays the batch's page lists out as a tree: a run of pages and the
// sequences that begin with it (kv_pages.hpp).  A run's rows are the (token,
// head of the group) pairs of all its sequences; its keys are split into
// chunks, and a workgroup takes 32 of the rows and one chunk.  Its 4 waves
// take the chunk's 32-key tiles in turn, each with a running softmax of its
// own, straight from memory into operand registers (the pool's tiles are the
// operands), and join at the end through LDS.  A row's results from its runs
// and chunks are (maximum, sum, values) in fp32, which a second kernel joins;
// where every row has one part the first writes the output itself.
#include <algorithm>
#include <cstring>

#include "attn_common.hpp"

namespace cvs {
namespace attn {
namespace {

constexpr int kTile = 32;     // rows and keys of a tile
constexpr int kWaves = 4;

struct Item {
  int32_t page_first;     // first of the run's pages in the plan's page list
  int32_t tile0, tiles;   // the chunk's tiles, counted from the run's first token
  int32_t key0;           // position in the sequence of the run's first token
  int32_t row0, rows;     // (token * group + head) rows, tokens in the plan's order
  int32_t slot0;          // of row0's partial result
  int32_t min_limit, max_limit;  // keys the rows see: positions below their limit
};

// A run of pages as the join sees it.
struct Run {
  int32_t parent;         // the run before it in its sequences, -1 for none
  int32_t slot0, chunks;  // chunk c of row row0 + i has slot slot0 + c * rows + i
  int32_t row0, rows;
};

struct CachedArgs {
  const char* pool;  // of the layer
  int64_t page_bytes, head_bytes;
  int page_shift;    // log2 of a page's tiles
  const Item* items;
  const int32_t* pages;
  const int32_t* limits;  // per token, in the plan's order
  const int32_t* q_rows;  // its row in q and out
  View q, out;
  float* lse;
  int64_t q_tokens;
  int kv_heads, group, dim;
  float c;
  float* part_o;  // kv head, slot, 32 NB values
  float2* part_ml;
  int64_t slots;  // 0: write the output
};

template <bool kBf, int NB>
__global__ __launch_bounds__(256, 2) void cached_attn_kernel(const CachedArgs a) {
  __shared__ float s_o[2][16 * NB][64];
  __shared__ float s_m[kWaves][64], s_l[kWaves][64];

  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = blockIdx.x % a.kv_heads;
  const Item it = a.items[blockIdx.x / a.kv_heads];

  const bool there = col < it.rows;
  const int row = it.row0 + min(col, it.rows - 1);
  const int tok = row / a.group, head = g * a.group + row % a.group;
  const int limit = a.limits[tok];
  const int64_t q_row = a.q_rows[tok];

  const int page_mask = (1 << a.page_shift) - 1;
  auto tile_at = [&](int i) CVS_INLINE {
    const int t = it.tile0 + i;
    const int64_t page = a.pages[it.page_first + (t >> a.page_shift)];
    return a.pool + page * a.page_bytes + g * a.head_bytes + (t & page_mask) * (2048 * NB) + lane * 16;
  };
  u32x4 kf[2 * NB], vf[2 * NB];
  auto load_keys = [&](const char* p) CVS_INLINE {
#pragma unroll
    for (int s = 0; s < 2 * NB; ++s) kf[s] = *reinterpret_cast<const u32x4*>(p + s * 1024);
  };
  auto load_values = [&](const char* p) CVS_INLINE {
#pragma unroll
    for (int s = 0; s < 2 * NB; ++s) vf[s] = *reinterpret_cast<const u32x4*>(p + a.head_bytes / 2 + s * 1024);
  };

  u32x4 q[2 * NB];
  {
    const char* src = a.q.p + 2 * (q_row * a.q.token + head * a.q.head);
#pragma unroll
    for (int s = 0; s < 2 * NB; ++s)
      q[s] = 16 * s + 8 * half < a.dim ? *reinterpret_cast<const u32x4*>(src + 32 * s + 16 * half) : u32x4{};
  }

  RowState<NB> st;
  st.init();
  uint32_t bad = 0;
  if (wave < it.tiles) {
    const char* p = tile_at(wave);
    load_keys(p);
    load_values(p);
    for (int i = wave; i < it.tiles; i += kWaves) {
      f32x16 s{};
#pragma unroll
      for (int k = 0; k < 2 * NB; ++k) s = mfma<kBf>(kf[k], q[k], s);
      p = tile_at(i + kWaves < it.tiles ? i + kWaves : i);
      load_keys(p);
      const int key0 = it.key0 + kTile * (it.tile0 + i);
      const bool mixed = key0 + kTile > it.min_limit;
      if (mixed) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (key0 + 8 * (r / 4) + 4 * half + r % 4 >= limit) s[r] = -INFINITY;
      }
      raise_max(s, st, a.c);
      exponentials(s, st, a.c);
      if (mixed) {
        // Past the largest limit the page holds whatever was there: zeros instead.  Infinities and NaNs in keys that
        // some rows see go around the product.
        const int left = it.max_limit - key0 - 4 * half;
#pragma unroll
        for (int k = 0; k < 2 * NB; ++k) {
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const int t = 16 * (k & 1) + 8 * (w / 2) + 2 * (w % 2);
            vf[k][w] &= (t < left ? 0xffffu : 0u) | (t + 1 < left ? 0xffff0000u : 0u);
          }
          vf[k] = clean<kBf>(vf[k], bad);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const u32x4 pr = prob_operand<kBf>(s, h);
#pragma unroll
        for (int b = 0; b < NB; ++b) st.o[b] = mfma<kBf>(vf[2 * b + h], pr, st.o[b]);
      }
      load_values(p);
    }
  }

  // The waves' states joined, in the order 0 + 2, 1 + 3, then both.
  s_m[wave][lane] = st.m;
  const bool met = __syncthreads_or(bad != 0);  // infinities or NaNs that some rows do not see
  float m = s_m[0][lane];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) m = fmaxf(m, s_m[w][lane]);
  const float alpha = __builtin_amdgcn_exp2f(st.m - (m == -INFINITY ? 0.f : m));
  s_l[wave][lane] = st.l * alpha;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) st.o[b][r] *= alpha;
#pragma unroll
  for (int step = 2; step >= 1; step >>= 1) {
    if (wave >= step && wave < 2 * step) {
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) s_o[wave - step][16 * b + r][lane] = st.o[b][r];
    }
    __syncthreads();
    if (wave < step) {
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) st.o[b][r] += s_o[wave][16 * b + r][lane];
    }
    __syncthreads();
  }
  if (wave != 0) return;
  const float l = both_sum((s_l[0][lane] + s_l[2][lane]) + (s_l[1][lane] + s_l[3][lane]));
  auto value = [&](int key, int d) CVS_INLINE {
    const int rel = key - it.key0, j = rel & 31, t = rel / kTile;
    const int64_t page = a.pages[it.page_first + (t >> a.page_shift)];
    const char* const v = a.pool + page * a.page_bytes + g * a.head_bytes + a.head_bytes / 2 +
                          (t & page_mask) * (2048 * NB);
    const int at = (d & 31) + 32 * ((j >> 2) & 1), e = 4 * ((j >> 3) & 1) + (j & 3);
    return *reinterpret_cast<const uint16_t*>(v + (2 * (d >> 5) + (j >> 4)) * 1024 + 16 * at + 2 * e);
  };
  const int first = it.key0 + kTile * it.tile0;
  const int last = there && l == l ? min(first + kTile * it.tiles, limit) : 0;
  if (a.slots == 0) {
    uint16_t* const out = reinterpret_cast<uint16_t*>(a.out.p) + q_row * a.out.token + head * a.out.head;
    store_row<kBf, NB>(st, 1.f / l, out, a.dim, there);
    if (met)
      store_nonfinite<kBf>(first, last, a.dim, value,
                           [&](int d, float x) CVS_INLINE { out[d] = uint16_t(pack2<kBf>(x, x)); });
    if (a.lse && there && half == 0)
      a.lse[int64_t(head) * a.q_tokens + q_row] = (m + __builtin_amdgcn_logf(l)) * kLn2;
    return;
  }
  const int64_t slot = g * a.slots + it.slot0 + col;
  float* const o = a.part_o + slot * (32 * NB);
  if (there) {
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<float4*>(o + 32 * b + 8 * j + 4 * half) =
            float4{st.o[b][4 * j], st.o[b][4 * j + 1], st.o[b][4 * j + 2], st.o[b][4 * j + 3]};
    if (half == 0) a.part_ml[slot] = float2{m, l};
  }
  if (met) store_nonfinite<kBf>(first, last, a.dim, value, [&](int d, float x) CVS_INLINE { o[d] = x; });
}

struct JoinArgs {
  const Run* runs;
  const int32_t* leaves;  // per token, the last of its runs
  const int32_t* q_rows;
  const float* part_o;
  const float2* part_ml;
  int64_t slots, rows;    // rows: tokens * heads
  View out;
  float* lse;
  int64_t q_tokens;
  int heads, group, dim, nb;
};

// One wave a (token, head) row: lanes take 2 columns each.
template <bool kBf>
__global__ __launch_bounds__(256) void join_parts_kernel(const JoinArgs a) {
  const int64_t i = int64_t(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (i >= a.rows) return;
  const int lane = threadIdx.x & 63;
  const int tok = int(i / a.heads), head = int(i % a.heads);
  const int64_t base = int64_t(head / a.group) * a.slots;
  const int row = tok * a.group + head % a.group;
  const int leaf = a.leaves[tok];
  float m = -INFINITY;
  for (int r = leaf; r >= 0;) {
    const Run run = a.runs[r];
    const int64_t s = base + run.slot0 + row - run.row0;
    for (int c = lane; c < run.chunks; c += 64) m = fmaxf(m, a.part_ml[s + int64_t(c) * run.rows].x);
    r = run.parent;
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) m = fmaxf(m, xor_lanes_f(m, o));
  const float from = m == -INFINITY ? 0.f : m;
  float l = 0.f, o0 = 0.f, o1 = 0.f;
  const int d = 2 * lane, width = 32 * a.nb;
  const int dl = d < width ? d : 0;
  for (int r = leaf; r >= 0;) {
    const Run run = a.runs[r];
    const int64_t s = base + run.slot0 + row - run.row0;
#pragma unroll 4
    for (int c = 0; c < run.chunks; ++c) {
      const int64_t at = s + int64_t(c) * run.rows;
      const float2 ml = a.part_ml[at];
      const float2 o = *reinterpret_cast<const float2*>(a.part_o + at * width + dl);
      const float w = __builtin_amdgcn_exp2f(ml.x - from);
      l += w * ml.y;
      o0 += w * o.x;
      o1 += w * o.y;
    }
    r = run.parent;
  }
  const float inv = 1.f / l;
  const int64_t q_row = a.q_rows[tok];
  if (d < a.dim)
    *reinterpret_cast<uint32_t*>(a.out.p + 2 * (q_row * a.out.token + head * a.out.head + d)) =
        pack2<kBf>(o0 * inv, o1 * inv);
  if (a.lse && lane == 0) a.lse[int64_t(head) * a.q_tokens + q_row] = (m + __builtin_amdgcn_logf(l)) * kLn2;
}

template <typename T>
size_t append(std::vector<char>& blob, const std::vector<T>& v) {
  const size_t at = (blob.size() + 15) / 16 * 16;
  blob.resize(at + v.size() * sizeof(T));
  if (!v.empty()) std::memcpy(blob.data() + at, v.data(), v.size() * sizeof(T));
  return at;
}

template <bool kBf>
void launch(cvs_context* ctx, const CachedArgs& a, int nb, int64_t blocks) {
  const TimerSpan ts = timer_span(ctx, "kv_attention");
  auto go = [&](auto kernel) {
    hipExtLaunchKernelGGL(kernel, dim3(unsigned(blocks)), dim3(256), 0, ctx->stream, ts.start, ts.stop, 0, a);
  };
  switch (nb) {
    case 1: go(cached_attn_kernel<kBf, 1>); break;
    case 2: go(cached_attn_kernel<kBf, 2>); break;
    case 3: go(cached_attn_kernel<kBf, 3>); break;
    default: go(cached_attn_kernel<kBf, 4>); break;
  }
  after_launch("cached_attn_kernel");
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
  std::vector<int64_t> order;
  const std::vector<kv::SharedRun> shared = kv::shared_runs(lists, counts, order);

  const size_t n = order.size();
  std::vector<int32_t> limits, q_rows, leaves;
  std::vector<int64_t> tok0(n + 1, 0);
  for (size_t p = 0; p < n; ++p) {
    const int64_t s = order[p], len = lengths[from[size_t(s)]], new_tokens = tokens[from[size_t(s)]];
    for (int64_t j = 0; j < new_tokens; ++j) {
      limits.push_back(int32_t(len - new_tokens + j + 1));
      q_rows.push_back(int32_t(first_row[size_t(s)] + j));
    }
    tok0[p + 1] = tok0[p] + new_tokens;
  }

  // Work in (32 rows, 32 keys) tiles of one kv head, and the chunk that spreads it over the device: enough
  // workgroups for four a compute unit, but at least two tiles a wave.
  std::vector<int64_t> run_tiles(shared.size());
  int64_t work = 0;
  for (size_t r = 0; r < shared.size(); ++r) {
    const kv::SharedRun& s = shared[r];
    int64_t most = 0;
    for (int64_t p = s.lo; p < s.hi; ++p) most = std::max(most, lengths[from[size_t(order[size_t(p)])]]);
    run_tiles[r] = (std::min((s.first + s.count) * pt, most) - s.first * pt + kTile - 1) / kTile;
    const int64_t rows = (tok0[size_t(s.hi)] - tok0[size_t(s.lo)]) * group;
    work += run_tiles[r] * ((rows + kTile - 1) / kTile);
  }
  const int64_t target = std::max<int64_t>(1, int64_t(4) * c->ctx->compute_units / c->kv_heads);
  const int64_t chunk = std::max<int64_t>(2 * kWaves, (work + target - 1) / target);

  std::vector<Item> items;
  std::vector<Run> runs;
  std::vector<int32_t> pages, cur(n, -1);
  int64_t slots = 0;
  bool one_part = true;
  for (size_t r = 0; r < shared.size(); ++r) {
    const kv::SharedRun& s = shared[r];
    const int64_t t0 = tok0[size_t(s.lo)], t1 = tok0[size_t(s.hi)], rows = (t1 - t0) * group;
    const int64_t chunks = (run_tiles[r] + chunk - 1) / chunk;
    const int64_t each = (run_tiles[r] + chunks - 1) / chunks;
    const int32_t parent = cur[size_t(s.lo)];
    if (parent >= 0 || chunks > 1) one_part = false;
    for (int64_t p = s.lo; p < s.hi; ++p) cur[size_t(p)] = int32_t(r);
    if (slots + rows * chunks > (int64_t(1) << 31) - 1) fail(CVS_ERR_UNSUPPORTED, "too many partial results");
    const int32_t page_first = int32_t(pages.size());
    const int32_t* const list = lists[size_t(s.member)];
    pages.insert(pages.end(), list + s.first, list + s.first + s.count);
    runs.push_back({parent, int32_t(slots), int32_t(chunks), int32_t(t0 * group), int32_t(rows)});
    for (int64_t k = 0; k < chunks; ++k) {
      const int64_t tile0 = k * each, tiles = std::min(each, run_tiles[r] - tile0);
      for (int64_t row = 0; row < rows; row += kTile) {
        const int64_t in = std::min<int64_t>(kTile, rows - row);
        int32_t lo = INT32_MAX, hi = 0;
        for (int64_t t = t0 + row / group; t <= t0 + (row + in - 1) / group; ++t) {
          lo = std::min(lo, limits[size_t(t)]);
          hi = std::max(hi, limits[size_t(t)]);
        }
        items.push_back({page_first, int32_t(tile0), int32_t(tiles), int32_t(s.first * pt), int32_t(t0 * group + row),
                         int32_t(in), int32_t(slots + k * rows + row), lo, hi});
      }
    }
    slots += rows * chunks;
  }
  if (int64_t(items.size()) * c->kv_heads > (int64_t(1) << 31) - 1) fail(CVS_ERR_UNSUPPORTED, "too much work");
  for (size_t p = 0; p < n; ++p)
    for (int64_t t = tok0[p]; t < tok0[p + 1]; ++t) leaves.push_back(cur[p]);
  plan->items = int(items.size());
  plan->slots = one_part ? 0 : slots;
  plan->at_items = append(blob, items);
  plan->at_pages = append(blob, pages);
  plan->at_limits = append(blob, limits);
  plan->at_rows = append(blob, q_rows);
  plan->at_leaves = append(blob, leaves);
  plan->at_runs = append(blob, runs);
}

}  // namespace attn
}  // namespace cvs

using namespace cvs;
using namespace cvs::attn;

extern "C" int cvs_kv_attention_async(cvs_kv_cache* cache, cvs_kv_plan* plan, int layer, const cvs_heads* q,
                                      const cvs_heads* out, float* lse, float scale) {
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
    const float c = scale_log2(scale, cache->dim);
    if (plan->items == 0) return;
    const char* const blob = plan->blob.as<char>();
    const int group = plan->heads / cache->kv_heads;
    float* part_o = nullptr;
    float2* part_ml = nullptr;
    const size_t slots = size_t(plan->slots) * size_t(cache->kv_heads), width = size_t(32 * cache->nb);
    if (slots) {
      ctx->ws_attn.reserve(slots * (width * sizeof(float) + sizeof(float2)));
      part_o = ctx->ws_attn.as<float>();
      part_ml = reinterpret_cast<float2*>(part_o + slots * width);
    }
    int shift = 0;
    while ((kTile << shift) < cache->book->page_tokens()) ++shift;
    const CachedArgs a{cache->pool + layer * cache->layer_bytes, cache->page_bytes, cache->head_bytes, shift,
                       reinterpret_cast<const Item*>(blob + plan->at_items),
                       reinterpret_cast<const int32_t*>(blob + plan->at_pages),
                       reinterpret_cast<const int32_t*>(blob + plan->at_limits),
                       reinterpret_cast<const int32_t*>(blob + plan->at_rows), view_of(q), view_of(out), lse,
                       plan->tokens, cache->kv_heads, group, cache->dim, c, part_o, part_ml, plan->slots};
    const int64_t blocks = int64_t(plan->items) * cache->kv_heads;
    const bool is_bf = cache->type == CVS_BF16;
    if (is_bf) launch<true>(ctx, a, cache->nb, blocks);
    else launch<false>(ctx, a, cache->nb, blocks);
    if (!slots) return;
    const JoinArgs j{reinterpret_cast<const Run*>(blob + plan->at_runs),
                     reinterpret_cast<const int32_t*>(blob + plan->at_leaves),
                     reinterpret_cast<const int32_t*>(blob + plan->at_rows), part_o, part_ml, plan->slots,
                     plan->tokens * plan->heads, view_of(out), lse, plan->tokens, plan->heads, group, cache->dim,
                     cache->nb};
    const TimerSpan ts = timer_span(ctx, "kv_join");
    const dim3 grid(unsigned((j.rows + 3) / 4));
    if (is_bf) hipExtLaunchKernelGGL(join_parts_kernel<true>, grid, dim3(256), 0, ctx->stream, ts.start, ts.stop, 0, j);
    else hipExtLaunchKernelGGL(join_parts_kernel<false>, grid, dim3(256), 0, ctx->stream, ts.start, ts.stop, 0, j);
    after_launch("join_parts_kernel");
  });
}
