// Attention of a batch's newest tokens over a paged cache, with what the
// sequences share read once for all of them.
//
// The plan lays the batch's page lists out as a tree: a run of pages and the
// sequences that begin with it (kv_pages.hpp).  A run's rows are the (token,
// head of the group) pairs of all its sequences, taken in blocks; a block's
// keys are cut into segments, so that every workgroup has about as many tiles
// of 32 keys to go through.  Two shapes of block:
//   up to 32 rows (the decoding of a sequence's own tokens, bound by the
//   reading of the cache): the 4 waves take the segment's tiles in turn, each
//   with a running softmax of its own, straight from memory into operand
//   registers (the pool's tiles are the operands), and join through LDS;
//   33 to 128 rows (many sequences on one prefix, or many new tokens, bound by
//   the matrix cores as well): each wave has 32 of the rows, and the tiles go
//   through LDS once for all of them (attend_tiles).
// A row's results from its runs and segments are (maximum, sum, values) in
// fp32, which a second kernel joins; where every row has one part the first
// writes the output itself.
//
// Bounds: long sequences the memory (48 of 100 to 6,000 tokens, 8 kv heads of
// 128, bf16, a token each: 103 us = 6.3 TB/s of distinct cache bytes; 8 over
// 100,003 shared tokens: 69 us = 5.9 TB/s of the shared ones alone), short ones
// latency: one sequence of 777 tokens, 16/4 heads of 64, takes 7.1 us, in which
// the plan, a page's id and its tiles are loaded one after another.
#pragma once

#include "attn_common.hpp"

namespace cvs {
namespace attn {
constexpr int kTile = 32;       // keys of a tile, rows of a wave
constexpr int kWaves = 4;
constexpr int kBlock = kTile * kWaves;  // rows of a large block

struct Segment {
  int32_t page_first;     // first of the run's pages in the plan's page list
  int32_t tile0, tiles;   // the segment's tiles, counted from the run's first token
  int32_t key0;           // position in the sequence of the run's first token
  int32_t row0, rows;     // (token * group + head) rows, tokens in the plan's order
  int32_t slot0;          // of row0's partial result
  int32_t min_limit, max_limit;  // keys the rows see: positions below their limit
};

struct CachedArgs {
  const char* pool;  // of the layer
  int64_t page_bytes, head_bytes;
  int page_shift;    // log2 of a page's tiles
  const Segment* segments;
  const int32_t* pages;
  const int32_t* limits;  // per token, in the plan's order
  const int32_t* q_rows;  // its row in q and out
  View q, out;
  float* lse;
  int64_t q_tokens;
  int kv_heads, group, dim;
  float* part_o;  // kv head, slot, 32 NB values
  float2* part_ml;
  int64_t slots;  // 0: write the output
  ScoreArgs scores;
};

// Words of the plan: written before the kernel starts and never by it, which
// the constant address space tells the compiler, so that a word at the same
// place for all lanes is loaded to a scalar register.
__device__ CVS_INLINE int32_t word(const int32_t* p, int64_t i) {
  return reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(reinterpret_cast<uintptr_t>(p))[i];
}
template <typename T>
__device__ CVS_INLINE T words(const T* p, int64_t i) {
  constexpr int n = sizeof(T) / 4;
  int32_t x[n];
#pragma unroll
  for (int k = 0; k < n; ++k) x[k] = word(reinterpret_cast<const int32_t*>(p + i), k);
  T t;
  __builtin_memcpy(&t, x, sizeof(T));
  return t;
}

// A lane's query row.
struct Row {
  bool there;
  int head, limit;
  int64_t q_row;
};

// Everything of a segment that both shapes of block use.
template <bool kBf, int NB>
struct Work {
  const CachedArgs& a;
  const Segment& it;
  int g, lane, half;

  __device__ CVS_INLINE const char* tile(int i) const {  // of the segment, this kv head's keys
    const int t = it.tile0 + i;
    return at(word(a.pages, it.page_first + (t >> a.page_shift)), t);
  }
  __device__ CVS_INLINE const char* at(int64_t page, int t) const {
    return a.pool + page * a.page_bytes + g * a.head_bytes + (t & ((1 << a.page_shift) - 1)) * (4096 * NB);
  }
  __device__ CVS_INLINE Row row(int i) const {  // past the last row, the last one's again (not stored)
    const int r = it.row0 + min(i, it.rows - 1), tok = r / a.group;
    return {i < it.rows, g * a.group + r % a.group, a.limits[tok], a.q_rows[tok]};
  }
  __device__ CVS_INLINE void load_q(const Row& r, u32x4 (&q)[2 * NB]) const {
    load_row<2 * NB>(a.q.p + 2 * (r.q_row * a.q.token + r.head * a.q.head), a.dim, q);
  }
  // A tile's values that no row sees may be anything (the page's memory as it was): zeros instead.  key0: of the tile.
  __device__ CVS_INLINE u32x4 hide(u32x4 v, int k16, int key0, int end) const {
    const int left = end - key0 - 4 * half;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int t = 16 * k16 + 8 * (w / 2) + 2 * (w % 2);
      v[w] &= (t < left ? 0xffffu : 0u) | (t + 1 < left ? 0xffff0000u : 0u);
    }
    return v;
  }
  // Stores row i of the segment: the output, or a part.  met: whether some row's values had infinities or NaNs in keys
  // that others do not see.
  __device__ CVS_INLINE void store(const RowState<NB>& st, float m, float l, const Row& r, int i, bool met) const {
    auto value = [&](int key, int d) CVS_INLINE {
      const int rel = key - it.key0 - kTile * it.tile0, j = rel & 31;
      const char* const v = tile(rel / kTile) + 2048 * NB;
      const int at = (d & 31) + 32 * ((j >> 2) & 1), e = 4 * ((j >> 3) & 1) + (j & 3);
      return *reinterpret_cast<const uint16_t*>(v + (2 * (d >> 5) + (j >> 4)) * 1024 + 16 * at + 2 * e);
    };
    const int key0 = it.key0 + kTile * it.tile0, keys = kTile * it.tiles;
    const int first = key0 + first_cleaned(it.min_limit - key0, keys);
    const int last = r.there && l == l ? min(key0 + keys, r.limit) : 0;
    if (a.slots == 0) {
      uint16_t* const out = reinterpret_cast<uint16_t*>(a.out.p) + r.q_row * a.out.token + r.head * a.out.head;
      store_row<kBf, NB>(st, 1.f / l, out, a.dim, r.there);
      if (met)
        add_nonfinite<kBf>(first, last, a.dim, value, [&](int d, float x) CVS_INLINE {
          x += to_float<kBf>(out[d]);
          out[d] = uint16_t(pack2<kBf>(x, x));
        });
      if (a.lse && r.there && half == 0)
        a.lse[int64_t(r.head) * a.q_tokens + r.q_row] = (m + __builtin_amdgcn_logf(l)) * kLn2;
      return;
    }
    const int64_t slot = g * a.slots + it.slot0 + i;
    float* const o = a.part_o + slot * (32 * NB);
    if (r.there) {
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<float4*>(o + 32 * b + 8 * j + 4 * half) =
              float4{st.o[b][4 * j], st.o[b][4 * j + 1], st.o[b][4 * j + 2], st.o[b][4 * j + 3]};
      if (half == 0) a.part_ml[slot] = float2{m, l};
    }
    if (met) add_nonfinite<kBf>(first, last, a.dim, value, [&](int d, float x) CVS_INLINE { o[d] += x; });
  }
};

// The segment's tiles in ascending order, or descending, page ids 64 at a time
// in a lane each: in the loops a page is then a register away, where a load of
// its own would be waited for at every tile.
template <bool kBf, int NB, bool kDown>
struct Tiles {
  const Work<kBf, NB>& w;
  int first, ids;  // of the pages held

  __device__ CVS_INLINE explicit Tiles(const Work<kBf, NB>& w) : w(w) {
    hold((kDown ? max(w.it.tile0, w.it.tile0 + w.it.tiles - 1) : w.it.tile0) >> w.a.page_shift);
  }
  __device__ CVS_INLINE void hold(int page) {
    first = kDown ? max(page - 63, w.it.tile0 >> w.a.page_shift) : page;
    page = first;
    // Lanes past the segment's last page hold that one again.
    const int last = max(page, (w.it.tile0 + w.it.tiles - 1) >> w.a.page_shift);
    ids = w.a.pages[w.it.page_first + min(page + w.lane, last)];
  }
  __device__ CVS_INLINE const char* operator()(int i) {
    const int t = w.it.tile0 + i, page = t >> w.a.page_shift;
    if (kDown ? page < first : page >= first + 64) hold(page);
    return w.at(__builtin_amdgcn_readlane(ids, page - first), t);
  }
};

// The scores of a lane's row, whose keys are counted from key0.
template <typename Scoring>
__device__ CVS_INLINE Scoring scoring_of(const CachedArgs& a, const Row& r, int key0) {
  if constexpr (Scoring::kPlain) return {a.scores.c};
  else return {a.scores, Scoring::kDown ? slope_log2(a.scores.slopes[r.head]) : 0.f, r.limit - 1 - key0};
}

// Up to 32 rows: the waves share the tiles.
template <bool kBf, int NB, typename Scoring>
__device__ CVS_INLINE void few_rows(const Work<kBf, NB>& w, int wave, char* lds) {
  const CachedArgs& a = w.a;
  const Segment& it = w.it;
  const int lane = w.lane, half = w.half;
  typedef float lanes_t[64];
  lanes_t* const s_m = reinterpret_cast<lanes_t*>(lds);
  lanes_t* const s_l = s_m + kWaves;
  lanes_t* const s_o = s_l + kWaves;  // two states

  const Row r = w.row(lane & 31);
  const Scoring scoring = scoring_of<Scoring>(a, r, 0);
  u32x4 kf[2 * NB], vf[2 * NB], q[2 * NB];
  auto load_keys = [&](const char* p) CVS_INLINE {
#pragma unroll
    for (int s = 0; s < 2 * NB; ++s) kf[s] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p + lane * 16 + s * 1024));
  };
  auto load_values = [&](const char* p) CVS_INLINE {
#pragma unroll
    for (int s = 0; s < 2 * NB; ++s)
      vf[s] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p + 2048 * NB + lane * 16 + s * 1024));
  };
  RowState<NB> st;
  st.init();
  bool bad = false;
  if (wave < it.tiles) {
    Tiles<kBf, NB, Scoring::kDown> tile(w);
    auto nth = [&](int i) CVS_INLINE { return Scoring::kDown ? it.tiles - 1 - i : i; };
    const char* p = tile(nth(wave));
    load_keys(p);
    load_values(p);
    w.load_q(r, q);
    for (int i = wave; i < it.tiles; i += kWaves) {
      f32x16 s{};
#pragma unroll
      for (int k = 0; k < 2 * NB; ++k) s = mfma<kBf>(kf[k], q[k], s);
      p = tile(nth(i + kWaves < it.tiles ? i + kWaves : i));
      load_keys(p);
      const int key0 = it.key0 + kTile * (it.tile0 + nth(i));
      if constexpr (!Scoring::kPlain) scoring.finish(s, key0 + 4 * half);
      if (key0 + kTile > it.min_limit) {
#pragma unroll
        for (int k = 0; k < 16; ++k)
          if (key0 + 8 * (k / 4) + 4 * half + k % 4 >= r.limit) s[k] = -INFINITY;
#pragma unroll
        for (int k = 0; k < 2 * NB; ++k) vf[k] = w.hide(vf[k], k & 1, key0, it.max_limit);
        if (it.min_limit < it.max_limit) bad |= clean<kBf>(vf);
      }
      if (i == wave) st.m = largest(s, scoring.c) - kLift<kBf>;
      probabilities<kBf, !Scoring::kPlain>(s, st, scoring.c);
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
  const bool met = __syncthreads_or(bad);
  float m = s_m[0][lane];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) m = fmaxf(m, s_m[i][lane]);
  const float alpha = __builtin_amdgcn_exp2f(st.m - (m == -INFINITY ? 0.f : m));
  s_l[wave][lane] = st.l * alpha;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int k = 0; k < 16; ++k) st.o[b][k] *= alpha;
#pragma unroll
  for (int step = 2; step >= 1; step >>= 1) {
    if (wave >= step && wave < 2 * step) {
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int k = 0; k < 16; ++k) s_o[(wave - step) * 16 * NB + 16 * b + k][lane] = st.o[b][k];
    }
    __syncthreads();
    if (wave < step) {
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int k = 0; k < 16; ++k) st.o[b][k] += s_o[wave * 16 * NB + 16 * b + k][lane];
    }
    if (step > 1) __syncthreads();
  }
  if (wave == 0) {
    const float l = both_sum((s_l[0][lane] + s_l[2][lane]) + (s_l[1][lane] + s_l[3][lane]));
    w.store(st, m, l, r, lane & 31, met);
  }
}

// The tiles of a segment through LDS, for attend_tiles: 64-key tile t is tiles 2 t and 2 t + 1.
template <bool kBf, int NB, bool kDown>
struct PageSource {
  static constexpr int kHalf = 2048 * NB;  // a 32-key tile, keys or values
  const Work<kBf, NB>& w;
  Tiles<kBf, NB, kDown> tile;
  const char* asked[2];  // where the keys of the last two tiles asked for are: their values are asked for later
  char *lds_k, *lds_v;
  int to_k, to_v, at_wave, wave, end;

  __device__ CVS_INLINE PageSource(const Work<kBf, NB>& w, int wave, char* lds, int end)
      : w(w), tile(w), lds_k(lds), lds_v(lds + 4 * kHalf), wave(wave), end(end) {
    // A wave loads half of one of the two tiles.
    at_wave = (wave & 1) * (kHalf / 2);
    const int to = (wave >> 1) * kHalf + at_wave;
    to_k = lds_addr(lds_k) + to;
    to_v = lds_addr(lds_v) + to;
  }
  __device__ CVS_INLINE void load(const char* from, int to) {
    const rsrc4 rs = make_rsrc(from + at_wave, kHalf / 2);
#pragma unroll
    for (int i = 0; i < NB; ++i) dma16(rs, to + i * 1024, i * 1024 + w.lane * 16);
  }
  __device__ CVS_INLINE void load_keys(int n, int t) {
    // The last tile again where the segment has an odd number; its keys are past the end.
    const char* const from = tile(min(2 * t + (wave >> 1), w.it.tiles - 1));
    asked[0] = asked[1];
    asked[1] = from;
    load(from, to_k + (n & 1) * 2 * kHalf);
  }
  // Called for each tile when the next one's keys have been asked for, or, for the last, its own.
  __device__ CVS_INLINE void load_values(int n, int) {
    load((2 * n + 2 < w.it.tiles ? asked[0] : asked[1]) + 2048 * NB, to_v + (n & 1) * 2 * kHalf);
  }
  __device__ CVS_INLINE u32x4 keys(int n, int h, int i) {
    return *reinterpret_cast<const u32x4*>(lds_k + (2 * (n & 1) + h) * kHalf + i * 1024 + w.lane * 16);
  }
  __device__ CVS_INLINE u32x4 values(int n, int h, int b, int k) {
    return *reinterpret_cast<const u32x4*>(lds_v + (2 * (n & 1) + h) * kHalf + (2 * b + k) * 1024 + w.lane * 16);
  }
  __device__ CVS_INLINE u32x4 hide(u32x4 v, int t, int h, int k) { return w.hide(v, k, 64 * t + 32 * h, end); }
};

// Up to 128 rows: each wave has its own.
template <bool kBf, int NB, typename Scoring>
__device__ CVS_INLINE void many_rows(const Work<kBf, NB>& w, int wave, char* lds) {
  const Segment& it = w.it;
  const int i = 32 * wave + (w.lane & 31);
  const Row r = w.row(i);
  u32x4 q[2 * NB];
  w.load_q(r, q);
  RowState<NB> st;
  st.init();
  bool bad = false;
  // Positions from the segment's first key on.
  const int key0 = it.key0 + kTile * it.tile0, keys = kTile * it.tiles;
  PageSource<kBf, NB, Scoring::kDown> src(w, wave, lds, min(it.max_limit - key0, keys));
  const Scoring scoring = scoring_of<Scoring>(w.a, r, key0);
  const int tiles = (it.tiles + 1) / 2, open = max(0, min(it.min_limit - key0, keys)) / 64;
  std::conditional_t<Scoring::kDown, FromTheMiddle, Ascending> order;
  if constexpr (Scoring::kDown) order.top = order.before = tiles;  // open tiles lie before all rows
  attend_tiles<kBf, NB, 2 * NB>(st, q, src, tiles, open, it.min_limit < it.max_limit, min(r.limit - key0, keys), scoring,
                                order, bad);
  const float l = both_sum(st.l);
  if (32 * wave < it.rows) w.store(st, st.m, l, r, i, bad);
}

template <bool kBf, int NB, typename Scoring>
__global__ __launch_bounds__(256, 2) void cached_attn_kernel(const CachedArgs a) {
  __shared__ __align__(16) char lds[16384 * NB];  // of many_rows; few_rows takes 8192 NB + 2048
  static_assert(8192 * NB + 2048 <= 16384 * NB, "LDS of few_rows");
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = blockIdx.x % a.kv_heads, wg = blockIdx.x / a.kv_heads;
  const Segment it = words(a.segments, wg);
  const Work<kBf, NB> w{a, it, g, lane, lane >> 5};
  if (it.rows > kTile) many_rows<kBf, NB, Scoring>(w, wave, lds);
  else few_rows<kBf, NB, Scoring>(w, wave, lds);
}

template <bool kBf, typename Scoring>
void launch_cached(cvs_context* ctx, const CachedArgs& a, int nb, int64_t blocks) {
  const TimerSpan ts = timer_span(ctx, "kv_attention");
  auto go = [&](auto kernel) {
    hipExtLaunchKernelGGL(kernel, dim3(unsigned(blocks)), dim3(256), 0, ctx->stream, ts.start, ts.stop, 0, a);
  };
  switch (nb) {
    case 1: go(cached_attn_kernel<kBf, 1, Scoring>); break;
    case 2: go(cached_attn_kernel<kBf, 2, Scoring>); break;
    case 3: go(cached_attn_kernel<kBf, 3, Scoring>); break;
    default: go(cached_attn_kernel<kBf, 4, Scoring>); break;
  }
  after_launch("cached_attn_kernel");
}

// With capped or biased scores, attn_cached_scored.hip.
void launch_cached_scored(cvs_context* ctx, const CachedArgs& a, int nb, int64_t blocks, int type);

}  // namespace attn
}  // namespace cvs
