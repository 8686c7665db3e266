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
#include <algorithm>
#include <cstring>

#include "attn_common.hpp"

namespace cvs {
namespace attn {
namespace {

constexpr int kTile = 32;       // keys of a tile, rows of a wave
constexpr int kWaves = 4;
constexpr int kBlock = kTile * kWaves;  // rows of a large block
constexpr int kJoin = 4;        // parts of a row that a lane reads at a time

struct Segment {
  int32_t page_first;     // first of the run's pages in the plan's page list
  int32_t tile0, tiles;   // the segment's tiles, counted from the run's first token
  int32_t key0;           // position in the sequence of the run's first token
  int32_t row0, rows;     // (token * group + head) rows, tokens in the plan's order
  int32_t slot0;          // of row0's partial result
  int32_t min_limit, max_limit;  // keys the rows see: positions below their limit
};

// The parts that a run gives the rows of its sequences: part p of row r has
// slot slot0 + p * rows + r.  parent: the run that its pages follow, or -1.
struct Parts {
  int32_t slot0, rows, count, parent;
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
  float c;
  float* part_o;  // kv head, slot, 32 NB values
  float2* part_ml;
  int64_t slots;  // 0: write the output
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

// The segment's tiles in ascending order, page ids 64 at a time in a lane
// each: in the loops a page is then a register away, where a load of its own
// would be waited for at every tile.
template <bool kBf, int NB>
struct Tiles {
  const Work<kBf, NB>& w;
  int first, ids;  // of the pages held

  __device__ CVS_INLINE explicit Tiles(const Work<kBf, NB>& w) : w(w) { hold(w.it.tile0 >> w.a.page_shift); }
  __device__ CVS_INLINE void hold(int page) {
    first = page;
    // Lanes past the segment's last page hold that one again.
    const int last = max(page, (w.it.tile0 + w.it.tiles - 1) >> w.a.page_shift);
    ids = w.a.pages[w.it.page_first + min(page + w.lane, last)];
  }
  __device__ CVS_INLINE const char* operator()(int i) {
    const int t = w.it.tile0 + i, page = t >> w.a.page_shift;
    if (page >= first + 64) hold(page);
    return w.at(__builtin_amdgcn_readlane(ids, page - first), t);
  }
};

// Up to 32 rows: the waves share the tiles.
template <bool kBf, int NB>
__device__ CVS_INLINE void few_rows(const Work<kBf, NB>& w, int wave, char* lds) {
  const CachedArgs& a = w.a;
  const Segment& it = w.it;
  const int lane = w.lane, half = w.half;
  typedef float lanes_t[64];
  lanes_t* const s_m = reinterpret_cast<lanes_t*>(lds);
  lanes_t* const s_l = s_m + kWaves;
  lanes_t* const s_o = s_l + kWaves;  // two states

  const Row r = w.row(lane & 31);
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
    Tiles<kBf, NB> tile(w);
    const char* p = tile(wave);
    load_keys(p);
    load_values(p);
    w.load_q(r, q);
    for (int i = wave; i < it.tiles; i += kWaves) {
      f32x16 s{};
#pragma unroll
      for (int k = 0; k < 2 * NB; ++k) s = mfma<kBf>(kf[k], q[k], s);
      p = tile(i + kWaves < it.tiles ? i + kWaves : i);
      load_keys(p);
      const int key0 = it.key0 + kTile * (it.tile0 + i);
      if (key0 + kTile > it.min_limit) {
#pragma unroll
        for (int k = 0; k < 16; ++k)
          if (key0 + 8 * (k / 4) + 4 * half + k % 4 >= r.limit) s[k] = -INFINITY;
#pragma unroll
        for (int k = 0; k < 2 * NB; ++k) vf[k] = w.hide(vf[k], k & 1, key0, it.max_limit);
        if (it.min_limit < it.max_limit) bad |= clean<kBf>(vf);
      }
      if (i == wave) st.m = largest(s, a.c) - kLift<kBf>;
      probabilities<kBf>(s, st, a.c);
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
template <bool kBf, int NB>
struct PageSource {
  static constexpr int kHalf = 2048 * NB;  // a 32-key tile, keys or values
  const Work<kBf, NB>& w;
  Tiles<kBf, NB> tile;
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
    for (int i = 0; i < NB; ++i) lds_dma<16, false>(rs, to + i * 1024, i * 1024 + w.lane * 16, 0);
  }
  __device__ CVS_INLINE void load_keys(int t) {
    // The last tile again where the segment has an odd number; its keys are past the end.
    const char* const from = tile(min(2 * t + (wave >> 1), w.it.tiles - 1));
    asked[0] = asked[1];
    asked[1] = from;
    load(from, to_k + (t & 1) * 2 * kHalf);
  }
  // Called for each tile when the next one's keys have been asked for, or, for the last, its own.
  __device__ CVS_INLINE void load_values(int t) {
    load((2 * t + 2 < w.it.tiles ? asked[0] : asked[1]) + 2048 * NB, to_v + (t & 1) * 2 * kHalf);
  }
  __device__ CVS_INLINE u32x4 keys(int t, int h, int i) {
    return *reinterpret_cast<const u32x4*>(lds_k + (2 * (t & 1) + h) * kHalf + i * 1024 + w.lane * 16);
  }
  __device__ CVS_INLINE u32x4 values(int t, int h, int b, int k) {
    return *reinterpret_cast<const u32x4*>(lds_v + (2 * (t & 1) + h) * kHalf + (2 * b + k) * 1024 + w.lane * 16);
  }
  __device__ CVS_INLINE u32x4 hide(u32x4 v, int t, int h, int k) { return w.hide(v, k, 64 * t + 32 * h, end); }
};

// Up to 128 rows: each wave has its own.
template <bool kBf, int NB>
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
  PageSource<kBf, NB> src(w, wave, lds, min(it.max_limit - key0, keys));
  attend_tiles<kBf, NB, 2 * NB>(st, q, src, (it.tiles + 1) / 2, max(0, min(it.min_limit - key0, keys)) / 64, it.min_limit < it.max_limit,
                        min(r.limit - key0, keys), w.a.c, bad);
  const float l = both_sum(st.l);
  if (32 * wave < it.rows) w.store(st, st.m, l, r, i, bad);
}

template <bool kBf, int NB>
__global__ __launch_bounds__(256, 2) void cached_attn_kernel(const CachedArgs a) {
  __shared__ __align__(16) char lds[16384 * NB];  // of many_rows; few_rows takes 8192 NB + 2048
  static_assert(8192 * NB + 2048 <= 16384 * NB, "LDS of few_rows");
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = blockIdx.x % a.kv_heads, wg = blockIdx.x / a.kv_heads;
  const Segment it = words(a.segments, wg);
  const Work<kBf, NB> w{a, it, g, lane, lane >> 5};
  if (it.rows > kTile) many_rows<kBf, NB>(w, wave, lds);
  else few_rows<kBf, NB>(w, wave, lds);
}

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
    const float c = scale_log2(scale, cache->dim);
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
                       plan->tokens, cache->kv_heads, group, cache->dim, c, part_o, part_ml, plan->slots};
    const int64_t blocks = int64_t(plan->workgroups) * cache->kv_heads;
    const bool is_bf = cache->type == CVS_BF16;
    if (is_bf) launch<true>(ctx, a, cache->nb, blocks);
    else launch<false>(ctx, a, cache->nb, blocks);
    if (!slots) return;
    const JoinArgs j{reinterpret_cast<const Parts*>(blob + plan->at_parts),
                     reinterpret_cast<const int32_t*>(blob + plan->at_runs),
                     reinterpret_cast<const int32_t*>(blob + plan->at_rows), part_o, part_ml, plan->slots,
                     plan->tokens * plan->heads, view_of(out), lse, plan->tokens, plan->heads, group, cache->dim};
    if (is_bf) launch_join<true>(ctx, j, cache->nb);
    else launch_join<false>(ctx, j, cache->nb);
  });
}
