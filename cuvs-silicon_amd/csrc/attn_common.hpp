// Definitions shared by the attention kernels (attn_prompt.hip, attn_cached.hip)
// and the paged cache (kv_cache.hip).
//
// All attention kernels compute, for a tile of 32 query rows a wave and 32
// keys, S^T = K Q^T and O^T += V^T P^T with v_mfma_f32_32x32x16.  A query row
// is a column of both accumulators, so everything that belongs to a row (its
// maximum, its sum, its rescaling) is a per-lane value shared by lanes l and
// l + 32, and the probabilities that leave the first product are the B operand
// of the second without moving between lanes: accumulator register r of lane l
// is key 8 (r / 4) + 4 (l / 32) + r % 4 of column l % 32, and the eight
// consecutive registers 8 s .. 8 s + 7 are the lane's B operand of the s-th 16
// keys when the A operand (V^T) orders its keys the same way.
#pragma once

#include <cmath>
#include <cstdint>
#include <memory>
#include <type_traits>
#include <vector>

#include "bf_common.hpp"
#include "cvs_internal.hpp"
#include "device_util.hpp"
#include "kv_pages.hpp"

namespace cvs {
namespace attn {

using bf::f32x16;
using bf::lds_addr;
using bf::make_rsrc;
using bf::rsrc4;
using bf::u32x4;

constexpr int kMaxDim = 128;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// 16 bytes a lane from a buffer straight to LDS address to + 16 lane, as
// bf::lds_dma, but five wait states before it: a descriptor that the compiler
// has spilled comes back through vector instructions just before the load,
// which it does not look into, and a scalar register that a vector instruction
// has written is there for a load after five.  (With one, a kernel of capped and
// biased scores read through descriptors of before, and gave other results from
// run to run.)
__device__ CVS_INLINE void dma16(rsrc4 rs, int to, uint32_t off) {
  asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(off), "s"(rs), "{m0}"(to) : "memory");
}

// One 16-byte MFMA operand: 8 elements of fp16 or bf16.
template <bool kBf>
__device__ CVS_INLINE f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (kBf) {
    typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(bf::half8, a), __builtin_bit_cast(bf::half8, b),
                                                  c, 0, 0, 0);
  }
}

// Two floats rounded to nearest even, packed.
template <bool kBf>
__device__ CVS_INLINE uint32_t pack2(float a, float b) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  const f32x2_t f = {a, b};
  if constexpr (kBf) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, bf16x2));
  } else {
    typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, half2_t));
  }
}

template <bool kBf>
__device__ CVS_INLINE float to_float(uint16_t x) {
  if constexpr (kBf) return __uint_as_float(uint32_t(x) << 16);
  return float(__builtin_bit_cast(_Float16, x));
}

// Bits 15 and 31 set where the half-word is an infinity or NaN (all exponent
// bits set: adding one unit of the exponent to the magnitude carries into
// bit 15, and never past it); the other bits are anything.
template <bool kBf>
__device__ CVS_INLINE uint32_t carries(uint32_t x) {
  return (x & 0x7fff7fffu) + (kBf ? 0x00800080u : 0x04000400u);
}
template <bool kBf>
__device__ CVS_INLINE bool nonfinite(uint16_t x) {
  return (carries<kBf>(x) & 0x8000u) != 0;
}

// Zeroes the infinities and NaNs among a wave's operands; whether there were any.
template <bool kBf, int N>
__device__ CVS_INLINE bool clean(u32x4 (&v)[N]) {
  uint32_t any = 0;
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) any |= carries<kBf>(v[j][i]);
  if (__ballot((any & 0x80008000u) != 0) == 0) return false;
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) v[j][i] &= ~((((carries<kBf>(v[j][i]) & 0x80008000u)) >> 15) * 0xffffu);
  return true;
}

// Running softmax of a lane's query row over the keys seen so far: m a
// log2-scaled score, or a little less (kLift), to count from, l this lane's share (its half of the keys) of
// the sum of 2^(score - m), o the weighted values.  All in fp32.
template <int NB>
struct RowState {
  f32x16 o[NB];
  float m, l;
  __device__ CVS_INLINE void init() {
#pragma unroll
    for (int b = 0; b < NB; ++b) o[b] = f32x16{};
    m = -INFINITY;
    l = 0.f;
  }
};

// The largest of a row's two lanes.
__device__ CVS_INLINE float both_max(float x) { return fmaxf(x, xor_lanes_f(x, 32)); }
__device__ CVS_INLINE float both_sum(float x) { return x + xor_lanes_f(x, 32); }

// A row's largest score among 32 keys, over its two lanes.
__device__ CVS_INLINE float largest(const f32x16& s, float c) {
  float top = fmaxf(s[0], s[1]);
#pragma unroll
  for (int r = 2; r < 16; ++r) top = fmaxf(top, s[r]);
  return both_max(top) * c;
}

// What becomes of a product s = q.k on its way to a score, in log2 units.
// Plain: c s, c = scale log2(e).  Otherwise (scored_probabilities):
//
//   cap: log2(e) C tanh(scale s / C).  With u = scale s / C, y = s^2: up to |u| =
//   1/2 that is s P(y), P of degree 3 fitted to c tanh(u) / u (least squares
//   weighted to an even relative error: 6e-7), with the powers of scale / C in
//   its coefficients (of lower degree, up to a smaller |u|, where those would
//   leave the range of fp32: score_args); above, C (1 - 2 / (1 + e^2u)), off by
//   its last places, 2^-22 C, which is as much beside the score.  A tile with no
//   |u| above 1/2, all of them in models whose scores stay within half of the cap,
//   takes five instructions a score more than a plain one and no exponential;
//
//   bias: minus log2(e) slope |place - key|, by the row's place and slope: linear
//   in the key where all of a tile's keys lie on one side of all rows, one
//   instruction a score, two elsewhere.
struct ScoreArgs {
  float c;
  float cap;            // log2(e) C
  float twice;          // log2(e) 2 scale / C
  float largest_y;      // of P's range; -1: P is not used
  float a[3];           // P's coefficients behind c
  int apart;            // scores may pass 2^24: they are finished before their row's m is taken off (attend_tiles)
  const float* slopes;  // of the heads, natural units; null: none
};
struct PlainScores {
  static constexpr bool kPlain = true, kDown = false;
  float c;
};
template <bool kCap_, bool kBias_>
struct Scores {
  static constexpr bool kPlain = false, kCap = kCap_, kBias = kBias_;
  // Scores fall with the distance: the nearest keys first, or every tile would have a larger maximum than the one before.
  static constexpr bool kDown = kBias;
  static constexpr float c = 1.f;  // of finished scores
  const ScoreArgs& a;
  float slope;  // log2(e) times the row's
  int place;    // the row's, counted like the keys

  // P(s^2), or c.
  __device__ CVS_INLINE float factor(float y) const {
    if constexpr (!kCap) return a.c;
    else return __builtin_fmaf(y, __builtin_fmaf(y, __builtin_fmaf(y, a.a[2], a.a[1]), a.a[0]), a.c);
  }
  // What is added to a product's score r of a lane's 16: rise (r's place) + from.  In a tile that lies before all of a
  // wave's rows, or behind them, the bias is linear in the key, and one instruction a score.
  static __device__ CVS_INLINE float added(float from, float rise, int r) {
    if constexpr (kBias) return __builtin_fmaf(rise, float(8 * (r / 4) + r % 4), from);
    else return from;
  }
  // Score r plus `from`, up to the cap's small scores.
  __device__ CVS_INLINE float score(float s, float from, float rise, int r) const {
    return __builtin_fmaf(s, factor(s * s), added(from, rise, r));
  }
  // The same, of any score.  one: 1, which the compiler does not know: it would keep what this has in common with
  // `score`, 16 registers of it, for a pass that hardly ever comes.
  __device__ CVS_INLINE float any_score(float s, float from, float rise, int r, float one) const {
    const float t = s * one, y = s * t, add = added(from, rise * one, r);
    const float x = __builtin_fmaf(t, factor(y), add);
    if constexpr (kCap) return y <= a.largest_y ? x : large(t) + add;
    else return x;
  }
  // Products of keys key + 8 (r / 4) + r % 4 to scores, in place: for `probabilities` with a c of 1.
  __device__ CVS_INLINE void finish(f32x16& s, int key) const {
    const float far = kBias ? float(place - key) : 0.f;
    f32x16 x;
    float top = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      if constexpr (kCap) top = fmaxf(top, s[r] * s[r]);
      x[r] = s[r] * factor(s[r] * s[r]);
    }
    if constexpr (kCap) {
      if (__ballot(!(top <= a.largest_y))) {
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = s[r] * s[r] <= a.largest_y ? x[r] : large(s[r]);
      }
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      if constexpr (kBias) s[r] = __builtin_fmaf(-slope, __builtin_fabsf(far - float(8 * (r / 4) + r % 4)), x[r]);
      else s[r] = x[r];
    }
  }
  __device__ CVS_INLINE float large(float s) const {
    const float e = 1.f + __builtin_amdgcn_exp2f(s * a.twice);
    return __builtin_fmaf(-2.f * a.cap, __builtin_amdgcn_rcpf(e), a.cap);
  }
};
// A head's slope in log2 units, from -kSteepest to kSteepest natural ones: of those a key a token nearer has all the weight
// already, and their products with 2^31 tokens are numbers of 32 bits (with a slope of 3e38 a row's own key, 0 tokens away,
// was at 0 times infinity).
constexpr float kSteepest = 1e28f;
__device__ CVS_INLINE float slope_log2(float slope) {
  return (slope > kSteepest ? kSteepest : slope < -kSteepest ? -kSteepest : slope) * kLog2e;
}
// A call's scores, checked; cap 0 for none.
ScoreArgs score_args(const cvs_scores* scores, float scale, int dim);
// Calls go with the type of a call's capped or biased scores (a std::common_type of it).
template <typename Go>
void pick_scores(const ScoreArgs& a, const Go& go) {
  if (a.cap > 0.f && a.slopes) go(std::common_type<Scores<true, true>>{});
  else if (a.slopes) go(std::common_type<Scores<false, true>>{});
  else go(std::common_type<Scores<true, false>>{});
}

// The order in which a row's tiles are taken: ascending, or from tile `top` - 1
// down to 0 and then up from `top`; tiles below `before` lie before the places of
// all rows, those from `top` on behind them.
struct Ascending {
  static constexpr int top = 0, before = 0;
  __device__ CVS_INLINE int operator()(int step) const { return step; }
};
struct FromTheMiddle {
  int top, before;
  __device__ CVS_INLINE int operator()(int step) const { return step < top ? top - 1 - step : step; }
};

// Scores of 32 keys -> probabilities 2^(c s - m), summed up.  Masked scores
// come in as -inf and leave as 0.
//
// A row's m is a score's: of its first tile's largest (the caller sets it so),
// or of a later tile's, not always of the largest of all: as long as the
// probabilities of a tile sum to no more than kMost a lane, they fit the type
// that they are rounded to and are as precise as any (a larger one has the same
// number of bits), so m stays and nothing needs rescaling.  The sum is needed
// anyway, so nearly all tiles take no maximum at all, and the matrix products
// before are in one block with the exponentials.  Where the sum is larger, or
// the row has not seen a score yet (m is -inf, and 0 stands in for it, so that
// -inf - (-inf) does not arise), the row takes its m from the tile's largest
// score and the tile's probabilities are computed again.
//
// bf16 has the range of fp32, and m is the score itself.  fp16 ends at 2^-24, so
// m stands kLift below the score, whose probability is then 2^kLift: those of
// 2^-22 of it keep all bits, and smaller ones are off by 2^-33 of it at most
// (counted from 1, 100,000 keys of 2^-26 each beside one heavy key were all
// rounded to 0).  What kLift takes from the room above it costs rows that meet
// much larger scores late: 8,000 causal tokens, 16/4 heads of 64, take 161 us at
// a lift of 0, 8 or 10 where scores are spread by 1, and 162, 170 or 176 us where
// they are spread by 2.6 (natural units).  A tile that sums to more than kMost
// has a probability above kMost / 16 > 2^(kLift + 1), so its row does rise.
//
// Scores that pass kFar are rounded before m is taken off: in one multiply-add,
// what m, a rounded score, lacks of its own passes 1 there, and from 2^31 on would
// make the exponential infinite, or leave the row nothing.  (Finished scores are
// rounded already.)  Nor has m a lift there, which could be rounded to twice itself.
constexpr float kFar = 16777216.f;
template <bool kBf>
constexpr float kLift = kBf ? 0.f : 8.f;
template <bool kBf>
constexpr float kMost = kBf ? 4096.f : 65504.f;
template <bool kBf, bool kFinished, int NB>
__device__ CVS_INLINE void probabilities(f32x16& s, RowState<NB>& st, float c) {
  f32x16 p;
  auto exponentials = [&](float c) CVS_INLINE {
    const float base = st.m == -INFINITY ? 0.f : st.m;
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c, -base));
      sum[r & 1] += p[r];
    }
    return sum[0] + sum[1];
  };
  float sum = exponentials(c);
  const bool over = !(sum <= kMost<kBf>) || (kFinished ? st.m == -INFINITY : !(__builtin_fabsf(st.m) < kFar));
  if (__ballot(over)) {
    const float most = largest(s, c), top = __builtin_fabsf(most) < kFar ? most - kLift<kBf> : most;
    // Either of the row's two lanes (exchanged by all lanes, before any condition); the other rows stay as they are, so
    // that a row's result depends on itself alone.
    const uint32_t either = uint32_t(over) | xor_lanes(uint32_t(over), 32);
    const bool raise = either != 0 && top > st.m;
    const float alpha = raise ? __builtin_amdgcn_exp2f(st.m - top) : 1.f;
    st.l *= alpha;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) st.o[b][r] *= alpha;
    st.m = raise ? top : st.m;
    const bool far = !kFinished && !(__builtin_fabsf(st.m) < kFar);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = far ? s[r] * c : s[r];
    sum = exponentials(far ? 1.f : c);
  }
  st.l += sum;
  s = p;
}

// `probabilities` of products s of capped or biased scores of keys key + 8 (r /
// 4) + r % 4, which lie before the row's place (behind it: `behind`).  Where all are P's, and nothing has to rise, one pass does, in one
// block with the matrix products before it; else the scores are taken once more,
// larger ones by their exponential.  Which of the two is used changes no bit of
// a row whose own scores are small.
template <bool kBf, int NB, typename Scoring>
__device__ CVS_INLINE void scored_probabilities(f32x16& s, RowState<NB>& st, const Scoring& sc, int key, bool behind) {
  const float rise = Scoring::kBias ? (behind ? -sc.slope : sc.slope) : 0.f;
  auto from = [&](float base) CVS_INLINE {
    return Scoring::kBias ? __builtin_fmaf(rise, float(key - sc.place), -base) : -base;
  };
  f32x16 p;
  float sum;
  {
    const float f = from(st.m == -INFINITY ? 0.f : st.m);
    float part[2] = {0.f, 0.f}, top = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      if constexpr (Scoring::kCap) top = fmaxf(top, s[r] * s[r]);
      p[r] = __builtin_amdgcn_exp2f(sc.score(s[r], f, rise, r));
      part[r & 1] += p[r];
    }
    sum = part[0] + part[1];
    const bool over = !(sum <= kMost<kBf>) | !(__builtin_fabsf(st.m) < kFar), large = Scoring::kCap & !(top <= sc.a.largest_y);
    if (__ballot(over | large) == 0) {
      st.l += sum;
      s = p;
      return;
    }
  }
  float most;
  auto pass = [&]() CVS_INLINE {
    const float base = st.m == -INFINITY ? 0.f : st.m, f = from(base);
    float one = 1.f, part[2] = {0.f, 0.f};
    asm volatile("" : "+s"(one));
    most = -INFINITY;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float x = sc.any_score(s[r], f, rise, r, one);
      most = fmaxf(most, x);
      p[r] = __builtin_amdgcn_exp2f(x);
      part[r & 1] += p[r];
    }
    sum = part[0] + part[1];
    return base;
  };
  const float base = pass();
  const bool over = !(sum <= kMost<kBf>) || !(__builtin_fabsf(st.m) < kFar);
  if (__ballot(over)) {
    float m = both_max(most) + base - kLift<kBf>;
    // Rows whose scores pass kFar, or did so far: biased ones (of capped ones there are none here).
    const bool far = Scoring::kBias && !(fmaxf(__builtin_fabsf(m), __builtin_fabsf(base)) < kFar);
    const bool any_far = __ballot(far) != 0;
    if (any_far) {
      float one = 1.f, top = -INFINITY;
      asm volatile("" : "+s"(one));
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float x = sc.any_score(s[r], from(0.f), rise, r, one);
        top = fmaxf(top, x);
        s[r] = far ? x : s[r];
      }
      top = both_max(top);
      m = far ? top : m;
    }
    const uint32_t either = uint32_t(over) | xor_lanes(uint32_t(over), 32);
    const bool raise = either != 0 && m > st.m;
    const float alpha = raise ? __builtin_amdgcn_exp2f(st.m - m) : 1.f;
    st.l *= alpha;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) st.o[b][r] *= alpha;
    st.m = raise ? m : st.m;
    pass();  // from the scores again: less the m of before they have its last place
    if (any_far) {
      float part[2] = {0.f, 0.f};
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        p[r] = far ? __builtin_amdgcn_exp2f(s[r] - (st.m == -INFINITY ? 0.f : st.m)) : p[r];
        part[r & 1] += p[r];
      }
      sum = part[0] + part[1];
    }
  }
  st.l += sum;
  s = p;
}

// B operand of the 16 keys `step` (0 or 1) of a probability tile.  The
// probabilities are rounded to the values' type here, the product's operand
// type: each is off by at most half a unit of its own last place (in fp16, of
// 2^-24 for those below 2^-14), which the sum over keys averages; the sum l
// keeps them unrounded.
template <bool kBf>
__device__ CVS_INLINE u32x4 prob_operand(const f32x16& p, int step) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = pack2<kBf>(p[8 * step + 2 * i], p[8 * step + 2 * i + 1]);
  return r;
}

// Attention of a workgroup's 4 x 32 query rows, of KS 16-column steps and NB
// 32-column blocks, over `tiles` 64-key tiles that go through LDS,
// double-buffered.  A row sees the keys below `limit`, counted from the first
// tile; in the first `open_tiles` tiles all rows see all keys, and `mixed` says
// that the tiles behind them may hold values that `hide` leaves and that some
// row does not see.
// Tiles are taken in `order`, an open one behind a masked one only where scores
// fall with the distance.
// The source moves the data: load_keys(n, t) and load_values(n, t) ask for the
// n-th tile, which is tile t, of either (buffer n & 1; the workgroup's waves
// share the work; in this order, a tile's values after the next one's keys),
// keys(n, h, i) is the A operand of columns 16 i of half h's 32 keys, values(n,
// h, b, k) of columns 32 b of its k-th 16 keys; hide(v, t, h, k) clears what a
// masked tile's values must not show.
//
// Half tiles go through a pipeline of three: the products of one with the
// values and of the next with the keys run while the one between goes through
// its exponentials.  In the middle of tile t everyone is done with its keys
// and with the values before it; what was asked for one tile ago, the next
// keys and its values, has to be there.
template <bool kBf, int NB, int KS, typename Source, typename Scoring, typename Order>
__device__ CVS_INLINE void attend_tiles(RowState<NB>& st, const u32x4 (&q)[KS], Source& src, int tiles,
                                        int open_tiles, bool mixed, int limit, const Scoring& scoring,
                                        const Order& order, bool& bad) {
  const int half = __lane_id() >> 5;
  int unmasked_tiles = open_tiles;
  f32x16 s[2];    // scores of a tile's two halves
  u32x4 p[2][2];  // and their probabilities
  auto scores = [&](int n, int h) CVS_INLINE {
    f32x16 x{};
#pragma unroll
    for (int i = 0; i < KS; ++i) x = mfma<kBf>(src.keys(n, h, i), q[i], x);
    return x;
  };
  auto add_values = [&](int n, int h, auto masked) CVS_INLINE {
    if constexpr (!masked) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int b = 0; b < NB; ++b) st.o[b] = mfma<kBf>(src.values(n, h, b, k), p[h][k], st.o[b]);
    } else {
      const int t = order(n);
      u32x4 v[2 * NB];
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i) v[i] = src.hide(src.values(n, h, i / 2, i % 2), t, h, i % 2);
      if (mixed && (Scoring::kPlain || t >= open_tiles)) bad |= clean<kBf>(v);
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i) st.o[i / 2] = mfma<kBf>(v[i], p[h][i % 2], st.o[i / 2]);
    }
  };
  auto mask = [&](int n, int h) CVS_INLINE {
    if constexpr (!Scoring::kPlain) scoring.finish(s[h], 64 * order(n) + 32 * h + 4 * half);
    const int seen = limit - 64 * order(n) - 32 * h - 4 * half;
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if (8 * (r / 4) + r % 4 >= seen) s[h][r] = -INFINITY;
  };
  auto soften = [&](int n, int h, auto masked) CVS_INLINE {
    if constexpr (Scoring::kPlain || masked) probabilities<kBf, !Scoring::kPlain>(s[h], st, scoring.c);
    else scored_probabilities<kBf>(s[h], st, scoring, 64 * order(n) + 32 * h + 4 * half, n >= order.top);
#pragma unroll
    for (int k = 0; k < 2; ++k) p[h][k] = prob_operand<kBf>(s[h], k);
  };
  auto step = [&](int n, auto masked, auto first) CVS_INLINE {
    if constexpr (!Scoring::kPlain) {
      if constexpr (!first) add_values(n - 1, 1, masked);
    } else if (n > 0) {
      add_values(n - 1, 1, masked);
    }
    if constexpr (masked) mask(n, 0);
    s[1] = scores(n, 1);
    soften(n, 0, masked);
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    __syncthreads();
    if (n + 2 < tiles) src.load_keys(n + 2, order(n + 2));
    if (n + 1 < tiles) src.load_values(n + 1, order(n + 1));
    add_values(n, 0, masked);
    if constexpr (masked) mask(n, 1);
    s[0] = scores(n + 1, 0);  // past the last tile: of whatever is there, and not used
    soften(n, 1, masked);
  };
  if (tiles <= 0) return;
  src.load_keys(0, order(0));
  if (tiles > 1) src.load_keys(1, order(1));
  src.load_values(0, order(0));
  __builtin_amdgcn_s_waitcnt(0x0F70);
  __syncthreads();
  s[0] = scores(0, 0);
  if constexpr (Scoring::kPlain) {  // others find the first tile's maximum as any later one's
    mask(0, 0);
    st.m = largest(s[0], scoring.c) - kLift<kBf>;
  }
  // Steps of open tiles take m off in the multiply-add that makes a score.  What the rounded m lacks of its own score
  // passes 1 where scores pass 2^24, and from 2^31 on makes the exponential infinite, or leaves the row nothing: calls whose
  // cap allows such scores take masked steps, which round a score first.
  if constexpr (!Scoring::kPlain) {
    if (Scoring::kCap && scoring.a.apart) unmasked_tiles = 0;
  }
  int n = 0;
  auto steps = [&](int end, auto masked) CVS_INLINE {
    for (; n < end; ++n) step(n, masked, std::false_type{});
  };
  // The first step has no values to add.  The compiler takes it out of loops of plain scores, and not out of others, where
  // a branch would split the blocks that overlap products and exponentials; it is there a masked one, of any tile.
  if constexpr (!Scoring::kPlain) step(n++, std::true_type{}, std::true_type{});
  if constexpr (!Scoring::kDown) {
    steps(unmasked_tiles, std::false_type{});
    steps(tiles, std::true_type{});
  } else {
    // Masked tiles come first, with those that lie neither before all rows nor behind them, and last; a step behind a
    // masked one still adds its values.
    const int sure = min(unmasked_tiles, order.before);
    const int first = order.top > sure ? order.top - sure + 1 : 0, last = max(order.top, unmasked_tiles);
    for (int masked = min(first, tiles), open = min(last, tiles);; masked = open = tiles) {
      steps(masked, std::true_type{});
      steps(open, std::false_type{});
      if (n >= tiles) break;
    }
  }
  add_values(tiles - 1, 1, std::true_type{});
}

// A query row as the B operand of the scores' product, zeros past its end.
// Every lane loads, from within the row: a load under a lane's condition
// would be waited for before the next one.
template <int KS>
__device__ CVS_INLINE void load_row(const char* src, int dim, u32x4 (&q)[KS]) {
  const int half = __lane_id() >> 5;
#pragma unroll
  for (int s = 0; s < KS; ++s) q[s] = *reinterpret_cast<const u32x4*>(src + min(32 * s + 16 * half, 2 * dim - 16));
#pragma unroll
  for (int s = 0; s < KS; ++s)
    if (16 * s + 8 * half >= dim) q[s] = u32x4{};
}

// Writes a lane's half of a row's 32 NB outputs, scaled.  Lanes l and l + 32
// hold alternate groups of 4 elements; the pair exchanges them so that each
// stores 16 bytes at a time.
template <bool kBf, int NB>
__device__ CVS_INLINE void store_row(const RowState<NB>& st, float scale, uint16_t* out, int dim, bool there) {
  const int half = __lane_id() >> 5;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      uint32_t w[2][2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k)
          w[i][k] = pack2<kBf>(st.o[b][4 * (j + i) + 2 * k] * scale, st.o[b][4 * (j + i) + 2 * k + 1] * scale);
      // Upper lanes take their partner's group j + 1, lower lanes their partner's group j.
      const auto x = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
      const auto y = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
      const int d = 32 * b + 8 * (j + half);
      if (there && d < dim) *reinterpret_cast<u32x4*>(out + d) = u32x4{x[0], y[0], x[1], y[1]};
    }
}

// Puts right the outputs of a wave whose values had infinities or NaNs in keys
// that some of its rows do not see (`clean` took them out of the product: 0 *
// inf there would reach those rows), after its rows have been stored: an
// infinity or NaN of any positive weight is its element's result, so the
// weights are not needed.  value(j, d) is element d of key j; a lane's row sees
// keys below `last`, and those below `first` were not cleaned; add(d, x) adds x
// to the row's stored element d.  What the product has kept may be added again:
// the sum of infinities and NaNs is the same.  Such a wave reads the values of
// its masked tiles again, one element at a time, 8 keys under way at once; no
// other wave comes here.  2,048 causal tokens, 8/2 heads of 64: 47 us with finite
// values, 63 us with NaNs in all of them, 209 us with infinities (7 ms where every
// key that a row sees was read again, one at a time).
template <bool kBf, typename Value, typename Add>
__device__ CVS_INLINE void add_nonfinite(int first, int last, int dim, const Value& value, const Add& add) {
  // The rows' stores come first, also of other lanes, which have written half of this lane's row.
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll 1
  for (int d = __lane_id() >> 5; d < dim; d += 2) {
    float sum = 0.f;
#pragma unroll 1
    for (int j = first; j < last && sum == sum; j += 8) {
      uint16_t x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = value(min(j + k, last - 1), d);  // past the last, that one again
#pragma unroll
      for (int k = 0; k < 8; ++k) sum += nonfinite<kBf>(x[k]) ? to_float<kBf>(x[k]) : 0.f;
    }
    if (sum != 0.f) add(d, sum);
  }
}

// First of keys [0, keys), of which all rows see `open`, that may have been
// cleaned, or one before it: masked tiles begin at up to 63 keys before key
// `open`, and the half tile before them is multiplied as one of them.
__device__ CVS_INLINE int first_cleaned(int open, int keys) { return max(0, min(open, keys) - 96); }

// A heads view as the kernels take it: strides in elements.
struct View {
  char* p;
  int64_t token, head;
};

// Checks a view's geometry; `what` names it in messages.
void check_view(const cvs_heads* x, const char* what);
// Checks that no two rows of an output lie over each other; layers of them, layer_stride apart.
void check_rows_apart(const cvs_heads* x, const char* what, int64_t layers = 1, int64_t layer_stride = 0);
inline View view_of(const cvs_heads* x) {
  // The stride of a single token or head is not looked at.
  return {static_cast<char*>(x->data), x->tokens > 1 ? x->token_stride : 0, x->heads > 1 ? x->head_stride : 0};
}

// Workgroups of 256 threads that a launch's x dimension holds.
constexpr int64_t kMaxBlocks = (int64_t(1) << 24) - 1;

// The softmax scale in log2 units: 0 stands for 1 / sqrt(dim).
float scale_log2(float scale, int dim);

// Memory for a plan: of those that destroyed plans left in `pool`, the
// smallest that fits, or new.  Plans are made and destroyed at every step of a
// program; all that reads or writes their memory is on one stream, in order,
// so it passes from one plan to the next without a wait.
DeviceBuffer take_blob(std::vector<DeviceBuffer>& pool, int live_plans, size_t bytes);

// Whether the context's stream is being captured into a HIP graph.  What a
// captured call has been given is read again at every replay, which no one
// tells the library of: the memory of its plan and of its parts goes to a
// `kept` list and is neither used for anything else nor freed before the
// context's or cache's end.
bool capturing(const cvs_context* ctx);
// Refuses what would be done at every replay, and not now.
void need_no_capture(const cvs_context* ctx, const char* what);

// Copies host bytes to device memory as arguments of kernels, kUploadBytes a
// launch: the host buffer is free on return and nothing is pinned, staged or
// waited for.
constexpr size_t kUploadBytes = 3840;
void upload(cvs_context* ctx, void* dst, const void* src, size_t bytes);

// Tokens [begin, end) of a page, rows row0 and on of the caller's arrays; the
// page is its sequence's index-th.
struct Span {
  int32_t page, range, row0, index;
  static Span of(int32_t page, int64_t begin, int64_t end, int64_t row0, int64_t index) {
    return {page, int32_t(begin | end << 16), int32_t(row0), int32_t(index)};  // both are at most 4096
  }
  __host__ __device__ int begin() const { return range & 0xffff; }
  __host__ __device__ int end() const { return range >> 16; }
};

// Spans of a small plan go to the kernels as arguments, others are read from the plan's memory.
constexpr int kInlineSpans = 192;
struct Spans {
  Span s[kInlineSpans];
};

}  // namespace attn
}  // namespace cvs

// A cache of key and value rows in pages, kv_cache.hip.
struct cvs_kv_cache {
  cvs_context* ctx = nullptr;
  int layers = 0, kv_heads = 0, dim = 0, type = 0;
  int nb = 0;                  // 32-element blocks of a padded row
  int64_t head_bytes = 0;      // one head's keys and values of a page: 2 * page_tokens * 64 nb
  int64_t page_bytes = 0;      // kv_heads * head_bytes
  int64_t layer_bytes = 0;     // pages * page_bytes
  char* pool = nullptr;
  std::unique_ptr<cvs::kv::PageBook> book;
  int live_plans = 0;
  std::vector<cvs::DeviceBuffer> blobs;  // device memory of destroyed plans, for the next ones
  std::vector<cvs::DeviceBuffer> kept;   // of plans of captured calls, until the cache's end
};

struct cvs_kv_plan {
  cvs_kv_cache* cache = nullptr;
  std::vector<int64_t> seqs;
  std::vector<uint64_t> versions;
  std::vector<cvs::attn::Span> spans;  // where the tokens lie, a page each
  int64_t tokens = 0;            // of all sequences
  int heads = 0;                 // query heads; 0: for reading and writing alone
  cvs::DeviceBuffer blob;
  bool captured = false;  // the blob is the cache's to keep
  // Offsets into the blob, in bytes.
  size_t at_spans = 0;
  int workgroups = 0;  // of attention, a kv head (attn_cached.hip)
  int64_t slots = 0;   // rows of partial results a kv head; 0: every row has one part
  size_t at_segments = 0, at_pages = 0, at_limits = 0, at_rows = 0, at_runs = 0, at_parts = 0;
};

namespace cvs {
namespace attn {
// The attention part of a plan's blob, appended to `blob`.
void plan_attention(cvs_kv_plan* plan, const int64_t* lengths, const int64_t* tokens, std::vector<char>& blob);
// The plan is the cache's and its sequences are as they were when it was made.
void check_plan(const cvs_kv_plan* plan);
// Before a call with the plan is launched: whether it is being captured; the plan's memory is then kept.
bool captured_call(cvs_kv_plan* plan);
}  // namespace attn
}  // namespace cvs
