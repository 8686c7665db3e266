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
using bf::lds_dma;
using bf::make_rsrc;
using bf::rsrc4;
using bf::u32x4;

constexpr int kMaxDim = 128;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

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
template <bool kBf>
constexpr float kLift = kBf ? 0.f : 8.f;
template <bool kBf>
constexpr float kMost = kBf ? 4096.f : 65504.f;
template <bool kBf, int NB>
__device__ CVS_INLINE void probabilities(f32x16& s, RowState<NB>& st, float c) {
  f32x16 p;
  auto exponentials = [&]() CVS_INLINE {
    const float base = st.m == -INFINITY ? 0.f : st.m;
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c, -base));
      sum[r & 1] += p[r];
    }
    return sum[0] + sum[1];
  };
  float sum = exponentials();
  const bool over = !(sum <= kMost<kBf>) || st.m == -INFINITY;
  if (__ballot(over)) {
    const float top = largest(s, c) - kLift<kBf>;
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
    sum = exponentials();
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
// The source moves the data: load_keys(t) and load_values(t) ask for a tile of
// either (buffer t & 1; the workgroup's waves share the work; in ascending
// order, a tile's values after the next one's keys), keys(t, h, i)
// is the A operand of columns 16 i of half h's 32 keys, values(t, h, b, k) of
// columns 32 b of its k-th 16 keys; hide(v, t, h, k) clears what a masked
// tile's values must not show.
//
// Half tiles go through a pipeline of three: the products of one with the
// values and of the next with the keys run while the one between goes through
// its exponentials.  In the middle of tile t everyone is done with its keys
// and with the values before it; what was asked for one tile ago, the next
// keys and its values, has to be there.
template <bool kBf, int NB, int KS, typename Source>
__device__ CVS_INLINE void attend_tiles(RowState<NB>& st, const u32x4 (&q)[KS], Source& src, int tiles,
                                        int open_tiles, bool mixed, int limit, float c, bool& bad) {
  const int half = __lane_id() >> 5;
  f32x16 s[2];    // scores of a tile's two halves
  u32x4 p[2][2];  // and their probabilities
  auto scores = [&](int t, int h) CVS_INLINE {
    f32x16 x{};
#pragma unroll
    for (int i = 0; i < KS; ++i) x = mfma<kBf>(src.keys(t, h, i), q[i], x);
    return x;
  };
  auto add_values = [&](int t, int h, auto masked) CVS_INLINE {
    if constexpr (!masked) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int b = 0; b < NB; ++b) st.o[b] = mfma<kBf>(src.values(t, h, b, k), p[h][k], st.o[b]);
    } else {
      u32x4 v[2 * NB];
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i) v[i] = src.hide(src.values(t, h, i / 2, i % 2), t, h, i % 2);
      if (mixed) bad |= clean<kBf>(v);
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i) st.o[i / 2] = mfma<kBf>(v[i], p[h][i % 2], st.o[i / 2]);
    }
  };
  auto mask = [&](int t, int h) CVS_INLINE {
    const int seen = limit - 64 * t - 32 * h - 4 * half;
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if (8 * (r / 4) + r % 4 >= seen) s[h][r] = -INFINITY;
  };
  auto soften = [&](int h) CVS_INLINE {
    probabilities<kBf>(s[h], st, c);
#pragma unroll
    for (int k = 0; k < 2; ++k) p[h][k] = prob_operand<kBf>(s[h], k);
  };
  auto step = [&](int t, auto masked) CVS_INLINE {
    if (t > 0) add_values(t - 1, 1, masked);
    if constexpr (masked) mask(t, 0);
    s[1] = scores(t, 1);
    soften(0);
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    __syncthreads();
    if (t + 2 < tiles) src.load_keys(t + 2);
    if (t + 1 < tiles) src.load_values(t + 1);
    add_values(t, 0, masked);
    if constexpr (masked) mask(t, 1);
    s[0] = scores(t + 1, 0);  // past the last tile: of whatever is there, and not used
    soften(1);
  };
  if (tiles <= 0) return;
  src.load_keys(0);
  if (tiles > 1) src.load_keys(1);
  src.load_values(0);
  __builtin_amdgcn_s_waitcnt(0x0F70);
  __syncthreads();
  s[0] = scores(0, 0);
  mask(0, 0);
  st.m = largest(s[0], c) - kLift<kBf>;
  int t = 0;
  for (; t < open_tiles; ++t) step(t, std::false_type{});
  for (; t < tiles; ++t) step(t, std::true_type{});
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

// Tokens [begin, end) of a page, rows row0 and on of the caller's arrays.
struct Span {
  int32_t page, begin, end, row0;
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
