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
// cycles, the vector unit 52%: 12,000 causal tokens, 32/8 heads, bf16, in 1.03
// to 1.05 ms from card to card = 1.13 PFLOP/s, 0.80 of the vendor's plain
// product).  Prompts with smaller heads no one unit: 64 passages of 40 to 512
// tokens, 12 heads of 64, take 45 us with the vector unit busy 51% of the cycles
// (193 instructions a 64-key step, 32 exponentials among them), the matrix cores
// 27%, the waves 27% of their time waiting, and 146 MB fetched for 88 MB of
// inputs: row blocks that share keys run on different XCDs, each with an L2 of
// its own.  Short prompts each workgroup's first loads.
#pragma once

#include "attn_common.hpp"

namespace cvs {
namespace attn {
constexpr int kRows = 128;  // query rows of a workgroup
constexpr int kKeys = 64;   // keys of a step

struct PromptItem {
  int32_t q0, q_len;  // the sequence's tokens in q
  int32_t k0, k_len;  // and in k, v
  int32_t row0;       // first of the item's rows (token * group + head of the group)
  int32_t prefix;     // keys that all of a causal sequence's queries see
};

struct PromptArgs {
  View q, k, v, out;
  float* lse;
  const PromptItem* items;
  int64_t q_tokens;  // lse rows are heads of q_tokens
  int kv_heads, group, dim, causal;
  ScoreArgs scores;
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
  __device__ CVS_INLINE void load(const char* base, int64_t step, int to, const uint32_t (&off)[kLoads], int n, int t) {
    const rsrc4 rs = make_rsrc(base + t * step, 0x7fffffff);
    const int left = k_len - t * kKeys;
    to += (n & 1) * kBuf;
    if (left >= kKeys) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) dma16(rs, to + i * 1024, off[i]);
    } else {
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
        dma16(rs, to + i * 1024, (first + i * 64) / P < left ? off[i] : kNowhere);
    }
  }
  __device__ CVS_INLINE void load_keys(int n, int t) { load(base_k, step_k, to_k, off_k, n, t); }
  __device__ CVS_INLINE void load_values(int n, int t) { load(base_v, step_v, to_v, off_v, n, t); }
  __device__ CVS_INLINE u32x4 keys(int n, int h, int i) {
    const int at = P == 12 ? (i & 1 ? k_odd : k_even) + 64 * (i / 2) : k_even ^ 32 * i;
    return *reinterpret_cast<const u32x4*>(lds_k + (n & 1) * kBuf + h * 32 * kPitch + at);
  }
  __device__ CVS_INLINE u32x4 values(int n, int h, int b, int k) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
    typedef __attribute__((address_space(3))) s16x4* lds_ptr;
    char* const from = lds_v + (n & 1) * kBuf + (32 * h + 16 * k) * kPitch + (P == 12 ? v_first + 64 * b : v_first ^ 64 * b);
    const auto x = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)from));
    const auto y = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(from + 8 * kPitch)));
    return u32x4{x[0], x[1], y[0], y[1]};
  }
  __device__ CVS_INLINE u32x4 hide(u32x4 v, int, int, int) { return v; }  // past the sequence's end are zeros
};

// Capped and biased scores leave a SIMD a wave less where heads are small: with the registers of plain ones they spill in
// the loop (64 passages of heads of 64, biased: 114 us, 51 so).  A few are spilled all the same: 2 for heads of 64 with
// both, 5 (biased) and 7 (both) for heads of 128; two to four of them come back in a step.
template <bool kBf, int NB, int KS, typename Scoring>
__global__ __launch_bounds__(256, NB == 4 ? 2 : NB == 3 ? (Scoring::kPlain ? 3 : 2) : (Scoring::kPlain ? 4 : 3)) void prompt_attn_kernel(const PromptArgs a) {
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
    return a.causal ? max(it.prefix, min(it.k_len, it.k_len + (t + 1 - it.q_len))) : it.k_len;
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
  const int tiles = (wg_max + kKeys - 1) / kKeys, open = wg_min / kKeys;
  const bool mixed = wg_min < it.k_len;
  float shift = 0.f;  // of the scores, by what all of the row's keys lie behind its place
  if constexpr (Scoring::kPlain) {
    attend_tiles<kBf, NB, KS>(st, q, src, tiles, open, mixed, limit, Scoring{a.scores.c}, Ascending{}, bad);
  } else {
    // Rows before the first key count from it, so that distances are as exact for them as for others.
    const int place = it.k_len - it.q_len + tok;
    const float slope = Scoring::kDown ? slope_log2(a.scores.slopes[head]) : 0.f;
    if (Scoring::kDown && place < 0) shift = slope * float(place);
    const Scoring scoring{a.scores, slope, max(place, 0)};
    if constexpr (Scoring::kDown) {
      const int place0 = it.k_len - it.q_len + it.row0 / a.group;  // of the first row
      const int last = it.k_len - it.q_len + (min(it.row0 + kRows, rows) - 1) / a.group;
      attend_tiles<kBf, NB, KS>(st, q, src, tiles, open, mixed, limit, scoring,
                                FromTheMiddle{min(max(last, 0) / kKeys + 1, tiles), (max(place0, 0) + 1) / kKeys}, bad);
    } else {
      attend_tiles<kBf, NB, KS>(st, q, src, tiles, open, mixed, limit, scoring, Ascending{}, bad);
    }
  }
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
    a.lse[int64_t(head) * a.q_tokens + it.q0 + tok] = limit > 0 ? (st.m + shift + __builtin_amdgcn_logf(l)) * kLn2 : -INFINITY;
}

template <bool kBf, typename Scoring>
void launch_prompt(cvs_context* ctx, const PromptArgs& a, int64_t blocks) {
  const TimerSpan ts = timer_span(ctx, "prompt_attention");
  auto go = [&](auto kernel) {
    hipExtLaunchKernelGGL(kernel, dim3(unsigned(blocks)), dim3(256), 0, ctx->stream, ts.start, ts.stop, 0, a);
  };
  // Blocks of 32 columns for the values, steps of 16 for the scores: heads of 72 and 80, 104 and 112 go without a step
  // that would multiply zeros.
  if (a.dim <= 64) go(prompt_attn_kernel<kBf, 2, 4, Scoring>);
  else if (a.dim <= 80) go(prompt_attn_kernel<kBf, 3, 5, Scoring>);
  else if (a.dim <= 96) go(prompt_attn_kernel<kBf, 3, 6, Scoring>);
  else if (a.dim <= 112) go(prompt_attn_kernel<kBf, 4, 7, Scoring>);
  else go(prompt_attn_kernel<kBf, 4, 8, Scoring>);
  after_launch("prompt_attn_kernel");
}

// With capped or biased scores, attn_prompt_scored.hip.
void launch_prompt_scored(cvs_context* ctx, const PromptArgs& a, int64_t blocks, int type);

}  // namespace attn
}  // namespace cvs
