// Tokens of a page's tile between the caller's rows and the pool's operand
// blocks (kv_cache.hip has the layout), a wave a tile of 32 tokens and kv
// head: shared by the kernels that move tokens as they are (kv_cache.hip) and
// that norm and rotate keys on the way (kv_append.hip).
#pragma once

#include "attn_common.hpp"

namespace cvs {
namespace attn {

// Rows 2 w and 2 w + 1 of an 8 x 8 matrix of 16-bit elements are x[2 w], x[2 w + 1]; transposed in place.
__device__ CVS_INLINE void transpose8(u32x4 (&x)[8]) {
  u32x4 y[8];
#pragma unroll
  for (int c = 0; c < 8; ++c)
#pragma unroll
    for (int k = 0; k < 4; ++k)
      y[c][k] = __builtin_amdgcn_perm(x[2 * k + 1][c / 2], x[2 * k][c / 2], c & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
  for (int c = 0; c < 8; ++c) x[c] = y[c];
}

// A lane's part of a tile's values: columns 8 c and on of tokens t0 + {0, 1, 2,
// 3, 8, 9, 10, 11}, whose elements stand together in the pool.  The tile's
// tokens [lo, hi) are the call's.
template <int NB>
struct TileValues {
  static constexpr int P = 4 * NB;  // 16-byte pieces of a row
  int lo, hi, c, t0;
  bool mine;
  u32x4* slots;
  u32x4 x[8];

  __device__ CVS_INLINE TileValues(char* vt, int lo, int hi) : lo(lo), hi(hi) {
    const int lane = __lane_id();
    c = lane % P;
    t0 = 16 * (lane / P >> 1) + 4 * (lane / P & 1);
    mine = lane < 4 * P && t0 < hi && t0 + 11 >= lo;
    slots = reinterpret_cast<u32x4*>(vt + (2 * (c / 4) + (lane / P >> 1)) * 1024 + (32 * (lane / P & 1) + 8 * (c % 4)) * 16);
  }
  __device__ CVS_INLINE int token(int j) const { return t0 + 8 * (j / 4) + j % 4; }
  __device__ CVS_INLINE int held(int t) const { return min(max(t, lo), hi - 1); }
  // From the caller's rows (vs: of the tile's token 0), all under way at once, of clamped tokens.
  __device__ CVS_INLINE void load(const char* vs, int64_t stride, int pieces) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      x[j] = *reinterpret_cast<const u32x4*>(vs + 2 * (held(token(j)) * stride + 8 * min(c, pieces - 1)));
  }
  // To the pool.  Tokens before the call's keep what they hold: where they share 16 bytes with new ones, those are written
  // one by one, as there are few of them and reading the old ones first would be one more wait.
  __device__ CVS_INLINE void store(int pieces) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c >= pieces) x[j] = u32x4{};
    transpose8(x);
    if (!mine) return;
    if (t0 >= lo) {
#pragma unroll
      for (int j = 0; j < 8; ++j) slots[j] = x[j];
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (token(k) < lo || token(k) >= hi) continue;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          reinterpret_cast<uint16_t*>(slots + j)[k] = uint16_t(x[j][k / 2] >> (16 * (k % 2)));
      }
    }
  }
};

// Where piece p of a tile's token t stands in the wave's LDS while keys change places.
template <int NB>
__device__ CVS_INLINE int staged(int t, int p) {
  return t * (4 * NB) + (p ^ (t & 3));
}

// What a wave has written to its LDS is there for all of its lanes.
__device__ CVS_INLINE void wave_lds_ready() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A tile's staged keys, tokens [lo, hi), to the pool.
template <int NB>
__device__ CVS_INLINE void store_keys(const u32x4* s, char* kt, int lo, int hi) {
  const int lane = __lane_id(), t = lane & 31;
  u32x4 y[2 * NB];
#pragma unroll
  for (int i = 0; i < 2 * NB; ++i) y[i] = s[staged<NB>(t, 2 * i + (lane >> 5))];
  if (t >= lo && t < hi) {
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) *reinterpret_cast<u32x4*>(kt + 1024 * i + 16 * lane) = y[i];
  }
}

// What a plan's tokens ask of move_tokens and append: checks the plan, the
// layers, k and v, and, for writing, that no other sequence has their pages.
void check_move(cvs_kv_plan* plan, int first_layer, int layers, const cvs_heads* k, const cvs_heads* v, bool write);
// Spans fill few of a page's tiles: tiles are then counted span by span within each tile of the page, and not tile by
// tile within each span.
inline bool spans_by_tile(const cvs_kv_plan* plan) {
  return 2 * plan->tokens < int64_t(plan->spans.size()) * plan->cache->book->page_tokens();
}

}  // namespace attn
}  // namespace cvs
