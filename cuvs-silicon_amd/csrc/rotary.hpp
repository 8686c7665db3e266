// Rotary positions and norms of heads, shared by rotary.hip (from array to
// array) and kv_append.hip (into the cache).
//
//   n = w x / sqrt(mean x^2 + eps)                     the norm of a head, if there is one
//   y_a = m (n_a cos t - n_b sin t)                    for each pair (a, b) of its first `dims`
//   y_b = m (n_b cos t + n_a sin t),  t = p f_i        channels, at position p; y = n elsewhere
//
// all in fp32, rounded once.  A frequency is held as the turns that a position
// adds, in units of 2^-64 modulo whole turns, and the angle is the integer
// product of both modulo 2^64: what is left of a turn is off by at most
// |p| 2^-63 turns however many whole ones there are, where p f in fp32 would be
// off by 0.004 radians at position 100,000.
#pragma once

#include "attn_common.hpp"

// Rotary positions of a model, rotary.hip.
struct cvs_rotary {
  cvs_context* ctx = nullptr;
  int dims = 0, layout = 0;
  float magnitude = 1.f;
  cvs::DeviceBuffer turns;        // dims / 2 frequencies
  mutable bool captured = false;  // the frequencies are the context's to keep
};

namespace cvs {
namespace attn {

// cos and sin of `phase` / 2^64 turns: the nearest quarter turn is taken off,
// and the rest, at most pi / 4, goes through polynomials fitted to sin(t) / t
// and cos(t) over that range (weighted least squares, errors of 1.8e-9 and
// 1e-10 before rounding; a float holds the rest to 2^-25 of it).
__device__ CVS_INLINE float2 cos_sin(uint64_t phase) {
  const uint64_t quarter = (phase + (uint64_t(1) << 61)) >> 62;
  const int32_t rest = int32_t(uint32_t((phase - (quarter << 62)) >> 32));
  const float t = float(rest) * 1.4629180792671596e-9f;  // 2 pi / 2^32
  const float y = t * t;
  const float s = __builtin_fmaf(
      t * y, __builtin_fmaf(y, __builtin_fmaf(y, -1.949563609e-4f, 8.331978662e-3f), -1.666665067e-1f), t);
  const float c = __builtin_fmaf(
      y * y, __builtin_fmaf(y, __builtin_fmaf(y, 2.443845141e-5f, -1.388736751e-3f), 4.166664687e-2f),
      __builtin_fmaf(y, -0.5f, 1.f));
  const uint32_t q = uint32_t(quarter);
  const float cs = q & 1 ? s : c, sn = q & 1 ? c : s;
  return float2{(q + 1) & 2 ? -cs : cs, q & 2 ? -sn : sn};
}

// The eight elements of a 16-byte piece.
template <bool kBf>
__device__ CVS_INLINE void unpack8(u32x4 x, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = to_float<kBf>(uint16_t(x[i]));
    f[2 * i + 1] = to_float<kBf>(uint16_t(x[i] >> 16));
  }
}
template <bool kBf>
__device__ CVS_INLINE u32x4 pack8(const float (&f)[8]) {
  return u32x4{pack2<kBf>(f[0], f[1]), pack2<kBf>(f[2], f[3]), pack2<kBf>(f[4], f[5]), pack2<kBf>(f[6], f[7])};
}

// How pairs lie in a head: neighbours within a piece; halves whose channels
// lie whole pieces apart; or halves any number of channels apart.
enum Pairs { kNeighbours, kPieces, kChannels };
inline Pairs pairs_of(const cvs_rotary* r) {
  if (!r || r->layout == CVS_ROTARY_NEIGHBOURS) return kNeighbours;
  return r->dims % 16 == 0 ? kPieces : kChannels;
}

// A norm as kernels take it: null weight for none.
struct Norm {
  const void* weight;
  int fp32;  // the weight's type: fp32, or the heads'
  float eps;
};

// Checks a norm of heads of `type`; null: none.
Norm norm_of(const cvs_head_norm* norm, int type, const char* what);
// Checks that a rotary belongs to the context and fits heads of `dim`.
void check_rotary(const cvs_rotary* rotary, const cvs_context* ctx, int dim);
// Before a call with the rotary is launched: keeps its memory for the replays of a capture.
void captured_rotary(const cvs_rotary* rotary);

}  // namespace attn
}  // namespace cvs
