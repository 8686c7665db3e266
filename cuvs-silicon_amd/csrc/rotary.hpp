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

#include "kv_tiles.hpp"

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

// A head is a row of 16-byte pieces, one a lane; the power of two of lanes that
// holds the largest head of a kernel has a row.
template <int kLanes>
struct HeadLane {
  int in, piece, pieces;  // lanes past the row's end repeat its last piece
  int dim, half;          // half: pairs that turn
  float inv_dim;
  __device__ CVS_INLINE HeadLane(int dim, int dims)
      : in(threadIdx.x % kLanes), piece(min(in, dim / 8 - 1)), pieces(dim / 8), dim(dim), half(dims / 2),
        inv_dim(1.f / float(dim)) {}
};

// A norm's weights to LDS in fp32.
template <bool kBf>
__device__ CVS_INLINE void load_weight(float* s, const Norm& n, int dim) {
  if (!n.weight) return;
  for (int i = threadIdx.x; i < dim; i += blockDim.x)
    s[i] = n.fp32 ? static_cast<const float*>(n.weight)[i] : to_float<kBf>(static_cast<const uint16_t*>(n.weight)[i]);
}

// The lane's piece x of a head, normed and rotated.  cs, sn: the head's cosines
// and sines, times the magnitude; w: its norm's weights, null for none; scratch:
// a place in LDS for each lane of the wave, this one's (kChannels alone).
template <bool kBf, int kLanes, Pairs kPairs, bool kNorm>
__device__ CVS_INLINE u32x4 ready(u32x4 x, const HeadLane<kLanes>& l, const float* cs, const float* sn, const float* w,
                                  float eps, u32x4* scratch) {
  const int half = l.half, piece = l.piece;
  float f[8], o[8];
  unpack8<kBf>(x, f);
  float inv = 1.f;
  if constexpr (kNorm) {
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = __builtin_fmaf(f[e], f[e], sum);
    if (l.in >= l.pieces) sum = 0.f;
#pragma unroll
    for (int m = 1; m < kLanes; m <<= 1) sum += xor_lanes_f(sum, m);
    if (w) {
      inv = 1.f / __builtin_sqrtf(__builtin_fmaf(sum, l.inv_dim, eps));
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] *= w[8 * piece + e];
    }
  }
  if constexpr (kPairs == kNeighbours) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const int p = 4 * piece + e / 2;
      const bool turned = p < half;
      const float c = cs[turned ? p : 0], s = sn[turned ? p : 0];
      o[e] = turned ? f[e] * c - f[e + 1] * s : f[e];
      o[e + 1] = turned ? f[e + 1] * c + f[e] * s : f[e + 1];
    }
  } else if constexpr (kPairs == kPieces) {
    // A piece of the first half, of the second, or behind both.
    const bool turned = 8 * piece < 2 * half, low = 8 * piece < half;
    const int to = !turned ? 0 : low ? half / 8 : -half / 8;  // where its partner is
    u32x4 px;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      px[k] = uint32_t(__builtin_amdgcn_ds_bpermute(4 * (int(__lane_id()) + to), int(x[k])));
    float g[8];
    unpack8<kBf>(px, g);
    const int p = !turned ? 0 : low ? 8 * piece : 8 * piece - half;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (kNorm) {
        if (w) g[e] *= w[8 * (piece + to) + e];
      }
      const float s = low ? -sn[p + e] : sn[p + e];
      o[e] = turned ? f[e] * cs[p + e] + g[e] * s : f[e];
    }
  } else {
    // The row's pieces side by side.
    *scratch = x;
    wave_lds_ready();
    const uint16_t* const row = reinterpret_cast<const uint16_t*>(scratch - l.in);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = 8 * piece + e;
      const bool turned = c < 2 * half, low = c < half;
      const int other = !turned ? c : low ? c + half : c - half, p = !turned ? 0 : low ? c : c - half;
      float g = to_float<kBf>(row[other]);
      if constexpr (kNorm) {
        if (w) g *= w[other];
      }
      const float s = low ? -sn[p] : sn[p];
      o[e] = turned ? f[e] * cs[p] + g * s : f[e];
    }
    wave_lds_ready();  // read before the next row's pieces are written
  }
  if constexpr (kNorm) {
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] *= inv;
  }
  return pack8<kBf>(o);
}

// A head on its way.
struct HeadRow {
  const char* in;
  char* out;
  const float *cs, *sn, *w;
  float eps;
};

// Rows [0, rows) by a workgroup, kAhead of each group of lanes under way at
// once; place(r) is row r, before() is run behind the first loads.  A row's
// input may be its own output and no other row's.
constexpr int kAhead = 4;
template <bool kBf, int kLanes, Pairs kPairs, bool kNorm, typename Place, typename Before>
__device__ CVS_INLINE void ready_rows(const HeadLane<kLanes>& l, int rows, u32x4* scratch, const Place& place,
                                      const Before& before) {
  const int groups = blockDim.x / kLanes, group = threadIdx.x / kLanes;
  u32x4 x[kAhead];
  auto load = [&](int first) CVS_INLINE {
#pragma unroll
    for (int i = 0; i < kAhead; ++i)  // past the last row, that one again (not stored)
      x[i] = *reinterpret_cast<const u32x4*>(place(min(first + i * groups, rows - 1)).in + 16 * l.piece);
  };
  load(group);
  before();
  for (int first = group; first - group < rows; first += kAhead * groups) {
    u32x4 y[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const HeadRow r = place(min(first + i * groups, rows - 1));
      y[i] = ready<kBf, kLanes, kPairs, kNorm>(x[i], l, r.cs, r.sn, r.w, r.eps, scratch);
    }
    load(first + kAhead * groups);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int r = first + i * groups;
      if (r < rows && l.in < l.pieces) *reinterpret_cast<u32x4*>(place(r).out + 16 * l.piece) = y[i];
    }
  }
}

// Checks a norm of heads of `type`; null: none.
Norm norm_of(const cvs_head_norm* norm, int type, const char* what);
// Checks that a rotary belongs to the context and fits heads of `dim`.
void check_rotary(const cvs_rotary* rotary, const cvs_context* ctx, int dim);
// Before a call with the rotary is launched: keeps its memory for the replays of a capture.
void captured_rotary(const cvs_rotary* rotary);

}  // namespace attn
}  // namespace cvs
