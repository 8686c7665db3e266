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
// |p| 2^-64 turns however many whole ones there are, where p f in fp32 would be
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
// 1e-10 before rounding; a float holds the rest to 2^-25 of it).  The rest's
// lower 32 bits are left out, 2^-32 turns or 1.5e-9 radians at most.
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

// A weight of a norm, 1 without one.
template <bool kBf>
__device__ CVS_INLINE float weight_of(const Norm& n, int c) {
  if (!n.weight) return 1.f;
  return n.fp32 ? static_cast<const float*>(n.weight)[c] : to_float<kBf>(static_cast<const uint16_t*>(n.weight)[c]);
}

typedef float f32x4 __attribute__((ext_vector_type(4)));

// What turns a token's heads: y_c = x_c own[c] + x_partner other[c], with the
// norm's weights, the magnitude and the sign of the sine in both.  A channel
// that does not turn has own = w and other = -0 for a partner of 0, which
// leaves x w as it is, its sign included.  In LDS, `dim` floats each.
struct Turning {
  const uint64_t* turns;
  float magnitude;
  int dim, half;  // half: pairs that turn
};
// Tokens [lo, hi) by a workgroup: a thread has one of the dim / 2 pairs (turned
// ones, then the rest by twos) of every so many tokens; position(t) is a token's.
template <bool kBf, Pairs kPairs, typename Position>
__device__ CVS_INLINE void make_turning(const Turning& a, const Norm& n, int lo, int hi, float* own, float* other,
                                        const Position& position) {
  const int slots = a.dim / 2, step = blockDim.x / slots, first = threadIdx.x / slots, p = threadIdx.x % slots;
  if (first >= step) return;
  const bool turned = p < a.half;
  const int c0 = kPairs == kNeighbours || !turned ? 2 * p : p;
  const int c1 = kPairs == kNeighbours || !turned ? 2 * p + 1 : p + a.half;
  const float w0 = weight_of<kBf>(n, c0), w1 = weight_of<kBf>(n, c1);
  const uint64_t each = turned ? a.turns[p] : 0;
  for (int t = lo + first; t < hi; t += step) {
    const float2 cs = turned ? cos_sin(each * uint64_t(position(t))) : float2{1.f, 0.f};
    const float m = turned ? a.magnitude : 1.f, c = m * cs.x, s = m * cs.y;
    float* const o = own + t * a.dim;
    float* const r = other + t * a.dim;
    o[c0] = c * w0;
    o[c1] = c * w1;
    r[c0] = turned ? -s * w1 : -0.f;
    r[c1] = turned ? s * w0 : -0.f;
  }
}

// A head is a row of 16-byte pieces, one a lane; the power of two of lanes that
// holds the largest head of a kernel has a row.
template <int kLanes>
struct HeadLane {
  int in, piece, pieces;  // lanes past the row's end repeat its last piece
  int dim, half;
  float inv_dim;
  bool turned, low;  // kPieces: a piece of either half, of the first
  int from;          // 4 times the lane that has its partners
  __device__ CVS_INLINE HeadLane(int dim, int half)
      : in(threadIdx.x % kLanes), piece(min(in, dim / 8 - 1)), pieces(dim / 8), dim(dim), half(half),
        inv_dim(1.f / float(dim)), turned(piece < half / 4), low(piece < half / 8) {
    const int to = !turned ? 0 : low ? half / 8 : -half / 8;
    from = 4 * (int(__lane_id()) + piece - in + to);
  }
};

// 1 / sqrt(x) for a row's lanes; the instruction takes subnormal numbers for 0.
__device__ CVS_INLINE float inverse_root(float x) {
  const bool tiny = x < 1e-35f;
  const float r = __builtin_amdgcn_rsqf(tiny ? x * 1.2676506002282294e30f : x);  // 2^100
  return tiny ? r * 1.125899906842624e15f : r;                                    // 2^50
}

// The lane's piece x of a head, normed (if kNorm and `normed`) and turned.
// scratch: the wave's lanes' places in LDS, this one's (kChannels alone).
template <bool kBf, int kLanes, Pairs kPairs, bool kNorm>
__device__ CVS_INLINE u32x4 ready(u32x4 x, const HeadLane<kLanes>& l, const float* own, const float* other, bool normed,
                                  float eps, u32x4* scratch) {
  float f[8], g[8], o[8];
  unpack8<kBf>(x, f);
  float inv = 1.f;
  if constexpr (kNorm) {
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = __builtin_fmaf(f[e], f[e], sum);
    if (l.in >= l.pieces) sum = 0.f;
#pragma unroll
    for (int m = 1; m < kLanes; m <<= 1) sum += xor_lanes_f(sum, m);
    const float root = inverse_root(__builtin_fmaf(sum, l.inv_dim, eps));
    // Before the factors: a product of them and a large channel could be infinite, and 0 times that is NaN.
    inv = normed ? root : 1.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] *= inv;
  }
  if constexpr (kPairs == kNeighbours) {
    // Whole pairs are in or out.
#pragma unroll
    for (int e = 0; e < 8; ++e) g[e] = 4 * l.piece + e / 2 < l.half ? f[e ^ 1] : 0.f;
  } else if constexpr (kPairs == kPieces) {
    u32x4 px;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t w = uint32_t(__builtin_amdgcn_ds_bpermute(l.from, int(x[k])));
      px[k] = l.turned ? w : 0;
    }
    unpack8<kBf>(px, g);
    if constexpr (kNorm) {
#pragma unroll
      for (int e = 0; e < 8; ++e) g[e] *= inv;
    }
  } else {
    // The row's pieces side by side.
    *scratch = x;
    wave_lds_ready();
    const uint16_t* const row = reinterpret_cast<const uint16_t*>(scratch - l.in);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = 8 * l.piece + e;
      const float v = to_float<kBf>(row[c < l.half ? c + l.half : c < 2 * l.half ? c - l.half : c]);
      g[e] = c < 2 * l.half ? (kNorm ? v * inv : v) : 0.f;
    }
    wave_lds_ready();  // read before the next row's pieces are written
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const f32x4 a = reinterpret_cast<const f32x4*>(own)[2 * l.piece + i];
    const f32x4 b = reinterpret_cast<const f32x4*>(other)[2 * l.piece + i];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int e = 4 * i + k;
      o[e] = __builtin_fmaf(f[e], a[k], g[e] * b[k]);
    }
  }
  return pack8<kBf>(o);
}

// A row's result here and not where it is stored: left to the compiler, the
// factors of all rows under way are read first and kept, in registers that
// leave a SIMD two or three waves.
__device__ CVS_INLINE void row_done(u32x4& y) {
  asm volatile("" : "+v"(y));
  __builtin_amdgcn_sched_barrier(0);
}

// Rows of an array by a workgroup: offsets in bytes from its first token and
// head, within 31 bits.
struct RowView {
  char* p;
  uint32_t token, head;
};
// Whether `heads` heads of up to 32 tokens lie within 31 bits of bytes.
inline bool rows_near(const View& v, int64_t heads) {
  return 2 * (31 * v.token + kMaxDim) + 2 * __int128(heads - 1) * v.head < (int64_t(1) << 31);
}

// Rows [0, rows) of tokens x heads by a workgroup, kAhead of each group of
// lanes under way at once.  before() is run behind the first loads.  A row's
// input may be its own output and no other row's.
constexpr int kAhead = 4;
struct Rows {
  int rows, heads;
  uint32_t magic;  // magic_of(heads)
  RowView in, out;
  const float *own, *other;  // of the first token
  bool normed;
  float eps;
};
// r / heads is 2 r magic / 2^32 for r below 2^16.
inline uint32_t magic_of(int heads) { return ((uint32_t(1) << 31) + uint32_t(heads) - 1) / uint32_t(heads); }
template <bool kBf, int kLanes, Pairs kPairs, bool kNorm, typename Before>
__device__ CVS_INLINE void ready_rows(const HeadLane<kLanes>& l, const Rows& a, u32x4* scratch, const Before& before) {
  const int groups = blockDim.x / kLanes, group = threadIdx.x / kLanes;
  auto token_of = [&](int r) CVS_INLINE { return __umulhi(2u * uint32_t(r), a.magic); };
  auto place = [&](const RowView& v, int r) CVS_INLINE {
    const uint32_t t = token_of(r), h = uint32_t(r) - t * uint32_t(a.heads);
    return v.p + (t * v.token + h * v.head + 16u * uint32_t(l.piece));
  };
  u32x4 x[kAhead];
  auto load = [&](int first) CVS_INLINE {
#pragma unroll
    for (int i = 0; i < kAhead; ++i)  // past the last row, that one again (not stored)
      x[i] = *reinterpret_cast<const u32x4*>(place(a.in, min(first + i * groups, a.rows - 1)));
  };
  load(group);
  before();
  for (int first = group; first - group < a.rows; first += kAhead * groups) {
    u32x4 y[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int at = int(token_of(min(first + i * groups, a.rows - 1))) * l.dim;
      y[i] = ready<kBf, kLanes, kPairs, kNorm>(x[i], l, a.own + at, a.other + at, a.normed, a.eps, scratch);
      row_done(y[i]);
    }
    if (first - group + kAhead * groups < a.rows) load(first + kAhead * groups);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int r = first + i * groups;
      if (r < a.rows && l.in < l.pieces) *reinterpret_cast<u32x4*>(place(a.out, r)) = y[i];
    }
  }
}

// Checks a norm of heads of `type`; null: none.
Norm norm_of(const cvs_head_norm* norm, int type, const char* what);
// Checks that a rotary belongs to the context and fits heads of `dim`.
void check_rotary(const cvs_rotary* rotary, const cvs_context* ctx, int dim);
// Checks positions in device memory.
void check_positions(const int64_t* positions);
// Before a call with the rotary is launched: keeps its memory for the replays of a capture.
void captured_rotary(const cvs_rotary* rotary);

}  // namespace attn
}  // namespace cvs
