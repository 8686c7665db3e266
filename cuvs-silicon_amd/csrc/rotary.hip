// Rotary positions of heads, with or without the norm of each head before
// them, from array to array: queries and keys in one launch.
//
// A workgroup takes a few tokens, all of their query or key heads or a part of
// them.  Its threads first make the factors of those tokens' channels, a pair
// each, for all heads (rotary.hpp); then a head is a row of 16-byte pieces, one
// a lane, and 4 to 16 lanes (the power of two that holds the head) have a row.
// The sum of squares goes over those lanes, a channel's partner comes from its
// own piece, from the lane that has it, or, where the halves are no whole pieces
// apart, through LDS.  Rows are read kAhead at a time, the first of them before
// the factors are made.
//
// Bounds: long prompts the memory (12,000 tokens, 32/8 heads of 128, bf16, normed
// and rotated: 53 us with inputs from memory, 4.6 TB/s read and write, where a
// copy by the vendor's library reaches 4.9; 41 us with inputs still in the
// last-level cache; the vector unit is busy 54% of the cycles then).  With cosines
// and sines in LDS, and weights applied to each row, it took 74 us.  Few tokens a
// chain of loads, the factors and a barrier: 2.9 us for one token of 16 heads of
// 64, 4.7 us for 48 of 40 heads of 128, normed; 8.8 us for 3,001 of 24 heads of 80.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "rotary.hpp"

namespace cvs {
namespace attn {
namespace {

constexpr int kTokens = 16;  // of a workgroup at most

// Queries or keys.
struct Part {
  View in, out;
  Norm norm;
  int heads, per_block, chunk, chunks;  // tokens and heads of a workgroup, workgroups of the heads
  uint32_t magic, last_magic;           // of a chunk's heads, and of the last one's
  int blocks;
};

struct RotateArgs {
  Part part[2];
  const int64_t* positions;
  Turning turning;
  int64_t tokens;
};

template <bool kBf, int kLanes, Pairs kPairs, bool kNorm>
__global__ __launch_bounds__(256) void rotate_kernel(const RotateArgs a) {
  __shared__ __align__(16) float s_own[kTokens * kMaxDim], s_other[kTokens * kMaxDim];
  __shared__ __align__(16) u32x4 s_rows[kPairs == kChannels ? 256 : 1];
  const bool second = int(blockIdx.x) >= a.part[0].blocks;
  const Part& p = a.part[second];
  const int block = blockIdx.x - (second ? a.part[0].blocks : 0);
  const int64_t t0 = int64_t(block / p.chunks) * p.per_block;
  const int nt = int(min(int64_t(p.per_block), a.tokens - t0));
  const int h0 = block % p.chunks * p.chunk, nh = min(p.chunk, p.heads - h0);
  const HeadLane<kLanes> l(a.turning.dim, a.turning.half);
  auto first = [&](const View& v) CVS_INLINE {
    return RowView{v.p + 2 * (t0 * v.token + h0 * v.head), uint32_t(2 * v.token), uint32_t(2 * v.head)};
  };
  const Rows rows{nt * nh, nh, nh == p.chunk ? p.magic : p.last_magic, first(p.in), first(p.out), s_own, s_other,
                  p.norm.weight != nullptr, p.norm.eps};
  ready_rows<kBf, kLanes, kPairs, kNorm>(l, rows, s_rows + (kPairs == kChannels ? threadIdx.x : 0), [&]() CVS_INLINE {
    make_turning<kBf, kPairs>(a.turning, p.norm, 0, nt, s_own, s_other,
                              [&](int t) CVS_INLINE { return a.positions[t0 + t]; });
    __syncthreads();
  });
}

template <bool kBf, int kLanes>
void launch(cvs_context* ctx, const RotateArgs& a, Pairs pairs, bool norm, dim3 grid) {
  const TimerSpan ts = timer_span(ctx, "rotate");
  auto go = [&](auto kernel) {
    hipExtLaunchKernelGGL(kernel, grid, dim3(256), 0, ctx->stream, ts.start, ts.stop, 0, a);
  };
  switch (pairs) {
    case kNeighbours: norm ? go(rotate_kernel<kBf, kLanes, kNeighbours, true>) : go(rotate_kernel<kBf, kLanes, kNeighbours, false>); break;
    case kPieces: norm ? go(rotate_kernel<kBf, kLanes, kPieces, true>) : go(rotate_kernel<kBf, kLanes, kPieces, false>); break;
    default: norm ? go(rotate_kernel<kBf, kLanes, kChannels, true>) : go(rotate_kernel<kBf, kLanes, kChannels, false>); break;
  }
  after_launch("rotate_kernel");
}

template <bool kBf>
void launch(cvs_context* ctx, const RotateArgs& a, Pairs pairs, bool norm, dim3 grid) {
  if (a.turning.dim > 64) launch<kBf, 16>(ctx, a, pairs, norm, grid);
  else if (a.turning.dim > 32) launch<kBf, 8>(ctx, a, pairs, norm, grid);
  else launch<kBf, 4>(ctx, a, pairs, norm, grid);
}

// The part of a turn that a position adds, in units of 2^-64 modulo whole turns, rounded: the radians' 53 bits times 1 / 2 pi
// in 128, of which the whole turns of 1024 radians take 8.
uint64_t turns_of(double radians) {
  constexpr uint64_t hi = 0x28be60db9391054aull, lo = 0x7f09d5f47d4d3770ull;  // 2^128 / 2 pi
  int exponent;
  const uint64_t m = uint64_t(std::ldexp(std::frexp(std::abs(radians), &exponent), 53));
  const int shift = 53 - exponent;  // radians = m 2^-shift; 42 and more, as they are at most 1024
  if (shift > 120) return 0;
  typedef unsigned __int128 u128;
  const u128 product = u128(m) * hi + (u128(m) * lo >> 64);  // m / 2 pi in units of 2^-64: 118 bits at most
  const uint64_t turns = uint64_t((product + (u128(1) << (shift - 1))) >> shift);
  return radians < 0 ? -turns : turns;
}

// Checks and launches; q or k may be null.
void rotate(cvs_context* ctx, const cvs_rotary* rotary, const int64_t* positions, const cvs_heads* const (&in)[2],
            const cvs_heads* const (&out)[2], const cvs_head_norm* const (&norm)[2], const char* const (&names)[2]) {
  RotateArgs a{};
  const cvs_heads* first = nullptr;
  for (int i = 0; i < 2; ++i) {
    const std::string w(names[i]);
    if (!in[i]) {
      if (out[i] || norm[i]) fail(CVS_ERR_INVALID_ARGUMENT, "an output or a norm of " + w + " without " + w);
      continue;
    }
    check_view(in[i], names[i]);
    check_view(out[i], (w + "_out").c_str());
    if (out[i]->tokens != in[i]->tokens || out[i]->heads != in[i]->heads || out[i]->head_dim != in[i]->head_dim ||
        out[i]->type != in[i]->type)
      fail(CVS_ERR_INVALID_ARGUMENT, w + " and its output must have one shape and type");
    if (!first) first = in[i];
    if (in[i]->tokens != first->tokens || in[i]->head_dim != first->head_dim || in[i]->type != first->type)
      fail(CVS_ERR_INVALID_ARGUMENT, "q and k must have the same tokens, head_dim and type");
    check_rows_apart(out[i], (w + "_out").c_str());
    if (in[i]->heads > 65535) fail(CVS_ERR_UNSUPPORTED, "too many heads");
    a.part[i].in = view_of(in[i]);
    a.part[i].out = view_of(out[i]);
    a.part[i].norm = norm_of(norm[i], in[i]->type, names[i]);
    a.part[i].heads = in[i]->heads;
  }
  if (!first) fail(CVS_ERR_INVALID_ARGUMENT, "neither q nor k");
  if (rotary) check_rotary(rotary, ctx, first->head_dim);
  if (positions && !rotary) fail(CVS_ERR_INVALID_ARGUMENT, "positions without a rotary");
  check_positions(positions);
  if (first->tokens == 0) return;
  if (rotary && !positions) fail(CVS_ERR_INVALID_ARGUMENT, "null positions");
  a.positions = positions;
  a.tokens = first->tokens;
  a.turning.dim = first->head_dim;
  if (rotary) {
    captured_rotary(rotary);
    a.turning.half = rotary->dims / 2;
    a.turning.turns = rotary->turns.as<uint64_t>();
    a.turning.magnitude = rotary->magnitude;
  }
  // A workgroup makes its tokens' factors once for all of its rows, about 128.  Fewer tokens are spread over two
  // workgroups a compute unit, queries' and keys' by their heads, and few ones' heads over more, down to 16 rows each.
  const int64_t all = int64_t(a.part[0].heads) + a.part[1].heads;
  int64_t blocks = 0;
  for (Part& p : a.part) {
    if (!p.heads) continue;
    const int64_t least = std::max<int64_t>(1, 2 * ctx->compute_units * p.heads / all);
    p.per_block = int(std::clamp<int64_t>(std::min<int64_t>(128 / p.heads, a.tokens / least), 1, kTokens));
    const int64_t groups = (a.tokens + p.per_block - 1) / p.per_block;
    const int64_t fit = std::clamp<int64_t>(least / groups, 1, (p.heads + 15) / 16);
    p.chunk = int(std::min<int64_t>((p.heads + fit - 1) / fit, 1024));
    if (!rows_near(p.in, p.chunk) || !rows_near(p.out, p.chunk)) p.chunk = 1;
    p.chunks = (p.heads + p.chunk - 1) / p.chunk;
    p.magic = magic_of(p.chunk);
    p.last_magic = magic_of(p.heads - (p.chunks - 1) * p.chunk);
    if (groups * p.chunks > kMaxBlocks) fail(CVS_ERR_UNSUPPORTED, "too many tokens");
    p.blocks = int(groups * p.chunks);
    blocks += p.blocks;
  }
  if (blocks > kMaxBlocks) fail(CVS_ERR_UNSUPPORTED, "too many tokens");
  const dim3 grid{unsigned(blocks)};
  const bool is_norm = a.part[0].norm.weight || a.part[1].norm.weight;
  if (first->type == CVS_BF16) launch<true>(ctx, a, pairs_of(rotary), is_norm, grid);
  else launch<false>(ctx, a, pairs_of(rotary), is_norm, grid);
}

}  // namespace

Norm norm_of(const cvs_head_norm* norm, int type, const char* what) {
  if (!norm) return {};
  const std::string w(what);
  if (!norm->weight) fail(CVS_ERR_INVALID_ARGUMENT, "null weight of the norm of " + w);
  if (norm->type != CVS_FP32 && norm->type != type)
    fail(CVS_ERR_UNSUPPORTED, "the norm's weight must be fp32 or of the type of " + w);
  if (reinterpret_cast<uintptr_t>(norm->weight) % (norm->type == CVS_FP32 ? 4 : 2) != 0)
    fail(CVS_ERR_UNSUPPORTED, "the norm's weight must be aligned to its type");
  if (!(norm->eps >= 0.f) || std::isinf(norm->eps))
    fail(CVS_ERR_INVALID_ARGUMENT, "eps must be finite and not negative");
  return {norm->weight, norm->type == CVS_FP32, norm->eps};
}

void check_rotary(const cvs_rotary* rotary, const cvs_context* ctx, int dim) {
  if (rotary->ctx != ctx) fail(CVS_ERR_INVALID_ARGUMENT, "the rotary belongs to another context");
  if (rotary->dims > dim)
    fail(CVS_ERR_INVALID_ARGUMENT, "the rotary turns " + std::to_string(rotary->dims) + " channels, heads have " +
                                       std::to_string(dim));
}

void check_positions(const int64_t* positions) {
  if (reinterpret_cast<uintptr_t>(positions) % 8 != 0)
    fail(CVS_ERR_UNSUPPORTED, "positions must be aligned to 8 bytes");
}

void captured_rotary(const cvs_rotary* rotary) {
  if (rotary->captured || !capturing(rotary->ctx)) return;
  rotary->ctx->kept.push_back(rotary->turns);
  rotary->captured = true;
}

}  // namespace attn
}  // namespace cvs

using namespace cvs;
using namespace cvs::attn;

extern "C" {

int cvs_rotary_frequencies(int dims, double base, const cvs_rotary_scaling* scaling, double* out_radians) {
  return guarded([&] {
    if (!out_radians) fail(CVS_ERR_INVALID_ARGUMENT, "null out_radians");
    if (dims < 2 || dims % 2 != 0 || dims > kMaxDim)
      fail(CVS_ERR_UNSUPPORTED, "a rotary turns an even number of channels from 2 to " + std::to_string(kMaxDim));
    if (!(base >= 1.0) || std::isinf(base)) fail(CVS_ERR_INVALID_ARGUMENT, "base must be finite and at least 1");
    const int kind = scaling ? scaling->kind : CVS_SCALING_NONE;
    const double factor = scaling ? scaling->factor : 1.0;
    if (kind < CVS_SCALING_NONE || kind > CVS_SCALING_TURNS) fail(CVS_ERR_INVALID_ARGUMENT, "unknown scaling");
    if (kind != CVS_SCALING_NONE && (!(factor > 0.0) || std::isinf(factor)))
      fail(CVS_ERR_INVALID_ARGUMENT, "a scaling's factor must be finite and positive");
    if (kind == CVS_SCALING_BASE && dims == 2)
      fail(CVS_ERR_INVALID_ARGUMENT, "a base cannot be scaled for a single pair of channels");
    if (kind == CVS_SCALING_TURNS &&
        (!(scaling->original_length > 0.0) || std::isinf(scaling->original_length) || !(scaling->low >= 0.0) ||
         !(scaling->high > scaling->low) || std::isinf(scaling->high)))
      fail(CVS_ERR_INVALID_ARGUMENT, "a scaling by turns needs a positive original length and 0 <= low < high");
    constexpr double two_pi = 6.283185307179586;
    for (int i = 0; i < dims / 2; ++i) {
      double f = std::pow(base, -2.0 * i / dims);
      if (kind == CVS_SCALING_LINEAR) f /= factor;
      if (kind == CVS_SCALING_BASE) f *= std::pow(factor, -2.0 * i / (dims - 2));
      if (kind == CVS_SCALING_TURNS) {
        const double turns = scaling->original_length * f / two_pi;
        const double share = std::clamp((turns - scaling->low) / (scaling->high - scaling->low), 0.0, 1.0);
        f *= share + (1.0 - share) / factor;
      }
      out_radians[i] = f;
    }
  });
}

int cvs_rotary_create(cvs_context* ctx, int dims, int layout, const double* radians, float magnitude,
                      cvs_rotary** out_rotary) {
  return guarded([&] {
    bind(ctx);
    if (!out_rotary) fail(CVS_ERR_INVALID_ARGUMENT, "null out_rotary");
    *out_rotary = nullptr;
    if (!radians) fail(CVS_ERR_INVALID_ARGUMENT, "null radians");
    if (dims < 2 || dims % 2 != 0 || dims > kMaxDim)
      fail(CVS_ERR_UNSUPPORTED, "a rotary turns an even number of channels from 2 to " + std::to_string(kMaxDim));
    if (layout != CVS_ROTARY_HALVES && layout != CVS_ROTARY_NEIGHBOURS)
      fail(CVS_ERR_INVALID_ARGUMENT, "layout must be CVS_ROTARY_HALVES or CVS_ROTARY_NEIGHBOURS");
    if (!std::isfinite(magnitude)) fail(CVS_ERR_INVALID_ARGUMENT, "magnitude must be finite");
    std::vector<uint64_t> turns;
    for (int i = 0; i < dims / 2; ++i) {
      if (!(std::abs(radians[i]) <= 1024.0))
        fail(CVS_ERR_UNSUPPORTED, "frequencies must be from -1024 to 1024 radians a position");
      turns.push_back(turns_of(radians[i]));
    }
    need_no_capture(ctx, "a rotary cannot be made");
    auto r = std::make_unique<cvs_rotary>();
    r->ctx = ctx;
    r->dims = dims;
    r->layout = layout;
    r->magnitude = magnitude;
    const size_t bytes = turns.size() * sizeof(uint64_t);
    r->turns = take_blob(ctx->plan_blobs, ctx->live_prompt_plans, bytes);
    try {
      upload(ctx, r->turns.ptr, turns.data(), bytes);
    } catch (...) {
      ctx->plan_blobs.push_back(r->turns);
      throw;
    }
    ++ctx->live_prompt_plans;
    ++ctx->live_children;
    *out_rotary = r.release();
  });
}

int cvs_rotary_destroy(cvs_rotary* rotary) {
  return guarded([&] {
    if (!rotary) return;
    // Later plans use the memory on the same stream, after whatever still reads it.
    if (!rotary->captured) rotary->ctx->plan_blobs.push_back(rotary->turns);
    --rotary->ctx->live_prompt_plans;
    --rotary->ctx->live_children;
    delete rotary;
  });
}

int cvs_rotate_async(cvs_context* ctx, const cvs_rotary* rotary, const int64_t* positions, const cvs_heads* x,
                     const cvs_heads* out) {
  return guarded([&] {
    bind(ctx);
    if (!rotary) fail(CVS_ERR_INVALID_ARGUMENT, "null rotary");
    if (!x) fail(CVS_ERR_INVALID_ARGUMENT, "null x");
    rotate(ctx, rotary, positions, {x, nullptr}, {out, nullptr}, {nullptr, nullptr}, {"x", "k"});
  });
}

int cvs_norm_rotate_async(cvs_context* ctx, const cvs_rotary* rotary, const int64_t* positions, const cvs_heads* q,
                          const cvs_heads* q_out, const cvs_head_norm* q_norm, const cvs_heads* k,
                          const cvs_heads* k_out, const cvs_head_norm* k_norm) {
  return guarded([&] {
    bind(ctx);
    rotate(ctx, rotary, positions, {q, k}, {q_out, k_out}, {q_norm, k_norm}, {"q", "k"});
  });
}

}  // extern "C"
