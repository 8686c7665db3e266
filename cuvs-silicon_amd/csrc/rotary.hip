// Rotary positions of heads, with or without the norm of each head before
// them, from array to array: queries and keys in one launch.
//
// A workgroup takes a few tokens, all of their heads or a part of them.  Its
// threads first make the cosines and sines of those tokens, one each, for all
// heads; then a head is a row of 16-byte pieces, one a lane, and 1 to 16 lanes
// (the power of two that holds the head) have a row.  The sum of squares goes
// over those lanes, a channel's partner comes from its own piece, from the
// lane that has it, or, where the halves are no whole pieces apart, through
// LDS.  Rows are read kAhead at a time, the first of them before the cosines
// are made.  Bound by the memory.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "rotary.hpp"

namespace cvs {
namespace attn {
namespace {

constexpr int kTokens = 16;  // of a workgroup at most
constexpr int kMaxPairs = kMaxDim / 2;

struct RotateArgs {
  View in[2], out[2];  // queries, keys
  Norm norm[2];
  int heads[2];
  const int64_t* positions;
  const uint64_t* turns;
  int64_t tokens;
  int dim, dims;
  float magnitude;
  int per_block;  // tokens of a workgroup
  int chunk;      // heads of a workgroup
};

template <bool kBf, int kLanes, Pairs kPairs, bool kNorm>
__global__ __launch_bounds__(256) void rotate_kernel(const RotateArgs a) {
  __shared__ __align__(16) float s_cos[kTokens * kMaxPairs], s_sin[kTokens * kMaxPairs];
  __shared__ __align__(16) float s_w[kNorm ? 2 * kMaxDim : 1];
  __shared__ __align__(16) u32x4 s_rows[kPairs == kChannels ? 256 : 1];
  const int64_t t0 = int64_t(blockIdx.x) * a.per_block;
  const int nt = int(min(int64_t(a.per_block), a.tokens - t0));
  const int h0 = blockIdx.y * a.chunk, nh = min(a.chunk, a.heads[0] + a.heads[1] - h0);
  const HeadLane<kLanes> l(a.dim, a.dims);
  auto place = [&](int r) CVS_INLINE {
    const int t = r / nh, h = h0 + r % nh, k = h >= a.heads[0], head = k ? h - a.heads[0] : h;
    const View& in = k ? a.in[1] : a.in[0];
    const View& out = k ? a.out[1] : a.out[0];
    const Norm& n = k ? a.norm[1] : a.norm[0];
    return HeadRow{in.p + 2 * ((t0 + t) * in.token + head * in.head),
                   out.p + 2 * ((t0 + t) * out.token + head * out.head), s_cos + t * kMaxPairs, s_sin + t * kMaxPairs,
                   kNorm && n.weight ? s_w + k * kMaxDim : nullptr, n.eps};
  };
  auto before = [&]() CVS_INLINE {
    for (int i = threadIdx.x; i < nt * l.half; i += 256) {
      const int t = i / l.half, p = i % l.half;
      const float2 cs = cos_sin(a.turns[p] * uint64_t(a.positions[t0 + t]));
      s_cos[t * kMaxPairs + p] = a.magnitude * cs.x;
      s_sin[t * kMaxPairs + p] = a.magnitude * cs.y;
    }
    if constexpr (kNorm) {
      load_weight<kBf>(s_w, a.norm[0], a.dim);
      load_weight<kBf>(s_w + kMaxDim, a.norm[1], a.dim);
    }
    __syncthreads();
  };
  ready_rows<kBf, kLanes, kPairs, kNorm>(l, nt * nh, s_rows + (kPairs == kChannels ? threadIdx.x : 0), place, before);
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
  if (a.dim > 64) launch<kBf, 16>(ctx, a, pairs, norm, grid);
  else if (a.dim > 32) launch<kBf, 8>(ctx, a, pairs, norm, grid);
  else launch<kBf, 4>(ctx, a, pairs, norm, grid);
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
    a.in[i] = view_of(in[i]);
    a.out[i] = view_of(out[i]);
    a.norm[i] = norm_of(norm[i], in[i]->type, names[i]);
    a.heads[i] = in[i]->heads;
  }
  if (!first) fail(CVS_ERR_INVALID_ARGUMENT, "neither q nor k");
  if (rotary) check_rotary(rotary, ctx, first->head_dim);
  if (first->tokens == 0) return;
  if (rotary && !positions) fail(CVS_ERR_INVALID_ARGUMENT, "null positions");
  const int64_t heads = int64_t(a.heads[0]) + a.heads[1];
  if (heads > 65536) fail(CVS_ERR_UNSUPPORTED, "too many heads");
  a.positions = positions;
  a.tokens = first->tokens;
  a.dim = first->head_dim;
  if (rotary) {
    captured_rotary(rotary);
    a.dims = rotary->dims;
    a.turns = rotary->turns.as<uint64_t>();
    a.magnitude = rotary->magnitude;
  }
  // A workgroup makes its tokens' cosines once for all rows, about 128 of them; few tokens' heads are spread over more
  // workgroups, down to 16 rows each.
  a.per_block = int(std::clamp<int64_t>(128 / heads, 1, kTokens));
  const int64_t blocks = (a.tokens + a.per_block - 1) / a.per_block;
  if (blocks > kMaxBlocks) fail(CVS_ERR_UNSUPPORTED, "too many tokens");
  const int64_t fit = std::max<int64_t>(1, 2 * ctx->compute_units / blocks);
  a.chunk = int(std::max<int64_t>(std::min<int64_t>(heads, 16), (heads + fit - 1) / fit));
  const dim3 grid(unsigned(blocks), unsigned((heads + a.chunk - 1) / a.chunk));
  const bool is_norm = a.norm[0].weight || a.norm[1].weight;
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
      // 64 bits of the part behind the point; a long double has them for all that is less than a turn.
      constexpr long double two_pi = 6.283185307179586476925286766559L;
      const long double t = static_cast<long double>(radians[i]) / two_pi;
      const long double part = (t - std::floor(t)) * 18446744073709551616.0L;
      turns.push_back(part >= 18446744073709551615.0L ? 0 : uint64_t(std::llroundl(part / 2) * 2));
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
