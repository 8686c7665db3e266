// A paged cache of attention keys and values: sequences as lists of pages
// that they may share, and the device work on pages - writing new tokens,
// reading tokens back, copying pages.
//
// Layout of the pool: layer, page, kv head, then the head's tokens in tiles of
// 32, the keys of a tile followed by its values.  Either is a run of 1 KiB
// blocks that are operands of v_mfma_f32_32x32x16 as they stand, 16 bytes a lane, as the
// datasets' tiles are, so that attention streams whole blocks from memory
// into operand registers:
//   keys:   block s holds columns [16 s, 16 s + 16); lane l has token l % 32, columns 16 s + 8 (l / 32) + [0, 8);
//   values: block 2 b + s holds columns [32 b, 32 b + 32) of tokens [16 s, 16 s + 16); lane l has column 32 b + l % 32
//           of tokens 16 s + 4 (l / 32) + {0, 1, 2, 3, 8, 9, 10, 11}, the order in which the first product leaves
//           its probabilities (attn_common.hpp).
// Rows are padded to whole 32-column blocks with zeros.
#include <cstring>

#include "attn_common.hpp"

namespace cvs {
namespace attn {
namespace {

// A plan's bytes as a kernel's arguments: a copy from pageable memory may wait
// for the stream, and a pinned buffer could not be filled again before its copy
// has ended.
struct Upload {
  uint32_t words[kUploadBytes / 4];
};

__global__ __launch_bounds__(256) void upload_kernel(uint32_t* __restrict__ dst, const Upload u, int words) {
  for (int i = threadIdx.x; i < words; i += 256) dst[i] = u.words[i];
}

// Up to kCopies page copies of a launch, passed as arguments.
constexpr int kCopies = 448;
struct Copies {
  kv::PageCopy c[kCopies];
};

// Bound by the memory: 24 pages of 256 KiB in 16 layers, 201 MB read and
// written in 37 us, 5.4 TB/s.
constexpr int kCopyBytes = 16384;  // of a workgroup: 4 loads of 16 bytes a thread in flight

__global__ __launch_bounds__(256) void copy_pages_kernel(char* __restrict__ pool, int64_t layer_bytes,
                                                         int64_t page_bytes, const Copies copies) {
  const kv::PageCopy c = copies.c[blockIdx.x];
  char* const layer = pool + int64_t(blockIdx.y) * layer_bytes;
  const int64_t at = int64_t(blockIdx.z) * kCopyBytes + threadIdx.x * 16;
  const char* const src = layer + c.src * page_bytes;
  char* const dst = layer + c.dst * page_bytes;
  u32x4 v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (at + i * 4096 < page_bytes) v[i] = *reinterpret_cast<const u32x4*>(src + at + i * 4096);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (at + i * 4096 < page_bytes) *reinterpret_cast<u32x4*>(dst + at + i * 4096) = v[i];
}

void copy_pages(cvs_kv_cache* cache, const std::vector<kv::PageCopy>& copies) {
  for (size_t at = 0; at < copies.size(); at += kCopies) {
    const size_t n = std::min(copies.size() - at, size_t(kCopies));
    Copies c;
    std::memcpy(c.c, copies.data() + at, n * sizeof(kv::PageCopy));
    const unsigned chunks = unsigned((cache->page_bytes + kCopyBytes - 1) / kCopyBytes);
    hipLaunchKernelGGL(copy_pages_kernel, dim3(unsigned(n), unsigned(cache->layers), chunks), dim3(256), 0,
                       cache->ctx->stream, cache->pool, cache->layer_bytes, cache->page_bytes, c);
    after_launch("copy_pages_kernel");
  }
}

// Spans of a small plan go to the kernel as arguments, others are read from the plan's memory.
constexpr int kInlineSpans = 192;
struct Spans {
  Span s[kInlineSpans];
};

struct MoveArgs {
  char* pool;  // of the first layer
  int64_t layer_bytes, page_bytes, head_bytes;
  const Span* spans;  // null: inline
  View k, v;
  int64_t k_layer, v_layer;  // strides of the caller's arrays from layer to layer
  int n_spans, page_tiles, by_tile, dim, kv_heads;
  int units;  // spans * tiles of a page * kv_heads
};

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

// Between rows of the caller's arrays and tiles of the pool, one wave a tile
// of 32 tokens, kv head and layer; no wave waits for another.  Rows are read
// and written along the row.  Keys change places 16 bytes at a time, through
// LDS of the wave's own; values by transposing, in a lane's registers, 8
// columns of the 8 tokens whose elements stand together.  A tile's tokens
// before the span's keep what they hold, also where their values share 16
// bytes with new ones; those after it are past the sequence's end.  A wave's
// loads are all under way at once: of clamped rows, or all under one condition.
// Bound by the memory: 12 sequences of 700 tokens, 16 layers of 8 heads of
// 128, 1.1 GB read and written in 206 us (write) and 207 us (read), 5.3 TB/s.
template <int NB, bool kWrite>
__global__ __launch_bounds__(256) void move_tokens_kernel(const MoveArgs a, const Spans inl) {
  constexpr int P = 4 * NB;  // 16-byte pieces of a row
  __shared__ __align__(16) u32x4 s[4][32 * P];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int unit = blockIdx.x * 4 + wave;
  if (unit >= a.units) return;
  // Span by span, or, where spans fill few of a page's tiles, all spans' first tiles, then all second ones, so that
  // whole ranges of workgroups are without work and not every other one, which would be every other XCD: 64 spans of 9
  // tokens in pages of 64 are written in 22 us by tiles and 38 by spans, 12 times 700 tokens in 217 and 211.
  const int g = unit % a.kv_heads, n = unit / a.kv_heads;
  const int at = a.by_tile ? n % a.n_spans : n / a.page_tiles, tile = a.by_tile ? n / a.n_spans : n % a.page_tiles;
  const Span sp = a.spans ? a.spans[at] : inl.s[at];
  const int lo = max(sp.begin - 32 * tile, 0), hi = min(sp.end - 32 * tile, 32);
  if (lo >= hi) return;
  char* const kt = a.pool + blockIdx.y * a.layer_bytes + sp.page * a.page_bytes + g * a.head_bytes +
                   int64_t(tile) * 4096 * NB;
  char* const vt = kt + 2048 * NB;
  const int64_t row = int64_t(sp.row0) + 32 * tile - sp.begin;  // of the tile's token 0
  char* const ks = a.k.p + 2 * (blockIdx.y * a.k_layer + row * a.k.token + g * a.k.head);
  char* const vs = a.v.p + 2 * (blockIdx.y * a.v_layer + row * a.v.token + g * a.v.head);
  const int pieces = a.dim / 8;
  auto held = [&](int t) CVS_INLINE { return min(max(t, lo), hi - 1); };

  // Values: lane = (columns 8 c and on, tokens t0 + {0, 1, 2, 3, 8, 9, 10, 11}).
  const int c = lane % P, t0 = 16 * (lane / P >> 1) + 4 * (lane / P & 1);
  const bool mine = lane < 4 * P && t0 < hi && t0 + 11 >= lo;
  u32x4* const slots = reinterpret_cast<u32x4*>(
      vt + (2 * (c / 4) + (lane / P >> 1)) * 1024 + (32 * (lane / P & 1) + 8 * (c % 4)) * 16);
  u32x4 x[8], y[P / 2];
  auto token = [&](int j) CVS_INLINE { return t0 + 8 * (j / 4) + j % 4; };
  if constexpr (kWrite) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      x[j] = *reinterpret_cast<const u32x4*>(vs + 2 * (held(token(j)) * a.v.token + 8 * min(c, pieces - 1)));
#pragma unroll
    for (int i = 0; i < P / 2; ++i) {
      const int n = 64 * i + lane;
      y[i] = *reinterpret_cast<const u32x4*>(ks + 2 * (held(n / P) * a.k.token + 8 * min(n % P, pieces - 1)));
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c >= pieces) x[j] = u32x4{};
    transpose8(x);
    if (mine && t0 < lo) {
      uint32_t keep[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) keep[k] = (token(2 * k) < lo ? 0xffffu : 0u) | (token(2 * k + 1) < lo ? 0xffff0000u : 0u);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const u32x4 old = slots[j];
#pragma unroll
        for (int k = 0; k < 4; ++k) x[j][k] = (x[j][k] & ~keep[k]) | (old[k] & keep[k]);
      }
    }
    if (mine) {
#pragma unroll
      for (int j = 0; j < 8; ++j) slots[j] = x[j];
    }
#pragma unroll
    for (int i = 0; i < P / 2; ++i) {
      const int n = 64 * i + lane, t = n / P, p = n % P;
      s[wave][t * P + (p ^ (t & 3))] = p < pieces ? y[i] : u32x4{};
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    const int t = lane & 31;
#pragma unroll
    for (int i = 0; i < P / 2; ++i) y[i] = s[wave][t * P + ((2 * i + (lane >> 5)) ^ (t & 3))];
    if (t >= lo && t < hi) {
#pragma unroll
      for (int i = 0; i < P / 2; ++i) *reinterpret_cast<u32x4*>(kt + 1024 * i + 16 * lane) = y[i];
    }
  } else {
    const int t = lane & 31;
    const bool key = t >= lo && t < hi;
    if (key) {
#pragma unroll
      for (int i = 0; i < P / 2; ++i) y[i] = *reinterpret_cast<const u32x4*>(kt + 1024 * i + 16 * lane);
    }
    if (mine) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = slots[j];
    }
    if (key) {
#pragma unroll
      for (int i = 0; i < P / 2; ++i) s[wave][t * P + ((2 * i + (lane >> 5)) ^ (t & 3))] = y[i];
    }
    transpose8(x);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (mine && token(j) >= lo && token(j) < hi && c < pieces)
        *reinterpret_cast<u32x4*>(vs + 2 * (token(j) * a.v.token + 8 * c)) = x[j];
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int i = 0; i < P / 2; ++i) {
      const int n = 64 * i + lane, t = n / P, p = n % P;
      if (t >= lo && t < hi && p < pieces)
        *reinterpret_cast<u32x4*>(ks + 2 * (t * a.k.token + 8 * p)) = s[wave][t * P + (p ^ (t & 3))];
    }
  }
}

void move_tokens(cvs_kv_plan* plan, int first_layer, int layers, const cvs_heads* k, int64_t k_layer,
                 const cvs_heads* v, int64_t v_layer, bool write) {
  check_plan(plan);
  cvs_kv_cache* const c = plan->cache;
  if (first_layer < 0 || layers < 1 || first_layer > c->layers - layers)
    fail(CVS_ERR_INVALID_ARGUMENT, "layers outside the cache's " + std::to_string(c->layers));
  for (const cvs_heads* x : {k, v}) {
    const char* const what = x == k ? "k" : "v";
    check_view(x, what);
    if (x->tokens != plan->tokens)
      fail(CVS_ERR_INVALID_ARGUMENT, std::string(what) + " must have the plan's " + std::to_string(plan->tokens) +
                                         " tokens");
    if (x->heads != c->kv_heads || x->head_dim != c->dim || x->type != c->type)
      fail(CVS_ERR_INVALID_ARGUMENT, std::string(what) + " must have the cache's heads, head_dim and type");
  }
  if (layers > 1 && (k_layer % 8 != 0 || v_layer % 8 != 0 || k_layer < 0 || v_layer < 0))
    fail(CVS_ERR_UNSUPPORTED, "layer strides must be non-negative multiples of 8 elements");
  if (!write) {
    check_rows_apart(k, "k", layers, k_layer);
    check_rows_apart(v, "v", layers, v_layer);
  }
  for (const Span& sp : plan->spans)
    if (write && c->book->refs(sp.page) > 1)
      fail(CVS_ERR_INVALID_ARGUMENT, "the plan's tokens lie in a page that sequences share: extend first");
  if (plan->spans.empty()) return;
  captured_call(plan);
  const int tiles = int(c->book->page_tokens() / 32);
  const int64_t units = int64_t(plan->spans.size()) * tiles * c->kv_heads;
  if (units > kMaxBlocks * 4) fail(CVS_ERR_UNSUPPORTED, "too many tokens");
  Spans inl;
  const bool small = plan->spans.size() <= size_t(kInlineSpans);
  if (small) std::memcpy(inl.s, plan->spans.data(), plan->spans.size() * sizeof(Span));
  const MoveArgs a{c->pool + first_layer * c->layer_bytes, c->layer_bytes, c->page_bytes, c->head_bytes,
                   small ? nullptr : reinterpret_cast<const Span*>(plan->blob.as<char>() + plan->at_spans),
                   view_of(k), view_of(v), k_layer, v_layer, int(plan->spans.size()), tiles,
                   2 * plan->tokens < int64_t(plan->spans.size()) * c->book->page_tokens(), c->dim, c->kv_heads, int(units)};
  const dim3 grid(unsigned((units + 3) / 4), unsigned(layers));
  const TimerSpan ts = timer_span(c->ctx, write ? "kv_write" : "kv_read");
  auto go = [&](auto kernel) {
    hipExtLaunchKernelGGL(kernel, grid, dim3(256), 0, c->ctx->stream, ts.start, ts.stop, 0, a, inl);
  };
  switch (c->nb) {
    case 1: write ? go(move_tokens_kernel<1, true>) : go(move_tokens_kernel<1, false>); break;
    case 2: write ? go(move_tokens_kernel<2, true>) : go(move_tokens_kernel<2, false>); break;
    case 3: write ? go(move_tokens_kernel<3, true>) : go(move_tokens_kernel<3, false>); break;
    default: write ? go(move_tokens_kernel<4, true>) : go(move_tokens_kernel<4, false>); break;
  }
  after_launch("move_tokens_kernel");
}

// Runs fn on the cache's bookkeeping with its errors as status codes.
template <typename Fn>
int on_book(cvs_kv_cache* cache, Fn&& fn) {
  return guarded([&] {
    if (!cache) fail(CVS_ERR_INVALID_ARGUMENT, "null cache");
    try {
      fn();
    } catch (const kv::PageError& e) {
      fail(e.full ? CVS_ERR_OUT_OF_MEMORY : CVS_ERR_INVALID_ARGUMENT, e.what);
    }
  });
}

void need(const void* p, const char* what) {
  if (!p) fail(CVS_ERR_INVALID_ARGUMENT, std::string("null ") + what);
}

void need_list(const void* p, int64_t n, const char* what) {
  if (n < 0) fail(CVS_ERR_INVALID_ARGUMENT, std::string("negative count of ") + what);
  if (n > 0) need(p, what);
}

}  // namespace

DeviceBuffer take_blob(std::vector<DeviceBuffer>& pool, int live_plans, size_t bytes) {
  size_t best = pool.size();
  for (size_t i = 0; i < pool.size(); ++i)
    if (pool[i].bytes >= bytes && (best == pool.size() || pool[i].bytes < pool[best].bytes)) best = i;
  DeviceBuffer b;
  if (best < pool.size()) {
    b = pool[best];
    pool.erase(pool.begin() + int64_t(best));
    return b;
  }
  pool.reserve(pool.size() + size_t(live_plans) + 1);  // destroying a plan does not allocate
  b.reserve(std::max(bytes, size_t(65536)));
  return b;
}

void upload(cvs_context* ctx, void* dst, const void* src, size_t bytes) {
  for (size_t at = 0; at < bytes; at += kUploadBytes) {
    const size_t n = std::min(bytes - at, kUploadBytes);
    Upload u;
    std::memcpy(u.words, static_cast<const char*>(src) + at, n);
    hipLaunchKernelGGL(upload_kernel, dim3(1), dim3(256), 0, ctx->stream,
                       reinterpret_cast<uint32_t*>(static_cast<char*>(dst) + at), u, int(n / 4));
    after_launch("upload_kernel");
  }
}

bool capturing(const cvs_context* ctx) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(ctx->stream, &status) != hipSuccess) {
    // The default stream while another one is captured: a launch on it says so itself, and the status is anything.
    (void)hipGetLastError();
    return false;
  }
  return status != hipStreamCaptureStatusNone;
}

void need_no_capture(const cvs_context* ctx, const char* what) {
  if (capturing(ctx))
    fail(CVS_ERR_INVALID_ARGUMENT, std::string(what) + " while the context's stream is being captured into a graph");
}

bool captured_call(cvs_kv_plan* plan) {
  if (!capturing(plan->cache->ctx)) return false;
  if (!plan->captured && plan->blob.ptr) {
    plan->cache->kept.push_back(plan->blob);
    plan->captured = true;
  }
  return true;
}

void check_plan(const cvs_kv_plan* plan) {
  if (!plan) fail(CVS_ERR_INVALID_ARGUMENT, "null plan");
  try {
    for (size_t i = 0; i < plan->seqs.size(); ++i)
      if (plan->cache->book->at(plan->seqs[i]).version != plan->versions[i])
        fail(CVS_ERR_INVALID_ARGUMENT, "sequence " + std::to_string(plan->seqs[i]) +
                                           " has changed since the plan was made: make a new one");
  } catch (const kv::PageError& e) {
    fail(CVS_ERR_INVALID_ARGUMENT, e.what);
  }
}

}  // namespace attn
}  // namespace cvs

using namespace cvs;
using namespace cvs::attn;

extern "C" {

int cvs_kv_cache_create(cvs_context* ctx, int layers, int64_t pages, int page_tokens, int kv_heads, int head_dim,
                        int type, cvs_kv_cache** out_cache) {
  return guarded([&] {
    bind(ctx);
    need(out_cache, "out_cache");
    *out_cache = nullptr;
    if (type != CVS_FP16 && type != CVS_BF16) fail(CVS_ERR_UNSUPPORTED, "a cache holds fp16 or bf16");
    if (layers < 1 || pages < 1 || kv_heads < 1)
      fail(CVS_ERR_INVALID_ARGUMENT, "a cache needs at least one layer, page and kv head");
    if (layers > 65535 || kv_heads > 65535 || pages > (int64_t(1) << 30))
      fail(CVS_ERR_UNSUPPORTED, "too many layers, pages or heads");
    if (page_tokens < 32 || page_tokens > 4096 || (page_tokens & (page_tokens - 1)) != 0)
      fail(CVS_ERR_UNSUPPORTED, "page_tokens must be a power of two from 32 to 4096");
    if (head_dim < 8 || head_dim % 8 != 0 || head_dim > kMaxDim)
      fail(CVS_ERR_UNSUPPORTED, "head_dim must be a multiple of 8 from 8 to " + std::to_string(kMaxDim));
    auto c = std::make_unique<cvs_kv_cache>();
    c->ctx = ctx;
    c->layers = layers;
    c->kv_heads = kv_heads;
    c->dim = head_dim;
    c->type = type;
    c->nb = (head_dim + 31) / 32;
    c->head_bytes = int64_t(2) * page_tokens * 64 * c->nb;
    c->page_bytes = c->head_bytes * kv_heads;
    if (c->page_bytes > (int64_t(1) << 29)) fail(CVS_ERR_UNSUPPORTED, "a page of a layer must not exceed 512 MiB");
    c->layer_bytes = c->page_bytes * pages;
    if (c->layer_bytes > (int64_t(1) << 50) / layers) fail(CVS_ERR_OUT_OF_MEMORY, "the pages exceed the memory");
    c->book = std::make_unique<kv::PageBook>(pages, page_tokens);
    CVS_HIP(hipMalloc(reinterpret_cast<void**>(&c->pool), size_t(c->layer_bytes) * size_t(layers)));
    ++ctx->live_children;
    *out_cache = c.release();
  });
}

int cvs_kv_cache_destroy(cvs_kv_cache* cache) {
  return guarded([&] {
    if (!cache) return;
    if (cache->live_plans > 0)
      fail(CVS_ERR_INVALID_ARGUMENT, "cache still has " + std::to_string(cache->live_plans) +
                                         " plan(s): destroy them first");
    bind(cache->ctx);
    (void)hipStreamSynchronize(cache->ctx->stream);
    for (auto& b : cache->blobs) b.release();
    for (auto& b : cache->kept) b.release();
    (void)hipFree(cache->pool);
    --cache->ctx->live_children;
    delete cache;
  });
}

int cvs_kv_cache_pages(cvs_kv_cache* cache, int64_t* out_pages, int64_t* out_free) {
  return on_book(cache, [&] {
    if (out_pages) *out_pages = cache->book->pages();
    if (out_free) *out_free = cache->book->free_pages();
  });
}

int cvs_kv_sequence_create(cvs_kv_cache* cache, int64_t n, int64_t* out_seqs) {
  return on_book(cache, [&] {
    need_list(out_seqs, n, "sequences");
    for (int64_t i = 0; i < n; ++i) out_seqs[i] = cache->book->create();
  });
}

int cvs_kv_sequence_fork(cvs_kv_cache* cache, int64_t parent, int64_t length, int64_t n, int64_t* out_seqs) {
  return on_book(cache, [&] {
    need_list(out_seqs, n, "sequences");
    const int64_t len = length < 0 ? cache->book->at(parent).length : length;
    for (int64_t i = 0; i < n; ++i) out_seqs[i] = cache->book->fork(parent, len);
  });
}

int cvs_kv_sequence_extend(cvs_kv_cache* cache, const int64_t* seqs, const int64_t* tokens, int64_t n) {
  return on_book(cache, [&] {
    need_list(seqs, n, "sequences");
    need_list(tokens, n, "tokens");
    bind(cache->ctx);
    need_no_capture(cache->ctx, "sequences cannot be extended");
    copy_pages(cache, cache->book->extend(seqs, tokens, n));
  });
}

int cvs_kv_sequence_truncate(cvs_kv_cache* cache, int64_t seq, int64_t length) {
  return on_book(cache, [&] { cache->book->truncate(seq, length); });
}

int cvs_kv_sequence_free(cvs_kv_cache* cache, const int64_t* seqs, int64_t n) {
  return on_book(cache, [&] {
    need_list(seqs, n, "sequences");
    cache->book->release(seqs, n);
  });
}

int cvs_kv_sequence_pages(cvs_kv_cache* cache, const int64_t* seqs, int64_t n, int64_t* out_lengths,
                          uint32_t* out_pages, int64_t room, int64_t* out_count) {
  return on_book(cache, [&] {
    need_list(seqs, n, "sequences");
    int64_t total = 0;
    for (int64_t i = 0; i < n; ++i) {
      const kv::Sequence& s = cache->book->at(seqs[i]);
      if (out_lengths) out_lengths[i] = s.length;
      for (const int32_t pg : s.pages) {
        if (out_pages && total < room) out_pages[total] = uint32_t(pg);
        ++total;
      }
    }
    if (out_count) *out_count = total;
    if (out_pages && total > room) fail(CVS_ERR_INVALID_ARGUMENT, "room for fewer pages than the sequences have");
  });
}

int cvs_kv_cache_compact(cvs_kv_cache* cache, int64_t* out_live) {
  return on_book(cache, [&] {
    bind(cache->ctx);
    need_no_capture(cache->ctx, "a cache cannot be compacted");
    copy_pages(cache, cache->book->compact());
    if (out_live) *out_live = cache->book->pages() - cache->book->free_pages();
  });
}

int cvs_kv_plan_create(cvs_kv_cache* cache, const int64_t* seqs, const int64_t* tokens, int64_t n, int heads,
                       cvs_kv_plan** out_plan) {
  return on_book(cache, [&] {
    need(out_plan, "out_plan");
    *out_plan = nullptr;
    need_list(seqs, n, "sequences");
    need_list(tokens, n, "tokens");
    if (heads < 0 || heads % cache->kv_heads != 0)
      fail(CVS_ERR_INVALID_ARGUMENT, "heads must be a multiple of the cache's kv heads (0: no attention)");
    bind(cache->ctx);
    kv::PageBook& book = *cache->book;
    const std::vector<kv::Sequence*> found = book.find(seqs, n);
    auto plan = std::make_unique<cvs_kv_plan>();
    plan->cache = cache;
    plan->heads = heads;
    std::vector<int64_t> lengths;
    auto& spans = plan->spans;
    const int64_t pt = book.page_tokens();
    for (int64_t i = 0; i < n; ++i) {
      const kv::Sequence& s = *found[size_t(i)];
      if (tokens[i] < 0 || tokens[i] > s.length)
        fail(CVS_ERR_INVALID_ARGUMENT, "sequence " + std::to_string(seqs[i]) + " has " + std::to_string(s.length) +
                                           " tokens, the plan asks for " + std::to_string(tokens[i]));
      if (plan->tokens + tokens[i] > kv::PageBook::kMaxTokens) fail(CVS_ERR_UNSUPPORTED, "tokens must fit 31 bits");
      plan->seqs.push_back(seqs[i]);
      plan->versions.push_back(s.version);
      lengths.push_back(s.length);
      for (int64_t t = s.length - tokens[i]; t < s.length;) {
        const int64_t in = t % pt, end = std::min(pt, in + s.length - t);
        const int32_t pg = s.pages[size_t(t / pt)];
        spans.push_back({pg, int32_t(in), int32_t(end), int32_t(plan->tokens)});
        plan->tokens += end - in;
        t += end - in;
      }
    }
    std::vector<char> blob;
    if (spans.size() > size_t(kInlineSpans)) {
      blob.resize(spans.size() * sizeof(Span));
      std::memcpy(blob.data(), spans.data(), blob.size());
    }
    if (heads > 0) plan_attention(plan.get(), lengths.data(), tokens, blob);
    if (!blob.empty()) {
      need_no_capture(cache->ctx, "plans cannot be made");
      plan->blob = take_blob(cache->blobs, cache->live_plans, blob.size());
      try {
        upload(cache->ctx, plan->blob.ptr, blob.data(), blob.size());
      } catch (...) {
        cache->blobs.push_back(plan->blob);
        throw;
      }
    }
    ++cache->live_plans;
    *out_plan = plan.release();
  });
}

int cvs_kv_plan_destroy(cvs_kv_plan* plan) {
  return guarded([&] {
    if (!plan) return;
    // Later plans use the memory on the same stream, after whatever still reads it.
    if (plan->blob.ptr && !plan->captured) plan->cache->blobs.push_back(plan->blob);
    --plan->cache->live_plans;
    delete plan;
  });
}

int cvs_kv_write_async(cvs_kv_cache* cache, cvs_kv_plan* plan, int first_layer, int layers, const cvs_heads* k,
                       int64_t k_layer_stride, const cvs_heads* v, int64_t v_layer_stride) {
  return on_book(cache, [&] {
    need(plan, "plan");
    if (plan->cache != cache) fail(CVS_ERR_INVALID_ARGUMENT, "the plan belongs to another cache");
    bind(cache->ctx);
    move_tokens(plan, first_layer, layers, k, k_layer_stride, v, v_layer_stride, true);
  });
}

int cvs_kv_read_async(cvs_kv_cache* cache, cvs_kv_plan* plan, int first_layer, int layers, const cvs_heads* k,
                      int64_t k_layer_stride, const cvs_heads* v, int64_t v_layer_stride) {
  return on_book(cache, [&] {
    need(plan, "plan");
    if (plan->cache != cache) fail(CVS_ERR_INVALID_ARGUMENT, "the plan belongs to another cache");
    bind(cache->ctx);
    move_tokens(plan, first_layer, layers, k, k_layer_stride, v, v_layer_stride, false);
  });
}

}  // extern "C"
