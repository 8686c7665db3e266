// Attention over a paged cache with capped scores, a bias by distance, or both:
// the kernels of attn_cached.hpp.
//
// Bounds: the memory, as with plain scores: 48 sequences of 100 to 6,000 tokens,
// 32/8 heads of 128, bf16, cap 30, 104 us = 6.2 TB/s (plain 103).  One sequence of
// 777 tokens, 16/4 heads of 64, biased: 7.6 us, latency.  64 sequences over 8,000
// shared tokens, a token each: 22.5 us capped, 22.2 biased, 26.4 both (plain 21.7),
// latency; 8 of 40 new tokens over 8,000: 71, 62, 75 and 62 us, the vector unit busy
// 40% of the cycles with a cap, the matrix cores 25%.
#include "attn_cached.hpp"

namespace cvs {
namespace attn {

void launch_cached_scored(cvs_context* ctx, const CachedArgs& a, int nb, int64_t blocks, int type) {
  auto go = [&](auto scoring) {
    typedef decltype(scoring) S;
    if (type == CVS_BF16) launch_cached<true, typename S::type>(ctx, a, nb, blocks);
    else launch_cached<false, typename S::type>(ctx, a, nb, blocks);
  };
  pick_scores(a.scores, go);
}

}  // namespace attn
}  // namespace cvs
