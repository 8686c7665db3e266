// Attention over a paged cache with capped scores, a bias by distance, or both: the kernels of attn_cached.hpp.
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
