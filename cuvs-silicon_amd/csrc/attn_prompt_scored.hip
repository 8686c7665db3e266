// Attention over packed sequences with capped scores, a bias by distance, or both: the kernels of attn_prompt.hpp.
#include "attn_prompt.hpp"

namespace cvs {
namespace attn {

void launch_prompt_scored(cvs_context* ctx, const PromptArgs& a, int64_t blocks, int type) {
  auto go = [&](auto scoring) {
    typedef decltype(scoring) S;
    if (type == CVS_BF16) launch_prompt<true, typename S::type>(ctx, a, blocks);
    else launch_prompt<false, typename S::type>(ctx, a, blocks);
  };
  pick_scores(a.scores, go);
}

}  // namespace attn
}  // namespace cvs
