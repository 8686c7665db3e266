// Attention over packed sequences with capped scores, a bias by distance, or
// both: the kernels of attn_prompt.hpp.
//
// Bounds: the vector unit.  8,000 causal tokens behind a prefix of 6,000, 32/8
// heads of 128, bf16: 954 us with a cap of 50 (the vector unit busy 63% of the
// cycles, the matrix cores 44%), 776 us biased, 918 us with both, 777 us plain, all
// in one session; 64 passages of 40 to 512 tokens, 12 heads of 64, fp16, in both
// directions: 49, 51, 55 and 40 us.  Scores beyond half of the cap take a second
// pass: 1.24 ms for a cap of 10 and 1.59 ms for one of 1 in the first case.
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
