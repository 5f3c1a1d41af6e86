// Attention over a prefix that a group of sequences shares: the kernels of the
// first part, all rows of a group against the group's pages.
#include "bfp_kv4_prompt.h"
#include "bfp_kv4_rows.h"

namespace bfp {

AttnKernel prefix_rows_kernel(int tiles, int terms, int waves, bool share) {
  return rows_kernel_for<SEES_PREFIX>(tiles, terms, waves, share);
}
AttnKernel prefix_prompt_kernel(int tiles, int terms, bool pairs) {
  if (pairs)
    return tiles <= 2   ? prompt_kernel_of<2, 4, SEES_PREFIX>(terms)
           : tiles <= 4 ? prompt_kernel_of<4, 4, SEES_PREFIX>(terms)
           : tiles <= 6 ? prompt_kernel_of<6, 4, SEES_PREFIX>(terms)
                        : prompt_kernel_of<8, 4, SEES_PREFIX>(terms);
  return prompt_kernel_for<SEES_PREFIX>(tiles, terms);
}

}  // namespace bfp
