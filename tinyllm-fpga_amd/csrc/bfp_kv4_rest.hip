// Attention over a prefix that a group of sequences shares: the kernels of the
// second part, every sequence's tokens behind the prefix.
#include "bfp_kv4_prompt.h"
#include "bfp_kv4_rows.h"

namespace bfp {

AttnKernel rest_rows_kernel(int tiles, int terms, int waves, bool share) {
  return rows_kernel_for<SEES_REST>(tiles, terms, waves, share);
}
AttnKernel rest_prompt_kernel(int tiles, int terms) { return prompt_kernel_for<SEES_REST>(tiles, terms); }

}  // namespace bfp
