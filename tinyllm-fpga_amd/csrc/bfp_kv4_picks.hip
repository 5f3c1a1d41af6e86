// Attention over the 4-bit cache's listed pages, a list for every row and KV
// head (bfp_kv4_rows.h).
#include "bfp_kv4_rows.h"

namespace bfp {

AttnKernel picks_kernel(int tiles, int terms, int waves, bool share) {
  return rows_kernel_for<SEES_PICKS>(tiles, terms, waves, share);
}

}  // namespace bfp
