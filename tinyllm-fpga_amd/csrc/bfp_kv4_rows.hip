// Attention over the 4-bit cache for few rows to a KV head (bfp_kv4_rows.h).
#include "bfp_kv4_rows.h"

namespace bfp {

AttnKernel rows_kernel(int tiles, int terms, int waves) { return rows_kernel_for<SEES_ALL>(tiles, terms, waves, true); }

}  // namespace bfp
