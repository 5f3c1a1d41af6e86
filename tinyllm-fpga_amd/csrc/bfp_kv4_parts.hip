// Attention over a prefix that a group of sequences shares: both parts of few
// rows in one launch (bfp_kv4_rows.h).
#include "bfp_kv4_rows.h"

namespace bfp {

PartsKernel parts_kernel(int tiles, int terms, int waves) {
  const int C = (tiles + 3) / 4;
  if (C == 1) return waves == 4 ? parts_kernel_of<1, 4>(tiles, terms) : parts_kernel_of<1, 16>(tiles, terms);
  if (C == 2) return waves == 4 ? parts_kernel_of<2, 4>(tiles, terms) : parts_kernel_of<2, 8>(tiles, terms);
  return C == 3 ? parts_kernel_of<3, 4>(tiles, terms) : parts_kernel_of<4, 4>(tiles, terms);
}

}  // namespace bfp
