// The rotation of a pair, for the kernels that turn heads.
#pragma once
#include <hip/hip_runtime.h>

namespace bfp {

__device__ __forceinline__ double2 rope_cs(float2 t) { return make_double2((double)t.x, (double)t.y); }

// y_a = a c - b s, y_b = b c + a s.  In float64: a product of a value and a
// float32 angle has at most 48 bits and is exact, so each result is rounded
// once, in the sum.  A rounding in float32 would move keys that lie next to a
// border between two 4-bit elements.
__device__ __forceinline__ void rope_pair(float a, float b, double2 cs, double &ya, double &yb) {
  ya = fma((double)a, cs.x, -((double)b * cs.y));
  yb = fma((double)b, cs.x, (double)a * cs.y);
}

}  // namespace bfp
