// The rotation of a pair, for the kernels that turn heads.
#pragma once
#include <hip/hip_runtime.h>

#include "bfp_rows.h"

namespace bfp {

// How the heads of rows are cut into units of work, for 16-byte accesses
// (`wide`: 8 pairs, that is two groups of 8 values, of the half layout, 4 of the
// interleaved one, or 8 values to copy) or value by value (a pair, or a value
// to copy): rows of any width, stride and alignment.
struct RopeShape {
  int half, interleaved, wide, turned, per_head;   // units that are turned, and all of them
};
inline RopeShape rope_shape(const bfp_rows &x, const bfp_rows &y, long long n_rows, int hd, int rot, int interleaved) {
  RopeShape s;
  s.half = rot / 2;
  s.interleaved = interleaved ? 1 : 0;
  s.wide = rows_aligned(x, 8, n_rows) && rows_aligned(y, 8, n_rows) && hd % 8 == 0 && (interleaved ? rot % 8 == 0 : s.half % 8 == 0);
  s.turned = s.wide ? (interleaved ? rot / 8 : s.half / 8) : s.half;
  s.per_head = s.turned + (s.wide ? (hd - rot) / 8 : hd - rot);
  return s;
}
// Heads a thread takes, one after the other, of wide units: their angles are
// the same, and their loads are under way together.  A call of few units is
// spread over more threads instead.  (5000 rows of 32 heads: 20.9 us with two
// heads a thread, 24.4 with four, 26 with one.)
constexpr int ROPE_HEADS = 2;

__device__ __forceinline__ double2 rope_cs(float2 t) { return make_double2((double)t.x, (double)t.y); }

// y_a = a c - b s, y_b = b c + a s.  In float64: a product of a value and a
// float32 angle has at most 48 bits and is exact, so each result is rounded
// once, in the sum.  A rounding in float32 would move keys that lie next to a
// border between two 4-bit elements.
__device__ __forceinline__ void rope_pair(float a, float b, double2 cs, double &ya, double &yb) {
  ya = fma((double)a, cs.x, -((double)b * cs.y));
  yb = fma((double)b, cs.x, (double)a * cs.y);
}

// The same in float32 for 16-bit results: b s is rounded to w, and the
// rounding error fma(b, s, -w), which is exact, taken off again (Kahan's
// difference of products): at most 1.5 float32 steps of the result off,
// also where the products cancel, far below a 16-bit step (5000 rows of 32
// heads, half of each turned: 24.4 us with float64, 20.9 so).  NaN where a
// product overflows.
__device__ __forceinline__ float diff_of_products(float a, float c, float b, float s) {
  const float w = b * s, e = fmaf(b, s, -w);
  return fmaf(a, c, -w) - e;
}
template <int M>
__device__ __forceinline__ void rope_pairs(const float *a, const float *b, int step, const float2 (&cs)[M], float *ya, float *yb) {
  bool bad = false;
#pragma unroll
  for (int i = 0; i < M; ++i) {
    ya[i * step] = diff_of_products(a[i * step], cs[i].x, b[i * step], cs[i].y);
    yb[i * step] = diff_of_products(b[i * step], cs[i].x, -a[i * step], cs[i].y);
    bad |= ya[i * step] != ya[i * step] || yb[i * step] != yb[i * step];
  }
  if (bad) {   // NaNs and infinities, and values near float32's end
#pragma unroll
    for (int i = 0; i < M; ++i) {
      double da, db;
      rope_pair(a[i * step], b[i * step], rope_cs(cs[i]), da, db);
      ya[i * step] = f64_to_f32_sticky(da);
      yb[i * step] = f64_to_f32_sticky(db);
    }
  }
}

// Unit j of head h of row t.  cs: the row's angles (null: it has none, NaN).
__device__ __forceinline__ void rope_unit(const RopeShape &s, const bfp_rows &x, const bfp_rows &y, long long t, int h,
                                          int j, const float2 *cs) {
  const long long xo = t * x.row_stride + h * x.head_stride, yo = t * y.row_stride + h * y.head_stride;
  if (j >= s.turned) {
    const int d = j + s.half;
    row_store(y, yo + d, row_load(x, xo + d));
    return;
  }
  const int da = s.interleaved ? 2 * j : j, db = s.interleaved ? 2 * j + 1 : j + s.half;
  double ya, yb;
  rope_pair(row_load(x, xo + da), row_load(x, xo + db), cs ? rope_cs(cs[j]) : make_double2(NAN, NAN), ya, yb);
  row_store(y, yo + da, ya);
  row_store(y, yo + db, yb);
}

// Wide unit j of heads h0 .. h0 + N - 1 (those below `heads`) of row t.
template <int N>
__device__ __forceinline__ void rope_wide_unit(const RopeShape &s, const bfp_rows &x, const bfp_rows &y, long long t,
                                               int h0, int heads, int j, const float2 *cs) {
  const bool turn = j < s.turned;
  const int da = turn ? 8 * j : 2 * s.half + (j - s.turned) * 8, db = da + s.half;
  const bool two = turn && !s.interleaved;
  float va[N][8], vb[N][8];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int h = h0 + n < heads ? h0 + n : heads - 1;
    row_load_n(x, t * x.row_stride + h * x.head_stride + da, va[n]);
    if (two) row_load_n(x, t * x.row_stride + h * x.head_stride + db, vb[n]);
  }
  if (!turn) {
#pragma unroll
    for (int n = 0; n < N; ++n)
      if (h0 + n < heads) row_store_n(y, t * y.row_stride + (h0 + n) * y.head_stride + da, va[n]);
    return;
  }
  if (two) {
    float2 c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = cs ? cs[8 * j + i] : make_float2(NAN, NAN);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (h0 + n >= heads) break;
      const long long yo = t * y.row_stride + (h0 + n) * y.head_stride;
      if (y.type == BFP_F32) {
        double ya[8], yb[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) rope_pair(va[n][i], vb[n][i], rope_cs(c[i]), ya[i], yb[i]);
        row_store_n(y, yo + da, ya);
        row_store_n(y, yo + db, yb);
      } else {
        float ya[8], yb[8];
        rope_pairs<8>(va[n], vb[n], 1, c, ya, yb);
        row_store_n(y, yo + da, ya);
        row_store_n(y, yo + db, yb);
      }
    }
  } else {
    float2 c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = cs ? cs[4 * j + i] : make_float2(NAN, NAN);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (h0 + n >= heads) break;
      const long long yo = t * y.row_stride + (h0 + n) * y.head_stride;
      if (y.type == BFP_F32) {
        double ya[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) rope_pair(va[n][2 * i], va[n][2 * i + 1], rope_cs(c[i]), ya[2 * i], ya[2 * i + 1]);
        row_store_n(y, yo + da, ya);
      } else {
        float ya[8];
        rope_pairs<4>(va[n], va[n] + 1, 2, c, ya, ya + 1);
        row_store_n(y, yo + da, ya);
      }
    }
  }
}

}  // namespace bfp
