// Rows of values in one of the types of bfp_rows (include/bfp.h): host
// checks, device loads and stores, and the division the kernels find their
// row and head with.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "bfp.h"
#include "bfp_internal.h"

namespace bfp {

// n / d for 0 <= n < 2^31 by a multiplication: sh = ceil(log2 d), mul =
// ceil(2^(31+sh) / d) < 2^32 (2^sh < 2 d), and n mul / 2^(31+sh) exceeds n / d
// by less than n / 2^(31+sh) <= 1/d, too little to reach the next whole
// number.
struct FastDiv {
  uint32_t mul = 0, d = 1;
  int sh = 0;
  FastDiv() = default;
  explicit FastDiv(uint32_t div) : d(div) {
    while ((1ull << sh) < div) ++sh;
    mul = (uint32_t)(((1ull << (31 + sh)) + div - 1) / div);
  }
  __host__ __device__ uint32_t div(uint32_t n) const {
    return (uint32_t)(((uint64_t)n * mul) >> (31 + sh));
  }
  __host__ __device__ uint32_t div(uint32_t n, uint32_t &rem) const {
    const uint32_t q = div(n);
    rem = n - q * d;
    return q;
  }
};

// The checks every operator makes of a bfp_rows; what: its name in messages.
inline int check_rows(const char *op, const char *what, const bfp_rows *r, int heads, int hd,
                      bool tiles, long long n_rows) {
  if (!r || !r->p) return set_err(BFP_EINVAL, "%s: %s is null", op, what);
  if (r->type < BFP_F32 || r->type > BFP_TILES)
    return set_err(BFP_EINVAL, "%s: %s has no such type (%d)", op, what, r->type);
  if (r->type == BFP_TILES && (!tiles || !r->e))
    return set_err(BFP_EINVAL, "%s: %s %s", op, what, tiles ? "has no exponents" : "cannot be tiles");
  if (r->heads != heads)
    return set_err(BFP_EINVAL, "%s: %s has %d heads, not %d", op, what, r->heads, heads);
  if (r->row_stride < 0 || r->head_stride < 0)
    return set_err(BFP_EINVAL, "%s: %s has a negative stride", op, what);
  if (r->head_stride < hd && heads > 1)
    return set_err(BFP_EINVAL, "%s: heads of %s overlap (stride %lld, hd %d)", op, what, r->head_stride, hd);
  if (r->type == BFP_TILES && (hd % 16 || (n_rows > 1 && r->row_stride % 16) || (heads > 1 && r->head_stride % 16)))
    return set_err(BFP_EINVAL, "%s: tiles of %s need hd and strides in multiples of 16", op, what);
  const int size = r->type == BFP_F32 ? 4 : 2;
  if ((uintptr_t)r->p % size) return set_err(BFP_EINVAL, "%s: %s is not aligned to its type", op, what);
  // offsets are 64-bit; the last one still has to fit
  const long long last = n_rows > 0 ? n_rows - 1 : 0;
  if ((r->row_stride > 0 && last > (1LL << 60) / r->row_stride) ||
      (r->head_stride > 0 && heads - 1 > (1LL << 60) / r->head_stride))
    return set_err(BFP_EINVAL, "%s: %s is too large", op, what);
  return BFP_OK;
}

// Whether two of n_rows x heads groups of hd values share a value: groups
// (t, h) and (t', h') do where |(t - t') row_stride + (h - h') head_stride| < hd.
// One dimension inside the other never does; strides between are looked at
// difference by difference, of the dimension that has fewer.
inline bool rows_share(long long row_stride, long long head_stride, long long n_rows, long long heads, long long hd) {
  long long s = row_stride, n = n_rows, t = head_stride, m = heads;
  if (n <= 1 || m <= 1) return n > 1 ? s < hd : m > 1 && t < hd;
  if (s < hd || t < hd) return true;
  if (s >= (m - 1) * t + hd || t >= (n - 1) * s + hd) return false;
  if (m > n) {
    const long long a = s, b = n;
    s = t, n = m, t = a, m = b;
  }
  for (long long j = 1; j < m; ++j) {   // j steps of t against the two nearest numbers of steps of s
    const long long i = j * t / s, rest = j * t - i * s;
    if ((i < n && rest < hd) || (i + 1 < n && s - rest < hd)) return true;
  }
  return false;
}

// The same for rows that are written: no two of them may share a value.
inline int check_out(const char *op, const char *what, const bfp_rows *r, int heads, int hd,
                     bool tiles, long long n_rows) {
  BFP_TRY(check_rows(op, what, r, heads, hd, tiles, n_rows));
  if (rows_share(r->row_stride, r->head_stride, n_rows, heads, hd))
    return set_err(BFP_EINVAL, "%s: rows of %s overlap (strides %lld and %lld, %d heads of %d)", op, what, r->row_stride,
                   r->head_stride, heads, hd);
  return BFP_OK;
}

// Rows in bytes: n rows s apart of m heads t apart, each w bytes from p on
// (0 apart where there is one).
struct RowPlaces {
  long long p, s, t, n, m, w;
};
inline RowPlaces row_places(const bfp_rows &r, long long n_rows, int hd, bool exponents) {
  const long long size = r.type == BFP_F32 ? 4 : 2, s = n_rows > 1 ? r.row_stride : 0, t = r.heads > 1 ? r.head_stride : 0;
  if (exponents) return {(long long)(uintptr_t)r.e, s / 16, t / 16, n_rows, r.heads, hd / 16};
  return {(long long)(uintptr_t)r.p, s * size, t * size, n_rows, r.heads, hd * size};
}
inline bool same_places(const RowPlaces &a, const RowPlaces &b) {
  return a.p == b.p && a.m == b.m && a.w == b.w && a.s == b.s && a.t == b.t;
}

// Whether a byte lies in both.  Exact where the rows are equally far apart,
// as in joined rows (and the heads, or there are few): a head of one against
// a head of the other is then a question of their distance modulo the rows'.
// Rows of another stride in the same memory count as sharing some.
inline bool places_share(const RowPlaces &a, const RowPlaces &b) {
  typedef __int128 wide;
  const auto row = [](const RowPlaces &r) { return (wide)(r.m - 1) * r.t + r.w; };
  const auto end = [&](const RowPlaces &r) { return (wide)r.p + (wide)(r.n - 1) * r.s + row(r); };
  if (end(a) <= b.p || end(b) <= a.p) return false;
  if (a.n > 1 && a.s != b.s) return true;
  const long long s = a.s, most = a.n - 1;
  if (s > 0) {   // b's rows in the gaps between a's: joined rows, without the search
    const long long gap = (b.p - a.p) % s, at = gap < 0 ? gap + s : gap;
    if (at >= row(a) && at + row(b) <= s) return false;
  }
  const auto meet = [&](wide d) {   // b's bytes d behind a's, in any two rows: -b.w < d + k s < a.w, |k| <= most
    if (most == 0 || s == 0) return -b.w < d && d < a.w;
    const wide x = -b.w - d;
    wide k = x / s - (x % s < 0 ? 1 : 0) + 1;   // the least with k s > x
    k = k < -most ? -most : k;
    return k <= most && k * s + d < a.w;
  };
  const wide d = (wide)b.p - a.p;
  if (a.m == 1 || b.m == 1 || a.t == b.t) {
    const long long t = a.m == 1 ? b.t : a.t;
    for (long long j = 1 - a.m; j < b.m; ++j)
      if (meet(d + (wide)j * t)) return true;
    return false;
  }
  if (a.m * b.m > 65536) return true;
  for (long long i = 0; i < a.m; ++i)
    for (long long j = 0; j < b.m; ++j)
      if (meet(d + (wide)j * b.t - (wide)i * a.t)) return true;
  return false;
}

// Results may lie on operands where each value takes its own operand's place
// (in_place), or nowhere near them.
inline int check_apart(const char *op, const char *what, const bfp_rows &y, const char *other, const bfp_rows &x,
                       long long n_rows, int hd, bool in_place) {
  if (n_rows <= 0) return BFP_OK;
  for (int i = 0; i < 4; ++i) {
    const bool ye = i & 1, xe = i & 2;
    if ((ye && y.type != BFP_TILES) || (xe && x.type != BFP_TILES)) continue;
    const RowPlaces a = row_places(y, n_rows, hd, ye), b = row_places(x, n_rows, hd, xe);
    if (in_place && ye == xe && same_places(a, b)) continue;
    if (places_share(a, b))
      return set_err(BFP_EINVAL, "%s: %s lies on %s%s", op, what, other, in_place ? ", but not in its place" : "");
  }
  return BFP_OK;
}

// Whether groups of n values (n values a multiple of 16 bytes) that start at
// multiples of n in a head can be moved with 16-byte accesses.  The stride of
// a single row or head is not used, and may be anything.
inline bool rows_aligned(const bfp_rows &r, int n, long long n_rows) {
  return (uintptr_t)r.p % 16 == 0 && (n_rows <= 1 || r.row_stride % n == 0) && (r.heads <= 1 || r.head_stride % n == 0);
}

__device__ __forceinline__ float bf16_to_f32(uint32_t b) { return __uint_as_float(b << 16); }
// Round to nearest even; NaN stays NaN.
__device__ __forceinline__ uint16_t f32_to_bf16(float f) {
  const __bf16 b = (__bf16)f;
  return __builtin_bit_cast(uint16_t, b);
}
__device__ __forceinline__ float f16_to_f32(uint32_t b) {
  return (float)__builtin_bit_cast(_Float16, (uint16_t)b);
}
__device__ __forceinline__ uint16_t f32_to_f16(float f) {
  const _Float16 h = (_Float16)f;
  return __builtin_bit_cast(uint16_t, h);
}
// float64 to 16 bits with one rounding: float32 first, toward zero with the
// lost bits gathered in the last one (so that no value moves onto a point
// halfway between two 16-bit numbers), then to nearest.
__device__ __forceinline__ float f64_to_f32_sticky(double d) {
  const float f = (float)d;
  const double back = (double)f;
  uint32_t b = __float_as_uint(f);
  if (fabs(back) > fabs(d)) --b;      // also from infinity to the largest float
  if (back != d && d == d) b |= 1u;
  return __uint_as_float(b);
}

// A tile's values are m 2^(e-15): exact in float32 (|m| <= 2^15, e >= -128).
__device__ __forceinline__ float tile_value(int m, int e) { return ldexpf((float)m, e - 15); }

// One value.
__device__ __forceinline__ float row_load(const bfp_rows &r, long long o) {
  switch (r.type) {
    case BFP_F32: return ((const float *)r.p)[o];
    case BFP_BF16: return bf16_to_f32(((const uint16_t *)r.p)[o]);
    case BFP_F16: return f16_to_f32(((const uint16_t *)r.p)[o]);
    default: return tile_value(((const int16_t *)r.p)[o], r.e[o >> 4]);
  }
}

// N values (8 or 16) from a 16-byte-aligned offset; all lie in one tile.
template <int N>
__device__ __forceinline__ void row_load_n(const bfp_rows &r, long long o, float (&v)[N]) {
  static_assert(N == 8 || N == 16, "");
  if (r.type == BFP_F32) {
    const float4 *p = (const float4 *)((const float *)r.p + o);
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const float4 x = p[i];
      v[4 * i] = x.x, v[4 * i + 1] = x.y, v[4 * i + 2] = x.z, v[4 * i + 3] = x.w;
    }
    return;
  }
  const uint4 *p = (const uint4 *)((const uint16_t *)r.p + o);
  uint32_t w[N / 2];
#pragma unroll
  for (int i = 0; i < N / 8; ++i) {
    const uint4 x = p[i];
    w[4 * i] = x.x, w[4 * i + 1] = x.y, w[4 * i + 2] = x.z, w[4 * i + 3] = x.w;
  }
  if (r.type == BFP_BF16) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else if (r.type == BFP_F16) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      v[2 * i] = f16_to_f32(w[i] & 0xffffu);
      v[2 * i + 1] = f16_to_f32(w[i] >> 16);
    }
  } else {
    const int e = r.e[o >> 4];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      v[2 * i] = tile_value((int16_t)(w[i] & 0xffffu), e);
      v[2 * i + 1] = tile_value((int16_t)(w[i] >> 16), e);
    }
  }
}

// One value out (never tiles).
__device__ __forceinline__ void row_store(const bfp_rows &r, long long o, float v) {
  switch (r.type) {
    case BFP_F32: ((float *)r.p)[o] = v; break;
    case BFP_BF16: ((uint16_t *)r.p)[o] = f32_to_bf16(v); break;
    default: ((uint16_t *)r.p)[o] = f32_to_f16(v); break;
  }
}
__device__ __forceinline__ void row_store(const bfp_rows &r, long long o, double v) {
  row_store(r, o, r.type == BFP_F32 ? (float)v : f64_to_f32_sticky(v));
}

// Non-temporal stores, for results that pass the caches once: 5000 rows of
// joined q, k and v appended 43 -> 37 us.  (Loads that way were slower: rope
// of 5000 rows 27 -> 31 us.)
__device__ __forceinline__ void st_nt(uint4 *p, uint4 v) {
  typedef unsigned u4 __attribute__((ext_vector_type(4)));
  __builtin_nontemporal_store(u4{v.x, v.y, v.z, v.w}, (u4 *)p);
}
__device__ __forceinline__ void st_nt(float4 *p, float4 v) {
  typedef float f4 __attribute__((ext_vector_type(4)));
  __builtin_nontemporal_store(f4{v.x, v.y, v.z, v.w}, (f4 *)p);
}
// N values out to a 16-byte-aligned offset.
template <int N, typename F>
__device__ __forceinline__ void row_store_n(const bfp_rows &r, long long o, const F (&v)[N]) {
  static_assert(N == 8 || N == 16, "");
  if (r.type == BFP_F32) {
    float4 *p = (float4 *)((float *)r.p + o);
#pragma unroll
    for (int i = 0; i < N / 4; ++i)
      st_nt(p + i, make_float4((float)v[4 * i], (float)v[4 * i + 1], (float)v[4 * i + 2], (float)v[4 * i + 3]));
    return;
  }
  uint32_t w[N / 2];
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    float a, b;
    if constexpr (sizeof(F) == 8)
      a = f64_to_f32_sticky(v[2 * i]), b = f64_to_f32_sticky(v[2 * i + 1]);
    else
      a = v[2 * i], b = v[2 * i + 1];
    w[i] = r.type == BFP_BF16 ? (uint32_t)f32_to_bf16(a) | ((uint32_t)f32_to_bf16(b) << 16)
                              : (uint32_t)f32_to_f16(a) | ((uint32_t)f32_to_f16(b) << 16);
  }
  uint4 *p = (uint4 *)((uint16_t *)r.p + o);
#pragma unroll
  for (int i = 0; i < N / 8; ++i) st_nt(p + i, make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]));
}

}  // namespace bfp
