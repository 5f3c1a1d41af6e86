// Rotary positions beside rope_fp (rtl/vc707/host/gen_smollm_blockfp_full.py:
// 250-258): the angles of scaled contexts, and the rotation of rows of heads
// of any even width in either pairing.
#include <math.h>

#include "bfp.h"
#include "bfp_internal.h"
#include "bfp_rotary.h"
#include "bfp_rows.h"

namespace bfp {

constexpr int ROPE_BS = 256;
constexpr int ROPE_MAX_FREQ = 256;

// The frequencies ride in the launch's arguments (2 KB): a call needs no
// copy to the device and no buffer that outlives it.
struct RopeFreqs {
  double inv[ROPE_MAX_FREQ];
};

// sin and cos in float64 for results that are rounded to float32: x less k
// quarter turns (pi/2 in two parts: off by 2^-53 for k up to 2^31), then the
// power series at |r| <= pi/4, cut where its next term is below 2^-63 (sine)
// and 2^-58 (cosine), far below half a step of the float32 they become.  A
// third of the library's work, which also serves larger arguments: 131072
// positions of 64 frequencies 22.4 -> 18.6 us.
__device__ __forceinline__ void sin_cos(double x, double &s, double &c) {
  if (!(fabs(x) <= 0x1p31)) {   // frequencies above one
    sincos(x, &s, &c);
    return;
  }
  const double k = rint(x * 0x1.45f306dc9c883p-1);
  const double r = fma(-k, 0x1.1a62633145c07p-54, fma(-k, 0x1.921fb54442d18p+0, x)), z = r * r;
  constexpr double f[] = {1, 1, 2, 6, 24, 120, 720, 5040, 40320, 362880, 3628800, 39916800, 479001600, 6227020800.0,
                          87178291200.0, 1307674368000.0, 20922789888000.0, 355687428096000.0};   // n!
  double a = 1.0 / f[17], b = 1.0 / f[16];
#pragma unroll
  for (int n = 15; n >= 3; n -= 2) a = fma(-a, z, 1.0 / f[n]);
#pragma unroll
  for (int n = 14; n >= 2; n -= 2) b = fma(-b, z, 1.0 / f[n]);
  const double sr = fma(-a * z, r, r), cr = fma(-b, z, 1.0);
  const int q = (int)(long long)k & 3;
  s = q & 1 ? cr : sr;
  c = q & 1 ? sr : cr;
  s = q & 2 ? -s : s;
  c = (q + 1) & 2 ? -c : c;
}

// (cos, sin) of one position and frequency a thread.
__global__ __launch_bounds__(ROPE_BS) void k_rope_table(RopeFreqs f, FastDiv n_freq, double mscale,
                                                        long long first, uint32_t n,
                                                        float2 *__restrict__ table) {
  const uint32_t u = blockIdx.x * ROPE_BS + threadIdx.x;
  if (u >= n) return;
  uint32_t j;
  const uint32_t i = n_freq.div(u, j);
  double s, c;
  sin_cos((double)(first + i) * f.inv[j], s, c);
  table[u] = make_float2((float)(c * mscale), (float)(s * mscale));
}

struct RopeArgs {
  bfp_rows x, y;
  RopeShape shape;
  const int32_t *pos;
  const float2 *table;
  int n_pos, row0;
  FastDiv per_row, per_head;   // units of work of a row, of N heads
  uint32_t units;
};

// N = 0: value by value.
template <int N>
__global__ __launch_bounds__(ROPE_BS) void k_rope(RopeArgs a) {
  const uint32_t u = blockIdx.x * ROPE_BS + threadIdx.x;
  if (u >= a.units) return;
  uint32_t rest, j;
  const long long t = a.row0 + (long long)a.per_row.div(u, rest);
  const int h = (int)a.per_head.div(rest, j);
  const int p = a.pos[t];
  const float2 *cs = (unsigned)p < (unsigned)a.n_pos ? a.table + (long long)p * a.shape.half : nullptr;
  if constexpr (N == 0)
    rope_unit(a.shape, a.x, a.y, t, h, (int)j, cs);
  else
    rope_wide_unit<N>(a.shape, a.x, a.y, t, h * N, a.x.heads, (int)j, cs);
}

}  // namespace bfp

using namespace bfp;

extern "C" {

int bfp_rope_freqs(int rot, double base, int scaling, double factor, int orig_ctx,
                   double *inv_freq, double *mscale) {
  if (!inv_freq || !mscale) return set_err(BFP_EINVAL, "rope_freqs: null pointer");
  if (rot < 2 || rot % 2 || rot > 2 * ROPE_MAX_FREQ)
    return set_err(BFP_EINVAL, "rope_freqs: rot=%d must be even, 2..%d", rot, 2 * ROPE_MAX_FREQ);
  if (!(base > 1.0) || !isfinite(base)) return set_err(BFP_EINVAL, "rope_freqs: base=%g", base);
  if (scaling < BFP_ROPE_NONE || scaling > BFP_ROPE_BANDS)
    return set_err(BFP_EINVAL, "rope_freqs: no such scaling (%d)", scaling);
  if (scaling != BFP_ROPE_NONE && (!(factor >= 1.0) || !isfinite(factor)))
    return set_err(BFP_EINVAL, "rope_freqs: factor=%g must be at least 1", factor);
  if (scaling >= BFP_ROPE_PARTS && orig_ctx <= 0)
    return set_err(BFP_EINVAL, "rope_freqs: orig_ctx=%d", orig_ctx);
  if (scaling == BFP_ROPE_NTK && rot == 2)
    return set_err(BFP_EINVAL, "rope_freqs: this scaling needs more than one pair");
  const double turn = 2.0 * M_PI;
  if (scaling == BFP_ROPE_NTK) base *= pow(factor, (double)rot / (double)(rot - 2));
  // the pair (a real number) that turns `turns` times over orig_ctx
  auto pair_of = [&](double turns) {
    return rot * log((double)orig_ctx / (turns * turn)) / (2.0 * log(base));
  };
  double low = 0.0, high = 0.0;
  if (scaling == BFP_ROPE_PARTS) {
    low = fmax(floor(pair_of(32.0)), 0.0);
    high = fmin(ceil(pair_of(1.0)), rot - 1.0);
  }
  for (int j = 0; j < rot / 2; ++j) {
    const double w = pow(base, -(double)(2 * j) / (double)rot);
    double keep = 1.0;   // the share of the unscaled frequency
    if (scaling == BFP_ROPE_LINEAR) keep = 0.0;
    if (scaling == BFP_ROPE_PARTS)
      keep = 1.0 - fmin(fmax((j - low) / fmax(high - low, 0.001), 0.0), 1.0);
    if (scaling == BFP_ROPE_BANDS)
      keep = fmin(fmax(((double)orig_ctx * w / turn - 1.0) / (4.0 - 1.0), 0.0), 1.0);
    inv_freq[j] = keep == 1.0 ? w : keep == 0.0 ? w / factor : w * keep + w / factor * (1.0 - keep);
  }
  *mscale = scaling == BFP_ROPE_PARTS ? 0.1 * log(factor) + 1.0 : 1.0;
  return BFP_OK;
}

int bfp_rope_table_d(const double *inv_freq, int n_freq, double mscale, long long first, int n_pos,
                     float *table, void *stream) {
  if (!inv_freq || !table) return set_err(BFP_EINVAL, "rope_table: null pointer");
  if (n_freq < 1 || n_freq > ROPE_MAX_FREQ)
    return set_err(BFP_EINVAL, "rope_table: n_freq=%d must be in [1, %d]", n_freq, ROPE_MAX_FREQ);
  if (n_pos < 0 || first < 0 || first > (1LL << 31) - n_pos)
    return set_err(BFP_EINVAL, "rope_table: first=%lld, n_pos=%d", first, n_pos);
  if ((uintptr_t)table % 8) return set_err(BFP_EINVAL, "rope_table: table is not 8-byte aligned");
  RopeFreqs f;
  for (int j = 0; j < ROPE_MAX_FREQ; ++j) f.inv[j] = j < n_freq ? inv_freq[j] : 0.0;
  // launches of fewer than 2^31 pairs
  const int step = (int)(0x7fffff00LL / n_freq);
  for (int i = 0; i < n_pos; i += step) {
    const int rows = n_pos - i < step ? n_pos - i : step;
    const uint32_t n = (uint32_t)rows * (uint32_t)n_freq;
    hipLaunchKernelGGL(k_rope_table, dim3((n + ROPE_BS - 1) / ROPE_BS), dim3(ROPE_BS), 0,
                       (hipStream_t)stream, f, FastDiv(n_freq), mscale, first + i, n,
                       (float2 *)table + (long long)i * n_freq);
    BFP_TRY(launch_status("rope_table"));
    if (n_pos - i <= step) break;
  }
  return BFP_OK;
}

int bfp_rope_d(const bfp_rows *x, int n_rows, int hd, const int32_t *pos, const float *table,
               int n_pos, int rot, int interleaved, const bfp_rows *y, void *stream) {
  if (n_rows < 0 || hd < 2 || hd > (1 << 20))
    return set_err(BFP_EINVAL, "rope: n_rows=%d, hd=%d", n_rows, hd);
  if (!x || x->heads < 1 || x->heads > (1 << 20))
    return set_err(BFP_EINVAL, "rope: x %s", x ? "has no heads, or too many" : "is null");
  BFP_TRY(check_rows("rope", "x", x, x->heads, hd, true, n_rows));
  BFP_TRY(check_out("rope", "y", y, x->heads, hd, false, n_rows));
  BFP_TRY(check_apart("rope", "y", *y, "x", *x, n_rows, hd, true));   // who writes a value has read its pair
  if (rot < 2 || rot % 2 || rot > hd) return set_err(BFP_EINVAL, "rope: rot=%d, hd=%d", rot, hd);
  if (!pos || !table || n_pos < 1) return set_err(BFP_EINVAL, "rope: no positions or no table");
  if ((uintptr_t)table % 8) return set_err(BFP_EINVAL, "rope: table is not 8-byte aligned");
  if ((uintptr_t)pos % 4) return set_err(BFP_EINVAL, "rope: pos is not aligned");
  if (n_rows == 0) return BFP_OK;
  const RopeShape shape = rope_shape(*x, *y, n_rows, hd, rot, interleaved);
  // two heads a thread once that still leaves eight waves a CU
  const long long all = (long long)n_rows * x->heads * shape.per_head;
  const int n = shape.wide && x->heads >= ROPE_HEADS && all >= (long long)ROPE_HEADS * 256 * 8 * 64 ? ROPE_HEADS : 1;
  const long long per_row = (long long)shape.per_head * ((x->heads + n - 1) / n);
  if (per_row > 0x3fffffffLL) return set_err(BFP_EINVAL, "rope: rows of %lld units", per_row);
  RopeArgs a{*x, *y, shape, pos, (const float2 *)table, n_pos, 0, FastDiv((uint32_t)per_row), FastDiv((uint32_t)shape.per_head), 0};
  auto *fn = !shape.wide ? k_rope<0> : n == 1 ? k_rope<1> : k_rope<ROPE_HEADS>;
  const int step = (int)(0x7fffff00LL / per_row);
  for (int r = 0; r < n_rows;) {
    const int rows = n_rows - r < step ? n_rows - r : step;
    a.row0 = r;
    a.units = (uint32_t)((long long)rows * per_row);
    hipLaunchKernelGGL(fn, dim3((a.units + ROPE_BS - 1) / ROPE_BS), dim3(ROPE_BS), 0, (hipStream_t)stream, a);
    BFP_TRY(launch_status("rope"));
    r += rows;
  }
  return BFP_OK;
}

}  // extern "C"
