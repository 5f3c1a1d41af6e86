// The 4-bit key/value cache: where a token's tiles lie, which rows a
// sequence has, and the conversion of a tile.
//
// Why this format: the E2M1 elements of a tile share a power of two, which is
// what v_cvt_scalef32_pk_bf16_fp4 takes: two elements and their exponent to
// two bfloat16 in one full-rate instruction (measured 5 clocks a wave, as a
// plain and/or takes), exactly.  Whole 4-bit mantissas of the 16-bit tiles'
// kind would need three times the instructions and lose 0.5 to 1.4 dB on
// normal and heavy-tailed data (18.7 and 17.1 dB against 19.2 and 18.5).
//
// Why tile by tile, token after token within a page (not head rows): four
// tokens of a tile are then 32 contiguous bytes and their exponents one
// word, whatever the head width, so a lane of the attention reads two 16-byte
// words and one exponent word; appended prompts write whole lines too.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "bfp.h"

namespace bfp {

constexpr int KV4_E_MIN = -100, KV4_E_MAX = 100;   // exponents of a tile
constexpr int KV4_BIAS = 127, KV4_NAN = 255;
// Exponent bytes from here on can pass bfloat16's range (6 x 2^126).  Only
// KV4_NAN is ever written; the attention takes values with the others as NaN,
// too, since an infinity times a probability of zero would reach rows that do
// not see it.
constexpr int KV4_PAST = 253;
constexpr int KV4_TILE_BYTES = 8;
constexpr int KV4_MAX_POS = 0x7fff0000;   // that a table of pages has room for

// The rows of a sequence in a batch, clamped to what the row arrays hold:
// rows row0 .. row0 + n - 1, row i at position at + i (which may be negative, or
// past the last page: kv4_page finds no page for it then).
struct Kv4Span {
  int row0, n, at;
};
__host__ __device__ inline Kv4Span kv4_span(int start, int stop, int len, int n_rows, int max_q) {
  Kv4Span s;
  const int r0 = start < 0 ? 0 : (start > n_rows ? n_rows : start);
  const int all = stop < r0 ? 0 : stop - r0, n = all < n_rows - r0 ? all : n_rows - r0;
  s.row0 = r0;
  s.n = n < max_q ? n : max_q;
  s.at = (len < 0 ? 0 : len) - all;   // also of rows that are not there
  return s;
}

// The tile index of (page, head, tile, slot): its exponent's byte offset, and
// its data at 8 times that.
__host__ __device__ inline long long kv4_tile(long long page_id, int heads, int head, int tiles,
                                              int tile, int page, int slot) {
  return ((page_id * heads + head) * tiles + tile) * page + slot;
}

// The page number p_page of a sequence, or -1 where it has none.
__host__ __device__ inline int kv4_page(const int32_t *pages, int width, int n_pages, int p_page) {
  if ((unsigned)p_page >= (unsigned)width) return -1;
  const int id = pages[p_page];
  return (unsigned)id < (unsigned)n_pages ? id : -1;
}

#if defined(__HIP_DEVICE_COMPILE__) || defined(__HIPCC__)
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// 2^(E-127) as the conversions take it (their scale operand is read for its
// exponent field only; 255 gives NaNs).
__device__ __forceinline__ float kv4_scale(uint32_t E) { return __uint_as_float(E << 23); }

// Eight elements (a word) to bfloat16: element 2 significant bits, exponent
// at least -100, so exact.
__device__ __forceinline__ bf16x8 kv4_decode8(uint32_t w, float scale) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Sixteen values to a tile.  The values are exact, or rounded toward zero
// with a set last bit where something was lost, so every comparison with a
// border between two elements comes out as it would on the exact value.  The
// largest magnitude a = f 2^x (f in [1, 2)) takes exponent x - 2, or x - 1
// from f = 1.75 on, where it would round past 6.
__device__ __forceinline__ uint2 kv4_encode(const float (&v)[16], uint32_t &E) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint32_t b = __float_as_uint(v[i]) & 0x7fffffffu;
    top = b > top ? b : top;
  }
  if (top >= 0x7f800000u) {   // a NaN or an infinity
    E = KV4_NAN;
    return make_uint2(0, 0);
  }
  int e = (int)(top >> 23) - 127 - 2 + ((top & 0x7fffffu) >= 0x600000u ? 1 : 0);
  e = e < KV4_E_MIN ? KV4_E_MIN : (e > KV4_E_MAX ? KV4_E_MAX : e);
  if (top == 0) e = 0;
  E = (uint32_t)(e + KV4_BIAS);
  const float s = kv4_scale(E);
  uint2 w = make_uint2(0, 0);
  w.x = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w.x, v[0], v[1], s, 0);
  w.x = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w.x, v[2], v[3], s, 1);
  w.x = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w.x, v[4], v[5], s, 2);
  w.x = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w.x, v[6], v[7], s, 3);
  w.y = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w.y, v[8], v[9], s, 0);
  w.y = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w.y, v[10], v[11], s, 1);
  w.y = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w.y, v[12], v[13], s, 2);
  w.y = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w.y, v[14], v[15], s, 3);
  return w;
}

// A tile as sixteen float32 (exact).
__device__ __forceinline__ void kv4_decode(uint2 w, uint32_t E, float (&v)[16]) {
  const float s = kv4_scale(E);
#define KV4_PAIR(i, word, sel)                                                     \
  {                                                                                \
    const f32x2 p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, s, sel);        \
    v[i] = p[0], v[i + 1] = p[1];                                                  \
  }
  KV4_PAIR(0, w.x, 0) KV4_PAIR(2, w.x, 1) KV4_PAIR(4, w.x, 2) KV4_PAIR(6, w.x, 3)
  KV4_PAIR(8, w.y, 0) KV4_PAIR(10, w.y, 1) KV4_PAIR(12, w.y, 2) KV4_PAIR(14, w.y, 3)
#undef KV4_PAIR
}
#endif

// The checks every entry point of the cache makes (bfp_kv4.hip).
int check_kv4(const char *op, const bfp_kv4 *c, const bfp_kv4_batch *b);
// Of those, the batch's, for pages of `page` tokens.
int check_batch(const char *op, const bfp_kv4_batch *b, int page);

}  // namespace bfp
