// What the kernels of the attention over the 4-bit cache share: their
// arguments, masks, the terms values are split into, and how work is placed.
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>

#include "bfp.h"
#include "bfp_device.h"
#include "bfp_f64.h"
#include "bfp_internal.h"
#include "bfp_kv4.h"
#include "bfp_rows.h"

namespace bfp {

constexpr int KEYS = 64;             // keys a wave takes at a time
// The running maximum is raised only when a score passes it, and then to this
// many powers of two above the score: the sums are rescaled a few times in a
// whole context instead of whenever a new maximum turns up.  No probability
// passes 1, so a sum of n values stays below n times the largest; the largest
// probability is 2^-8 where the maximum was set, which a float holds as well.
constexpr float M_SLACK = 8.0f;

typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

struct Kv4AttnArgs {
  bfp_kv4 c;
  bfp_kv4_batch b;
  bfp_rows q, out;
  int tiles, group, page_shift, window, row_tiles;
  int splits, chunk;   // k_kv4_prompt: pieces of the keys, and their length in tiles
  int stream;          // k_kv4_rows: workgroups that share all tiles (0: one takes all keys of its rows)
  int out_wide;        // out takes 16-byte stores
  FastDiv by_seq, by_head, by_split, by_group;
  // A workgroup's piece: one sequence after the other, its last rows, which
  // see the most keys, first.  Neighbouring workgroups take different KV heads
  // of the same rows and keys: workgroups go to the XCDs and their shader
  // engines in turn, whether one is ready sooner or not, so neighbours should
  // take equally long.
  __device__ void place(int &seq, int &head, int &split, int &rt) const {
    uint32_t u, h, s;
    seq = (int)by_seq.div(blockIdx.x, u);
    u = by_head.div(u, h);
    rt = row_tiles - 1 - (int)by_split.div(u, s);
    split = (int)s;
    head = (int)h + split % c.heads;
    head = head < c.heads ? head : head - c.heads;
  }
  float scale2;        // |scale| * log2(e), kept above 0
  float slack;         // M_SLACK in scores: M_SLACK / scale2, above the score that raises the maximum
  float q_sign;        // the scale's sign, or 0, which the queries take
  // unfinished rows: the sums, and (maximum, sum of probabilities)
  float *part_o;       // k_kv4_prompt [sequence][row of max_q][query head][split][hd]; k_kv4_rows [slot][R][hd]
  float2 *part_ml;     // without [hd]
  unsigned long long *there, number;   // k_kv4_rows: which slots are filled, and this call's number
};

// Position p's visible keys are [lo, hi).
__device__ __forceinline__ int key_hi(int p) { return p < 0 ? 0 : p + 1; }
__device__ __forceinline__ int key_lo(int hi, int window) {
  return window > 0 && hi > window ? hi - window : 0;
}

// The tiles of split `split` out of a row tile's n: chunks as long as the
// longest sequence's splits are, so that workgroups take equally long
// whatever the lengths; the last split takes what is left, where a sequence
// is longer than the batch says.
struct KeyPart {
  int first, stop;
};
__device__ __forceinline__ KeyPart key_part(int n, int split, int splits, int chunk) {
  const long long a = (long long)split * chunk, b = a + chunk;
  KeyPart p;
  p.first = a < n ? (int)a : n;
  p.stop = split + 1 == splits || b > n ? n : (int)b;
  return p;
}

// x cut to bfloat16 toward zero: the rest is exact, and has the sign of x.
__device__ __forceinline__ float cut_bf16(float x) {
  return __uint_as_float(__float_as_uint(x) & 0xffff0000u);
}

// Term t of T of a query's value x: split by cuts (three hold any float32).
// An infinite query has no score but infinities and NaN, so its row is NaN
// whatever it sees: as a NaN it says so itself, where infinities of one sign
// would leave probabilities of nothing but zeros.
template <int T>
__device__ __forceinline__ float query_term(float x, int t) {
  if (!(fabsf(x) < INFINITY)) return t == 0 ? NAN : 0.0f;
  if (T == 1) return x;
  for (int i = 0; i < t; ++i) x -= cut_bf16(x);
  return cut_bf16(x);
}

__device__ __forceinline__ bf16x8 pack8(const float (&v)[8]) {
  bf16x8 r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = (__bf16)v[i];
  return r;
}

// Term t of eight probabilities.  Two terms: the first cut, the second
// rounded (2^-16 of the value at most).  Three (of four places): all cut,
// which holds a float32 exactly; what the fourth place gets is not used.
template <int T>
__device__ __forceinline__ bf16x8 pack_terms(float (&p)[8], int t) {
  if constexpr (T == 1) {
    return pack8(p);
  } else if constexpr (T == 2) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float c = cut_bf16(p[i]), rest = p[i] - c;
      p[i] = t == 0 ? c : rest;
    }
    return pack8(p);
  } else {
    const uint32_t m1 = t >= 1 ? 0xffff0000u : 0u, m2 = t >= 2 ? 0xffff0000u : 0u;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      p[i] -= __uint_as_float(__float_as_uint(p[i]) & m1);
      p[i] -= __uint_as_float(__float_as_uint(p[i]) & m2);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)   // the upper halves of two
      w[i] = __builtin_amdgcn_perm(__float_as_uint(p[2 * i + 1]), __float_as_uint(p[2 * i]), 0x07060302u);
    return __builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
  }
}

template <int M>
__device__ __forceinline__ float fpeer(float v) {
  return __int_as_float(peer<M>(__float_as_int(v)));
}

// A sum over the T columns that hold the terms of a row (columns R apart).
// The wider step first: the result is then the same in all of them.
template <int T>
__device__ __forceinline__ float term_sum(float v) {
  if constexpr (T >= 2) v += fpeer<8>(v);
  if constexpr (T >= 4) v += fpeer<4>(v);
  return v;
}

// Over 16 neighbouring lanes, and over the wave.
__device__ __forceinline__ float max16(float v) {
  v = fmaxf(v, fpeer<8>(v));
  v = fmaxf(v, fpeer<4>(v));
  v = fmaxf(v, fpeer<2>(v));
  return fmaxf(v, fpeer<1>(v));
}
__device__ __forceinline__ float sum16(float v) {
  v += fpeer<8>(v);
  v += fpeer<4>(v);
  v += fpeer<2>(v);
  return v + fpeer<1>(v);
}
__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, fpeer<32>(v));
  return max16(fmaxf(v, fpeer<16>(v)));
}
__device__ __forceinline__ float wave_sum(float v) {
  v += fpeer<32>(v);
  return sum16(v + fpeer<16>(v));
}

// Whether a byte of w is at least KV4_PAST: its lower seven bits carry into the
// eighth, which is set.
__device__ __forceinline__ bool has_byte_past(uint32_t w) {
  return ((w & 0x7f7f7f7fu) + 0x01010101u * (256 - KV4_PAST)) & w & 0x80808080u;
}
// w with its bytes kept where keep has a bit (byte i: bit i).
__device__ __forceinline__ uint32_t byte_mask(uint32_t keep) {
  return (((keep & 1) | ((keep & 2) << 7) | ((keep & 4) << 14) | ((keep & 8) << 21)) * 255u);
}

// Tiles have no NaN and no infinity: -2^127 (mantissa -32768, exponent 127),
// the largest magnitude they hold, stands for a NaN, so that whatever reads the
// row sees that it is no result; infinities stand as far out as tiles go.
__device__ __forceinline__ float tile_holds(float v) {
  return fabsf(v) <= 0x1.fffffep127f ? v : v > 0.0f ? 0x1.fffffep127f : -0x1.fffffep127f;
}

// Value o of a finished row: one of 16 neighbouring lanes with neighbouring o.
__device__ __forceinline__ void out_store(const bfp_rows &r, long long o, float v) {
  if (r.type != BFP_TILES) {
    row_store(r, o, v);
    return;
  }
  int e;
  const int m = quantize16_lanes((double)tile_holds(v), e);
  ((int16_t *)r.p)[o] = (int16_t)m;
  if ((threadIdx.x & 15) == 0) r.e[o >> 4] = (int8_t)e;
}

// Eight values from o on; of a tile, the other eight are lane ^ 1's.
__device__ __forceinline__ void out_store8(const bfp_rows &r, long long o, const float (&v)[8], bool wide) {
  if (r.type != BFP_TILES) {
    if (wide) {
      row_store_n(r, o, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) row_store(r, o + i, v[i]);
    }
    return;
  }
  float x[8], top = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = tile_holds(v[i]);
    top = fmaxf(top, fabsf(x[i]));
  }
  const int e = tile_exp_of((double)fmaxf(top, __shfl_xor(top, 1, 64)));
#pragma unroll
  for (int i = 0; i < 8; ++i) ((int16_t *)r.p)[o + i] = (int16_t)tile_mant_of((double)x[i], e);
  if (!(threadIdx.x & 1)) r.e[o >> 4] = (int8_t)e;
}

// What a row tile of k_kv4_rows costs beside its tiles (the queries, the first
// loads, the results: about 4 us), in tiles of the list that hold nothing:
// pieces of many short sequences hold fewer tiles.
constexpr int ROWS_EXTRA = 4;

typedef void (*attn_fn)(Kv4AttnArgs);
// The kernel for heads of `tiles` tiles (k_kv4_rows: with 4 waves, or the 16
// or 8 that rows_waves says) and its dynamic LDS.
struct AttnKernel {
  attn_fn fn;
  int lds;
};
AttnKernel rows_kernel(int tiles, int terms, int waves);
AttnKernel prompt_kernel(int tiles, int terms);
inline int rows_waves(int tiles) { return tiles <= 4 ? 16 : tiles <= 8 ? 8 : 4; }
inline int prompt_waves(int tiles, int terms) { return tiles <= 8 && terms < 3 ? 8 : 4; }
// Queues the kernel that joins what k_kv4_prompt left in pieces.
void launch_join_prompt(const Kv4AttnArgs &a, hipStream_t s);

}  // namespace bfp
