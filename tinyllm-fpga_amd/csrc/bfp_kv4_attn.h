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

// What a launch's rows see.
enum Kv4Sees {
  SEES_ALL,      // their sequence up to their position
  SEES_PICKS,    // of that the pages that a list of each row and KV head names
  SEES_PREFIX,   // of that what their sequence's group shares: one "sequence" is a group's rows
  SEES_REST      // of that what lies behind the shared tokens
};

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
  __device__ void place(uint32_t block, int &seq, int &head, int &split, int &rt) const {
    uint32_t u, h, s;
    seq = (int)by_seq.div(block, u);
    u = by_head.div(u, h);
    rt = row_tiles - 1 - (int)by_split.div(u, s);
    split = (int)s;
    head = (int)h + split % c.heads;
    head = head < c.heads ? head : head - c.heads;
  }
  __device__ bool piece(int rows, int &g, int &head, int &split, int &rt, int &splits, int &chunk) const;
  float scale2;        // |scale| * log2(e), kept above 0
  float slack;         // M_SLACK in scores: M_SLACK / scale2, above the score that raises the maximum
  float q_sign;        // the scale's sign, or 0, which the queries take
  // unfinished rows: the sums, and (maximum, sum of probabilities)
  float *part_o;       // k_kv4_prompt [sequence][row of max_q][query head][split][hd]; k_kv4_rows [slot][R][hd]
  float2 *part_ml;     // without [hd]
  unsigned long long *there, number;   // k_kv4_rows: which slots are filled, and this call's number
  // listed pages: n_picks a row and KV head, and the row tiles of a token's query heads
  const int32_t *picks;
  int n_picks, token_tiles;
  // Shared prefixes.  SEES_PREFIX: b's sequences are the groups (pages, width,
  // n_seq, max_q), its start and len still the batch's.  Both launches leave
  // unfinished rows in part_o [place][hd] and part_ml, the prefix's places first
  // (prefix_place), then the rest's (rest_place); k_kv4_rows its own parts in slot_o,
  // slot_ml.
  bfp_kv4_shared sh;
  int sh_seqs;   // sequences of the batch
  int prefix_splits, rest_splits;   // at most, a row
  long long rest_first;             // the rest's first place
  int pieces, piece_shift, piece_blocks;   // k_kv4_prompt: workgroups that share the keys of up to 64 groups (0: splits of one length), log2 of each one's rows, and the launch's
  int4 *piece_of;   // with them, of each group: splits, first workgroup, row tiles, first row
  float *slot_o;
  float2 *slot_ml;
};

// Position p's visible keys are [lo, hi).
__device__ __forceinline__ int key_hi(int p) { return p < 0 ? 0 : p + 1; }
__device__ __forceinline__ int key_lo(int hi, int window) {
  return window > 0 && hi > window ? hi - window : 0;
}

// Group g's sequences, within the batch.
struct Kv4Group {
  int first, stop;
};
__device__ __forceinline__ Kv4Group kv4_group(const Kv4AttnArgs &a, int g) {
  const int f = a.sh.start[g], t = a.sh.start[g + 1];
  Kv4Group x;
  x.first = f < 0 ? 0 : f < a.sh_seqs ? f : a.sh_seqs;
  x.stop = t < x.first ? x.first : t < a.sh_seqs ? t : a.sh_seqs;
  return x;
}
// The rows of a group, as one sequence's, and the tokens that they share and
// the pages have room for (at).
__device__ __forceinline__ Kv4Span kv4_group_span(const Kv4AttnArgs &a, int g, Kv4Group &x) {
  x = kv4_group(a, g);
  Kv4Span s = kv4_span(a.b.start[x.first], a.b.start[x.stop], 0, a.b.n_rows, a.b.max_q);
  const long long cap = (long long)a.b.width << a.page_shift;
  const int len = a.sh.len[g];
  s.at = len < 0 ? 0 : len < cap ? len : (int)cap;
  return s;
}
// The least position that any row of a group sees.
__device__ __forceinline__ int kv4_group_low(const Kv4AttnArgs &a, const Kv4Group &x) {
  if (a.window == 0) return 0;
  int low = 0x7fffffff;
#pragma unroll 4
  for (int b = x.first; b < x.stop; ++b) {
    const int len = a.b.len[b], n = a.b.start[b + 1] - a.b.start[b];
    const int at = len > n ? len - n : 0;
    if (len > 0 && n > 0) low = key_lo(key_hi(at), a.window) < low ? key_lo(key_hi(at), a.window) : low;
  }
  return low == 0x7fffffff ? 0 : low;
}
// The tokens that sequence b's group (g) shares, 0 outside every group.
__device__ __forceinline__ int kv4_shared_len(const Kv4AttnArgs &a, int b, int &g) {
  int past = a.sh.n_groups;   // the last group that begins at b or before
  g = 0;
  while (past - g > 1) {
    const int mid = g + (past - g) / 2;
    (a.sh.start[mid] <= b ? g : past) = mid;
  }
  const int n = a.sh.len[g];
  return a.sh.start[g] <= b && b < a.sh.start[g + 1] && n > 0 ? (n < KV4_MAX_POS ? n : KV4_MAX_POS) : 0;
}
__device__ __forceinline__ int kv4_shared_len(const Kv4AttnArgs &a, int b) {
  int g;
  return kv4_shared_len(a, b, g);
}
// The position of row t of a group: of the sequence in which it lies.  Lane x
// < N of every N neighbouring ones has the wave's x-th row; each gets its own's.
template <int N>
__device__ __forceinline__ int kv4_row_position(const Kv4AttnArgs &a, const Kv4Group &x, int t) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int b0 = x.first; b0 < x.stop; b0 += 64) {
    const int past = b0 + lane < x.stop ? a.b.start[b0 + lane + 1] : 0x7fffffff;   // the first row behind sequence b0 + lane
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int c = __popcll(__ballot(past <= __builtin_amdgcn_readlane(t, k)));
      n += lane % N == k ? c : 0;
    }
  }
  const int b = x.first + n < x.stop ? x.first + n : x.stop - 1;
  if (b < x.first) return -1;
  const int len = a.b.len[b];
  const long long p = (long long)(len < 0 ? 0 : len) - a.b.start[b + 1] + t;
  return p < 0 ? -1 : (int)(p < KV4_MAX_POS ? p : KV4_MAX_POS);
}

// Where a row's unfinished sums lie.  The prefix's, where pieces of the groups'
// keys are shared out: by workgroup and row in it, since how many splits there are
// depends on how many rows; else by row, head and split.
__device__ __forceinline__ long long prefix_place(const Kv4AttnArgs &a, long long tok, int qh, int split) {
  return (tok * a.q.heads + qh) * a.prefix_splits + split;
}
// The rest's: of row i of a sequence (k_kv4_prompt splits only what few row tiles see,
// and rows that belong to no sequence should not take splits' room).
__device__ __forceinline__ long long rest_place(const Kv4AttnArgs &a, int seq, int i, long long tok, int qh, int split) {
  return a.rest_first + (a.rest_splits > 1 ? (((long long)seq * a.b.max_q + i) * a.q.heads + qh) * a.rest_splits + split : tok * a.q.heads + qh);
}

// Over N neighbouring lanes (16 or 32).
template <int N>
__device__ __forceinline__ int min_lanes(int v) {
  if (N == 32) v = min(v, peer<16>(v));
  v = min(v, peer<8>(v));
  v = min(v, peer<4>(v));
  v = min(v, peer<2>(v));
  return min(v, peer<1>(v));
}
template <int N>
__device__ __forceinline__ int max_lanes(int v) { return -min_lanes<N>(-v); }

// Workgroup blockIdx.x's part of the groups' prefixes, at most 64 of them,
// where the longest takes its keys in prefix_splits splits at most: all workgroups
// take equally many tiles, whatever the groups' lengths, as long as a round of
// them (a.pieces) has room for every row tile.  False: there is nothing for it.
__device__ __forceinline__ bool Kv4AttnArgs::piece(int rows, int &g, int &head, int &split, int &rt, int &splits, int &chunk) const {
  const int lane = threadIdx.x & 63;
  int units = 0, tiles = 0, row0 = 0;   // row tiles x KV heads, key tiles, and the first row
  if (lane < b.n_seq) {
    Kv4Group x;
    const Kv4Span s = kv4_group_span(*this, lane, x);
    const int low = kv4_group_low(*this, x) / KEYS;
    row0 = s.row0;
    units = (int)(((long long)s.n * group + rows - 1) / rows) * c.heads;
    tiles = s.at > low * KEYS ? (s.at + KEYS - 1) / KEYS - low : 1;
  }
  const auto sum = [](int v) { return (int)psum<1>(psum<2>(psum<4>(psum<8>(psum<16>(psum<32>(v)))))); };
  int most = units ? tiles : 0;
#pragma unroll
  for (int d = 32; d > 0; d /= 2) most = max(most, __shfl_xor(most, d, 64));
  const int places = sum(min(units, 1 << 20));
  int least = max((most + prefix_splits - 1) / prefix_splits, 4);
  chunk = max(most, 1);
  if (places <= pieces && least < chunk) {   // the shortest pieces of which there are no more than `pieces`
    int too_short = least - 1;
    while (chunk - too_short > 1) {
      const int mid = too_short + (chunk - too_short) / 2;
      (sum(units * ((tiles + mid - 1) / mid)) <= pieces ? chunk : too_short) = mid;   // (units are 256 at most here, and tiles / mid 48)
    }
  }
  const int mine = (tiles + chunk - 1) / chunk;
  int up = units * mine;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int x = __shfl_up(up, d, 64);
    up += lane >= d ? x : 0;
  }
  if (blockIdx.x == 0 && threadIdx.x < b.n_seq) piece_of[lane] = make_int4(mine, up - units * mine, units / c.heads, row0);
  const unsigned long long past = __ballot(up > (int)blockIdx.x);
  if (!past) return false;
  g = __ffsll((long long)past) - 1;
  splits = __builtin_amdgcn_readlane(mine, g);
  chunk = __builtin_amdgcn_readfirstlane(chunk);
  const int before = __builtin_amdgcn_readlane(up - units * mine, g), its = __builtin_amdgcn_readlane(units, g) / c.heads;
  uint32_t h;
  const uint32_t u = by_head.div(blockIdx.x - (uint32_t)before, h);
  head = (int)h;
  split = (int)(u / (uint32_t)its);
  rt = (int)(u - (uint32_t)split * its);
  return true;
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
AttnKernel picks_kernel(int tiles, int terms, int waves, bool share);
AttnKernel prompt_kernel(int tiles, int terms);
// Of a shared prefix, and of what lies behind it.
AttnKernel prefix_rows_kernel(int tiles, int terms, int waves, bool share);
AttnKernel prefix_prompt_kernel(int tiles, int terms, bool pairs);
AttnKernel rest_rows_kernel(int tiles, int terms, int waves, bool share);
AttnKernel rest_prompt_kernel(int tiles, int terms);
// Both parts of few rows in one launch, the prefix's workgroups first: they
// have nothing to wait for in each other.
typedef void (*attn_parts_fn)(Kv4AttnArgs prefix, Kv4AttnArgs rest, uint32_t prefix_blocks);
struct PartsKernel {
  attn_parts_fn fn;
  int lds;
};
PartsKernel parts_kernel(int tiles, int terms, int waves);
inline int rows_waves(int tiles) { return tiles <= 4 ? 16 : tiles <= 8 ? 8 : 4; }
inline int prompt_waves(int tiles, int terms) { return tiles <= 8 && terms < 3 ? 8 : 4; }
// Two workgroups of four waves a CU instead of one of eight: registers and LDS hold them.
inline bool prompt_pairs(int tiles, int terms) { return tiles <= 8 && terms < 3; }
// Queues the kernel that joins what k_kv4_prompt left in pieces.
void launch_join_prompt(const Kv4AttnArgs &a, hipStream_t s);
// The same of a row's two parts.
void launch_join_shared(const Kv4AttnArgs &a, hipStream_t s);

}  // namespace bfp
