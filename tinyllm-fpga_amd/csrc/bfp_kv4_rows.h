// Attention over the 4-bit cache for few rows to a KV head: decode steps, and
// the few tokens of a checked draft.
//
// A workgroup takes up to 16 columns (rows x terms) of one sequence and KV
// head, its waves take 64 keys in turn.  With S^T = K Q^T the keys are the
// matrix tile's rows and a lane's K operand is one tile of one key, straight
// from memory through the decoding conversion.  S^T leaves the probabilities
// in the layout in which O^T = V^T P^T takes them, with the keys in the order
// (lane group, register, key of four), so they never move between lanes.  V
// has to be turned over: its decoded tiles go through the wave's own piece of
// LDS and come back with the transposing reads.
//
// SEES_PICKS: every row and KV head sees the pages that a list of its own names
// (in any order; each once) instead of all up to its position.  The keys of
// the listed pages, one after the other, are the key tiles then, and a row
// tile is one token's query heads.  Every list decodes its own keys, so vector
// work bounds it: 1021 rows over 24 pages of 32 tokens, 32 + 4 heads of 128, take 78
// us, 165 TFLOP/s in one term (it has two).  Few rows wait for
// the chain list -> page number -> bytes: 8 rows over 32 pages of 64, 18 us.
// SEES_PREFIX, SEES_REST: the two parts of rows that share a prefix, left
// unfinished.  All rows of a group are one sequence in the first.  64 rows over
// up to 2048 own tokens, 32 + 8 heads of 128: 31 us, 105 MB at 3.4 TB/s, a chain
// of loads and products a key tile at two to three waves a SIMD.
#pragma once
#include "bfp_kv4_attn.h"

namespace bfp {

// A wave's side (K or V) of one 64-key tile: lane (r = lane % 16, g = lane /
// 16) holds keys 4r .. 4r+3 of head tiles g * C .. g * C + C - 1, four keys' exponents a
// word.
template <int C>
struct KvSide {
  uint4 w[C][2];
  uint32_t e[C];
};

__device__ __forceinline__ uint2 half_of(const uint4 (&w)[2], int j) {
  return j == 0 ? make_uint2(w[0].x, w[0].y) : j == 1 ? make_uint2(w[0].z, w[0].w)
         : j == 2 ? make_uint2(w[1].x, w[1].y) : make_uint2(w[1].z, w[1].w);
}

// Head tiles that do not exist are read as the last one; keys without a page
// as the first page's.
template <int C>
__device__ __forceinline__ void load_side(KvSide<C> &x, const uint8_t *data, const uint8_t *exps, long long o,
                                          int page, int t, int tiles) {
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const long long oc = o + (long long)(t + c < tiles ? t + c : tiles - 1) * page;
    const uint4 *p = (const uint4 *)(data + oc * KV4_TILE_BYTES);
    x.w[c][0] = ld_nt(p);
    x.w[c][1] = ld_nt(p + 1);
    x.e[c] = *(const uint32_t *)(exps + oc);
  }
}

// The exponent byte of key j as the conversions take it: they look at the
// exponent field only, whatever lies beside it.
__device__ __forceinline__ float scale_of(uint32_t e, int j) {
  return __uint_as_float(j == 0 ? e << 23 : j == 1 ? e << 15 : j == 2 ? e << 7 : e >> 1);
}

// LDS rows of 32 keys x hd bfloat16.  A row's bytes are an odd multiple of
// 32, so that the 32-byte pieces of neighbouring rows, which the transposing
// reads take, lie in different banks; the two 16-byte halves of every piece
// change places in each second group of four rows, so that eight lanes'
// writes do too (without that they took twice as long).
constexpr int v_pitch(int C) { return 32 * (4 * C | 1); }
constexpr int V_ROWS = 32;
// Floats of a wave's sums in LDS when the waves are joined: m and sum of 16
// columns, then R rows of hd (and 4 more, for the banks).
__host__ __device__ inline int join_floats(int R, int tiles) { return 32 + R * (16 * tiles + 4); }

// Shared work.  With `stream` workgroups, the batch's key tiles are one long
// list -- sequence by sequence, each one's row tiles and KV heads one after
// the other, each of those its keys in order -- and every workgroup takes an
// equally long piece of it, whatever the sequences' lengths.  A piece may end
// in the middle of a row tile's keys: then the sums of the row tile's parts go
// to slots of the workspace, and the workgroup that finishes the last of them
// joins them, always in the order of the keys.
constexpr int STREAM_SEQS = 256;   // sequences of such a batch: one a thread
constexpr int MAX_PARTS = 128;     // of a row tile: their factors are held in LDS
struct RowsSeq {
  int row0, n, at;     // Kv4Span
  int tile0, tiles;    // the keys that any of its rows sees, in tiles (at least one: somebody writes the zeros)
  int groups;          // row tiles x KV heads
  int low;             // SEES_REST: the first position
  Kv4Group of;         // SEES_PREFIX: the group
  __device__ uint32_t span() const { return (uint32_t)tiles + ROWS_EXTRA; }
};
template <Kv4Sees SEES>
__device__ __forceinline__ RowsSeq rows_seq(const Kv4AttnArgs &a, int R, int b) {
  RowsSeq s;
  const Kv4Span sp = SEES == SEES_PREFIX ? kv4_group_span(a, b, s.of)
                                         : kv4_span(a.b.start[b], a.b.start[b + 1], a.b.len[b], a.b.n_rows, a.b.max_q);
  s.row0 = sp.row0, s.n = sp.n, s.at = sp.at, s.tile0 = 0, s.tiles = 1, s.groups = 0;
  if (SEES == SEES_REST) s.low = kv4_shared_len(a, b);
  if (sp.n == 0) return s;
  if (SEES == SEES_PICKS) {
    s.tiles = (int)((((long long)a.n_picks << a.page_shift) + KEYS - 1) / KEYS);
    s.groups = sp.n * a.token_tiles * a.c.heads;
    return s;
  }
  const long long cap = (long long)a.b.width << a.page_shift;
  const int hi = SEES == SEES_PREFIX ? sp.at : key_hi(sp.at + sp.n - 1), end = hi < cap ? hi : (int)cap;
  int lo = SEES == SEES_PREFIX ? kv4_group_low(a, s.of) : key_lo(key_hi(sp.at), a.window);
  if (SEES == SEES_REST) lo = lo > s.low ? lo : s.low;
  s.tile0 = lo / KEYS;
  s.tiles = end > lo ? (end + KEYS - 1) / KEYS - s.tile0 : 1;
  s.groups = (sp.n * a.group + R - 1) / R * a.c.heads;
  return s;
}

// The list's offsets: before[b] tiles lie before sequence b, before[n_seq] are
// all; each workgroup takes `piece` of them.  256 threads.
struct Stream {
  uint32_t before[STREAM_SEQS + 1];
  uint32_t wave[4], longest[4];
  int last;
};
template <Kv4Sees SEES>
__device__ __forceinline__ uint32_t stream_plan(const Kv4AttnArgs &a, int R, Stream &st) {
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  uint32_t n = 0, most = 0;
  if (t < a.b.n_seq) {
    const RowsSeq s = rows_seq<SEES>(a, R, t);
    n = (uint32_t)s.groups * s.span();
    most = (uint32_t)s.tiles;
  }
  uint32_t up = n;   // inclusive sums over the wave
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint32_t x = __shfl_up(up, d, 64);
    up += lane >= d ? x : 0;
  }
  if (lane == 63) st.wave[w] = up;
#pragma unroll
  for (int d = 32; d > 0; d /= 2) {
    const uint32_t x = __shfl_xor(most, d, 64);
    most = x > most ? x : most;
  }
  if (lane == 0) st.longest[w] = most;
  __syncthreads();
  uint32_t base = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) base += k < w ? st.wave[k] : 0;
  if (t < a.b.n_seq) st.before[t + 1] = base + up;
  if (t == 0) st.before[0] = 0;
  __syncthreads();
  most = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) most = st.longest[k] > most ? st.longest[k] : most;
  const uint32_t all = st.before[a.b.n_seq], share = (all + a.stream - 1) / a.stream;
  // m tiles in pieces of at least m / (MAX_PARTS - 2): at most MAX_PARTS of them, wherever they begin
  const uint32_t least = (most + MAX_PARTS - 3) / (MAX_PARTS - 2);
  return ((share > least ? share : least) + 3) / 4 * 4;   // a tile for each of four waves
}

// What workgroups hand each other goes past the XCDs' L2 caches, store by
// store and load by load (device-scope accesses): a store is done when the
// wait for it is over, so a workgroup's arrival after that wait and a barrier
// says that its sums are there.  A device-scope fence instead would write back
// and drop all of an L2 each time: one sequence of 8192 tokens took 55 us with
// fences, 16 this way.
__device__ __forceinline__ void put(float *p, float v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void put(float2 *p, float2 v) {
  __hip_atomic_store((unsigned long long *)p, ((unsigned long long)__float_as_uint(v.y) << 32) | __float_as_uint(v.x),
                     __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float get(const float *p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 get(const float2 *p) {
  const unsigned long long u = __hip_atomic_load((const unsigned long long *)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return make_float2(__uint_as_float((uint32_t)u), __uint_as_float((uint32_t)(u >> 32)));
}
__device__ __forceinline__ void stores_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Wave 0: this part (number `mine` of a row tile's) is there; true for the
// wave that finds all parts there, which is at least the last one's.  A part
// is there if its flag holds the call's number (64 bits, from a random
// start), so the workspace needs no clearing; whoever joins the parts takes
// the flags away, so a replayed graph finds none.  Two workgroups may both
// find all parts: they write the same results.
__device__ __forceinline__ uint32_t part_slot(uint32_t p0, uint32_t k) { return 2 * (p0 + k) + (k == 0 ? 1 : 0); }
__device__ __forceinline__ bool arrive(unsigned long long *there, unsigned long long number, uint32_t p0, uint32_t mine,
                                       uint32_t parts) {
  const uint32_t lane = threadIdx.x & 63;
  if (lane == 0)
    __hip_atomic_store(there + part_slot(p0, mine), number, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  stores_done();
  bool all = true;
#pragma unroll
  for (uint32_t k = 0; k < MAX_PARTS; k += 64)
    if (k + lane < parts)
      all &= __hip_atomic_load(there + part_slot(p0, k + lane), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == number;
  if (!__all(all)) return false;
#pragma unroll
  for (uint32_t k = 0; k < MAX_PARTS; k += 64)
    if (k + lane < parts)
      __hip_atomic_store(there + part_slot(p0, k + lane), 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return true;
}

// C: head tiles a lane group holds (hd <= 64 C); T: terms of a row (columns
// R = 16 / T rows share); W: waves; SHARE: a.stream says whether workgroups
// share all tiles (W = 4).
template <int C, int R, Kv4Sees SEES>
__device__ void join_parts(const Kv4AttnArgs &a, char *lds, const RowsSeq &sp, int head, int rt, uint32_t p0, int parts);

// Where row tile rt's rows lie: rows rr0 .. rows - 1 of the KV head's, row rr
// being query head rr % G of token rr / G (SEES_PICKS: head rr of token i).
struct RowTile {
  int rr0, rows, i;
};
template <int R, Kv4Sees SEES>
__device__ __forceinline__ RowTile row_tile(const Kv4AttnArgs &a, const RowsSeq &sp, int rt) {
  if (SEES != SEES_PICKS) return {rt * R, sp.n * a.group, 0};
  const int i = rt / a.token_tiles, rr0 = (rt - i * a.token_tiles) * R;
  return {rr0, i < sp.n ? a.group : 0, i};
}
template <Kv4Sees SEES>
__device__ __forceinline__ int token_of(const Kv4AttnArgs &a, const RowTile &t, int rr) { return SEES == SEES_PICKS ? t.i : rr / a.group; }
template <Kv4Sees SEES>
__device__ __forceinline__ int head_of(const Kv4AttnArgs &a, int rr) { return SEES == SEES_PICKS ? rr : rr % a.group; }

// A lane's part of a column's query.
__device__ __forceinline__ void pack_query(const float (&x)[16], bf16x8 (&qf)[2]) {
  float y[8];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int d = 0; d < 8; ++d) y[d] = x[8 * h + d];
    qf[h] = pack8(y);
  }
}
// All head tiles of it, their loads under way together: behind a branch on the
// type each they follow one another.
template <int C, int T, int TYPE>
__device__ __forceinline__ void load_query(const Kv4AttnArgs &a, long long at, int tile0, bool mine, int t, bf16x8 (&qf)[C][2]) {
  bfp_rows q = a.q;
  q.type = TYPE;
  float x[C][16];
#pragma unroll
  for (int c = 0; c < C; ++c) {
#pragma unroll
    for (int d = 0; d < 16; ++d) x[c][d] = 0.0f;
    if (mine && tile0 + c < a.tiles) row_load_n(q, at + 16 * (tile0 + c), x[c]);
  }
#pragma unroll
  for (int c = 0; c < C; ++c) {
#pragma unroll
    for (int d = 0; d < 16; ++d) x[c][d] = query_term<T>(x[c][d], t) * a.q_sign;
    pack_query(x[c], qf[c]);
  }
}

// The workspace of a launch's own parts, and where unfinished rows go.
template <Kv4Sees SEES>
__device__ __forceinline__ float *slot_o(const Kv4AttnArgs &a) { return SEES >= SEES_PREFIX ? a.slot_o : a.part_o; }
template <Kv4Sees SEES>
__device__ __forceinline__ float2 *slot_ml(const Kv4AttnArgs &a) { return SEES >= SEES_PREFIX ? a.slot_ml : a.part_ml; }
template <Kv4Sees SEES>
__device__ __forceinline__ long long sum_place(const Kv4AttnArgs &a, long long tok, int qh) {   // (these launches split no row's keys)
  return SEES == SEES_PREFIX ? prefix_place(a, tok, qh, 0) : rest_place(a, 0, 0, tok, qh, 0);
}
template <Kv4Sees SEES>
__device__ __forceinline__ void leave_sum(const Kv4AttnArgs &a, long long tok, int qh, int d, float2 ml, float v) {
  const long long at = sum_place<SEES>(a, tok, qh);
  if (d == 0) a.part_ml[at] = ml;
  a.part_o[at * (16 * a.tiles) + d] = v;
}

// Waves a SIMD that the registers leave room for.  Without shared work (which
// takes 50 more) three of heads up to 128, four up to 64.
constexpr int rows_per_simd(int C, int W, Kv4Sees sees, bool share) {
  if (W > 8) return 4;
  if (sees != SEES_ALL && !share && C <= 2) return C == 1 ? 4 : 3;
  return C == 1 ? 3 : W > 4 || C == 2 ? 2 : 1;
}

template <int C, int T, int W, Kv4Sees SEES, bool SHARE>
__device__ __forceinline__ void rows_block(const Kv4AttnArgs &a, uint32_t block) {
  constexpr int R = 16 / T;
  constexpr bool PICK = SEES == SEES_PICKS;
  extern __shared__ __align__(16) char lds[];
  __shared__ Stream st;
  int seq, head, rt, split;
  uint32_t x = 0, x_stop = 1, piece = 0;
  if (SHARE && a.stream) {
    piece = stream_plan<SEES>(a, R, st);
    x = block * piece;
    const uint32_t all = st.before[a.b.n_seq];
    if (x >= all) return;
    x_stop = x + piece < all ? x + piece : all;
    seq = 0;
    for (int b = threadIdx.x & 63; b < a.b.n_seq; b += 64)   // every wave for itself
      seq += __popcll(__ballot(st.before[b + 1] <= x));
    seq = __builtin_amdgcn_readfirstlane(seq);
  } else {
    a.place(block, seq, head, split, rt);
  }
  const int G = a.group;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const int t = r / R;
  const int tiles = a.tiles;
  // one round takes keys of one row tile and KV head
  bool begun = false;
  while (x < x_stop) {
    const int32_t *pages = a.b.pages + (long long)seq * a.b.width;
    // Unsigned: of a wave that has no tile, whose first one may lie past 2^31 keys
    // (the place of a signed overflow's result in its page is not defined).
    auto slot_of = [&](int tile) { return (uint32_t)tile * KEYS + 4 * r; };
    auto offset_of = [&](int tile, int id) {
      return kv4_tile(id < 0 ? 0 : id, a.c.heads, head, tiles, 0, a.c.page, slot_of(tile) & (a.c.page - 1));
    };
    // Without a window a wave's first tile is known before the lengths are:
    // its page number and its bytes are on their way while those arrive.
    KvSide<C> k, v;
    int id = -1;
    long long at = 0;
    const bool early = SEES == SEES_ALL && !(SHARE && a.stream) && a.window == 0;
    if (early) {
      id = kv4_page(pages, a.b.width, a.c.n_pages, (w * KEYS + 4 * r) >> a.page_shift);
      at = offset_of(w, id);
      load_side(k, a.c.k, a.c.k_e, at, a.c.page, g * C, tiles);
      load_side(v, a.c.v, a.c.v_e, at, a.c.page, g * C, tiles);
    }
    const RowsSeq sp = rows_seq<SEES>(a, R, seq);
    int from = 0, upto = sp.tiles, slot = -1;
    uint32_t begin = 0;
    if (SHARE && a.stream) {
      const uint32_t y = x - st.before[seq], group = y / sp.span(), off = y - group * sp.span();
      const uint32_t left = x_stop - x, whole = sp.span() - off, take = left < whole ? left : whole;
      begin = x - off;
      x += take;
      from = (int)off;
      if (from >= sp.tiles) {   // nothing but the end of its span
        while (x < x_stop && x == st.before[seq + 1]) ++seq;
        continue;
      }
      upto = from + (int)take < sp.tiles ? from + (int)take : sp.tiles;
      // the first part of a row tile's keys goes to the workgroup's second slot, any other to its first
      if (from > 0 || upto < sp.tiles) slot = 2 * block + (from == 0 ? 1 : 0);
      head = (int)(group % (uint32_t)a.c.heads);
      rt = (int)(group / (uint32_t)a.c.heads);
      if (begun) __syncthreads();   // the last round's sums have been read
      begun = true;
    } else {
      x = x_stop;
    }
    const RowTile row_t = row_tile<R, SEES>(a, sp, rt);
    const int rows = row_t.rows, rr0 = row_t.rr0;   // rows of this KV head: (token, query head)
    if (rr0 >= rows) return;     // never with shared work

    // this lane's column
    const int rr = rr0 + r % R;
    const bool mine = rr < rows;
    const int i = mine ? token_of<SEES>(a, row_t, rr) : 0, qh = head * G + (mine ? head_of<SEES>(a, rr) : 0);
    int hi = mine ? key_hi(sp.at + i) : 0, lo = key_lo(hi, a.window);
    // what all of them see, and any of them
    const int last = (rr0 + R < rows ? rr0 + R : rows) - 1;
    int hi_min = key_hi(sp.at + rr0 / G), hi_max = key_hi(sp.at + last / G);
    int lo_min = key_lo(hi_min, a.window), lo_max = key_lo(hi_max, a.window);
    if constexpr (SEES == SEES_REST) {
      lo = lo > sp.low ? lo : sp.low;
      lo_min = lo_min > sp.low ? lo_min : sp.low;
      lo_max = lo_max > sp.low ? lo_max : sp.low;
    }
    bool blind = false;   // SEES_PREFIX: the row sees none of it; what is worked out for it is thrown away, not masked
    if constexpr (SEES == SEES_PREFIX) {   // rows of several sequences: by each one's position
      const int ends = key_hi(kv4_row_position<R>(a, sp.of, sp.row0 + (rr < rows ? rr : rows - 1) / G));
      lo = mine ? key_lo(ends, a.window) : 0;
      hi = mine ? (ends < sp.at ? ends : sp.at) : 0;
      blind = hi <= lo;
      hi_min = __builtin_amdgcn_readfirstlane(min_lanes<16>(blind ? 0x7fffffff : hi));
      hi_max = __builtin_amdgcn_readfirstlane(max_lanes<16>(hi));
      lo_min = __builtin_amdgcn_readfirstlane(min_lanes<16>(blind ? 0x7fffffff : lo));
      lo_max = __builtin_amdgcn_readfirstlane(max_lanes<16>(blind ? 0 : lo));
    }
    const long long cap = (long long)a.b.width << a.page_shift;
    const int end = hi_max < cap ? hi_max : (int)cap;
    const int first = PICK ? from : sp.tile0 + from > lo_min / KEYS ? sp.tile0 + from : lo_min / KEYS;
    const int past = end > lo_min ? (end + KEYS - 1) / KEYS : 0;
    const int stop = PICK ? upto : sp.tile0 + upto < past ? sp.tile0 + upto : past;
    // the row's list, and the positions that it sees
    const int32_t *list = PICK ? a.picks + ((long long)(sp.row0 + row_t.i) * a.c.heads + head) * a.n_picks : nullptr;
    const int sees = PICK ? key_hi(sp.at + row_t.i) : 0;

    // the listed pages of a wave's first tiles are asked for before the queries
    auto pick_of = [&](int tile) {
      const int p = (int)(((long long)tile * KEYS + 4 * r) >> a.page_shift);
      return tile < stop && p < a.n_picks ? list[p] : -1;
    };
    int tile = first + w;
    int pick = -1, next_pick = -1, after_pick = -1;
    if (PICK) {
      pick = pick_of(tile);
      next_pick = pick_of(tile + W);
      after_pick = pick_of(tile + 2 * W);
    }

    // the column's query, term t
    bf16x8 qf[C][2];
    const long long q_at = (long long)(sp.row0 + i) * a.q.row_stride + qh * a.q.head_stride;
    if constexpr (SEES == SEES_ALL) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float x[16];
        if (mine && g * C + c < tiles) {
          row_load_n(a.q, q_at + 16 * (g * C + c), x);
#pragma unroll
          for (int d = 0; d < 16; ++d) x[d] = query_term<T>(x[d], t) * a.q_sign;
        } else {
#pragma unroll
          for (int d = 0; d < 16; ++d) x[d] = 0.0f;
        }
        pack_query(x, qf[c]);
      }
    } else {
      switch (a.q.type) {
        case BFP_F32: load_query<C, T, BFP_F32>(a, q_at, g * C, mine, t, qf); break;
        case BFP_BF16: load_query<C, T, BFP_BF16>(a, q_at, g * C, mine, t, qf); break;
        case BFP_F16: load_query<C, T, BFP_F16>(a, q_at, g * C, mine, t, qf); break;
        default: load_query<C, T, BFP_TILES>(a, q_at, g * C, mine, t, qf); break;
      }
    }

    float m = -INFINITY, sum = 0.0f;
    f32x4 o[4 * C];
#pragma unroll
    for (int d = 0; d < 4 * C; ++d) o[d] = f32x4{0, 0, 0, 0};

    constexpr int PITCH = v_pitch(C);
    char *mylds = lds + w * V_ROWS * PITCH;
    const int swap = (r >> 2) & 1;
    char *vput0 = mylds + r * PITCH + g * C * 32 + 16 * swap, *vput1 = vput0 + 16 - 32 * swap;   // + 16 rows, + a tile
    const char *vget = mylds + (g * 4 + (r >> 2)) * PITCH + (((r & 3) ^ (2 * (g & 1))) * 8);        // + 16 rows, + a tile
    // The page number of a wave's tile is asked for two of its tiles ahead,
    // and looked at only when its bytes are asked for (8 sequences of 131072
    // tokens, 8 KV heads of 128: 151 us with one tile ahead, 149 so).
    auto page_of = [&](int tile) {
      const uint32_t p = slot_of(tile) >> a.page_shift;
      return tile < stop && p < (unsigned)a.b.width ? pages[p] : -1;
    };
    auto known = [&](int raw) { return (unsigned)raw < (unsigned)a.c.n_pages ? raw : -1; };
    // PICK: the listed pages are asked for three of the wave's tiles ahead
    auto picked = [&](int pick) { return (unsigned)pick < (unsigned)a.b.width ? pages[pick] : -1; };

    // K of the next tile is asked for when this one's scores are done, V when
    // this one's has gone to LDS: no second set of registers
    if (!early) {
      id = known(PICK ? picked(pick) : page_of(tile));
      at = offset_of(tile, id);
      load_side(k, a.c.k, a.c.k_e, at, a.c.page, g * C, tiles);
      load_side(v, a.c.v, a.c.v_e, at, a.c.page, g * C, tiles);
    }
    int next_raw = PICK ? picked(next_pick) : page_of(tile + W);
    for (; tile < stop; tile += W) {
      const int t0 = tile * KEYS;
      const int after_raw = PICK ? picked(after_pick) : page_of(tile + 2 * W), next_id = known(next_raw);
      const int third_pick = PICK ? pick_of(tile + 3 * W) : -1;
      const bool have = id >= 0;
      const unsigned long long okmask = __ballot(have);
      // PICK: how many of this lane's four keys the row sees
      const int seen = !PICK || !have ? 0 : sees - (pick << a.page_shift) - ((t0 + 4 * r) & (a.c.page - 1));
      const bool inner = PICK ? __all(seen >= 4) : t0 >= lo_max && t0 + KEYS <= hi_min && okmask == ~0ull;

      // scores: s[j][e] is key t0 + 16 g + 4 e + j of column r
      f32x4 s[4];
#pragma unroll
      for (int c = 0; c < C; ++c)   // a head tile that does not exist: its bytes must not make a NaN of 0 times them
        if (g * C + c >= tiles) k.e[c] = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[j] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < C; ++c) {
          const float sc = scale_of(k.e[c], j);
          const uint2 words = half_of(k.w[c], j);
          s[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kv4_decode8(words.x, sc), qf[c][0], s[j], 0, 0, 0);
          s[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kv4_decode8(words.y, sc), qf[c][1], s[j], 0, 0, 0);
        }
      }
      at = offset_of(tile + W, next_id);   // past the end: the first page, not used
      load_side(k, a.c.k, a.c.k_e, at, a.c.page, g * C, tiles);
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] = term_sum<T>(s[j][e]);
      if (!inner) {
        asm volatile("");   // a branch past all this, not selects every time
        if constexpr (PICK) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t ok = (uint32_t)__ballot(seen > j) >> (4 * g);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[j][e] = (ok >> e) & 1 ? s[j][e] : -INFINITY;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const bool ok = (okmask >> (4 * g + e)) & 1;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int key = t0 + 16 * g + 4 * e + j;
              s[j][e] = (ok & (key >= lo) & (key < hi)) ? s[j][e] : -INFINITY;
            }
          }
        }
        // values that no row of this workgroup sees become zeros, whatever their bytes
        uint32_t keep = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = t0 + 4 * r + j;
          keep |= (PICK ? seen > j : have & (key >= lo_min) & (key < end)) ? 1u << j : 0u;
        }
        const uint32_t bytes = byte_mask(keep);
        const uint32_t k0 = keep & 1 ? ~0u : 0u, k1 = keep & 2 ? ~0u : 0u, k2 = keep & 4 ? ~0u : 0u, k3 = keep & 8 ? ~0u : 0u;
#pragma unroll
        for (int c = 0; c < C; ++c) {
          v.e[c] &= bytes;
          v.w[c][0] = make_uint4(v.w[c][0].x & k0, v.w[c][0].y & k0, v.w[c][0].z & k1, v.w[c][0].w & k1);
          v.w[c][1] = make_uint4(v.w[c][1].x & k2, v.w[c][1].y & k2, v.w[c][1].z & k3, v.w[c][1].w & k3);
        }
      }

      // running maximum; a NaN score does not move it and makes its row NaN below
      float top = s[0][0];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, s[j][e]);
      top = fmaxf(top, fpeer<16>(top));
      top = fmaxf(top, fpeer<32>(top));
      const bool raise = top > m;
      if (__any(raise)) {
        const float mn = raise ? top + a.slack : m;
        const float f = raise ? exp2f((m - mn) * a.scale2) : 1.0f;   // from -infinity: 0
        m = mn;
        sum *= f;
#pragma unroll
        for (int d = 0; d < 4 * C; ++d) o[d] *= f;
      }
      const float m0 = m == -INFINITY ? 0.0f : -m * a.scale2;
      bf16x8 pb[2];
#pragma unroll
      for (int jp = 0; jp < 2; ++jp) {
        float pv[8];
#pragma unroll
        for (int jj = 0; jj < 2; ++jj)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p = __builtin_amdgcn_exp2f(fmaf(s[2 * jp + jj][e], a.scale2, m0));
            if (T > 1) sum += p;
            pv[4 * jj + e] = p;
          }
        pb[jp] = pack_terms<T>(pv, t);
        if constexpr (T == 1) {   // the sum takes the probabilities as the product takes them
#pragma unroll
          for (int e = 0; e < 8; e += 2)
            sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(s16x2, bf16x2{pb[jp][e], pb[jp][e + 1]}), s16x2{0x3f80, 0x3f80},
                                                  sum, false);
        }
      }

      // A tile of V that holds a NaN counts as zeros in the product, so that it
      // cannot reach a row that does not see it; the rows that do are set below.
      uint32_t bad = 0;
#pragma unroll
      for (int c = 0; c < C; ++c) bad |= has_byte_past(v.e[c]) && g * C + c < tiles ? 1u << c : 0u;
      const bool any_nan = __any(bad);
      uint32_t ve[C];
      if (any_nan) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
          ve[c] = v.e[c];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (((ve[c] >> (8 * j)) & 255u) < KV4_PAST) continue;
            v.e[c] &= ~(255u << (8 * j));
            (j & 1 ? v.w[c][j >> 1].z : v.w[c][j >> 1].x) = 0;
            (j & 1 ? v.w[c][j >> 1].w : v.w[c][j >> 1].y) = 0;
          }
        }
      }
#pragma unroll
      for (int jp = 0; jp < 2; ++jp) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int c = 0; c < C; ++c) {
#pragma unroll
          for (int jj = 0; jj < 2; ++jj) {
            const float sc = scale_of(v.e[c], 2 * jp + jj);
            const uint2 words = half_of(v.w[c], 2 * jp + jj);
            *(bf16x8 *)(vput0 + jj * 16 * PITCH + c * 32) = kv4_decode8(words.x, sc);
            *(bf16x8 *)(vput1 + jj * 16 * PITCH + c * 32) = kv4_decode8(words.y, sc);
          }
        }
        if (jp == 1) load_side(v, a.c.v, a.c.v_e, at, a.c.page, g * C, tiles);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int d = 0; d < 4 * C; ++d) {
          const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(vget + d * 32));
          const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(vget + 16 * PITCH + d * 32));
          const bf16x8 va = __builtin_bit_cast(bf16x8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
          o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, pb[jp], o[d], 0, 0, 0);
        }
      }
      if (any_nan) {
        uint8_t *le = (uint8_t *)mylds;   // exponents, (key, 16 tiles)
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int j = 0; j < 4; ++j) le[(4 * r + j) * 16 + g * C + c] = (uint8_t)(ve[c] >> (8 * j));
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int d = 0; d < 4 * C; ++d) {
          bool hit = false;
          if constexpr (PICK) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint32_t ok = (uint32_t)__ballot(seen > j);
#pragma unroll 1
              for (int k = 0; k < 16; ++k) hit |= (le[16 * (4 * k + j) + d] >= KV4_PAST) & (((ok >> k) & 1) != 0);
            }
          } else {
#pragma unroll 1
            for (int key = 0; key < KEYS; ++key) hit |= (le[16 * key + d] >= KV4_PAST) & (t0 + key >= lo) & (t0 + key < hi);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) o[d][e] = hit ? NAN : o[d][e];
        }
      }
      id = next_id;
      next_raw = after_raw;
      if (PICK) {
        pick = next_pick;
        next_pick = after_pick;
        after_pick = third_pick;
      }
    }

    if (SEES == SEES_PREFIX && blind) {
      m = -INFINITY;
      sum = 0.0f;
#pragma unroll
      for (int d = 0; d < 4 * C; ++d) o[d] = f32x4{0, 0, 0, 0};
    }

    // join the terms, then the waves
    sum += fpeer<16>(sum);
    sum += fpeer<32>(sum);
    __syncthreads();
    const int hd = 16 * tiles, stride = join_floats(R, tiles);
    float *jw = (float *)lds + w * stride;
    if (g == 0) {
      jw[r] = m * a.scale2;   // base-2 logarithm from here on
      jw[16 + r] = sum;
    }
#pragma unroll
    for (int d = 0; d < 4 * C; ++d) {
      if (d < tiles) {
        f32x4 v = o[d];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = term_sum<T>(T == 4 && t == 3 ? 0.0f : v[e]);
        if (r < R) *(f32x4 *)(jw + 32 + r * (hd + 4) + 16 * d + 4 * g) = v;
      }
    }
    __syncthreads();
    const float *jf = (const float *)lds;
    if constexpr (SEES != SEES_ALL && !SHARE && W <= 4) {
      // the rows' factors once, then eight values a thread: with few threads the
      // factors for every 16 values cost 5 us more (two waves, 8 rows of 128)
      float *factor = (float *)lds + W * stride, *top = factor + R * W, *total = top + R;
      for (int u = threadIdx.x; u < 16 * R; u += 64 * W) {
        const int row = u >> 4, k = u & 15;
        const float mk = k < W ? jf[k * stride + row] : -INFINITY, M = max16(mk);
        const float f = mk == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mk - M);
        const float L = sum16(k < W ? f * jf[k * stride + 16 + row] : 0.0f);
        if (k < W) factor[row * W + k] = f;
        if (k == 0) top[row] = M, total[row] = L;
      }
      __syncthreads();
      for (int u = threadIdx.x; u < R * 2 * tiles; u += 64 * W) {   // a tile's two halves in neighbouring lanes
        const int row = u / (2 * tiles), d = 8 * (u - row * 2 * tiles);
        if (rr0 + row >= rows) break;
        float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < W; ++k) {
          const float f = factor[row * W + k];
          const f32x4 *p = (const f32x4 *)(jf + k * stride + 32 + row * (hd + 4) + d);
          const f32x4 x = p[0], y = p[1];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[e] += f * x[e];
            v[4 + e] += f * y[e];
          }
        }
        const float L = total[row];
        const long long tok = sp.row0 + token_of<SEES>(a, row_t, rr0 + row);
        const int rh = head * G + head_of<SEES>(a, rr0 + row);
        if (SEES >= SEES_PREFIX) {
          const long long at = sum_place<SEES>(a, tok, rh);
          if (d == 0) a.part_ml[at] = make_float2(top[row], L);
          float4 *p = (float4 *)(a.part_o + at * hd + d);
          p[0] = make_float4(v[0], v[1], v[2], v[3]);
          p[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = L == 0.0f ? 0.0f : v[e] / L;
          out_store8(a.out, tok * a.out.row_stride + rh * a.out.head_stride + d, v, a.out_wide);
        }
      }
      return;
    }
    // 16 lanes to a row's tile; lane k of them works out wave k's factor
    const int l16 = threadIdx.x & 15;
    for (int u = threadIdx.x >> 4; u < R * tiles; u += 4 * W) {
      const int row = u / tiles, d = 16 * (u % tiles) + l16;
      if (rr0 + row >= rows) break;   // all 16 lanes
      const float mk = l16 < W ? jf[l16 * stride + row] : -INFINITY, M = max16(mk);
      const float f = mk == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mk - M);
      const float L = sum16(l16 < W ? f * jf[l16 * stride + 16 + row] : 0.0f);
      float acc = 0.0f;
#pragma unroll
      for (int k = 0; k < W; ++k)
        acc += __shfl(f, (lane & 48) + k, 64) * jf[k * stride + 32 + row * (hd + 4) + d];
      const int ri = token_of<SEES>(a, row_t, rr0 + row), rh = head * G + head_of<SEES>(a, rr0 + row);
      const long long tok = sp.row0 + ri;
      if (slot >= 0) {
        if (d == 0) put(slot_ml<SEES>(a) + slot * R + row, make_float2(M, L));
        put(slot_o<SEES>(a) + ((long long)slot * R + row) * hd + d, acc);
      } else if (SEES >= SEES_PREFIX) {
        leave_sum<SEES>(a, tok, rh, d, make_float2(M, L), acc);
      } else {
        out_store(a.out, tok * a.out.row_stride + rh * a.out.head_stride + d, L == 0.0f ? 0.0f : acc / L);
      }
    }
    if (!(SHARE && a.stream)) return;
    if (slot >= 0) {
      // the row tile's parts are the pieces from p0 on
      const uint32_t p0 = begin / piece, parts = (begin + sp.tiles - 1) / piece - p0 + 1;
      stores_done();
      __syncthreads();
      if (w == 0) {
        const bool all = arrive(a.there, a.number, p0, block - p0, parts);
        if (lane == 0) st.last = all;
      }
      __syncthreads();
      if (st.last) join_parts<C, R, SEES>(a, lds, sp, head, rt, p0, (int)parts);
    }
    while (x < x_stop && x == st.before[seq + 1]) ++seq;   // and past sequences without rows
  }
}

template <int C, int T, int W, Kv4Sees SEES, bool SHARE>
__global__ __launch_bounds__(64 * W, rows_per_simd(C, W, SEES, SHARE)) void k_kv4_rows(Kv4AttnArgs a) {
  rows_block<C, T, W, SEES, SHARE>(a, blockIdx.x);
}

// Both parts of rows that share a prefix.
template <int C, int T, int W>
__global__ __launch_bounds__(64 * W, rows_per_simd(C, W, SEES_REST, false)) void k_kv4_parts(Kv4AttnArgs prefix, Kv4AttnArgs rest,
                                                                                             uint32_t prefix_blocks) {
  if (blockIdx.x < prefix_blocks)
    rows_block<C, T, W, SEES_PREFIX, false>(prefix, blockIdx.x);
  else
    rows_block<C, T, W, SEES_REST, false>(rest, blockIdx.x - prefix_blocks);
}

// 64 E values of a part at a time, row after row; a lane has E of them under
// way for each of its wave's parts.
template <int E, Kv4Sees SEES>
__device__ __forceinline__ void join_values(const Kv4AttnArgs &a, const RowsSeq &sp, int head, const RowTile &row_t, uint32_t p0,
                                            int parts, int R, int values, const float *factor, const float *total,
                                            const float *top, float *sums) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, G = a.group, hd = 16 * a.tiles;
  for (int v0 = 0; v0 < values; v0 += 64 * E) {
    float acc[E];
    int at[E], row[E];   // past the last value: the last one, not taken
#pragma unroll
    for (int e = 0; e < E; ++e) {
      acc[e] = 0.0f;
      at[e] = v0 + 64 * e + lane < values ? v0 + 64 * e + lane : values - 1;
      row[e] = at[e] / hd;
    }
#pragma unroll 2
    for (int k = w; k < parts; k += 4) {
      const float *o = slot_o<SEES>(a) + (long long)part_slot(p0, (uint32_t)k) * R * hd;
      float x[E];
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = get(o + at[e]);
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] += factor[k * R + row[e]] * x[e];
    }
#pragma unroll
    for (int e = 0; e < E; ++e) sums[w * 64 * E + 64 * e + lane] = acc[e];
    __syncthreads();
    for (int u = threadIdx.x; u < 64 * E && v0 + u < values; u += 256) {   // whole groups of 16 lanes
      const int r = (v0 + u) / hd, rr = row_t.rr0 + r;
      const float L = total[r], sum = (sums[u] + sums[64 * E + u]) + (sums[128 * E + u] + sums[192 * E + u]);
      const long long tok = sp.row0 + token_of<SEES>(a, row_t, rr);
      const int qh = head * G + head_of<SEES>(a, rr);
      if (SEES >= SEES_PREFIX)
        leave_sum<SEES>(a, tok, qh, (v0 + u) % hd, make_float2(top[r], L), sum);
      else
        out_store(a.out, tok * a.out.row_stride + qh * a.out.head_stride + (v0 + u) % hd, L == 0.0f ? 0.0f : sum / L);
    }
    __syncthreads();
  }
}

// A row tile's rows from the parts of their keys.  All of a workgroup of four
// waves: the parts' factors first, then every wave takes each fourth part, a
// lane the same values of all of them.
template <int C, int R, Kv4Sees SEES>
__device__ void join_parts(const Kv4AttnArgs &a, char *lds, const RowsSeq &sp, int head, int rt, uint32_t p0, int parts) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, hd = 16 * a.tiles;
  const RowTile row_t = row_tile<R, SEES>(a, sp, rt);
  const int left = row_t.rows - row_t.rr0, rows = left < R ? left : R;
  float *factor = (float *)lds, *total = factor + MAX_PARTS * R, *top = total + R, *sums = top + R;   // [part][R], [R] x 2, [4][1024]
  auto slot = [&](int k) { return (long long)part_slot(p0, (uint32_t)k) * R; };
  for (int row = w; row < rows; row += 4) {
    float2 ml[MAX_PARTS / 64];
    float M = -INFINITY, L = 0.0f;
#pragma unroll
    for (int k = 0; k < MAX_PARTS / 64; ++k) {
      ml[k] = 64 * k + lane < parts ? get(slot_ml<SEES>(a) + slot(64 * k + lane) + row) : make_float2(-INFINITY, 0.0f);
      M = fmaxf(M, ml[k].x);
    }
    M = wave_max(M);
#pragma unroll
    for (int k = 0; k < MAX_PARTS / 64; ++k) {
      // a part that saw nothing (or NaN scores alone, whose sum is NaN): factor 0
      const float f = ml[k].x == -INFINITY ? 0.0f : exp2f(ml[k].x - M);
      L += f * ml[k].y;
      if (64 * k + lane < parts) factor[(64 * k + lane) * R + row] = f;
    }
    L = wave_sum(L);
    if (lane == 0) total[row] = L, top[row] = M;
  }
  __syncthreads();
  const int values = rows * hd;
  if (C == 1 || values <= 512)   // 16 need more registers than the narrow heads' kernels have
    join_values<8, SEES>(a, sp, head, row_t, p0, parts, R, values, factor, total, top, sums);
  else
    join_values<16, SEES>(a, sp, head, row_t, p0, parts, R, values, factor, total, top, sums);
}

static int rows_lds(int C, int W, int R, int tiles, bool share) {
  int lds = W * V_ROWS * v_pitch(C);
  for (int n : {(W * join_floats(R, tiles) + (W <= 4 ? R * (W + 2) : 0)) * 4, share ? (MAX_PARTS * R + 2 * R + 4096) * 4 : 0})
    lds = n > lds ? n : lds;
  return lds;
}

template <int C, int W, Kv4Sees SEES, bool SHARE = W == 4>
static AttnKernel rows_kernel_of(int tiles, int terms) {
  const int R = 16 / terms;
  const int lds = rows_lds(C, W, R, tiles, SHARE);
  return {terms == 1 ? k_kv4_rows<C, 1, W, SEES, SHARE> : terms == 2 ? k_kv4_rows<C, 2, W, SEES, SHARE> : k_kv4_rows<C, 4, W, SEES, SHARE>, lds};
}

template <Kv4Sees SEES>
static AttnKernel rows_kernel_for(int tiles, int terms, int waves, bool share) {
  const int C = (tiles + 3) / 4;
  if constexpr (SEES == SEES_PICKS) {
    if (waves == 2)
      return C == 1   ? rows_kernel_of<1, 2, SEES>(tiles, terms)
             : C == 2 ? rows_kernel_of<2, 2, SEES>(tiles, terms)
             : C == 3 ? rows_kernel_of<3, 2, SEES>(tiles, terms)
                      : rows_kernel_of<4, 2, SEES>(tiles, terms);
  }
  if (SEES == SEES_ALL) share = true;   // whether or not they do: one kernel
  if (waves == 4 && !share) {
    constexpr bool SHARE = SEES == SEES_ALL;
    return C == 1   ? rows_kernel_of<1, 4, SEES, SHARE>(tiles, terms)
           : C == 2 ? rows_kernel_of<2, 4, SEES, SHARE>(tiles, terms)
           : C == 3 ? rows_kernel_of<3, 4, SEES, SHARE>(tiles, terms)
                    : rows_kernel_of<4, 4, SEES, SHARE>(tiles, terms);
  }
  if (C == 1) return waves == 4 ? rows_kernel_of<1, 4, SEES>(tiles, terms) : rows_kernel_of<1, 16, SEES>(tiles, terms);
  if (C == 2) return waves == 4 ? rows_kernel_of<2, 4, SEES>(tiles, terms) : rows_kernel_of<2, 8, SEES>(tiles, terms);
  return C == 3 ? rows_kernel_of<3, 4, SEES>(tiles, terms) : rows_kernel_of<4, 4, SEES>(tiles, terms);
}

template <int C, int W>
static PartsKernel parts_kernel_of(int tiles, int terms) {
  return {terms == 4 ? k_kv4_parts<C, 4, W> : terms == 2 ? k_kv4_parts<C, 2, W> : k_kv4_parts<C, 1, W>,
          rows_lds(C, W, 16 / terms, tiles, false)};
}

}  // namespace bfp
