// Bounds of each page's keys, and the pages that a score picks for each row.
//
// lo_d and hi_d are the least and the largest key of channel d in a page.  No
// key of the page has a product with q above sum_d max(q_d lo_d, q_d hi_d), and
// summed over the heads that share the keys that is
//   score = sum_d hi_d P_d + lo_d N_d,  P_d = sum max(q_d, 0),  N_d = sum min(q_d, 0):
// one product of length 2 hd a page, whatever the heads.  Cached keys have two
// significant bits, so bounds are exact in bfloat16 and lie in memory as the
// matrix cores take them.
#include <math.h>

#include "bfp_kv4_attn.h"

namespace bfp {

constexpr int BOUND_T = 256;
constexpr uint32_t BOUND_NAN = 0x7fc07fc0u;

typedef short i16x2 __attribute__((ext_vector_type(2)));

struct Kv4BoundArgs {
  bfp_kv4 c;
  bfp_kv4_batch b;
  uint16_t *bounds;
  int touched, lanes_shift;   // pages that a sequence's new rows can lie in; log2 of page / 4
  FastDiv by_group, by_head, by_touched;   // groups of tiles, one a wave; heads; pages of a sequence
  long long n_units;
};

// bfloat16 as numbers that compare as whole ones do (and back).
__device__ __forceinline__ i16x2 sortable(i16x2 v) { return v ^ ((v >> 15) & (short)0x7fff); }
__device__ __forceinline__ i16x2 lane_xor(i16x2 v, int m) {
  return __builtin_bit_cast(i16x2, __shfl_xor(__builtin_bit_cast(int, v), m, 64));
}

// A lane takes four tokens of one tile, as they lie side by side; the lanes
// of a tile join.  Bound by one chain of loads (lengths, page number, bytes): three
// ragged prompts of up to 8192 tokens, 8 heads of 128, 6.4 us for 8.6 MB, 64
// sequences' last pages 4.2.
__global__ __launch_bounds__(BOUND_T) void k_kv4_bounds(Kv4BoundArgs a) {
  const long long u64 = (long long)blockIdx.x * (BOUND_T / 64) + (threadIdx.x >> 6);
  if (u64 >= a.n_units) return;
  uint32_t group, head, j;
  const uint32_t seq = a.by_touched.div(a.by_head.div(a.by_group.div((uint32_t)u64, group), head), j);
  const Kv4Span s = kv4_span(a.b.start[seq], a.b.start[seq + 1], a.b.len[seq], a.b.n_rows, a.b.max_q);
  const int stop = s.at + s.n, first = s.at > 0 ? s.at : 0;
  if (s.n == 0 || stop <= first) return;
  const int page = a.c.page, p = first / page + (int)j;
  if (p > (stop - 1) / page) return;
  const int id = kv4_page(a.b.pages + (long long)seq * a.b.width, a.b.width, a.c.n_pages, p);
  if (id < 0) return;
  const int lane = threadIdx.x & 63, tiles = a.c.hd / 16, lanes = 1 << a.lanes_shift;
  const int tile = (int)group * (64 >> a.lanes_shift) + (lane >> a.lanes_shift), slot = 4 * (lane & (lanes - 1));
  const bool mine = tile < tiles;
  const long long o = kv4_tile(id, a.c.heads, (int)head, tiles, mine ? tile : tiles - 1, page, slot);
  const uint4 *d = (const uint4 *)(a.c.k + o * KV4_TILE_BYTES);
  const uint4 w[2] = {d[0], d[1]};
  const uint32_t e = *(const uint32_t *)(a.c.k_e + o);
  const int held = stop - p * page;   // slots of this page that hold a token

  i16x2 lo[8], hi[8];
  uint32_t bad = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) lo[i] = i16x2{0x7fff, 0x7fff}, hi[i] = i16x2{-0x8000, -0x8000};
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const bool have = slot + t < held;
    const uint32_t E = (e >> (8 * t)) & 255u;
    bad |= have && E >= KV4_PAST ? 1u : 0u;
    const float sc = kv4_scale(E);
    const uint32_t words[2] = {t & 1 ? w[t >> 1].z : w[t >> 1].x, t & 1 ? w[t >> 1].w : w[t >> 1].y};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4 v = __builtin_bit_cast(uint4, kv4_decode8(words[h], sc));
      const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const i16x2 y = sortable(__builtin_bit_cast(i16x2, x[i]));
        if (have) {
          lo[4 * h + i] = __builtin_elementwise_min(lo[4 * h + i], y);
          hi[4 * h + i] = __builtin_elementwise_max(hi[4 * h + i], y);
        }
      }
    }
  }
  for (int m = 1; m < lanes; m *= 2) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      lo[i] = __builtin_elementwise_min(lo[i], lane_xor(lo[i], m));
      hi[i] = __builtin_elementwise_max(hi[i], lane_xor(hi[i], m));
    }
    bad |= __shfl_xor(bad, m, 64);
  }
  if (!mine || (lane & (lanes - 1)) > 1) return;
  // the tile's first lane writes the least ones, its second the largest
  const bool upper = lane & 1;
  uint32_t y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const i16x2 x = sortable(upper ? hi[i] : lo[i]);
    y[i] = bad ? BOUND_NAN : __builtin_bit_cast(uint32_t, x);
  }
  uint4 *to = (uint4 *)(a.bounds + (((long long)id * a.c.heads + head) * 2 + (upper ? 1 : 0)) * a.c.hd + 16 * tile);
  to[0] = make_uint4(y[0], y[1], y[2], y[3]);
  to[1] = make_uint4(y[4], y[5], y[6], y[7]);
}

// ------------------------------------------------------------------- scores
// Scores in float32 on the bfloat16 matrix cores, P and N in three terms of
// eight bits, and how far they may be from the exact ones.  The choice is
// exact all the same: with every score within e of its value, pages more than
// 2 e above the n-th largest are surely picked and those more than 2 e below it
// surely not; what lies between is scored again in float64 (k_kv4_pick).
struct Kv4PickArgs {
  bfp_kv4 c;
  bfp_kv4_batch b;
  bfp_rows q;
  const uint16_t *bounds;
  int group, i0, rows;        // rows i0 .. i0 + rows - 1 of every sequence
  int products;               // that are added up to a score
  int n, first, last;         // pages to pick; of these the first and the last ones, whatever their scores
  int chunks, chunk;          // pieces of the pages, and how many pages each has
  FastDiv by_head, by_chunk, by_tile;
  float *score;               // [sequence][row][head][width]
  float *off;                 // [sequence][row][head][chunk]: sums of the products' magnitudes, at most
  int32_t *picks;
};

constexpr int PICK_WIDTH = 16384;         // pages of a table: a bit each, twice, and scores have to fit the LDS
constexpr int SCORE_W = 4;                // waves

// The last page that row i of a span sees, -1: none.
__device__ __forceinline__ int own_page(const Kv4PickArgs &a, const Kv4Span &s, int i) {
  const int p = s.at + i;
  if (p < 0) return -1;
  const int q = p / a.c.page;
  return q < a.b.width ? q : a.b.width - 1;
}

// Eight values of N and P from offset o on, for query heads `stride` apart.
// One branch on the type, so that the heads' loads are under way together
// (behind a branch each they took a microsecond apiece).
template <int TYPE>
__device__ __forceinline__ void group_sums_of(bfp_rows q, long long o, long long stride, int group, float (&N)[8], float (&P)[8]) {
  q.type = TYPE;
#pragma unroll 4
  for (int h = 0; h < group; ++h) {
    float x[8];
    row_load_n(q, o + h * stride, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool is = x[e] == x[e];
      N[e] += is ? fminf(x[e], 0.0f) : NAN;
      P[e] += is ? fmaxf(x[e], 0.0f) : NAN;
    }
  }
}
__device__ __forceinline__ void group_sums(const bfp_rows &q, long long o, int group, float (&N)[8], float (&P)[8]) {
  switch (q.type) {
    case BFP_F32: group_sums_of<BFP_F32>(q, o, q.head_stride, group, N, P); break;
    case BFP_BF16: group_sums_of<BFP_BF16>(q, o, q.head_stride, group, N, P); break;
    case BFP_F16: group_sums_of<BFP_F16>(q, o, q.head_stride, group, N, P); break;
    default: group_sums_of<BFP_TILES>(q, o, q.head_stride, group, N, P); break;
  }
}

// R: rows of a wave's matrix tile.  16: their terms multiply one after the
// other; 4: the terms are columns of the tile.  K: steps of 32 values (hd / 16).
// The waves share P and N, each works out some of the steps, and each takes
// every fourth 16 pages, whose operands are loaded as they lie, the next ones
// while these are multiplied.  One row: bound by the bytes of the bounds (8 rows
// over up to 2048 pages, 8 heads of 128: 42 MB in 16 us, 2.6 TB/s; much of it is the
// first loads and the queries' sums).  Many: by four products a step where one
// is the score's (1021 rows of up to 1024 pages, 4 heads: 32 us).
template <int R, int K>
__global__ __launch_bounds__(64 * SCORE_W, K <= 8 ? 4 : 2) void k_kv4_score(Kv4PickArgs a) {
  constexpr int T = R == 16 ? 3 : 1;
  __shared__ bf16x8 coefs[T * K * 64];
  __shared__ float waves[SCORE_W][16];
  uint32_t chunk, rt, head;   // neighbours take the heads of the same pages
  const int seq = (int)a.by_tile.div(a.by_chunk.div(a.by_head.div(blockIdx.x, head), chunk), rt);
  const Kv4Span s = kv4_span(a.b.start[seq], a.b.start[seq + 1], a.b.len[seq], a.b.n_rows, a.b.max_q);
  const int i0 = a.i0 + (int)rt * R, stop = a.i0 + a.rows < s.n ? a.i0 + a.rows : s.n;
  if (i0 >= stop) return;
  const int ilast = i0 + R < stop ? i0 + R - 1 : stop - 1;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
  const int base = (int)chunk * a.chunk, all = own_page(a, s, ilast) + 1, pages = base + a.chunk < all ? base + a.chunk : all;
  // all of them are taken, or there are none here
  if (all <= a.n || base >= pages) return;
  const int hd = a.c.hd, i = i0 + col % R;
  const bool mine = i < stop;
  const int32_t *table = a.b.pages + (long long)seq * a.b.width;
  auto page_of = [&](int p0) { return p0 + col < pages ? kv4_page(table, a.b.width, a.c.n_pages, p0 + col) : -1; };
  auto fetch = [&](int id, bf16x8 (&v)[K]) {   // a page that does not exist: the first one's, not used
    const bf16x8 *from = (const bf16x8 *)(a.bounds + ((long long)(id < 0 ? 0 : id) * a.c.heads + head) * 2 * hd + 8 * g);
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = from[4 * k];
  };
  int p0 = base + 16 * w;
  constexpr int STEP = 16 * SCORE_W;
  int id = page_of(p0), next_id = page_of(p0 + STEP);
  bf16x8 v[2][K];
  fetch(id, v[0]);
  fetch(next_id, v[1]);
  // a column: dims 32 k + 8 g .. + 7 of [N | P]; eight dims' N and P by one lane
  auto put = [&](int at, const float (&sum)[8]) {
#pragma unroll
    for (int t = 0; t < T; ++t) {
      const int term = R == 16 ? t : col / R;
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = term < 3 ? query_term<3>(sum[e], term) : 0.0f;
      coefs[(t * K + at / 32) * 64 + 16 * (at / 8 % 4) + col] = pack8(y);
    }
  };
  constexpr bool HALF = K <= SCORE_W;   // as many waves for N alone, and for P
#pragma unroll
  for (int k0 = 0; 2 * k0 < K; k0 += SCORE_W) {
    const int d = 32 * (k0 + (HALF ? w / 2 : w)) + 8 * g;
    if (d >= hd) break;
    float N[8], P[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) N[e] = P[e] = 0.0f;
    if (mine)
      group_sums(a.q, (long long)(s.row0 + i) * a.q.row_stride + (long long)head * a.group * a.q.head_stride + d, a.group, N, P);
    if (!HALF || w % 2 == 0) put(d, N);
    if (!HALF || w % 2 == 1) put(hd + d, P);
  }
  __syncthreads();
  // (read again for every tile: in registers those of 16 rows leave room for two waves a SIMD)
  auto coef = [&](int t, int k) { return coefs[(t * K + k) * 64 + lane]; };
  const long long out = ((long long)seq * a.rows + (i - a.i0)) * a.c.heads + head;
  float most = 0.0f;
#pragma unroll 1
  for (; p0 < pages; p0 += 2 * STEP) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {   // the bytes of the tile after the next are asked for when this one's have been used
      const int first = p0 + u * STEP;
      if (first >= pages) break;
      asm volatile("" ::: "memory");   // the coefficients stay in LDS
      f32x4 sc = {0, 0, 0, 0}, mag = {0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int t = 0; t < T; ++t) sc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[u][k], coef(t, k), sc, 0, 0, 0);
        typedef unsigned u4 __attribute__((ext_vector_type(4)));
        const u4 va = __builtin_bit_cast(u4, v[u][k]) & 0x7fff7fffu, ca = __builtin_bit_cast(u4, coef(0, k)) & 0x7fff7fffu;
        mag = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, va), __builtin_bit_cast(bf16x8, ca), mag, 0, 0, 0);
      }
      const unsigned long long there = __ballot(id >= 0);
      id = next_id;
      if (first + 2 * STEP < pages) {
        next_id = page_of(first + 2 * STEP);
        fetch(next_id, v[u]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x = sc[e], m = mag[e];
        if (R == 4) {
          x = term_sum<4>(x);
          m = term_sum<4>(m);
        }
        const int page = first + 4 * g + e;
        if (!mine || page >= pages || (R == 4 && col >= R)) continue;
        const bool ok = (there >> (4 * g + e)) & 1;
        if (ok) most = fabsf(x) < INFINITY ? fmaxf(most, m) : INFINITY;
        a.score[out * a.b.width + page] = ok ? fmaxf(x, -0x1.fffffep127f) : -INFINITY;   // -infinity: no page
      }
    }
  }
  // over the column's four lanes, then the waves
  most = fmaxf(most, fpeer<16>(most));
  most = fmaxf(most, fpeer<32>(most));
  if (g == 0) waves[w][col] = most;
  __syncthreads();
  if (threadIdx.x < R && mine)
    a.off[out * a.chunks + chunk] = fmaxf(fmaxf(waves[0][col], waves[1][col]), fmaxf(waves[2][col], waves[3][col]));
}

// -------------------------------------------------------------------- picks
__device__ __forceinline__ uint32_t key_of(float f) {
  const uint32_t b = __float_as_uint(f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
__device__ __forceinline__ unsigned long long key_of(double f) {
  if (f != f) return ~0ull;   // a NaN counts as the largest
  const unsigned long long b = (unsigned long long)__double_as_longlong(f + 0.0);   // -0 is 0
  return b >> 63 ? ~b : b | 0x8000000000000000ull;
}

// Sums over a workgroup of W waves of three numbers that each wave counted
// (below 2^21 in all): one word a wave, which as many lanes read and add up.  Two
// sets of places in turn, one barrier a call.  (Every thread reading all of the
// waves' counts took 0.9 us a call with 16 waves.)
template <int W>
struct Counter {
  unsigned long long (*place)[W];
  int turn;
  __device__ void add(int (&n)[3]) {
    if ((threadIdx.x & 63) == 0)
      place[turn][threadIdx.x >> 6] = (unsigned long long)n[0] | (unsigned long long)n[1] << 21 | (unsigned long long)n[2] << 42;
    __syncthreads();
    long long v = (long long)place[turn][threadIdx.x & (W - 1)];
    if (W > 8) v += peer<8>(v);
    if (W > 4) v += peer<4>(v);
    v += peer<2>(v);
    v += peer<1>(v);
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)((unsigned long long)v >> 32));
    const unsigned long long u = (unsigned long long)hi << 32 | lo;
    n[0] = (int)(u & 0x1fffff);
    n[1] = (int)((u >> 21) & 0x1fffff);
    n[2] = (int)(u >> 42);
    turn ^= 1;
  }
};

// A key that exactly `want` of the n keys reach, or, where there is none, the
// largest that more do.  Two bits a round.
template <int W, typename Key>
__device__ __forceinline__ Key nth_key(int n, int want, const Key *key, Counter<W> &count) {
  Key at = 0;
#pragma unroll 1
  for (int bit = 8 * (int)sizeof(Key) - 2; bit >= 0; bit -= 2) {
    const Key q[3] = {at | (Key)1 << bit, at | (Key)2 << bit, at | (Key)3 << bit};
    int c[3] = {0, 0, 0};
    for (int p0 = 0; p0 < n; p0 += 64 * W) {
      const int p = p0 + threadIdx.x;
      const Key k = p < n ? key[p] : 0;
#pragma unroll
      for (int u = 0; u < 3; ++u) c[u] += __popcll(__ballot(k >= q[u]));
    }
    count.add(c);
    int reach = 0;
#pragma unroll
    for (int u = 0; u < 3; ++u)
      if (c[u] >= want) at = q[u], reach = c[u];
    if (reach == want) break;
  }
  return at;
}

// The least of the keys that reach `at` (there is one).
template <int W>
__device__ __forceinline__ uint32_t least_key(int n, uint32_t at, const uint32_t *key, uint32_t *waves) {
  uint32_t v = 0xffffffffu;
  for (int p = threadIdx.x; p < n; p += 64 * W) v = key[p] >= at && key[p] < v ? key[p] : v;
#pragma unroll
  for (int d = 32; d > 0; d /= 2) {
    const uint32_t x = __shfl_xor(v, d, 64);
    v = x < v ? x : v;
  }
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = v;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < W; ++k) v = waves[k] < v ? waves[k] : v;
  return v;
}

// The want-th largest of the n values whose keys are not 0, out of `count` of
// them, between least and most.  Bins of equal width first, then, in one wave,
// those of the bin in which it lies; by its bits where they are more than a
// wave's lanes.  (By bits alone: 9 us of 14 for 2048 pages.)
constexpr int BINS = 256;
struct BinSpace {
  int bins[BINS], n;
  uint32_t list[64], found;
};
template <int W>
__device__ __forceinline__ float nth_value(int n, int want, const uint32_t *key, float least, float most, BinSpace &b, uint32_t *waves,
                                           Counter<W> &count) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const float scale = (BINS - 1) / (most - least);   // 0, infinite or NaN: all in one bin
  auto bin_of = [&](uint32_t k) {
    const float x = (of_key(k) - least) * scale;     // does not fall where the value rises
    return x > 0.0f ? (int)fminf(x, (float)(BINS - 1)) : 0;
  };
  for (int i = threadIdx.x; i < BINS; i += 64 * W) b.bins[i] = 0;
  if (threadIdx.x == 0) b.n = 0;
  __syncthreads();
  for (int p = threadIdx.x; p < n; p += 64 * W)
    if (key[p]) atomicAdd(&b.bins[bin_of(key[p])], 1);
  __syncthreads();
  // every wave: the bin, from above, in which the count reaches `want`
  int mine[BINS / 64], sum = 0;   // lane l: bins from BINS - 1 - 4 l down
#pragma unroll
  for (int i = 0; i < BINS / 64; ++i) sum += mine[i] = b.bins[BINS - 1 - (BINS / 64 * lane + i)];
  int up = sum;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int x = __shfl_up(up, d, 64);
    up += lane >= d ? x : 0;
  }
  int above = up - sum, bin = -1, held = 0;
#pragma unroll
  for (int i = 0; i < BINS / 64; ++i) {
    if (bin < 0 && above + mine[i] >= want) bin = BINS - 1 - (BINS / 64 * lane + i), held = mine[i];
    if (bin < 0) above += mine[i];
  }
  const int from = __ffsll((unsigned long long)__ballot(bin >= 0)) - 1;   // the first lane that reaches it
  bin = __shfl(bin, from, 64);
  held = __shfl(held, from, 64);
  const int rank = want - __shfl(above, from, 64);   // in the bin, from 1
  if (held > 64) return of_key(least_key<W>(n, nth_key<W, uint32_t>(n, want, key, count), key, waves));
  for (int p = threadIdx.x; p < n; p += 64 * W)
    if (key[p] && bin_of(key[p]) == bin) b.list[atomicAdd(&b.n, 1)] = key[p];
  __syncthreads();
  if (w == 0) {
    const uint32_t x = lane < held ? b.list[lane] : 0;
    int r = 0, same = 0;   // how many are larger, and how many are alike
    for (int u = 0; u < held; ++u) {
      const uint32_t y = (uint32_t)__builtin_amdgcn_readlane((int)x, u);
      r += y > x;
      same += y == x;
    }
    if (lane < held && r < rank && rank <= r + same) b.found = x;   // all that write it write the same
  }
  __syncthreads();
  return of_key(b.found);
}

// The exact score of a page, by eight neighbouring lanes; coef: N and P in
// float64.
__device__ __forceinline__ double exact_score(const Kv4PickArgs &a, int id, int head, const double *coef) {
  const int hd = a.c.hd, l = threadIdx.x & 7;
  const uint16_t *v = a.bounds + ((long long)id * a.c.heads + head) * 2 * hd;
  double sum = 0.0;
  for (int d = 8 * l; d < 2 * hd; d += 64) {
    const uint4 x = *(const uint4 *)(v + d);
    const uint32_t y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sum = __builtin_fma((double)__uint_as_float(y[i] << 16), coef[d + 2 * i], sum);
      sum = __builtin_fma((double)__uint_as_float(y[i] & 0xffff0000u), coef[d + 2 * i + 1], sum);
    }
  }
  sum += __shfl_xor(sum, 1, 64);
  sum += __shfl_xor(sum, 2, 64);
  return sum + __shfl_xor(sum, 4, 64);
}

// One row and KV head a workgroup of W waves.  Bound by its rounds of the
// workgroup's waves, one after the other, each a barrier and a pass over LDS (64
// rows and heads over 2048 pages 13 us, 4084 over 1024 36).  words: a bit for every page
// that is taken, and for every one that may be; then the scores as keys, in
// float32 and, of those at the border, in float64.
template <int W>
__global__ __launch_bounds__(64 * W) void k_kv4_pick(Kv4PickArgs a) {
  extern __shared__ __align__(16) unsigned long long words[];
  __shared__ unsigned long long places[2][W];
  __shared__ float tops[W], ends[W][2];
  __shared__ uint32_t least[W];
  __shared__ BinSpace bins;
  __shared__ double coef[512];
  __shared__ int lie_before[PICK_WIDTH / 64];   // pages of the border before each word
  const int head = blockIdx.y, seq = (int)(blockIdx.x / (unsigned)a.rows), i = a.i0 + (int)(blockIdx.x % (unsigned)a.rows);
  const Kv4Span s = kv4_span(a.b.start[seq], a.b.start[seq + 1], a.b.len[seq], a.b.n_rows, a.b.max_q);
  if (i >= s.n) return;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int n = own_page(a, s, i) + 1;   // pages that it sees
  const int32_t *table = a.b.pages + (long long)seq * a.b.width;
  int32_t *to = a.picks + ((long long)(s.row0 + i) * a.c.heads + head) * a.n;
  const long long in = ((long long)seq * a.rows + (i - a.i0)) * a.c.heads + head;
  const float *score = a.score + in * a.b.width;
  const int n_words = (n + 63) / 64;
  unsigned long long *take = words, *border = words + n_words, *keys = border + n_words;
  uint32_t *key32 = (uint32_t *)keys;   // 0: not to be picked
  Counter<W> count{places, 0};
  auto forced = [&](int p) { return p < a.first || p >= n - a.last; };

  // The forced pages that exist, the others that do, and how far scores may be off.
  int c[3] = {0, 0, 0};
  const bool all = n <= a.n;
  float low = INFINITY, high = -INFINITY;
  for (int p0 = 0; p0 < n; p0 += 64 * W) {
    const int p = p0 + threadIdx.x;
    const float x = p < n && !all && !forced(p) ? score[p] : -INFINITY;
    const bool there = p < n && (all || forced(p) ? kv4_page(table, a.b.width, a.c.n_pages, p) >= 0 : x != -INFINITY);
    if (p < n) key32[p] = x == -INFINITY ? 0u : key_of(x);
    low = x == -INFINITY ? low : fminf(low, x);
    high = fmaxf(high, x);
    const unsigned long long f = __ballot(there && (all || forced(p)));
    c[0] += __popcll(f);
    c[1] += __popcll(__ballot(there && !all && !forced(p)));
    if (lane == 0 && p0 + 64 * w < n) take[p0 / 64 + w] = f;
  }
  if (!all) {
    low = -wave_max(-low);
    high = wave_max(high);
    if (lane == 0) ends[w][0] = low, ends[w][1] = high;
  }
  count.add(c);
  int want = a.n - c[0];
  want = want < c[1] ? want : c[1];
  if (want > 0 && want == c[1]) {
    for (int p0 = 0; p0 < n; p0 += 64 * W) {
      const int p = p0 + threadIdx.x;
      const unsigned long long f = __ballot(p < n && key32[p] != 0);
      if (lane == 0 && p0 + 64 * w < n) take[p0 / 64 + w] |= f;
    }
  } else if (want > 0) {
    float most = 0.0f;
    for (int k = threadIdx.x; k * a.chunk < n; k += 64 * W) most = fmaxf(most, a.off[in * a.chunks + k]);
    most = wave_max(most);
    if (lane == 0) tops[w] = most;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < W; ++k) most = fmaxf(most, tops[k]);
    // Every product that is added to a sum, 2^-23 of the sum of the magnitudes
    // each (the matrix cores may cut): 2 hd, or three times as many where the
    // terms go one after the other into one sum (a.products).  In what is
    // added: P and N themselves (sums of the group's queries in float32, 2^-24
    // each) and the joining of sums that hold a term each, of which the
    // second and third are 2^-7 and 2^-14 of the first.  Magnitudes are of the
    // first terms at least, 1 - 2^-7 of the whole.
    const float e2 = 2.0f * (a.products + a.group + 16) * 0x1.06p-23f * most + 0x1p-120f;
    const bool exact_all = !(e2 < 0x1p120f);
    float A = 0.0f;
    if (!exact_all) {
#pragma unroll
      for (int k = 0; k < W; ++k) low = fminf(low, ends[k][0]), high = fmaxf(high, ends[k][1]);
      A = nth_value<W>(n, want, key32, low, high, bins, least, count);
    }
    c[0] = c[1] = c[2] = 0;
    for (int p0 = 0; p0 < n; p0 += 64 * W) {
      const int p = p0 + threadIdx.x;
      const uint32_t k = p < n ? key32[p] : 0u;
      const bool free = exact_all ? p < n && !forced(p) && kv4_page(table, a.b.width, a.c.n_pages, p) >= 0 : k != 0;
      const float x = free && !exact_all ? of_key(k) - A : 0.0f;
      const unsigned long long in_set = __ballot(free && x > e2), between = __ballot(free && !(x > e2) && !(x < -e2));
      c[0] += __popcll(in_set);
      c[1] += __popcll(between);
      if (lane == 0 && p0 + 64 * w < n) {
        take[p0 / 64 + w] |= in_set;
        border[p0 / 64 + w] = between;
      }
    }
    count.add(c);
    want -= c[0];
    if (want >= c[1]) {   // all of them
      for (int k = threadIdx.x; k < n_words; k += 64 * W) take[k] |= border[k];
    } else {
      // P and N, then the border's scores in float64 over the approximate ones' keys
      for (int d = threadIdx.x; d < 2 * a.c.hd; d += 64 * W) {
        double sum = 0.0;
        const bool upper = d >= a.c.hd;
        for (int h = 0; h < a.group; ++h) {
          const double x = row_load(a.q, (long long)(s.row0 + i) * a.q.row_stride + (head * a.group + h) * a.q.head_stride + (upper ? d - a.c.hd : d));
          sum += x != x ? x : upper ? fmax(x, 0.0) : fmin(x, 0.0);
        }
        coef[d] = sum;
      }
      if (w == 0) {
        int before = 0;
        for (int k0 = 0; k0 < n_words; k0 += 64) {
          const int mine = k0 + lane < n_words ? __popcll(border[k0 + lane]) : 0;
          int up = mine;
#pragma unroll
          for (int d = 1; d < 64; d *= 2) {
            const int x = __shfl_up(up, d, 64);
            up += lane >= d ? x : 0;
          }
          if (k0 + lane < n_words) lie_before[k0 + lane] = before + up - mine;
          before += __shfl(up, 63, 64);
        }
      }
      __syncthreads();
      // Page u of the border: the last word with no more than u before it, and its bit.
      auto page_at = [&](int u) {
        int k = 0, past = n_words;
        while (past - k > 1) {
          const int mid = k + (past - k) / 2;
          (lie_before[mid] <= u ? k : past) = mid;
        }
        unsigned long long m = border[k];
        int left = u - lie_before[k], at = 0;
#pragma unroll
        for (int half = 32; half > 0; half /= 2) {
          const int low = __popcll(m & ((1ull << half) - 1));
          if (left >= low) left -= low, m >>= half, at += half;
        }
        return 64 * k + at;
      };
      const int m = c[1];   // pages of the border; keys: their scores, in order
      for (int u = threadIdx.x >> 3; u < m; u += 8 * W) {   // eight lanes a page
        const int id = kv4_page(table, a.b.width, a.c.n_pages, page_at(u));
        const double sc = exact_score(a, id < 0 ? 0 : id, head, coef);
        if ((threadIdx.x & 7) == 0) keys[u] = key_of(sc);
      }
      __syncthreads();
      if (m <= 64) {   // one wave: each page by how many come before it
        if (w == 0) {
          const unsigned long long mine = lane < m ? keys[lane] : 0;
          int r = 0;
          for (int u = 0; u < m; ++u) {
            const unsigned long long x = keys[u];
            r += x > mine || (x == mine && u < lane);
          }
          if (lane < m && r < want) {
            const int p = page_at(lane);
            atomicOr(take + p / 64, 1ull << (p & 63));
          }
        }
      } else {
        // T: what the last one taken has (or more reach: then the first of those at T)
        const unsigned long long T = nth_key<W, unsigned long long>(m, want, keys, count);
        c[0] = c[1] = c[2] = 0;
        for (int u0 = 0; u0 < m; u0 += 64 * W) {
          const int u = u0 + threadIdx.x;
          c[0] += __popcll(__ballot(u < m && keys[u] >= T));
          c[1] += __popcll(__ballot(u < m && keys[u] > T));
        }
        count.add(c);
        int ties = c[0] == want ? m : want - c[1];   // of those at T the first
        // page by page, in order: one wave
        if (w == 0) {
          for (int k = 0; k < n_words; ++k) {
            const unsigned long long b = border[k], below = (1ull << lane) - 1;
            const bool is = (b >> lane) & 1;
            const unsigned long long x = is ? keys[lie_before[k] + __popcll(b & below)] : 0;
            const unsigned long long equal = __ballot(is && x == T), above = __ballot(is && x > T);
            const bool tie = is && x == T && __popcll(equal & below) < ties;
            const unsigned long long got = above | __ballot(tie);
            const int used = __popcll(equal);
            ties = ties > used ? ties - used : 0;
            if (lane == 0) take[k] |= got;
          }
        }
      }
    }
  }
  __syncthreads();
  // in the pages' order: a wave takes 64 words at a time
  int before = 0;
  for (int k0 = 0; k0 < n_words; k0 += 64) {
    const unsigned long long m = k0 + lane < n_words ? take[k0 + lane] : 0;
    int up = __popcll(m);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int x = __shfl_up(up, d, 64);
      up += lane >= d ? x : 0;
    }
    const int mine = before + up - __popcll(m);
    for (int k = k0 + w; k < k0 + 64 && k < n_words; k += W) {
      const unsigned long long word = take[k];
      const int at = __shfl(mine, k - k0, 64) + __popcll(word & ((1ull << lane) - 1));
      if ((word >> lane) & 1) to[at] = 64 * k + lane;
    }
    before += __shfl(up, 63, 64);
  }
  for (int k = before + threadIdx.x; k < a.n; k += 64 * W) to[k] = -1;
}

// ---------------------------------------------------------------------- host
static int check_bounds(const char *op, const void *bounds) {
  if (!bounds || (uintptr_t)bounds % 16) return set_err(BFP_EINVAL, "%s: bounds are null or not 16-byte aligned", op);
  return BFP_OK;
}

constexpr size_t PICK_SCRATCH = (size_t)256 << 20;   // at most, unless one row of each sequence needs more
constexpr int PICK_CHUNKS = 256;

struct PickPlan {
  int rows, R, chunks, chunk;   // rows of a sequence in a piece, and of a matrix tile
  size_t scores, work;
};
static PickPlan plan_pick(const bfp_kv4 &c, const bfp_kv4_batch &b) {
  PickPlan p;
  const int rows = b.max_q < b.n_rows ? b.max_q : b.n_rows;
  const size_t row = (size_t)b.n_seq * c.heads * ((size_t)b.width + PICK_CHUNKS) * sizeof(float);
  size_t most = PICK_SCRATCH / row;
  if (most >= 16) most = most / 16 * 16;
  p.rows = most < 1 ? 1 : most < (size_t)rows ? (int)most : rows;
  p.R = p.rows > 4 ? 16 : 4;
  // 512 workgroups, each with 64 pages or more (1021 rows of 1024 pages, 4 heads: 34 us
  // with a thousand, 32 so, 36 with 256; 7 rows of 2048, 8 heads: 17.1, 16.1, 19.5)
  const long long tiles = (long long)((p.rows + p.R - 1) / p.R) * c.heads * b.n_seq;
  long long chunks = 512 / tiles;
  if (chunks > (b.width + 63) / 64) chunks = (b.width + 63) / 64;
  if (chunks > PICK_CHUNKS) chunks = PICK_CHUNKS;
  if (chunks < 1) chunks = 1;
  p.chunk = (int)((b.width + chunks - 1) / chunks + 63) / 64 * 64;
  p.chunks = (b.width + p.chunk - 1) / p.chunk;
  p.scores = (size_t)b.n_seq * p.rows * c.heads * b.width;
  p.work = (p.scores + (size_t)b.n_seq * p.rows * c.heads * p.chunks) * sizeof(float);
  return p;
}

static int check_pick(const char *op, const bfp_kv4 *cache, const bfp_kv4_batch *batch, const bfp_rows *q) {
  BFP_TRY(check_kv4(op, cache, batch));
  if (!q || q->heads < cache->heads || q->heads % cache->heads || q->heads > 65536)
    return set_err(BFP_EINVAL, "%s: q has %d heads, the cache %d", op, q ? q->heads : 0, cache->heads);
  BFP_TRY(check_rows(op, "q", q, q->heads, cache->hd, true, batch->n_rows));
  if (!rows_aligned(*q, 8, batch->n_rows)) return set_err(BFP_EINVAL, "%s: q needs 16-byte alignment and strides in multiples of 8", op);
  if (batch->width > PICK_WIDTH) return set_err(BFP_EINVAL, "%s: width=%d pages, at most %d", op, batch->width, PICK_WIDTH);
  return BFP_OK;
}

typedef void (*score_fn)(Kv4PickArgs);
template <int R>
static score_fn score_kernel(int k) {
  static const score_fn fn[16] = {k_kv4_score<R, 1>,  k_kv4_score<R, 2>,  k_kv4_score<R, 3>,  k_kv4_score<R, 4>,
                                  k_kv4_score<R, 5>,  k_kv4_score<R, 6>,  k_kv4_score<R, 7>,  k_kv4_score<R, 8>,
                                  k_kv4_score<R, 9>,  k_kv4_score<R, 10>, k_kv4_score<R, 11>, k_kv4_score<R, 12>,
                                  k_kv4_score<R, 13>, k_kv4_score<R, 14>, k_kv4_score<R, 15>, k_kv4_score<R, 16>};
  return fn[k - 1];
}

}  // namespace bfp

using namespace bfp;

extern "C" {

int bfp_kv4_bounds_d(const bfp_kv4 *cache, const bfp_kv4_batch *batch, uint16_t *bounds, void *stream) {
  const char *op = "kv4_bounds";
  BFP_TRY(check_kv4(op, cache, batch));
  BFP_TRY(check_bounds(op, bounds));
  if (batch->n_seq == 0 || batch->max_q == 0 || batch->n_rows == 0) return BFP_OK;
  Kv4BoundArgs a{};
  a.c = *cache;
  a.b = *batch;
  a.bounds = bounds;
  const int rows = batch->max_q < batch->n_rows ? batch->max_q : batch->n_rows;
  a.touched = (int)(((long long)rows + cache->page - 2) / cache->page + 1);
  a.touched = a.touched < batch->width ? a.touched : batch->width;
  a.lanes_shift = __builtin_ctz((unsigned)cache->page) - 2;
  const int each = 64 >> a.lanes_shift, groups = (cache->hd / 16 + each - 1) / each;
  a.by_group = FastDiv(groups);
  a.by_head = FastDiv(cache->heads);
  a.by_touched = FastDiv(a.touched);
  a.n_units = (long long)batch->n_seq * a.touched * cache->heads * groups;
  if (a.n_units > 0x3ffffff) return set_err(BFP_EINVAL, "%s: n_seq=%d of max_q=%d rows are too many for one call", op, batch->n_seq, batch->max_q);
  hipLaunchKernelGGL(k_kv4_bounds, dim3((unsigned)((a.n_units + BOUND_T / 64 - 1) / (BOUND_T / 64))), dim3(BOUND_T), 0,
                     (hipStream_t)stream, a);
  return launch_status(op);
}

size_t bfp_kv4_select_work(const bfp_kv4 *cache, const bfp_kv4_batch *batch, const bfp_rows *q) {
  if (check_pick("kv4_select_work", cache, batch, q) || batch->n_seq == 0 || batch->max_q == 0 || batch->n_rows == 0) return 0;
  return plan_pick(*cache, *batch).work;
}

int bfp_kv4_select_d(const bfp_kv4 *cache, const bfp_kv4_batch *batch, const uint16_t *bounds, const bfp_rows *q, int n, int first,
                     int last, int32_t *picks, void *work, size_t work_bytes, void *stream) {
  const char *op = "kv4_select";
  BFP_TRY(check_pick(op, cache, batch, q));
  BFP_TRY(check_bounds(op, bounds));
  if (n < 1 || (long long)n * cache->page > KV4_MAX_POS || first < 0 || last < 1 || first > n - last)
    return set_err(BFP_EINVAL, "%s: n=%d pages, first=%d and last=%d of them", op, n, first, last);
  if (batch->n_seq == 0 || batch->max_q == 0 || batch->n_rows == 0) return BFP_OK;
  if (!picks || (uintptr_t)picks % 4) return set_err(BFP_EINVAL, "%s: picks are null or not aligned", op);
  const PickPlan p = plan_pick(*cache, *batch);
  if (!work || (uintptr_t)work % 16 || work_bytes < p.work)
    return set_err(BFP_EINVAL, "%s: needs %zu bytes of 16-byte-aligned scratch, got %zu", op, p.work, work ? work_bytes : (size_t)0);
  const int rows = batch->max_q < batch->n_rows ? batch->max_q : batch->n_rows;
  const long long tiles = (p.rows + p.R - 1) / p.R, blocks = tiles * p.chunks * batch->n_seq, pick_blocks = (long long)p.rows * batch->n_seq;
  // 2^32 threads a launch
  if (blocks * cache->heads > 0xffffff || pick_blocks * cache->heads > 0x3fffff)
    return set_err(BFP_EINVAL, "%s: n_seq=%d of max_q=%d rows are too many for one call", op, batch->n_seq, batch->max_q);
  Kv4PickArgs a{};
  a.c = *cache;
  a.b = *batch;
  a.q = *q;
  a.bounds = bounds;
  a.group = q->heads / cache->heads;
  a.rows = p.rows;
  a.products = (p.R == 16 ? 3 : 1) * 2 * cache->hd;
  a.n = n, a.first = first, a.last = last;
  a.chunks = p.chunks;
  a.chunk = p.chunk;
  a.by_head = FastDiv(cache->heads);
  a.by_chunk = FastDiv(p.chunks);
  a.by_tile = FastDiv((uint32_t)tiles);
  a.score = (float *)work;
  a.off = a.score + p.scores;
  a.picks = picks;
  const score_fn score = p.R == 4 ? score_kernel<4>(cache->hd / 16) : score_kernel<16>(cache->hd / 16);
  const size_t lds = (size_t)(batch->width + 63) / 64 * 16 + (size_t)batch->width * 8;
  // few workgroups: more waves each (4084 rows of 1024 pages: 35 us with four, 56 with one)
  const int W = pick_blocks * cache->heads <= 512 ? 16 : 4;
  const score_fn pick = W == 16 ? k_kv4_pick<16> : k_kv4_pick<4>;
  if (lds > 49152) HIP_TRY(hipFuncSetAttribute((const void *)pick, hipFuncAttributeMaxDynamicSharedMemorySize, 136 * 1024));
  for (a.i0 = 0; a.i0 < rows; a.i0 += p.rows) {
    hipLaunchKernelGGL(score, dim3((unsigned)(blocks * cache->heads)), dim3(64 * SCORE_W), 0, (hipStream_t)stream, a);
    BFP_TRY(launch_status(op));
    hipLaunchKernelGGL(pick, dim3((unsigned)pick_blocks, cache->heads), dim3(64 * W), lds, (hipStream_t)stream, a);
    BFP_TRY(launch_status(op));
  }
  return BFP_OK;
}

}  // extern "C"
