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
  __device__ uint32_t span() const { return (uint32_t)tiles + ROWS_EXTRA; }
};
__device__ __forceinline__ RowsSeq rows_seq(const Kv4AttnArgs &a, int R, int b) {
  const Kv4Span sp = kv4_span(a.b.start[b], a.b.start[b + 1], a.b.len[b], a.b.n_rows, a.b.max_q);
  RowsSeq s{sp.row0, sp.n, sp.at, 0, 1, 0};
  if (sp.n == 0) return s;
  const long long cap = (long long)a.b.width << a.page_shift;
  const int hi = key_hi(sp.at + sp.n - 1), end = hi < cap ? hi : (int)cap, lo = key_lo(key_hi(sp.at), a.window);
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
__device__ __forceinline__ uint32_t stream_plan(const Kv4AttnArgs &a, int R, Stream &st) {
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  uint32_t n = 0, most = 0;
  if (t < a.b.n_seq) {
    const RowsSeq s = rows_seq(a, R, t);
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
// R = 16 / T rows share); W: waves.
template <int C, int R>
__device__ void join_parts(const Kv4AttnArgs &a, char *lds, const RowsSeq &sp, int head, int rr0, uint32_t p0, int parts);

template <int C, int T, int W>
__global__ __launch_bounds__(64 * W, W > 8 ? 4 : C == 1 ? 3 : W > 4 || C == 2 ? 2 : 1) void k_kv4_rows(Kv4AttnArgs a) {
  constexpr int R = 16 / T;
  extern __shared__ __align__(16) char lds[];
  __shared__ Stream st;
  int seq, head, rt, split;
  uint32_t x = 0, x_stop = 1, piece = 0;
  if (W == 4 && a.stream) {
    piece = stream_plan(a, R, st);
    x = blockIdx.x * piece;
    const uint32_t all = st.before[a.b.n_seq];
    if (x >= all) return;
    x_stop = x + piece < all ? x + piece : all;
    seq = 0;
    for (int b = threadIdx.x & 63; b < a.b.n_seq; b += 64)   // every wave for itself
      seq += __popcll(__ballot(st.before[b + 1] <= x));
    seq = __builtin_amdgcn_readfirstlane(seq);
  } else {
    a.place(seq, head, split, rt);
  }
  const int G = a.group;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const int t = r / R;
  const int tiles = a.tiles;
  // one round takes keys of one row tile and KV head
  bool begun = false;
  while (x < x_stop) {
    const int32_t *pages = a.b.pages + (long long)seq * a.b.width;
    auto offset_of = [&](int tile, int id) {
      return kv4_tile(id < 0 ? 0 : id, a.c.heads, head, tiles, 0, a.c.page, (tile * KEYS + 4 * r) & (a.c.page - 1));
    };
    // Without a window a wave's first tile is known before the lengths are:
    // its page number and its bytes are on their way while those arrive.
    KvSide<C> k, v;
    int id = -1;
    long long at = 0;
    const bool early = !(W == 4 && a.stream) && a.window == 0;
    if (early) {
      id = kv4_page(pages, a.b.width, a.c.n_pages, (w * KEYS + 4 * r) >> a.page_shift);
      at = offset_of(w, id);
      load_side(k, a.c.k, a.c.k_e, at, a.c.page, g * C, tiles);
      load_side(v, a.c.v, a.c.v_e, at, a.c.page, g * C, tiles);
    }
    const RowsSeq sp = rows_seq(a, R, seq);
    int from = 0, upto = sp.tiles, slot = -1;
    uint32_t begin = 0;
    if (W == 4 && a.stream) {
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
      if (from > 0 || upto < sp.tiles) slot = 2 * blockIdx.x + (from == 0 ? 1 : 0);
      head = (int)(group % (uint32_t)a.c.heads);
      rt = (int)(group / (uint32_t)a.c.heads);
      if (begun) __syncthreads();   // the last round's sums have been read
      begun = true;
    } else {
      x = x_stop;
    }
    const int rows = sp.n * G;   // rows of this KV head: (token, query head)
    const int rr0 = rt * R;
    if (rr0 >= rows) return;     // never with shared work

    // this lane's column
    const int rr = rr0 + r % R;
    const bool mine = rr < rows;
    const int i = mine ? rr / G : 0, qh = head * G + (mine ? rr % G : 0);
    const int hi = mine ? key_hi(sp.at + i) : 0, lo = key_lo(hi, a.window);
    // what all of them see, and any of them
    const int last = (rr0 + R < rows ? rr0 + R : rows) - 1;
    const int hi_min = key_hi(sp.at + rr0 / G), hi_max = key_hi(sp.at + last / G);
    const int lo_min = key_lo(hi_min, a.window), lo_max = key_lo(hi_max, a.window);
    const long long cap = (long long)a.b.width << a.page_shift;
    const int end = hi_max < cap ? hi_max : (int)cap;
    const int first = sp.tile0 + from > lo_min / KEYS ? sp.tile0 + from : lo_min / KEYS;
    const int past = end > lo_min ? (end + KEYS - 1) / KEYS : 0;
    const int stop = sp.tile0 + upto < past ? sp.tile0 + upto : past;

    // the column's query, term t
    bf16x8 qf[C][2];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float x[16];
      if (mine && g * C + c < tiles) {
        row_load_n(a.q, (long long)(sp.row0 + i) * a.q.row_stride + qh * a.q.head_stride + 16 * (g * C + c), x);
#pragma unroll
        for (int d = 0; d < 16; ++d) x[d] = query_term<T>(x[d], t) * a.q_sign;
      } else {
#pragma unroll
        for (int d = 0; d < 16; ++d) x[d] = 0.0f;
      }
      float y[8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int d = 0; d < 8; ++d) y[d] = x[8 * h + d];
        qf[c][h] = pack8(y);
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
      const int p = (tile * KEYS + 4 * r) >> a.page_shift;
      return tile < stop && (unsigned)p < (unsigned)a.b.width ? pages[p] : -1;
    };
    auto known = [&](int raw) { return (unsigned)raw < (unsigned)a.c.n_pages ? raw : -1; };

    // K of the next tile is asked for when this one's scores are done, V when
    // this one's has gone to LDS: no second set of registers
    int tile = first + w;
    if (!early) {
      id = known(page_of(tile));
      at = offset_of(tile, id);
      load_side(k, a.c.k, a.c.k_e, at, a.c.page, g * C, tiles);
      load_side(v, a.c.v, a.c.v_e, at, a.c.page, g * C, tiles);
    }
    int next_raw = page_of(tile + W);
    for (; tile < stop; tile += W) {
      const int t0 = tile * KEYS;
      const int after_raw = page_of(tile + 2 * W), next_id = known(next_raw);
      const bool have = id >= 0;
      const unsigned long long okmask = __ballot(have);
      const bool inner = t0 >= lo_max && t0 + KEYS <= hi_min && okmask == ~0ull;

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
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool ok = (okmask >> (4 * g + e)) & 1;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int key = t0 + 16 * g + 4 * e + j;
            s[j][e] = (ok & (key >= lo) & (key < hi)) ? s[j][e] : -INFINITY;
          }
        }
        // values that no row of this workgroup sees become zeros, whatever their bytes
        uint32_t keep = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = t0 + 4 * r + j;
          keep |= (have & (key >= lo_min) & (key < end)) ? 1u << j : 0u;
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
#pragma unroll 1
          for (int key = 0; key < KEYS; ++key) hit |= (le[16 * key + d] >= KV4_PAST) & (t0 + key >= lo) & (t0 + key < hi);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[d][e] = hit ? NAN : o[d][e];
        }
      }
      id = next_id;
      next_raw = after_raw;
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
      const int ri = (rr0 + row) / G, rh = head * G + (rr0 + row) % G;
      const long long tok = sp.row0 + ri;
      if (slot >= 0) {
        if (d == 0) put(a.part_ml + slot * R + row, make_float2(M, L));
        put(a.part_o + ((long long)slot * R + row) * hd + d, acc);
      } else {
        out_store(a.out, tok * a.out.row_stride + rh * a.out.head_stride + d, L == 0.0f ? 0.0f : acc / L);
      }
    }
    if (!(W == 4 && a.stream)) return;
    if (slot >= 0) {
      // the row tile's parts are the pieces from p0 on
      const uint32_t p0 = begin / piece, parts = (begin + sp.tiles - 1) / piece - p0 + 1;
      stores_done();
      __syncthreads();
      if (w == 0) {
        const bool all = arrive(a.there, a.number, p0, blockIdx.x - p0, parts);
        if (lane == 0) st.last = all;
      }
      __syncthreads();
      if (st.last) join_parts<C, R>(a, lds, sp, head, rr0, p0, (int)parts);
    }
    while (x < x_stop && x == st.before[seq + 1]) ++seq;   // and past sequences without rows
  }
}

// 64 E values of a part at a time, row after row; a lane has E of them under
// way for each of its wave's parts.
template <int E>
__device__ __forceinline__ void join_values(const Kv4AttnArgs &a, const RowsSeq &sp, int head, int rr0, uint32_t p0, int parts,
                                            int R, int values, const float *factor, const float *total, float *sums) {
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
      const float *o = a.part_o + (long long)part_slot(p0, (uint32_t)k) * R * hd;
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
      const int r = (v0 + u) / hd, rr = rr0 + r;
      const float L = total[r], sum = (sums[u] + sums[64 * E + u]) + (sums[128 * E + u] + sums[192 * E + u]);
      out_store(a.out, (long long)(sp.row0 + rr / G) * a.out.row_stride + (head * G + rr % G) * a.out.head_stride + (v0 + u) % hd,
                L == 0.0f ? 0.0f : sum / L);
    }
    __syncthreads();
  }
}

// A row tile's rows from the parts of their keys.  All of a workgroup of four
// waves: the parts' factors first, then every wave takes each fourth part, a
// lane the same values of all of them.
template <int C, int R>
__device__ void join_parts(const Kv4AttnArgs &a, char *lds, const RowsSeq &sp, int head, int rr0, uint32_t p0, int parts) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, G = a.group, hd = 16 * a.tiles;
  const int left = sp.n * G - rr0, rows = left < R ? left : R;
  float *factor = (float *)lds, *total = factor + MAX_PARTS * R, *sums = total + R;   // [part][R], [R], [4][1024]
  auto slot = [&](int k) { return (long long)part_slot(p0, (uint32_t)k) * R; };
  for (int row = w; row < rows; row += 4) {
    float2 ml[MAX_PARTS / 64];
    float M = -INFINITY, L = 0.0f;
#pragma unroll
    for (int k = 0; k < MAX_PARTS / 64; ++k) {
      ml[k] = 64 * k + lane < parts ? get(a.part_ml + slot(64 * k + lane) + row) : make_float2(-INFINITY, 0.0f);
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
    if (lane == 0) total[row] = L;
  }
  __syncthreads();
  const int values = rows * hd;
  if (C == 1 || values <= 512)   // 16 need more registers than the narrow heads' kernels have
    join_values<8>(a, sp, head, rr0, p0, parts, R, values, factor, total, sums);
  else
    join_values<16>(a, sp, head, rr0, p0, parts, R, values, factor, total, sums);
}

template <int C, int W>
static AttnKernel pick(int tiles, int terms) {
  const int R = 16 / terms;
  int lds = W * V_ROWS * v_pitch(C);
  for (int n : {W * join_floats(R, tiles) * 4, (MAX_PARTS * R + R + 4096) * 4}) lds = n > lds ? n : lds;
  return {terms == 1 ? k_kv4_rows<C, 1, W> : terms == 2 ? k_kv4_rows<C, 2, W> : k_kv4_rows<C, 4, W>, lds};
}

AttnKernel rows_kernel(int tiles, int terms, int waves) {
  const int C = (tiles + 3) / 4;
  if (C == 1) return waves == 4 ? pick<1, 4>(tiles, terms) : pick<1, 16>(tiles, terms);
  if (C == 2) return waves == 4 ? pick<2, 4>(tiles, terms) : pick<2, 8>(tiles, terms);
  return C == 3 ? pick<3, 4>(tiles, terms) : pick<4, 4>(tiles, terms);
}

}  // namespace bfp
