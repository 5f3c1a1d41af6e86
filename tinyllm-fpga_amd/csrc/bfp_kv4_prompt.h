// Attention over the 4-bit cache for prompts, whole or in pieces.
//
// A workgroup takes 32 rows a wave of one sequence and KV head (a row is a
// token and one of the query heads that share the KV head), all waves the
// same 64 keys.  Each key tile is decoded once into LDS as bfloat16 while the
// one before it is multiplied.  The matrix tiles are 32 x 32: an operand read
// from LDS (1 KB) feeds 16384 products.  As for few rows, the keys are the
// rows of S^T, and the probabilities stay in place.
//
// SEES_PREFIX, SEES_REST: the two parts of rows that share a prefix, left
// unfinished.  All rows of a group are one sequence in the first: a prefix is
// read and decoded once for up to 256 of them.  As in prompts, exponentials and
// products take turns (matrix cores busy 45%): three documents of up to 65536 tokens
// with 239 rows of 16 heads behind them 200-234 us, 0.6 of the matrix product's rate
// in two terms.  64 samples' rows behind 16384 tokens, 256 a KV head: 49 us in two
// terms, of which the eight key tiles a workgroup has are 30, its first loads and
// its results the rest.
#pragma once
#include "bfp_kv4_attn.h"

namespace bfp {

typedef float f32x16 __attribute__((ext_vector_type(16)));

// K rows: read 16 bytes a lane, 32 rows at a time; 16 bytes past the row put
// eight neighbouring rows in different banks.  V rows: read by transposing
// loads of 4 rows x 64 bytes, which an odd multiple of 64 bytes spreads.
constexpr int pk_pitch(int tb) { return 32 * tb + 16; }
constexpr int pv_pitch(int tb) { return 64 * ((tb / 2) | 1); }
// A tile of K, and of V with its exponent bytes (key, 16 tiles).
constexpr int k_bytes(int tb) { return KEYS * pk_pitch(tb); }
constexpr int v_bytes(int tb) { return KEYS * (pv_pitch(tb) + 16); }
// Two workgroups a CU: four waves of heads and terms for which there are eight too.
constexpr bool in_pairs(int tb, int t, int w) { return w == 4 && t < 3 && tb <= 8; }
// Tiles of V held: with three, one barrier a tile is enough; the widest heads,
// and pairs of wide ones, leave room for two, and take a second barrier.
constexpr int v_buffers(int tb, bool pair) { return tb <= (pair ? 6 : 12) ? 3 : 2; }
constexpr int OUT_PITCH = 36;   // floats: 32 values of a row, on their way out
constexpr int prompt_lds(int tb, int t, int waves) {
  const int in = 2 * k_bytes(tb) + v_buffers(tb, in_pairs(tb, t, waves)) * v_bytes(tb), out = waves * (32 * OUT_PITCH + 64) * 4;
  return in > out ? in : out;
}

// A lane's part of a row's query, all loads under way together: behind a branch
// on the type each, as where one row tile follows another, they take 3 us.
template <int TB, int T, int TYPE>
__device__ __forceinline__ void prompt_query(const Kv4AttnArgs &a, long long at, bool mine, bf16x8 (&qf)[T][TB]) {
  bfp_rows q = a.q;
  q.type = TYPE;
  float x[TB][8];
#pragma unroll
  for (int c = 0; c < TB; ++c) {
#pragma unroll
    for (int d = 0; d < 8; ++d) x[c][d] = 0.0f;
    if (mine && c < a.tiles) row_load_n(q, at + 16 * c, x[c]);
  }
#pragma unroll
  for (int c = 0; c < TB; ++c)
#pragma unroll
    for (int t = 0; t < T; ++t) {
      float y[8];
#pragma unroll
      for (int d = 0; d < 8; ++d) y[d] = query_term<T>(x[c][d], t) * a.q_sign;
      qf[t][c] = pack8(y);
    }
}

// TB: tiles of the head the loops are built for (even; a narrower head's
// missing tiles are zeros in K, and columns of V whose results nobody
// takes); T: terms; W: waves.
template <int TB, int T, int W, Kv4Sees SEES>
__global__ __launch_bounds__(64 * W, W == 8 || in_pairs(TB, T, W) ? 2 : 1) void k_kv4_prompt(Kv4AttnArgs a) {
  constexpr int ROWS = 32 * W, DT = TB / 2, UNITS = (TB + W - 1) / W;
  constexpr int KP = pk_pitch(TB), VP = pv_pitch(TB), NV = v_buffers(TB, in_pairs(TB, T, W));
  extern __shared__ __align__(16) char lds[];
  __shared__ int nan_tiles[4];
  int seq, head, rt, split, splits = a.splits, chunk = a.chunk;
  if (SEES == SEES_PREFIX && a.pieces) {
    if (!a.piece(ROWS, seq, head, split, rt, splits, chunk)) return;
  } else {
    a.place(blockIdx.x, seq, head, split, rt);
  }
  Kv4Group of{};
  const Kv4Span sp = SEES == SEES_PREFIX ? kv4_group_span(a, seq, of)
                                         : kv4_span(a.b.start[seq], a.b.start[seq + 1], a.b.len[seq], a.b.n_rows, a.b.max_q);
  const int low = SEES == SEES_REST ? kv4_shared_len(a, seq) : 0;
  const int G = a.group, rows = sp.n * G;
  if (rt >= (rows + ROWS - 1) / ROWS) return;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, h = lane >> 5;
  const int tiles = a.tiles;
  const int wg0 = rt * ROWS, rr0 = wg0 + 32 * w, rr = rr0 + n;
  const bool mine = rr < rows;
  uint32_t qg;
  const int i = (int)a.by_group.div((uint32_t)(mine ? rr : 0), qg), qh = head * G + (int)qg;
  // what any of the workgroup's rows sees
  const int glast = (wg0 + ROWS < rows ? wg0 + ROWS : rows) - 1;
  int begin = key_lo(key_hi(sp.at + wg0 / G), a.window);
  int top_hi = key_hi(sp.at + glast / G);
  if (SEES == SEES_REST) begin = begin > low ? begin : low;
  if (SEES == SEES_PREFIX) {
    begin = __builtin_amdgcn_readfirstlane(kv4_group_low(a, of));
    top_hi = sp.at;
  }
  const long long cap = (long long)a.b.width << a.page_shift;
  const int end = top_hi < cap ? top_hi : (int)cap;
  const int tile0 = begin / KEYS, n_tiles = end > begin ? (end + KEYS - 1) / KEYS - tile0 : 0;
  const KeyPart part = key_part(n_tiles, split, splits, chunk);
  const int first = tile0 + part.first, stop = tile0 + part.stop;

  // this lane's row, and what the wave's rows all see
  int hi = mine ? key_hi(sp.at + i) : 0, lo = key_lo(hi, a.window);
  const int wfirst = rr0 < rows ? rr0 : rows - 1, wlast = (rr0 + 32 < rows ? rr0 + 32 : rows) - 1;
  int hi_min = key_hi(sp.at + wfirst / G), lo_max = key_lo(rr0 < rows ? key_hi(sp.at + wlast / G) : 0, a.window);
  if (SEES == SEES_REST) {
    lo = lo > low ? lo : low;
    lo_max = lo_max > low ? lo_max : low;
  }
  bool blind = false;   // SEES_PREFIX: the row sees none of it; what is worked out for it is thrown away, not masked
  bf16x8 qf[T][TB];
  // SEES_PREFIX, whose rows are of several sequences: by each one's position
  auto take_rows = [&]() __attribute__((always_inline)) {
    uint32_t rest;
    const int row = (int)a.by_group.div((uint32_t)(mine ? rr : rows - 1), rest);
    const int ends = key_hi(kv4_row_position<32>(a, of, sp.row0 + row));
    lo = mine ? key_lo(ends, a.window) : 0;
    hi = mine ? (ends < sp.at ? ends : sp.at) : 0;
    blind = hi <= lo;
    hi_min = __builtin_amdgcn_readfirstlane(min_lanes<32>(blind ? 0x7fffffff : hi));
    lo_max = __builtin_amdgcn_readfirstlane(max_lanes<32>(blind ? 0 : lo));
    const long long q_at = (long long)(sp.row0 + i) * a.q.row_stride + qh * a.q.head_stride + 8 * h;
    switch (a.q.type) {
      case BFP_F32: prompt_query<TB, T, BFP_F32>(a, q_at, mine, qf); break;
      case BFP_BF16: prompt_query<TB, T, BFP_BF16>(a, q_at, mine, qf); break;
      case BFP_F16: prompt_query<TB, T, BFP_F16>(a, q_at, mine, qf); break;
      default: prompt_query<TB, T, BFP_TILES>(a, q_at, mine, qf); break;
    }
  };
  if constexpr (SEES != SEES_PREFIX) {
#pragma unroll
    for (int c = 0; c < TB; ++c) {
      float x[8];
      if (mine && c < tiles) {
        row_load_n(a.q, (long long)(sp.row0 + i) * a.q.row_stride + qh * a.q.head_stride + 16 * c + 8 * h, x);
      } else {
#pragma unroll
        for (int d = 0; d < 8; ++d) x[d] = 0.0f;
      }
#pragma unroll
      for (int t = 0; t < T; ++t) {
        float y[8];
#pragma unroll
        for (int d = 0; d < 8; ++d) y[d] = query_term<T>(x[d], t) * a.q_sign;
        qf[t][c] = pack8(y);
      }
    }
  }

  float m = -INFINITY, sum = 0.0f;
  f32x16 o[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[d][e] = 0.0f;

  const int32_t *pages = a.b.pages + (long long)seq * a.b.width;
  // wave w brings in head tiles w, w + W, ... of K and V, a key a lane
  struct Bytes {
    uint2 k[UNITS], v[UNITS];
    uint32_t ke[UNITS], ve[UNITS];
    bool there;
    unsigned long long ok;   // whose keys are there
  };
  // The page number of this lane's key, where some row sees the key; looked at
  // only when the page is fetched, a tile later: a use here would wait for it
  // and for the bytes asked for before it (two prompts of 8192 tokens, 32 heads
  // of 128: 870 us that way, 807 this way).
  auto page_of = [&](int tile) {
    if (tile >= stop) return -1;
    const int key = tile * KEYS + lane;
    int id = -1;
    if ((tile * KEYS >= begin && tile * KEYS <= end - KEYS) || (key >= begin && key < end)) id = pages[key >> a.page_shift];
    return id;
  };
  // a key without a page reads the first one's bytes; they are not used
  const uint32_t page_tiles = (uint32_t)a.c.heads * tiles * a.c.page;   // at most 2^24
  auto fetch = [&](Bytes &x, int tile, int id) __attribute__((always_inline)) {
    x.there = (unsigned)id < (unsigned)a.c.n_pages;
    const uint32_t slot = ((uint32_t)tile * KEYS + lane) & (a.c.page - 1);   // (unsigned: past the last tile)
    const unsigned long long at = (unsigned long long)(x.there ? (uint32_t)id : 0u) * page_tiles + slot;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int t = w + u * W;
      const long long from = kv4_tile(0, a.c.heads, head, tiles, t < tiles ? t : tiles - 1, a.c.page, 0);   // the same in every lane
      x.k[u] = ((const uint2 *)(a.c.k + from * KV4_TILE_BYTES))[at];
      x.v[u] = ((const uint2 *)(a.c.v + from * KV4_TILE_BYTES))[at];
      x.ke[u] = (a.c.k_e + from)[at];
      x.ve[u] = (a.c.v_e + from)[at];
    }
    x.ok = __ballot(x.there);
  };
  char *const k_lds = lds, *const v_lds = lds + 2 * k_bytes(TB);
  auto decode = [&](const Bytes &x, int t1) __attribute__((always_inline)) {   // tile first + t1
    char *kb = k_lds + (t1 & 1) * k_bytes(TB) + lane * KP, *vt = v_lds + t1 % NV * v_bytes(TB), *vb = vt + lane * VP;
    const int sw = (lane >> 1) & 3;   // 16-byte pieces of each 64 change places, for the writes' banks
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int t = w + u * W;
      if (UNITS * W > TB && t >= TB) break;
      const bool ok = x.there && t < tiles;   // zeros for what the head or the cache does not have
      const float ks = kv4_scale(x.ke[u]);
      bf16x8 *kd = (bf16x8 *)(kb + 32 * t);
      kd[0] = kv4_decode8(t < tiles ? x.k[u].x : 0u, ks);
      kd[1] = kv4_decode8(t < tiles ? x.k[u].y : 0u, ks);
      // NaN tiles of V count as zeros in the product; the rows that see them are set after
      const uint32_t E = ok ? x.ve[u] : 0u;
      const bool take = ok && E < KV4_PAST;
      vt[KEYS * VP + lane * 16 + t] = (char)E;
      if (E >= KV4_PAST) nan_tiles[t1 & 3] = 1;
      const float vs = kv4_scale(take ? E : 0u);
      *(bf16x8 *)(vb + 64 * (t >> 1) + 16 * ((2 * (t & 1)) ^ sw)) = kv4_decode8(take ? x.v[u].x : 0u, vs);
      *(bf16x8 *)(vb + 64 * (t >> 1) + 16 * ((2 * (t & 1) + 1) ^ sw)) = kv4_decode8(take ? x.v[u].y : 0u, vs);
    }
  };
  // scores of half a tile (32 keys), before any mask: s[e] is key 8 (e / 4) + 4 h + e % 4 of row n
  auto scores = [&](int t1, int u) {
    const char *kr = k_lds + (t1 & 1) * k_bytes(TB) + (32 * u + n) * KP + 16 * h;
    f32x16 s;
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] = 0.0f;
#pragma unroll
    for (int c = 0; c < TB; ++c) {
      const bf16x8 kf = *(const bf16x8 *)(kr + 32 * c);
#pragma unroll
      for (int t = 0; t < T; ++t) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[t][c], s, 0, 0, 0);
    }
    return s;
  };
  auto mask = [&](f32x16 &s, int tile, int u, unsigned long long ok) {
    const int t0 = tile * KEYS;
    if (t0 >= lo_max && t0 + KEYS <= hi_min && ok == ~0ull) return;
    asm volatile("");   // a branch past the selects, not selects every time
    const uint32_t okh = (uint32_t)(ok >> (32 * u)) >> (4 * h);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int k = 8 * (e >> 2) + (e & 3), key = t0 + 32 * u + 4 * h + k;
      s[e] = ((((okh >> k) & 1) != 0) & (key >= lo) & (key < hi)) ? s[e] : -INFINITY;
    }
  };
  auto top_of = [&](const f32x16 &s) {
    float top = s[0];
#pragma unroll
    for (int e = 0; e < 16; ++e) top = fmaxf(top, s[e]);
    return fmaxf(top, fpeer<32>(top));
  };

  const int vrow = 4 * h + ((lane & 15) >> 2);   // of 8: the rows and columns this lane reads V from
  const int vcol = 16 * ((2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) ^ (vrow >> 1)) + 8 * (lane & 1);

  // Steps of 32 keys.  A step takes the scores of its keys from the step
  // before it and multiplies the next step's (matrix cores) while it
  // exponentiates its own (vector units); then its probabilities and V.
  // A tile's bytes arrive and are decoded a tile ahead: barrier t lies
  // between the steps of tile t, decoding tile t + 1 before it.  So K of
  // tile t is read between barriers t - 1 and t and written between t - 2 and
  // t - 1, V is read between t - 1 and t + 1.  nan_tiles[t % 4] is cleared before
  // barrier t - 2, set between t - 2 and t - 1, read between t and t + 1.
  if (threadIdx.x < 4) nan_tiles[threadIdx.x] = 0;
  __syncthreads();
  Bytes next;
  int id = page_of(first);
  fetch(next, first, id);
  unsigned long long ok = next.ok;
  if constexpr (SEES == SEES_PREFIX) take_rows();   // while the first tile is under way
  decode(next, 0);
  id = page_of(first + 1);
  __syncthreads();
  f32x16 s = scores(0, 0);
  mask(s, first, 0, ok);
  float top = top_of(s);
  for (int tile = first; tile < stop; ++tile) {
    const int t1 = tile - first;
    fetch(next, tile + 1, id);
    id = page_of(tile + 2);
    if (threadIdx.x == 0) nan_tiles[(t1 + 2) & 3] = 0;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (u == 1) __syncthreads();
      const bool raise = top > m;
      if (__any(raise)) {
        const float mn = raise ? top + a.slack : m;
        const float f = raise ? exp2f((m - mn) * a.scale2) : 1.0f;
        m = mn;
        sum *= f;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[d][e] *= f;
      }
      const float m0 = m == -INFINITY ? 0.0f : -m * a.scale2;
      f32x16 sn = u == 0 ? scores(t1, 1) : scores(t1 + 1, 0);
      float p[16];
      bf16x8 pb[2][T];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int e = 8 * half; e < 8 * half + 8; ++e) p[e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.scale2, m0));
        if constexpr (T == 1) {
          // the sum takes the probabilities as the product takes them
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const bf16x2 two = {(__bf16)p[8 * half + e], (__bf16)p[8 * half + e + 1]};
            pb[half][0][e] = two[0];
            pb[half][0][e + 1] = two[1];
            sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(s16x2, two), s16x2{0x3f80, 0x3f80}, sum, false);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) sum += p[8 * half + e];
#pragma unroll
          for (int t = 0; t < T; ++t) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              pb[half][t][e] = (__bf16)p[8 * half + e];
              if (t + 1 < T) p[8 * half + e] -= (float)pb[half][t][e];
            }
          }
        }
      }
      const char *vr = v_lds + t1 % NV * v_bytes(TB) + (32 * u + vrow) * VP + vcol;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(vr + 16 * half * VP + 64 * d));
          const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(vr + (16 * half + 8) * VP + 64 * d));
          const bf16x8 va = __builtin_bit_cast(bf16x8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
          for (int t = 0; t < T; ++t) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va, pb[half][t], o[d], 0, 0, 0);
        }
      }
      if (u == 0) {
        decode(next, t1 + 1);
        mask(sn, tile, 1, ok);
      } else {
        mask(sn, tile + 1, 0, next.ok);
      }
      s = sn;
      top = top_of(s);
    }
    ok = next.ok;
    if (nan_tiles[t1 & 3]) {
      const uint8_t *ve = (const uint8_t *)v_lds + t1 % NV * v_bytes(TB) + KEYS * VP;
      const int t0 = tile * KEYS;
#pragma unroll
      for (int c = 0; c < TB; ++c) {
        bool hit = false;
#pragma unroll 1
        for (int k = 0; k < KEYS; ++k) hit |= (ve[16 * k + c] >= KV4_PAST) & (t0 + k >= lo) & (t0 + k < hi);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[c >> 1][8 * (c & 1) + e] = hit ? NAN : o[c >> 1][8 * (c & 1) + e];
      }
    }
    if constexpr (NV == 2) __syncthreads();   // before V of tile t - 1 gives way to t + 1
  }
  if (SEES == SEES_PREFIX && blind) {
    m = -INFINITY;
    sum = 0.0f;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][e] = 0.0f;
  }
  __syncthreads();

  // results: 32 values of the wave's rows at a time through LDS, 4 lanes to a
  // row with 8 values each
  sum += fpeer<32>(sum);
  float *ow = (float *)lds + w * 32 * OUT_PITCH, *ml = (float *)lds + W * 32 * OUT_PITCH + w * 64;
  if (h == 0) {
    ml[n] = m * a.scale2;
    ml[32 + n] = sum;
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
  const int hd = 16 * tiles, piece = 8 * (lane & 3);
  bool live[2];
  long long to[2];   // of the row's first value, in out or in the unfinished sums
  float over[2];     // 1 / sum (0: nothing seen), or 1
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int row = (lane >> 2) + 16 * k;
    live[k] = rr0 + row < rows;
    uint32_t rg;
    const int ri = (int)a.by_group.div((uint32_t)(live[k] ? rr0 + row : 0), rg), rh = head * G + (int)rg;
    const long long tok = sp.row0 + ri;
    const float L = ml[32 + row];
    if (SEES >= SEES_PREFIX) {
      const long long at = SEES == SEES_REST ? rest_place(a, seq, ri, tok, rh, split)
                           : a.pieces        ? (long long)blockIdx.x * ROWS + 32 * w + row
                                             : prefix_place(a, tok, rh, split);
      if (live[k] && piece == 0) a.part_ml[at] = make_float2(ml[row], L);
      to[k] = at * hd;
      over[k] = 1.0f;
    } else if (a.splits > 1) {   // by the row's place in its sequence: the scratch holds no more than they have
      const long long at = (((long long)seq * a.b.max_q + ri) * a.q.heads + rh) * a.splits + split;
      if (live[k] && piece == 0) a.part_ml[at] = make_float2(ml[row], L);
      to[k] = at * hd;
      over[k] = 1.0f;
    } else {
      to[k] = tok * a.out.row_stride + rh * a.out.head_stride;
      over[k] = L == 0.0f ? 0.0f : 1.0f / L;
    }
  }
#pragma unroll
  for (int d = 0; d < DT; ++d) {
    if (2 * d < tiles) {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int b = 0; b < 4; ++b)
        *(f32x4 *)(ow + n * OUT_PITCH + 8 * b + 4 * h) = f32x4{o[d][4 * b], o[d][4 * b + 1], o[d][4 * b + 2], o[d][4 * b + 3]};
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (!live[k] || 32 * d + piece >= hd) continue;   // all of a tile's lanes
        const float *from = ow + ((lane >> 2) + 16 * k) * OUT_PITCH + piece;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = from[e] * over[k];
        const long long at = to[k] + 32 * d + piece;
        if (SEES >= SEES_PREFIX || a.splits > 1) {
          float4 *p = (float4 *)(a.part_o + at);
          p[0] = make_float4(v[0], v[1], v[2], v[3]);
          p[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
          out_store8(a.out, at, v, a.out_wide);
        }
      }
    }
  }
}

template <int TB, int W, Kv4Sees SEES>
static AttnKernel prompt_kernel_of(int terms) {
  return {terms == 1 ? k_kv4_prompt<TB, 1, W, SEES> : terms == 2 ? k_kv4_prompt<TB, 2, W, SEES> : k_kv4_prompt<TB, 3, 4, SEES>,
          terms == 1 ? prompt_lds(TB, 1, W) : terms == 2 ? prompt_lds(TB, 2, W) : prompt_lds(TB, 3, 4)};
}

template <Kv4Sees SEES>
static AttnKernel prompt_kernel_for(int tiles, int terms) {
  return tiles <= 2    ? prompt_kernel_of<2, 8, SEES>(terms)
         : tiles <= 4  ? prompt_kernel_of<4, 8, SEES>(terms)
         : tiles <= 6  ? prompt_kernel_of<6, 8, SEES>(terms)
         : tiles <= 8  ? prompt_kernel_of<8, 8, SEES>(terms)
         : tiles <= 12 ? prompt_kernel_of<12, 4, SEES>(terms)
                       : prompt_kernel_of<16, 4, SEES>(terms);
}

}  // namespace bfp
