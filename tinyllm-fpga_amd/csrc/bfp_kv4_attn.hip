// Attention over the 4-bit paged cache.
//
// Per query row and head: out = sum_j p_j v_j / sum_j p_j, p_j = exp(scale
// q.k_j - m), one pass over the keys with the running maximum m and sum
// (softmax in base 2, float32).  Both products run on the bfloat16 matrix
// cores.  A cached value has two significant bits, so its bfloat16 is exact;
// queries and probabilities that need more than bfloat16's eight are split
// into terms of eight bits, and a row's terms are further columns of the same
// matrix tile: a decode step has few rows to a KV head (the query heads that
// share it), so the split costs no further matrix instruction.
//
// k_kv4_rows: a workgroup takes up to 16 columns (rows x terms) of one
// sequence and KV head, its waves take 64 keys in turn.  With S^T = K Q^T the
// keys are the matrix tile's rows and a lane's K operand is one tile of one
// key, straight from memory through the decoding conversion.  S^T leaves the
// probabilities in the layout in which O^T = V^T P^T takes them, with the keys
// in the order (lane group, register, key of four), so they never move
// between lanes.  V has to be turned over: its decoded tiles go through the
// wave's own piece of LDS and come back with the transposing reads.
#include <math.h>

#include "bfp.h"
#include "bfp_device.h"
#include "bfp_f64.h"
#include "bfp_internal.h"
#include "bfp_kv4.h"
#include "bfp_rows.h"

namespace bfp {

constexpr int KEYS = 64;             // keys a wave takes at a time
// The running maximum is raised only when a score passes it by this many
// powers of two: probabilities up to 2^8 are as exact as those up to 1, and
// the sums are rescaled a few times in a whole context instead of whenever a
// new maximum turns up.
constexpr float M_SLACK = 8.0f;

typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

struct Kv4AttnArgs {
  bfp_kv4 c;
  bfp_kv4_batch b;
  bfp_rows q, out;
  int tiles, group, page_shift, window, splits, row_tiles;
  FastDiv by_seq, by_head, by_split;   // k_kv4_prompt's workgroups
  float scale2;        // |scale| * log2(e), kept above 0; the queries take the sign
  float slack;         // M_SLACK in scores: M_SLACK / scale2
  float q_sign;
  float *part_o;       // [row][query head][split][hd], where splits > 1
  float2 *part_ml;     // [row][query head][split]: m, sum
};

// Position p's visible keys are [lo, hi).
__device__ __forceinline__ int key_hi(int p) { return p < 0 ? 0 : p + 1; }
__device__ __forceinline__ int key_lo(int hi, int window) {
  return window > 0 && hi > window ? hi - window : 0;
}

// x cut to bfloat16 toward zero: the rest is exact, and has the sign of x.
__device__ __forceinline__ float cut_bf16(float x) {
  return __uint_as_float(__float_as_uint(x) & 0xffff0000u);
}

// Term t of x's split by cuts (three hold any float32).  An infinity or a
// NaN is its own first term.
__device__ __forceinline__ float cut_term(float x, int t) {
  const bool good = fabsf(x) < INFINITY;
  if (!good) return t == 0 ? (x != x ? NAN : x) : 0.0f;
  for (int i = 0; i < t; ++i) x -= cut_bf16(x);
  return cut_bf16(x);
}

// Term t of x's split by rounding.
template <int T>
__device__ __forceinline__ float round_term(float x, int t) {
  if constexpr (T > 1) {
#pragma unroll
    for (int i = 1; i < T && i < 3; ++i) {
      const float r = x - (float)(__bf16)x;
      x = t >= i ? r : x;
    }
    if constexpr (T == 4) x = t == 3 ? 0.0f : x;
  }
  return x;
}

__device__ __forceinline__ bf16x8 pack8(const float (&v)[8]) {
  bf16x8 r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = (__bf16)v[i];
  return r;
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

__device__ __forceinline__ bool has_byte_255(uint32_t w) {
  return ((w & 0x7f7f7f7fu) + 0x01010101u) & w & 0x80808080u;
}
// w with its bytes kept where keep has a bit (byte i: bit i).
__device__ __forceinline__ uint32_t byte_mask(uint32_t keep) {
  return (((keep & 1) | ((keep & 2) << 7) | ((keep & 4) << 14) | ((keep & 8) << 21)) * 255u);
}

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
    x.w[c][0] = p[0];
    x.w[c][1] = p[1];
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

// Value o of a finished row: one of 16 neighbouring lanes with neighbouring o.
__device__ __forceinline__ void out_store(const bfp_rows &r, long long o, float v) {
  if (r.type != BFP_TILES) {
    row_store(r, o, v);
    return;
  }
  int e;
  const int m = quantize16_lanes((double)v, e);
  ((int16_t *)r.p)[o] = (int16_t)m;
  if ((threadIdx.x & 15) == 0) r.e[o >> 4] = (int8_t)e;
}

// C: head tiles a lane group holds (hd <= 64 C); T: terms of a row (columns
// R = 16 / T rows share); W: waves.
template <int C, int T, int W>
__global__ __launch_bounds__(64 * W, C == 1 ? 4 : C == 2 ? 2 : 1) void k_kv4_rows(Kv4AttnArgs a) {
  constexpr int R = 16 / T;
  extern __shared__ __align__(16) char lds[];
  const int seq = blockIdx.z, head = blockIdx.y;
  const int rt = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
  const Kv4Span sp = kv4_span(a.b.start[seq], a.b.start[seq + 1], a.b.len[seq], a.b.n_rows, a.b.max_q);
  const int G = a.group, rows = sp.n * G;   // rows of this KV head: (token, query head)
  const int rr0 = rt * R;
  if (rr0 >= rows) return;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const int t = r / R;
  const int tiles = a.tiles;

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
  const int tile0 = lo_min / KEYS, n_tiles = end > lo_min ? (end + KEYS - 1) / KEYS - tile0 : 0;
  const int per = (n_tiles + a.splits - 1) / a.splits;
  const int first = tile0 + split * per;
  const int stop = tile0 + (split + 1 < a.splits && (split + 1) * per < n_tiles ? (split + 1) * per : n_tiles);

  // the column's query, term t
  bf16x8 qf[C][2];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    float x[16];
    if (mine && g * C + c < tiles) {
      row_load_n(a.q, (long long)(sp.row0 + i) * a.q.row_stride + qh * a.q.head_stride + 16 * (g * C + c), x);
#pragma unroll
      for (int d = 0; d < 16; ++d) x[d] = (T == 1 ? x[d] : cut_term(x[d], t)) * a.q_sign;
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
  const int32_t *pages = a.b.pages + (long long)seq * a.b.width;
  auto page_of = [&](int tile) {
    return tile < stop ? kv4_page(pages, a.b.width, a.c.n_pages, (tile * KEYS + 4 * r) >> a.page_shift) : -1;
  };
  auto offset_of = [&](int tile, int id) {
    return kv4_tile(id < 0 ? 0 : id, a.c.heads, head, tiles, 0, a.c.page, (tile * KEYS + 4 * r) & (a.c.page - 1));
  };

  // K of the next tile is asked for when this one's scores are done, V when
  // this one's has gone to LDS: no second set of registers
  KvSide<C> k, v;
  int tile = first + w;
  int id = page_of(tile);
  long long at = offset_of(tile, id);
  load_side(k, a.c.k, a.c.k_e, at, a.c.page, g * C, tiles);
  load_side(v, a.c.v, a.c.v_e, at, a.c.page, g * C, tiles);
  for (; tile < stop; tile += W) {
    const int t0 = tile * KEYS;
    const int next_id = page_of(tile + W);
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
          s[j][e] = ok & (key >= lo) & (key < hi) ? s[j][e] : -INFINITY;
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
    const bool raise = top > m + a.slack;
    if (__any(raise)) {
      const float mn = raise ? top : m;
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
          sum += p;
          pv[4 * jj + e] = round_term<T>(p, t);
        }
      pb[jp] = pack8(pv);
    }

    // A tile of V that holds a NaN counts as zeros in the product, so that it
    // cannot reach a row that does not see it; the rows that do are set below.
    uint32_t bad = 0;
#pragma unroll
    for (int c = 0; c < C; ++c) bad |= has_byte_255(v.e[c]) && g * C + c < tiles ? 1u << c : 0u;
    const bool any_nan = __any(bad);
    uint32_t ve[C];
    if (any_nan) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        ve[c] = v.e[c];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (((ve[c] >> (8 * j)) & 255u) != KV4_NAN) continue;
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
        for (int key = 0; key < KEYS; ++key) hit |= (le[16 * key + d] == KV4_NAN) & (t0 + key >= lo) & (t0 + key < hi);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[d][e] = hit ? NAN : o[d][e];
      }
    }
    id = next_id;
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
      for (int e = 0; e < 4; ++e) v[e] = term_sum<T>(v[e]);
      if (r < R) *(f32x4 *)(jw + 32 + r * (hd + 4) + 16 * d + 4 * g) = v;
    }
  }
  __syncthreads();
  const float *jf = (const float *)lds;
  // 16 lanes to a row's tile
  for (int u = threadIdx.x >> 4; u < R * tiles; u += 4 * W) {
    const int row = u / tiles, d = 16 * (u % tiles) + (threadIdx.x & 15);
    if (rr0 + row >= rows) break;   // all 16 lanes
    float M = -INFINITY;
#pragma unroll
    for (int k = 0; k < W; ++k) M = fmaxf(M, jf[k * stride + row]);
    float L = 0.0f, acc = 0.0f;
#pragma unroll
    for (int k = 0; k < W; ++k) {
      const float mk = jf[k * stride + row];
      const float f = mk == -INFINITY ? 0.0f : exp2f(mk - M);
      L += f * jf[k * stride + 16 + row];
      acc += f * jf[k * stride + 32 + row * (hd + 4) + d];
    }
    const int ri = (rr0 + row) / G, rh = head * G + (rr0 + row) % G;
    const long long tok = sp.row0 + ri;
    if (a.splits > 1) {
      const long long at = (tok * a.q.heads + rh) * a.splits + split;
      if (d == 0) a.part_ml[at] = make_float2(M, L);
      a.part_o[at * hd + d] = acc;
    } else {
      out_store(a.out, tok * a.out.row_stride + rh * a.out.head_stride + d, L == 0.0f ? 0.0f : acc / L);
    }
  }
}

// ------------------------------------------------------------- many rows
// k_kv4_prompt: a workgroup takes 32 rows a wave of one sequence and KV head
// (a row is a token and one of the query heads that share the KV head), all
// waves the same 64 keys.  Each key tile is decoded once into LDS as
// bfloat16, two buffers deep: the next tile's bytes are on their way while
// this one is multiplied.  The matrix tiles are 32 x 32: an operand read
// from LDS (1 KB) then feeds 16384 products, so the waves together ask for
// what LDS delivers only when the matrix cores run without a pause.  As in
// k_kv4_rows, keys are the rows of S^T, and the probabilities stay in place.
typedef float f32x16 __attribute__((ext_vector_type(16)));

// K rows: read 16 bytes a lane, 32 rows at a time; 16 bytes past the row put
// eight neighbouring rows in different banks.  V rows: read by transposing
// loads of 4 rows x 64 bytes, which an odd multiple of 64 bytes spreads.
constexpr int pk_pitch(int tb) { return 32 * tb + 16; }
constexpr int pv_pitch(int tb) { return 64 * ((tb / 2) | 1); }
// A tile of K, and of V with its exponent bytes (key, 16 tiles).
constexpr int k_bytes(int tb) { return KEYS * pk_pitch(tb); }
constexpr int v_bytes(int tb) { return KEYS * (pv_pitch(tb) + 16); }
// Tiles of V held: with three, one barrier a tile is enough; the widest heads
// leave room for two, and take a second barrier.
constexpr int v_buffers(int tb) { return tb <= 12 ? 3 : 2; }
constexpr int OUT_PITCH = 36;   // floats: 32 values of a row, on their way out
constexpr int prompt_lds(int tb, int waves) {
  const int in = 2 * k_bytes(tb) + v_buffers(tb) * v_bytes(tb), out = waves * (32 * OUT_PITCH + 64) * 4;
  return in > out ? in : out;
}

// TB: tiles of the head the loops are built for (even; a narrower head's
// missing tiles are zeros in K, and columns of V whose results nobody
// takes); T: terms; W: waves.
template <int TB, int T, int W>
__global__ __launch_bounds__(64 * W, (W + 3) / 4) void k_kv4_prompt(Kv4AttnArgs a) {
  constexpr int ROWS = 32 * W, DT = TB / 2, UNITS = (TB + W - 1) / W;
  constexpr int KP = pk_pitch(TB), VP = pv_pitch(TB), NV = v_buffers(TB);
  extern __shared__ __align__(16) char lds[];
  __shared__ int nan_tiles[4];
  // One sequence after the other, its last rows, which see the most keys,
  // first.  Neighbouring workgroups take different KV heads and the same rows:
  // workgroups go to the XCDs and their shader engines in turn, whether one
  // is ready sooner or not, so neighbours should take equally long.
  uint32_t u, h1, s1;
  const int seq = (int)a.by_seq.div(blockIdx.x, u);
  u = a.by_head.div(u, h1);
  u = a.by_split.div(u, s1);
  const int head = (int)h1, split = (int)s1, rt = a.row_tiles - 1 - (int)u;
  const Kv4Span sp = kv4_span(a.b.start[seq], a.b.start[seq + 1], a.b.len[seq], a.b.n_rows, a.b.max_q);
  const int G = a.group, rows = sp.n * G;
  if (rt >= (rows + ROWS - 1) / ROWS) return;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, h = lane >> 5;
  const int tiles = a.tiles;
  const int wg0 = rt * ROWS, rr0 = wg0 + 32 * w, rr = rr0 + n;
  const bool mine = rr < rows;
  const int i = mine ? rr / G : 0, qh = head * G + (mine ? rr % G : 0);
  const int hi = mine ? key_hi(sp.at + i) : 0, lo = key_lo(hi, a.window);
  // what this wave's rows all see, and any of the workgroup's
  const int wfirst = rr0 < rows ? rr0 : rows - 1, wlast = (rr0 + 32 < rows ? rr0 + 32 : rows) - 1;
  const int hi_min = key_hi(sp.at + wfirst / G), hi_max = rr0 < rows ? key_hi(sp.at + wlast / G) : 0;
  const int lo_min = key_lo(hi_min, a.window), lo_max = key_lo(hi_max, a.window);
  const int glast = (wg0 + ROWS < rows ? wg0 + ROWS : rows) - 1;
  const int begin = key_lo(key_hi(sp.at + wg0 / G), a.window);
  const int top_hi = key_hi(sp.at + glast / G);
  const long long cap = (long long)a.b.width << a.page_shift;
  const int end = top_hi < cap ? top_hi : (int)cap;
  const int tile0 = begin / KEYS, n_tiles = end > begin ? (end + KEYS - 1) / KEYS - tile0 : 0;
  const int per = (n_tiles + a.splits - 1) / a.splits;
  const int first = tile0 + split * per;
  const int stop = tile0 + (split + 1 < a.splits && (split + 1) * per < n_tiles ? (split + 1) * per : n_tiles);

  bf16x8 qf[T][TB];
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
      for (int d = 0; d < 8; ++d) y[d] = (T == 1 ? x[d] : cut_term(x[d], t)) * a.q_sign;
      qf[t][c] = pack8(y);
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
  uint2 rk[UNITS], rv[UNITS];
  uint32_t rke[UNITS], rve[UNITS];
  bool there = false;
  auto page_of = [&](int tile) {
    const int key = tile * KEYS + lane;
    return tile < stop && key >= begin && key < end ? kv4_page(pages, a.b.width, a.c.n_pages, key >> a.page_shift) : -1;
  };
  // a key without a page reads the first one's bytes; they are not used
  auto fetch = [&](int tile, int id) {
    there = id >= 0;
    const long long at = kv4_tile(there ? id : 0, a.c.heads, head, tiles, 0, a.c.page, (tile * KEYS + lane) & (a.c.page - 1));
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int t = w + u * W;
      const long long o8 = at + (long long)(t < tiles ? t : tiles - 1) * a.c.page;
      rk[u] = *(const uint2 *)(a.c.k + o8 * KV4_TILE_BYTES);
      rv[u] = *(const uint2 *)(a.c.v + o8 * KV4_TILE_BYTES);
      rke[u] = a.c.k_e[o8];
      rve[u] = a.c.v_e[o8];
    }
  };
  char *const k_lds = lds, *const v_lds = lds + 2 * k_bytes(TB);
  auto decode = [&](int t1) {   // tile first + t1
    char *kb = k_lds + (t1 & 1) * k_bytes(TB) + lane * KP, *vt = v_lds + t1 % NV * v_bytes(TB), *vb = vt + lane * VP;
    const int sw = (lane >> 1) & 3;   // 16-byte pieces of each 64 change places, for the writes' banks
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int t = w + u * W;
      if (UNITS * W > TB && t >= TB) break;
      const bool ok = there && t < tiles;   // zeros for what the head or the cache does not have
      const float ks = kv4_scale(rke[u]);
      bf16x8 *kd = (bf16x8 *)(kb + 32 * t);
      kd[0] = kv4_decode8(t < tiles ? rk[u].x : 0u, ks);
      kd[1] = kv4_decode8(t < tiles ? rk[u].y : 0u, ks);
      // NaN tiles of V count as zeros in the product; the rows that see them are set after
      const uint32_t E = ok ? rve[u] : 0u;
      const bool take = ok && E != KV4_NAN;
      vt[KEYS * VP + lane * 16 + t] = (char)E;
      if (E == KV4_NAN) nan_tiles[t1 & 3] = 1;
      const float vs = kv4_scale(take ? E : 0u);
      *(bf16x8 *)(vb + 64 * (t >> 1) + 16 * ((2 * (t & 1)) ^ sw)) = kv4_decode8(take ? rv[u].x : 0u, vs);
      *(bf16x8 *)(vb + 64 * (t >> 1) + 16 * ((2 * (t & 1) + 1) ^ sw)) = kv4_decode8(take ? rv[u].y : 0u, vs);
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
      s[e] = (((okh >> k) & 1) != 0) & (key >= lo) & (key < hi) ? s[e] : -INFINITY;
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
  int id = page_of(first);
  fetch(first, id);
  unsigned long long ok = __ballot(there);
  decode(0);
  id = page_of(first + 1);
  __syncthreads();
  f32x16 s = scores(0, 0);
  mask(s, first, 0, ok);
  float top = top_of(s);
  for (int tile = first; tile < stop; ++tile) {
    const int t1 = tile - first;
    fetch(tile + 1, id);
    const unsigned long long ok_next = __ballot(there);
    id = page_of(tile + 2);
    if (threadIdx.x == 0) nan_tiles[(t1 + 2) & 3] = 0;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (u == 1) __syncthreads();
      const bool raise = top > m + a.slack;
      if (__any(raise)) {
        const float mn = raise ? top : m;
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
        decode(t1 + 1);
        mask(sn, tile, 1, ok);
      } else {
        mask(sn, tile + 1, 0, ok_next);
      }
      s = sn;
      top = top_of(s);
    }
    ok = ok_next;
    if (nan_tiles[t1 & 3]) {
      const uint8_t *ve = (const uint8_t *)v_lds + t1 % NV * v_bytes(TB) + KEYS * VP;
      const int t0 = tile * KEYS;
#pragma unroll
      for (int c = 0; c < TB; ++c) {
        bool hit = false;
#pragma unroll 1
        for (int k = 0; k < KEYS; ++k) hit |= (ve[16 * k + c] == KV4_NAN) & (t0 + k >= lo) & (t0 + k < hi);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[c >> 1][8 * (c & 1) + e] = hit ? NAN : o[c >> 1][8 * (c & 1) + e];
      }
    }
    if constexpr (NV == 2) __syncthreads();   // before V of tile t - 1 gives way to t + 1
  }
  __syncthreads();

  // results: 32 values of the wave's rows at a time through LDS, 16 lanes to a tile
  sum += fpeer<32>(sum);
  float *ow = (float *)lds + w * 32 * OUT_PITCH, *ml = (float *)lds + W * 32 * OUT_PITCH + w * 64;
  if (h == 0) {
    ml[n] = m * a.scale2;
    ml[32 + n] = sum;
  }
  const int hd = 16 * tiles;
#pragma unroll
  for (int d = 0; d < DT; ++d) {
    if (2 * d >= tiles) break;
    const f32x16 v = o[d];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int b = 0; b < 4; ++b)
      *(f32x4 *)(ow + n * OUT_PITCH + 8 * b + 4 * h) = f32x4{v[4 * b], v[4 * b + 1], v[4 * b + 2], v[4 * b + 3]};
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
#pragma unroll 1
    for (int k = lane >> 4; k < 64; k += 4) {
      const int row = k >> 1, dim = 32 * d + 16 * (k & 1) + (lane & 15);
      if (rr0 + row >= rows) break;
      if (dim >= hd) continue;   // all 16 lanes
      const int ri = (rr0 + row) / G, rh = head * G + (rr0 + row) % G;
      const long long tok = sp.row0 + ri;
      const float L = ml[32 + row], acc = ow[row * OUT_PITCH + dim - 32 * d];
      if (a.splits > 1) {
        const long long at = (tok * a.q.heads + rh) * a.splits + split;
        if (dim == 0) a.part_ml[at] = make_float2(ml[row], L);
        a.part_o[at * hd + dim] = acc;
      } else {
        out_store(a.out, tok * a.out.row_stride + rh * a.out.head_stride + dim, L == 0.0f ? 0.0f : acc / L);
      }
    }
  }
}

// Joins the splits: a wave takes one row and query head.
__global__ __launch_bounds__(256) void k_kv4_join(Kv4AttnArgs a) {
  const int seq = blockIdx.y;
  const Kv4Span sp = kv4_span(a.b.start[seq], a.b.start[seq + 1], a.b.len[seq], a.b.n_rows, a.b.max_q);
  const int u = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int i = u / a.q.heads, qh = u % a.q.heads;
  if (i >= sp.n) return;
  const long long tok = sp.row0 + i, at = (tok * a.q.heads + qh) * a.splits;
  const int hd = 16 * a.tiles;
  // lane k holds split k's maximum and sum (at most 64 splits)
  const float2 ml = lane < a.splits ? a.part_ml[at + lane] : make_float2(-INFINITY, 0.0f);
  float M = ml.x;
  M = fmaxf(M, fpeer<32>(M));
  M = fmaxf(M, fpeer<16>(M));
  M = fmaxf(M, fpeer<8>(M));
  M = fmaxf(M, fpeer<4>(M));
  M = fmaxf(M, fpeer<2>(M));
  M = fmaxf(M, fpeer<1>(M));
  // a split that saw nothing (or NaN scores alone, whose sum is NaN): factor 0
  const float f = ml.x == -INFINITY ? 0.0f : exp2f(ml.x - M);
  float L = f * ml.y;
  L += fpeer<32>(L);
  L += fpeer<16>(L);
  L += fpeer<8>(L);
  L += fpeer<4>(L);
  L += fpeer<2>(L);
  L += fpeer<1>(L);
  float acc[4] = {0, 0, 0, 0};
#pragma unroll 8
  for (int k = 0; k < a.splits; ++k) {
    const float fk = __shfl(f, k, 64);
#pragma unroll
    for (int d = 0; d < 4; ++d)
      if (64 * d + lane < hd) acc[d] += fk * a.part_o[(at + k) * hd + 64 * d + lane];
  }
#pragma unroll
  for (int d = 0; d < 4; ++d)
    if (64 * d + lane < hd)
      out_store(a.out, tok * a.out.row_stride + qh * a.out.head_stride + 64 * d + lane, L == 0.0f ? 0.0f : acc[d] / L);
}

// ------------------------------------------------------------------- host
struct Kv4Plan {
  bool prompt;       // k_kv4_prompt, else k_kv4_rows
  int terms, waves, row_tiles, splits;
  size_t work;
};

// The terms a row is carried in: one where queries, probabilities and results
// are bfloat16 and the rows fill the tile's 16 columns anyway; two hold a
// float16 or 16-bit-tile query and leave probabilities 2^-18 off; three
// (of four places) hold float32 queries and results.
static int terms_of(const bfp_rows &q, const bfp_rows &out, int rows) {
  if (q.type == BFP_F32 || out.type == BFP_F32 || out.type == BFP_TILES) return 4;
  return q.type == BFP_BF16 && out.type == BFP_BF16 && rows > 8 ? 1 : 2;
}

static Kv4Plan plan_attn(const bfp_kv4 &c, const bfp_kv4_batch &b, const bfp_rows &q, const bfp_rows &out, int window) {
  Kv4Plan p{};
  const int group = q.heads / c.heads, tiles = c.hd / 16;
  const long long rows = (long long)b.max_q * group;
  const long long cap = (long long)b.width * c.page;
  long long keys = b.max_len > 0 && b.max_len < cap ? b.max_len : cap;
  if (window > 0 && keys > (long long)window + b.max_q) keys = (long long)window + b.max_q;
  const long long key_tiles = (keys + KEYS - 1) / KEYS;
  p.prompt = rows > 64;
  if (p.prompt) {
    const bool wide = q.type == BFP_F32 || out.type == BFP_F32 || out.type == BFP_TILES;
    p.terms = wide ? 3 : (q.type == BFP_BF16 && out.type == BFP_BF16 ? 1 : 2);
    p.waves = tiles <= 8 && p.terms < 3 ? 8 : 4;
    p.row_tiles = (int)((rows + 32 * p.waves - 1) / (32 * p.waves));
  } else {
    p.terms = terms_of(q, out, (int)rows);
    p.waves = 4;
    const int R = 16 / p.terms;
    p.row_tiles = (int)((rows + R - 1) / R);
  }
  const long long groups = (long long)p.row_tiles * c.heads * b.n_seq;
  long long s = groups > 0 ? (p.prompt ? 512 : 1024) / groups : 1;
  if (s > key_tiles / 4) s = key_tiles / 4;
  if (s > 64) s = 64;   // a lane of k_kv4_join each
  p.splits = s < 1 ? 1 : (int)s;
  if (p.splits > 1) {
    const size_t cells = (size_t)b.n_rows * q.heads * p.splits;
    p.work = cells * (16 * tiles * sizeof(float) + sizeof(float2));
  }
  return p;
}

static int check_attn(const char *op, const bfp_kv4 *cache, const bfp_kv4_batch *batch, const bfp_rows *q,
                      const bfp_rows *out, int window) {
  BFP_TRY(check_kv4(op, cache, batch));
  if (!q || q->heads < cache->heads || q->heads % cache->heads || q->heads > 65536)
    return set_err(BFP_EINVAL, "%s: q has %d heads, the cache %d", op, q ? q->heads : 0, cache->heads);
  BFP_TRY(check_rows(op, "q", q, q->heads, cache->hd, true, batch->n_rows));
  BFP_TRY(check_out(op, "out", out, q->heads, cache->hd, true, batch->n_rows));
  if (!rows_aligned(*q, 8)) return set_err(BFP_EINVAL, "%s: q needs 16-byte alignment and strides in multiples of 8", op);
  if (window < 0) return set_err(BFP_EINVAL, "%s: window=%d", op, window);
  if ((long long)batch->max_q * (q->heads / cache->heads) > 0x3fffffffLL)
    return set_err(BFP_EINVAL, "%s: max_q=%d rows of %d heads are too many", op, batch->max_q, q->heads);
  return BFP_OK;
}

typedef void (*attn_fn)(Kv4AttnArgs);
template <int C>
static attn_fn pick_rows(int terms) {
  return terms == 1 ? k_kv4_rows<C, 1, 4> : terms == 2 ? k_kv4_rows<C, 2, 4> : k_kv4_rows<C, 4, 4>;
}
template <int TB, int W>
static attn_fn pick_prompt(int terms) {
  return terms == 1 ? k_kv4_prompt<TB, 1, W> : terms == 2 ? k_kv4_prompt<TB, 2, W> : k_kv4_prompt<TB, 3, 4>;
}

}  // namespace bfp

using namespace bfp;

extern "C" {

size_t bfp_kv4_attn_work(const bfp_kv4 *cache, const bfp_kv4_batch *batch, const bfp_rows *q,
                         const bfp_rows *out, int window) {
  if (check_attn("kv4_attn_work", cache, batch, q, out, window)) return 0;
  return plan_attn(*cache, *batch, *q, *out, window).work;
}

int bfp_kv4_attn_d(const bfp_kv4 *cache, const bfp_kv4_batch *batch, const bfp_rows *q,
                   const bfp_rows *out, double scale, int window, void *work, size_t work_bytes,
                   void *stream) {
  const char *op = "kv4_attn";
  BFP_TRY(check_attn(op, cache, batch, q, out, window));
  if (!isfinite(scale)) return set_err(BFP_EINVAL, "%s: scale=%g", op, scale);
  if (batch->n_seq == 0 || batch->max_q == 0 || batch->n_rows == 0) return BFP_OK;
  const Kv4Plan p = plan_attn(*cache, *batch, *q, *out, window);
  if (p.work && (!work || (uintptr_t)work % 16 || work_bytes < p.work))
    return set_err(BFP_EINVAL, "%s: needs %zu bytes of 16-byte-aligned scratch, got %zu", op, p.work, work ? work_bytes : (size_t)0);
  Kv4AttnArgs a{};
  a.c = *cache;
  a.b = *batch;
  a.q = *q;
  a.out = *out;
  a.tiles = cache->hd / 16;
  a.group = q->heads / cache->heads;
  a.page_shift = __builtin_ctz((unsigned)cache->page);
  a.window = window;
  a.splits = p.splits;
  // a scale of zero (all scores alike) is taken as one that leaves nothing of them
  a.scale2 = fmaxf((float)(fabs(scale) * 1.44269504088896340736), 0x1p-100f);
  a.slack = M_SLACK / a.scale2;
  a.q_sign = scale < 0 ? -1.0f : 1.0f;
  if (p.work) {
    const size_t cells = (size_t)batch->n_rows * q->heads * p.splits;
    a.part_o = (float *)work;
    a.part_ml = (float2 *)((float *)work + cells * 16 * a.tiles);
  }
  a.row_tiles = p.row_tiles;
  a.by_head = FastDiv(cache->heads);
  a.by_split = FastDiv(p.splits);
  long long blocks = (long long)p.row_tiles * p.splits * (p.prompt ? cache->heads : 1);
  if (blocks <= 0x7fffffLL && p.prompt) {
    a.by_seq = FastDiv((uint32_t)blocks);
    blocks *= batch->n_seq;
  }
  if (blocks > 0x7fffffLL) return set_err(BFP_EINVAL, "%s: max_q=%d is too large for one call", op, batch->max_q);
  attn_fn fn;
  int lds;
  if (p.prompt) {
    const int tb = a.tiles <= 2 ? 2 : a.tiles <= 4 ? 4 : a.tiles <= 6 ? 6 : a.tiles <= 8 ? 8 : a.tiles <= 12 ? 12 : 16;
    fn = tb == 2 ? pick_prompt<2, 8>(p.terms) : tb == 4 ? pick_prompt<4, 8>(p.terms) : tb == 6 ? pick_prompt<6, 8>(p.terms)
         : tb == 8 ? pick_prompt<8, 8>(p.terms) : tb == 12 ? pick_prompt<12, 4>(p.terms) : pick_prompt<16, 4>(p.terms);
    lds = prompt_lds(tb, p.waves);
  } else {
    const int C = (a.tiles + 3) / 4, R = 16 / p.terms;
    fn = C == 1 ? pick_rows<1>(p.terms) : C == 2 ? pick_rows<2>(p.terms) : C == 3 ? pick_rows<3>(p.terms) : pick_rows<4>(p.terms);
    const int in = p.waves * V_ROWS * v_pitch(C), res = p.waves * join_floats(R, a.tiles) * 4;
    lds = in > res ? in : res;
  }
  if (lds > 65536)   // one limit for a kernel, whatever the call
    HIP_TRY(hipFuncSetAttribute((const void *)fn, hipFuncAttributeMaxDynamicSharedMemorySize, 159 * 1024));
  hipLaunchKernelGGL(fn, p.prompt ? dim3((unsigned)blocks) : dim3((unsigned)blocks, cache->heads, batch->n_seq), dim3(64 * p.waves), lds, (hipStream_t)stream, a);
  BFP_TRY(launch_status(op));
  if (p.splits > 1) {
    const long long n = ((long long)batch->max_q * q->heads + 3) / 4;
    hipLaunchKernelGGL(k_kv4_join, dim3((unsigned)n, batch->n_seq), dim3(256), 0, (hipStream_t)stream, a);
    BFP_TRY(launch_status(op));
  }
  return BFP_OK;
}

}  // extern "C"
