// The 4-bit key/value cache's rows in and out: new tokens appended with
// their rotation, and read back.
#include <math.h>

#include "bfp.h"
#include "bfp_internal.h"
#include "bfp_kv4.h"
#include "bfp_rotary.h"
#include "bfp_rows.h"

namespace bfp {

constexpr int KV4_BS = 256;

int check_kv4(const char *op, const bfp_kv4 *c, const bfp_kv4_batch *b) {
  if (!c || !c->k || !c->k_e || !c->v || !c->v_e) return set_err(BFP_EINVAL, "%s: no cache", op);
  if (c->page < 16 || c->page > 256 || (c->page & (c->page - 1)))
    return set_err(BFP_EINVAL, "%s: page=%d must be 16, 32, 64, 128 or 256", op, c->page);
  if (c->n_pages < 1 || c->heads < 1 || c->heads > 4096)
    return set_err(BFP_EINVAL, "%s: n_pages=%d, heads=%d", op, c->n_pages, c->heads);
  if (c->hd < 16 || c->hd > 256 || c->hd % 16)
    return set_err(BFP_EINVAL, "%s: hd=%d must be a multiple of 16 up to 256", op, c->hd);
  if (((uintptr_t)c->k | (uintptr_t)c->k_e | (uintptr_t)c->v | (uintptr_t)c->v_e) % 16)
    return set_err(BFP_EINVAL, "%s: the cache's arrays must be 16-byte aligned", op);
  return check_batch(op, b, c->page);
}

int check_batch(const char *op, const bfp_kv4_batch *b, int page) {
  if (!b) return set_err(BFP_EINVAL, "%s: no batch", op);
  if (b->n_seq < 0 || b->n_seq > 65535 || b->n_rows < 0 || b->width < 1 || b->max_q < 0 || b->max_len < 0)
    return set_err(BFP_EINVAL, "%s: n_seq=%d (at most 65535), n_rows=%d, width=%d, max_q=%d, max_len=%d",
                   op, b->n_seq, b->n_rows, b->width, b->max_q, b->max_len);
  // positions, and the keys of the tiles that begin before the last one, are ints
  if ((long long)b->width * page > KV4_MAX_POS)
    return set_err(BFP_EINVAL, "%s: width=%d pages of %d are more than %d positions", op, b->width, page, KV4_MAX_POS);
  if (b->n_seq > 0 && (!b->pages || !b->start || !b->len))
    return set_err(BFP_EINVAL, "%s: the batch's arrays are null", op);
  if (((uintptr_t)b->pages | (uintptr_t)b->start | (uintptr_t)b->len) % 4)
    return set_err(BFP_EINVAL, "%s: the batch's arrays are not aligned", op);
  return BFP_OK;
}

// A unit of work is a tile (16 values) of one row and head: one lane loads,
// turns and converts it, so the shared exponent needs no other lane.  Units
// of a sequence are numbered so that 64 lanes cover `cols` neighbouring tiles
// of `block` neighbouring rows: with block 1 (few new rows) a row's tiles and
// heads one after the other, with block 16 (prompts) 16 rows x 4 tiles, whole
// 128-byte lines of the rows on one side and of the pages on the other.
struct Kv4Units {
  FastDiv cols, groups;   // tiles side by side; groups of them in a row (all heads)
  int block_shift;
  __device__ void of(uint32_t u, int &row, uint32_t &col) const {
    uint32_t c, g;
    u = cols.div(u, c);
    const uint32_t r = u & ((1u << block_shift) - 1);
    const uint32_t b = groups.div(u >> block_shift, g);
    row = (int)((b << block_shift) + r);
    col = g * cols.d + c;
  }
};

struct Kv4AppendArgs {
  bfp_kv4 c;
  bfp_kv4_batch b;
  bfp_rows k, v, q, q_out;
  const int32_t *pos;
  const float2 *table;
  int n_pos, half, interleaved;
  // workgroups [0, q_blocks) of a sequence turn queries, the others append
  RopeShape shape;
  FastDiv q_row, q_head;   // q's units of a row, of N heads
  int q_blocks;
  uint32_t q_units;
  Kv4Units units;
  FastDiv tiles;   // of a head
  uint32_t n_units;
};

// Sixteen values of a head from d0 on, turned by the angles cs (half of
// them; the first 2 * half values of the head are turned).
__device__ __forceinline__ void load_turned(const bfp_rows &r, long long o, int d0, const float2 *cs,
                                            int half, int interleaved, bool known, double (&y)[16]) {
  float x[16];
  row_load_n(r, o + d0, x);
  const int rot = 2 * half;
  if (d0 >= rot) {
#pragma unroll
    for (int i = 0; i < 16; ++i) y[i] = x[i];
    return;
  }
  if (!known) {   // no angle for this position
#pragma unroll
    for (int i = 0; i < 16; ++i) y[i] = d0 + i < rot ? (double)NAN : (double)x[i];
    return;
  }
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      if (d0 + i < rot) {
        rope_pair(x[i], x[i + 1], rope_cs(cs[(d0 + i) >> 1]), y[i], y[i + 1]);
      } else {
        y[i] = x[i];
        y[i + 1] = x[i + 1];
      }
    }
  } else if (half % 16 == 0) {   // the partners are another whole tile
    const bool second = d0 >= half;
    float p[16];
    row_load_n(r, o + (second ? d0 - half : d0 + half), p);
    const float2 *c = cs + (second ? d0 - half : d0);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      double a, b;
      rope_pair(second ? p[i] : x[i], second ? x[i] : p[i], rope_cs(c[i]), a, b);
      y[i] = second ? b : a;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int d = d0 + i;
      if (d >= rot) {
        y[i] = x[i];
        continue;
      }
      const bool second = d >= half;
      const float p = row_load(r, o + (second ? d - half : d + half));
      double a, b;
      rope_pair(second ? p : x[i], second ? x[i] : p, rope_cs(cs[second ? d - half : d]), a, b);
      y[i] = second ? b : a;
    }
  }
}

// Zeros where rope_unit or rope_wide_unit would write.
template <int N>
__device__ __forceinline__ void zero_unit(const RopeShape &s, const bfp_rows &y, long long t, int h0, int j) {
  const bool turn = j < s.turned;
  const int w = N ? 8 : 1, da = !turn ? 2 * s.half + (j - s.turned) * w : s.interleaved ? (N ? 8 : 2) * j : w * j;
  const int values = N ? 8 : turn && s.interleaved ? 2 : 1;
  for (int h = h0; h < y.heads && h < h0 + (N ? N : 1); ++h) {
    const long long yo = t * y.row_stride + h * y.head_stride + da;
    for (int i = 0; i < values; ++i) {
      row_store(y, yo + i, 0.0f);
      if (turn && !s.interleaved) row_store(y, yo + s.half + i, 0.0f);
    }
  }
}

// N: heads of q a thread turns (0: value by value).  Bound by the bytes of k,
// v and q in and of q and the tiles out.
template <int N>
__global__ __launch_bounds__(KV4_BS) void k_kv4_append(Kv4AppendArgs a) {
  const int seq = blockIdx.y;
  const bool is_q = (int)blockIdx.x < a.q_blocks;
  const uint32_t u = (blockIdx.x - (is_q ? 0 : a.q_blocks)) * KV4_BS + threadIdx.x;
  if (u >= (is_q ? a.q_units : a.n_units)) return;
  const Kv4Span s = kv4_span(a.b.start[seq], a.b.start[seq + 1], a.b.len[seq], a.b.n_rows, a.b.max_q);
  int i;
  uint32_t col, tile;
  if (is_q)
    i = (int)a.q_row.div(u, col);
  else
    a.units.of(u, i, col);
  if (i >= s.n) return;
  const long long t = s.row0 + i;
  const int at = s.at + i;
  const int id = at < 0 ? -1 : kv4_page(a.b.pages + (long long)seq * a.b.width, a.b.width, a.c.n_pages, at / a.c.page);
  const int p = a.pos ? a.pos[t] : at;
  const bool known = (unsigned)p < (unsigned)a.n_pos;
  const float2 *cs = a.table + (known ? (long long)p * a.half : 0);
  if (is_q) {
    uint32_t j;
    const int h = (int)a.q_head.div(col, j);
    if (id < 0) {
      zero_unit<N>(a.shape, a.q_out, t, h * (N ? N : 1), (int)j);
    } else if constexpr (N == 0) {
      rope_unit(a.shape, a.q, a.q_out, t, h, (int)j, known ? cs : nullptr);
    } else {
      rope_wide_unit<N>(a.shape, a.q, a.q_out, t, h * N, a.q.heads, (int)j, known ? cs : nullptr);
    }
    return;
  }
  if (id < 0) return;
  int head = (int)a.tiles.div(col, tile);
  const int d0 = 16 * (int)tile;
  const bool is_v = head >= a.c.heads;
  if (is_v) head -= a.c.heads;
  float x[16];
  if (is_v) {
    row_load_n(a.v, t * a.v.row_stride + head * a.v.head_stride + d0, x);
  } else {
    double y[16];
    load_turned(a.k, t * a.k.row_stride + head * a.k.head_stride, d0, cs, a.half, a.interleaved, known, y);
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = f64_to_f32_sticky(y[j]);
  }
  uint32_t E;
  const uint2 w = kv4_encode(x, E);
  const long long o = kv4_tile(id, a.c.heads, head, (int)a.tiles.d, (int)tile, a.c.page, at & (a.c.page - 1));
  *(uint2 *)((is_v ? a.c.v : a.c.k) + o * KV4_TILE_BYTES) = w;
  (is_v ? a.c.v_e : a.c.k_e)[o] = (uint8_t)E;
}

struct Kv4ReadArgs {
  bfp_kv4 c;
  bfp_kv4_batch b;
  bfp_rows k, v;
  int first, sides;   // 0: k, 1: v
  Kv4Units units;
  FastDiv tiles;
  uint32_t n_units;
};

__global__ __launch_bounds__(KV4_BS) void k_kv4_read(Kv4ReadArgs a) {
  const int seq = blockIdx.y;
  const uint32_t u = blockIdx.x * KV4_BS + threadIdx.x;
  if (u >= a.n_units) return;
  const Kv4Span s = kv4_span(a.b.start[seq], a.b.start[seq + 1], a.b.len[seq], a.b.n_rows, a.b.max_q);
  int i;
  uint32_t col, tile;
  a.units.of(u, i, col);
  if (i >= s.n) return;
  int head = (int)a.tiles.div(col, tile);
  const bool is_v = a.first || head >= a.c.heads;
  if (head >= a.c.heads) head -= a.c.heads;
  const long long t = s.row0 + i;
  const int at = s.at + i;
  const int id = at < 0 ? -1 : kv4_page(a.b.pages + (long long)seq * a.b.width, a.b.width, a.c.n_pages, at / a.c.page);
  float x[16];
  if (id < 0) {
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = 0.0f;
  } else {
    const long long o = kv4_tile(id, a.c.heads, head, (int)a.tiles.d, (int)tile, a.c.page, at & (a.c.page - 1));
    kv4_decode(*(const uint2 *)((is_v ? a.c.v : a.c.k) + o * KV4_TILE_BYTES), (is_v ? a.c.v_e : a.c.k_e)[o], x);
  }
  const bfp_rows &r = is_v ? a.v : a.k;
  row_store_n(r, t * r.row_stride + head * r.head_stride + 16 * (int)tile, x);
}

// Units of `sections` heads of a batch, and their launch's width.
static int plan_units(const char *op, const bfp_kv4 &c, const bfp_kv4_batch &b, int sections,
                      Kv4Units &units, FastDiv &tiles, uint32_t &n_units) {
  const int nt = c.hd / 16;
  const int block = b.max_q >= 16 ? 16 : 1;
  const int cols = block == 1 ? nt : (nt % 4 == 0 ? 4 : nt % 2 == 0 ? 2 : 1);
  units.cols = FastDiv(cols);
  units.groups = FastDiv((uint32_t)(sections * (nt / cols)));
  units.block_shift = block == 1 ? 0 : 4;
  tiles = FastDiv(nt);
  const long long rows = ((long long)b.max_q + block - 1) / block * block;
  const long long n = rows * sections * nt;
  if (n > 0x7fffff00LL) return set_err(BFP_EINVAL, "%s: max_q=%d rows of %d heads are too many for one call", op, b.max_q, sections);
  n_units = (uint32_t)n;
  return BFP_OK;
}

}  // namespace bfp

using namespace bfp;

extern "C" {

int bfp_kv4_append_d(const bfp_kv4 *cache, const bfp_kv4_batch *batch, const bfp_rows *k,
                     const bfp_rows *v, const bfp_rows *q, const bfp_rows *q_out, const int32_t *pos,
                     const float *table, int n_pos, int rot, int interleaved, void *stream) {
  const char *op = "kv4_append";
  BFP_TRY(check_kv4(op, cache, batch));
  const int hd = cache->hd, rows = batch->n_rows;
  BFP_TRY(check_rows(op, "k", k, cache->heads, hd, true, rows));
  BFP_TRY(check_rows(op, "v", v, cache->heads, hd, true, rows));
  if (!rows_aligned(*k, 8, rows) || !rows_aligned(*v, 8, rows))
    return set_err(BFP_EINVAL, "%s: k and v need 16-byte alignment and strides in multiples of 8", op);
  if (!q != !q_out) return set_err(BFP_EINVAL, "%s: q and q_out go together", op);
  if (q) {
    if (q->heads < 1 || q->heads > 65536) return set_err(BFP_EINVAL, "%s: q has %d heads", op, q->heads);
    BFP_TRY(check_rows(op, "q", q, q->heads, hd, true, rows));
    BFP_TRY(check_out(op, "q_out", q_out, q->heads, hd, false, rows));
    if (!rows_aligned(*q, 8, rows) || !rows_aligned(*q_out, 8, rows))
      return set_err(BFP_EINVAL, "%s: q and q_out need 16-byte alignment and strides in multiples of 8", op);
    // q_out may be q: who writes a value has read its pair (rope_wide_unit)
    BFP_TRY(check_apart(op, "q_out", *q_out, "q", *q, rows, hd, true));
    BFP_TRY(check_apart(op, "q_out", *q_out, "k", *k, rows, hd, false));
    BFP_TRY(check_apart(op, "q_out", *q_out, "v", *v, rows, hd, false));
  }
  if (table) {
    if (rot < 2 || rot % 2 || rot > hd) return set_err(BFP_EINVAL, "%s: rot=%d, hd=%d", op, rot, hd);
    if (n_pos < 1) return set_err(BFP_EINVAL, "%s: n_pos=%d", op, n_pos);
    if ((uintptr_t)table % 8) return set_err(BFP_EINVAL, "%s: table is not 8-byte aligned", op);
  }
  if ((uintptr_t)pos % 4) return set_err(BFP_EINVAL, "%s: pos is not aligned", op);
  if (batch->n_seq == 0 || batch->max_q == 0 || rows == 0) return BFP_OK;
  Kv4AppendArgs a{};
  a.c = *cache;
  a.b = *batch;
  a.k = *k;
  a.v = *v;
  a.pos = pos;
  a.table = (const float2 *)table;
  a.n_pos = table ? n_pos : 0;
  a.half = table ? rot / 2 : 0;
  a.interleaved = interleaved ? 1 : 0;
  BFP_TRY(plan_units(op, a.c, a.b, 2 * a.c.heads, a.units, a.tiles, a.n_units));
  int n = 1;
  if (q) {
    a.q = *q, a.q_out = *q_out;
    a.shape = rope_shape(*q, *q_out, rows, hd, 2 * a.half, interleaved);
    // two heads a thread once that still leaves eight waves a CU
    const long long all = (long long)rows * q->heads * a.shape.per_head;
    n = !a.shape.wide ? 0 : q->heads >= ROPE_HEADS && all >= (long long)ROPE_HEADS * 256 * 8 * 64 ? ROPE_HEADS : 1;
    const long long per_row = (long long)a.shape.per_head * (n > 1 ? (q->heads + n - 1) / n : q->heads);
    if (per_row * batch->max_q > 0x7fffff00LL)
      return set_err(BFP_EINVAL, "%s: max_q=%d rows of %d query heads are too many for one call", op, batch->max_q, q->heads);
    a.q_row = FastDiv((uint32_t)per_row);
    a.q_head = FastDiv((uint32_t)a.shape.per_head);
    a.q_units = (uint32_t)(per_row * batch->max_q);
    a.q_blocks = (int)((a.q_units + KV4_BS - 1) / KV4_BS);
  }
  hipLaunchKernelGGL(n == 0 ? k_kv4_append<0> : n == 1 ? k_kv4_append<1> : k_kv4_append<ROPE_HEADS>,
                     dim3(a.q_blocks + (a.n_units + KV4_BS - 1) / KV4_BS, batch->n_seq), dim3(KV4_BS), 0,
                     (hipStream_t)stream, a);
  return launch_status(op);
}

int bfp_kv4_read_d(const bfp_kv4 *cache, const bfp_kv4_batch *batch, const bfp_rows *k,
                   const bfp_rows *v, void *stream) {
  const char *op = "kv4_read";
  BFP_TRY(check_kv4(op, cache, batch));
  if (!k && !v) return set_err(BFP_EINVAL, "%s: neither k nor v", op);
  for (const bfp_rows *r : {k, v}) {
    if (!r) continue;
    BFP_TRY(check_out(op, r == k ? "k" : "v", r, cache->heads, cache->hd, false, batch->n_rows));
    if (!rows_aligned(*r, 8, batch->n_rows))
      return set_err(BFP_EINVAL, "%s: k and v need 16-byte alignment and strides in multiples of 8", op);
  }
  if (batch->n_seq == 0 || batch->max_q == 0 || batch->n_rows == 0) return BFP_OK;
  if (k && v) BFP_TRY(check_apart(op, "v", *v, "k", *k, batch->n_rows, cache->hd, false));
  Kv4ReadArgs a{};
  a.c = *cache;
  a.b = *batch;
  if (k) a.k = *k;
  if (v) a.v = *v;
  a.first = k ? 0 : 1;
  a.sides = (k ? 1 : 0) + (v ? 1 : 0);
  BFP_TRY(plan_units(op, a.c, a.b, a.sides * a.c.heads, a.units, a.tiles, a.n_units));
  hipLaunchKernelGGL(k_kv4_read, dim3((a.n_units + KV4_BS - 1) / KV4_BS, batch->n_seq), dim3(KV4_BS), 0,
                     (hipStream_t)stream, a);
  return launch_status(op);
}

}  // extern "C"
