// Attention over the 4-bit paged cache: which kernel takes a call, and the
// entry points.
//
// Per query row and head: out = sum_j p_j v_j / sum_j p_j, p_j = exp(scale
// q.k_j - m), one pass over the keys with the running maximum m and sum
// (softmax in base 2, float32).  Both products run on the bfloat16 matrix
// cores.  A cached value has two significant bits, so its bfloat16 is exact;
// queries and probabilities that need more than bfloat16's eight are split
// into terms of eight bits.  With few rows to a KV head the terms are further
// columns of the same matrix tile and cost no further matrix instruction;
// prompts multiply term by term.
#include "bfp_kv4_attn.h"

#include <atomic>
#include <chrono>

namespace bfp {

struct Kv4Plan {
  bool prompt;       // k_kv4_prompt, else k_kv4_rows
  int terms, waves, row_tiles, splits, chunk, stream;
  size_t cells;      // of the workspace: rows of unfinished sums
  size_t work;       // its bytes
  double us;
};

// The terms a row is carried in: three (of four places) hold float32 queries
// and results; two hold a float16 or 16-bit-tile query and leave probabilities
// 2^-16 off (cut, then rounded; k_kv4_prompt rounds both, 2^-17).  One, for
// bfloat16 queries and results of more than 8 rows, rounds probabilities to
// bfloat16 as the result is: a second term would need a second row tile (8
// documents of 131072 tokens with 4 new ones, 16 rows a KV head: 158 us; 32
// rows, two tiles: 250).  Prompts the same: two of 8192 tokens with 32 heads of
// 128 take 811 us in one term and 1250 in two (float16), with a relative error
// against 64 bits of 0.0021 where float32 probabilities leave 0.0016, the
// result's own rounding.  float32 results carry all of them.
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
  p.chunk = (int)key_tiles;
  p.splits = 1;
  // Both kernels' times in microseconds, from what a workgroup of each takes
  // for itself (the first loads, the results) and for a round of 64-key tiles,
  // one workgroup a CU at a time:
  //                     few rows: itself, 16 / 8 / 4 tiles    prompts: itself, a tile
  //   heads up to 64          7.0 (float32 8.9), 2.7                 8.8 (10.6), 1.4
  //   up to 128               7.5 (9.5), 2.6                         12, 1.8
  //   up to 192, 256          11, 13; 2.6                            16, 20; 2.1
  // Measured when the rule was made (prompts have become 2 to 7% faster since),
  // with both forced: 22 rows of 9 heads 7.4 against 8.8, 100 rows
  // over 2000 keys 12.8 / 16.0 + 5.2, 5 x 300 rows in float32 74 / 18.9, 64 rows
  // of 32 heads of 128 over 4000 keys 46 / 26 + 13.
  const bool wide = q.type == BFP_F32 || out.type == BFP_F32 || out.type == BFP_TILES;
  const int size = tiles <= 4 ? 0 : tiles <= 8 ? 1 : tiles <= 12 ? 2 : 3;
  const long long all_rows = (b.n_rows < (long long)b.n_seq * b.max_q ? b.n_rows : (long long)b.n_seq * b.max_q) * group * c.heads;
  const double seen = key_tiles - 0.5 * ((b.max_q < keys ? b.max_q : keys) / KEYS);   // on average
  const double cus = 256.0;
  Kv4Plan few = p;
  {
    static const double itself[4] = {7.0, 7.5, 11.0, 13.0};
    few.prompt = false;
    few.terms = terms_of(q, out, (int)(rows < 64 ? rows : 64));
    const int R = 16 / few.terms;
    few.row_tiles = (int)((rows + R - 1) / R);
    few.waves = rows_waves(tiles);
    const double each = itself[size] + (few.terms == 4 ? 2.0 : 0.0), per_tile = 2.65 / few.waves;
    const double groups = (double)((all_rows + R - 1) / R);
    const double rounds = groups < cus ? 1.0 : groups / cus;
    // Short contexts: one workgroup takes a row tile's keys, four tiles a wave
    // at most, and there is nothing to join.  Otherwise as many workgroups as
    // run at once share all keys equally.
    const long long most_groups = (long long)few.row_tiles * c.heads * b.n_seq, cap_tiles = (cap + KEYS - 1) / KEYS;
    few.us = rounds * (each + per_tile * few.waves * ceil(seen / few.waves));
    // (Four waves also where wider workgroups would be more than 2^32 threads.)
    if (key_tiles > 4 * few.waves || most_groups * few.waves > 0x3ffffff) {
      few.waves = 4;
      if (b.n_seq <= 256 && most_groups * (cap_tiles + ROWS_EXTRA) < 0x7fffffffLL) {
        const long long most = most_groups * (key_tiles + ROWS_EXTRA) / 4 + 1, slots = tiles <= 4 ? 768 : tiles <= 8 ? 512 : 256;
        few.stream = (int)(most < slots ? most : slots);
        few.cells = 2 * (size_t)few.stream * R;
        few.us = each + R * c.hd / 128.0 + per_tile * groups * (seen + ROWS_EXTRA) / cus;   // joined by one workgroup
      }
    }
  }
  {
    static const double itself[4] = {8.8, 12.0, 16.0, 20.0}, tile[4] = {1.4, 1.8, 2.1, 2.1};
    p.prompt = true;
    p.terms = wide ? 3 : (q.type == BFP_BF16 && out.type == BFP_BF16 ? 1 : 2);
    p.waves = prompt_waves(tiles, p.terms);
    p.row_tiles = (int)((rows + 32 * p.waves - 1) / (32 * p.waves));
    const long long groups = (long long)p.row_tiles * c.heads * b.n_seq;
    long long s = groups > 0 ? 256 / groups : 1;
    if (s > key_tiles / 4) s = key_tiles / 4;
    if (s > 64) s = 64;   // a lane of k_kv4_join_prompt each
    if (s > 1) {
      p.splits = (int)s;
      p.chunk = (int)((key_tiles + s - 1) / s);
      p.cells = (size_t)b.n_seq * b.max_q * q.heads * p.splits;   // at most 256 row tiles
    }
    const double work = (double)all_rows / (32 * p.waves) * p.splits, rounds = work < cus ? 1.0 : work / cus;
    p.us = rounds * (itself[size] + (p.terms == 3 ? 1.8 : 0.0) + tile[size] * (p.splits > 1 ? p.chunk : seen)) + (p.splits > 1 ? 5.0 : 0.0);
  }
  if (few.us <= p.us) p = few;
  p.work = p.cells * (16 * tiles * sizeof(float) + sizeof(float2)) + 2 * p.stream * sizeof(unsigned long long);
  return p;
}

// A number no other call has: what k_kv4_rows knows its flags in the
// workspace by, whatever the workspace held before.
static unsigned long long call_number() {
  static std::atomic<unsigned long long> next{[] {
    const unsigned long long t = (unsigned long long)std::chrono::steady_clock::now().time_since_epoch().count();
    return (t ^ (unsigned long long)(uintptr_t)&next) * 0x9E3779B97F4A7C15ull;
  }()};
  const unsigned long long n = next.fetch_add(1, std::memory_order_relaxed);
  return n ? n : next.fetch_add(1, std::memory_order_relaxed);   // 0 is no call's
}

static int check_attn(const char *op, const bfp_kv4 *cache, const bfp_kv4_batch *batch, const bfp_rows *q,
                      const bfp_rows *out, int window, bool placed) {
  BFP_TRY(check_kv4(op, cache, batch));
  if (!q || q->heads < cache->heads || q->heads % cache->heads || q->heads > 65536)
    return set_err(BFP_EINVAL, "%s: q has %d heads, the cache %d", op, q ? q->heads : 0, cache->heads);
  BFP_TRY(check_rows(op, "q", q, q->heads, cache->hd, true, batch->n_rows));
  BFP_TRY(check_out(op, "out", out, q->heads, cache->hd, true, batch->n_rows));
  if (!rows_aligned(*q, 8, batch->n_rows)) return set_err(BFP_EINVAL, "%s: q needs 16-byte alignment and strides in multiples of 8", op);
  // out may be q: a workgroup has read its rows' queries before anyone writes their results
  if (placed) BFP_TRY(check_apart(op, "out", *out, "q", *q, batch->n_rows, cache->hd, true));
  if (window < 0) return set_err(BFP_EINVAL, "%s: window=%d", op, window);
  if ((long long)batch->max_q * (q->heads / cache->heads) > 0x3fffffffLL)
    return set_err(BFP_EINVAL, "%s: max_q=%d rows of %d heads are too many", op, batch->max_q, q->heads);
  return BFP_OK;
}

}  // namespace bfp

using namespace bfp;

extern "C" {

size_t bfp_kv4_attn_work(const bfp_kv4 *cache, const bfp_kv4_batch *batch, const bfp_rows *q,
                         const bfp_rows *out, int window) {
  if (check_attn("kv4_attn_work", cache, batch, q, out, window, false)) return 0;
  return plan_attn(*cache, *batch, *q, *out, window).work;
}

int bfp_kv4_attn_d(const bfp_kv4 *cache, const bfp_kv4_batch *batch, const bfp_rows *q,
                   const bfp_rows *out, double scale, int window, void *work, size_t work_bytes,
                   void *stream) {
  const char *op = "kv4_attn";
  BFP_TRY(check_attn(op, cache, batch, q, out, window, true));
  const float scale2 = (float)(fabs(scale) * 1.44269504088896340736);
  if (!isfinite(scale2)) return set_err(BFP_EINVAL, "%s: scale=%g is not float32's", op, scale);
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
  a.chunk = p.chunk;
  // a scale of zero, or too small for float32: all scores alike, from queries of zeros
  a.scale2 = scale2 == 0.0f ? 1.0f : scale2;
  a.q_sign = scale2 == 0.0f ? 0.0f : scale < 0 ? -1.0f : 1.0f;
  // (kept finite, and so that no score below 2^126 passes float32 with it)
  a.slack = fminf(M_SLACK / a.scale2, 0x1p125f);
  a.stream = p.stream;
  if (p.work) {
    a.part_o = (float *)work;
    a.part_ml = (float2 *)((float *)work + p.cells * 16 * a.tiles);
    a.there = (unsigned long long *)(a.part_ml + p.cells);
    a.number = call_number();
  }
  a.row_tiles = p.row_tiles;
  a.by_head = FastDiv(cache->heads);
  a.by_split = FastDiv(p.splits);
  a.by_group = FastDiv((uint32_t)a.group);
  a.out_wide = rows_aligned(*out, 8, batch->n_rows);
  const long long each = (long long)p.row_tiles * p.splits * cache->heads, blocks = p.stream ? p.stream : each * batch->n_seq;
  if (blocks > 0x3ffffff / p.waves || each > 0x7fffffff)   // 2^32 threads
    return set_err(BFP_EINVAL, "%s: n_seq=%d of max_q=%d rows are too many for one call", op, batch->n_seq, batch->max_q);
  a.by_seq = FastDiv((uint32_t)each);
  const AttnKernel k = p.prompt ? prompt_kernel(a.tiles, p.terms) : rows_kernel(a.tiles, p.terms, p.waves);
  if (k.lds > 65536)   // one limit for a kernel, whatever the call
    HIP_TRY(hipFuncSetAttribute((const void *)k.fn, hipFuncAttributeMaxDynamicSharedMemorySize, 158 * 1024));
  hipLaunchKernelGGL(k.fn, dim3((unsigned)blocks), dim3(64 * p.waves), k.lds, (hipStream_t)stream, a);
  BFP_TRY(launch_status(op));
  if (p.splits == 1) return BFP_OK;
  launch_join_prompt(a, (hipStream_t)stream);
  return launch_status(op);
}

}  // extern "C"
