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

#include <algorithm>
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

// The longest sequence's keys that any of its rows sees, from position `from` on.
static long long keys_of(const bfp_kv4 &c, const bfp_kv4_batch &b, int window, long long from) {
  const long long cap = (long long)b.width * c.page;
  long long keys = (b.max_len > 0 && b.max_len < cap ? b.max_len : cap) - from;
  keys = keys < 1 ? 1 : keys;
  return window > 0 && keys > (long long)window + b.max_q ? (long long)window + b.max_q : keys;
}

// keys: of the longest sequence; whole: all rows see all of them, else up to
// their own; most: splits; row_terms: of every row, whatever the kernel (0:
// each kernel's own).
static Kv4Plan plan_keys(const bfp_kv4 &c, const bfp_kv4_batch &b, const bfp_rows &q, const bfp_rows &out, long long keys, bool whole,
                         int most, int row_terms = 0) {
  Kv4Plan p{};
  const int group = q.heads / c.heads, tiles = c.hd / 16;
  const long long rows = (long long)b.max_q * group;
  const long long cap = (long long)b.width * c.page;
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
  const double seen = whole ? key_tiles : key_tiles - 0.5 * ((b.max_q < keys ? b.max_q : keys) / KEYS);   // on average
  const double cus = 256.0;
  Kv4Plan few = p;
  {
    static const double itself[4] = {7.0, 7.5, 11.0, 13.0};
    few.prompt = false;
    few.terms = row_terms ? row_terms : terms_of(q, out, (int)(rows < 64 ? rows : 64));
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
        // A shared prefix takes 15 us more so (8 to 32 rows of 32 + 8 heads): heads of 128, 16384
        // keys 42, 41, 52, 58 against the prompts' 27, 29, 30, 31; 65536 keys 65, 85, 106,
        // 128 against 67, 68, 70, 71; heads of 64, 16384 keys 33 to 39 against 21 to 23.
        if (whole) few.us += 15.0;
      }
    }
  }
  {
    static const double itself[4] = {8.8, 12.0, 16.0, 20.0}, tile[4] = {1.4, 1.8, 2.1, 2.1};
    p.prompt = true;
    p.terms = wide ? 3 : row_terms ? row_terms : (q.type == BFP_BF16 && out.type == BFP_BF16 ? 1 : 2);
    p.waves = prompt_waves(tiles, p.terms);
    p.row_tiles = (int)((rows + 32 * p.waves - 1) / (32 * p.waves));
    const long long groups = (long long)p.row_tiles * c.heads * b.n_seq;
    long long s = groups > 0 ? 256 / groups : 1;
    if (s > key_tiles / 4) s = key_tiles / 4;
    if (s > most) s = most;   // a lane of the joining wave each
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

static Kv4Plan plan_attn(const bfp_kv4 &c, const bfp_kv4_batch &b, const bfp_rows &q, const bfp_rows &out, int window) {
  return plan_keys(c, b, q, out, keys_of(c, b, window, 0), false, 64);
}

// Shared prefixes: the groups' rows as sequences against the groups' tokens,
// then every sequence's tokens behind them; the parts of a row side by side.
struct SharedPlan {
  Kv4Plan prefix, rest;
  bfp_kv4_batch groups;
  int pieces;               // k_kv4_prompt of up to 64 groups: workgroups that share the keys
  long long blocks;         // and the launch's (0: its plan's)
  bool joined;              // both parts in one launch
  bool pairs;               // the prompts' kernel with two workgroups a CU
  size_t prefix_sums, sums, own, work;   // parts of rows, of the prefix and in all; bytes of the launches' own parts
};
static SharedPlan plan_shared(const bfp_kv4 &c, const bfp_kv4_batch &b, const bfp_kv4_shared &sh, const bfp_rows &q, const bfp_rows &out,
                              int window) {
  SharedPlan p;
  p.groups = b;
  p.groups.pages = sh.pages;
  p.groups.n_seq = sh.n_groups;
  p.groups.width = sh.width;
  p.groups.max_len = sh.max_len;
  p.groups.max_q = sh.max_rows > 0 && sh.max_rows < b.n_rows ? sh.max_rows : b.n_rows;
  // Both parts in the terms that a sequence's rows have by themselves, however
  // many the group has.  (64 samples of one problem, 4 rows a KV head, 256 a group,
  // 16384 tokens: the prefix takes 49 us in two terms and 38 in one, which leaves
  // bfloat16 results 1.3 times as far from the exact ones as without groups.)
  const long long seq_rows = (long long)(b.max_q < b.n_rows ? b.max_q : b.n_rows) * (q.heads / c.heads);
  const int terms = terms_of(q, out, (int)(seq_rows < 64 ? seq_rows : 64));
  const long long prefix = keys_of(c, p.groups, window, 0);
  p.prefix = plan_keys(c, p.groups, q, out, prefix, true, 48, terms);
  // Without a hint the rest may be anything: the keys of a stream are shared out on the device.
  const long long cap = (long long)sh.width * c.page;
  p.rest = plan_keys(c, b, q, out, keys_of(c, b, window, sh.max_len < cap ? sh.max_len : cap), false, 16, terms);
  long long few = 0;   // workgroups of few rows that take all keys of a row tile: more than the card has CUs, then four waves each
  for (const Kv4Plan *k : {&p.prefix, &p.rest})
    if (!k->prompt && !k->stream) few += (long long)k->row_tiles * c.heads * (k == &p.rest ? b.n_seq : sh.n_groups);
  for (Kv4Plan *k : {&p.prefix, &p.rest})
    if (!k->prompt && !k->stream && few > 256) k->waves = 4;
  // Both such, a prefix of few keys or rows and few keys behind it: one launch (5
  // chats behind 304 tokens, 9 heads of 64: 23 us in two launches, 15 in one).
  // (One kernel then: a row tile's rows follow from the terms, which are the same.)
  p.joined = !p.prefix.prompt && !p.prefix.stream && !p.rest.prompt && !p.rest.stream && p.prefix.waves == p.rest.waves;
  // Prompts' kernel: 128 rows a workgroup where that leaves fewer rows empty
  // than 256 (groups of 320 rows, heads of 96, two terms: 217 us against 260; of 128
  // rows, heads of 128, 65536 keys: 72 against 86; where both fill them alike 550
  // against 520).
  const long long group_rows = (long long)p.groups.max_q * (q.heads / c.heads), in_8 = (group_rows + 255) / 256 * 256, in_4 = (group_rows + 127) / 128 * 128;
  p.pairs = p.prefix.prompt && prompt_pairs(c.hd / 16, p.prefix.terms) && in_4 + in_4 / 8 < in_8;
  if (p.pairs) {
    p.prefix.waves = 4;
    p.prefix.row_tiles = (int)(in_4 / 128);
  }
  // Up to 64 groups: the device shares the keys out, whatever the groups'
  // lengths; no group has more splits than workgroups a KV head.  Either all
  // row tiles' keys are whole, or they are split into `pieces` at most.  The
  // launch has room for both, and each workgroup a place for its rows' sums:
  // with places by row, as many as a row can have splits, 64 suffixes of 512
  // tokens behind 16384 would take 18 GB of scratch instead of 1.1.
  p.pieces = p.blocks = 0;
  if (p.prefix.prompt && sh.n_groups <= 64) {
    const int group = q.heads / c.heads, rows = 32 * p.prefix.waves;
    const long long key_tiles = (prefix + KEYS - 1) / KEYS;
    const long long in_groups = std::min<long long>(b.n_rows, (long long)sh.n_groups * p.groups.max_q);
    const long long most = ((in_groups * group + rows - 1) / rows + sh.n_groups) * c.heads;
    p.pieces = p.pairs ? 512 : 256;
    int s = p.pieces / c.heads;
    if (s > key_tiles / 4) s = (int)(key_tiles / 4);
    p.prefix.splits = s < 1 ? 1 : s < 48 ? s : 48;
    p.blocks = std::max(most, std::min<long long>(p.pieces, most * p.prefix.splits));
  }
  const size_t rows = (size_t)b.n_rows * q.heads;
  p.prefix_sums = p.pieces ? (size_t)p.blocks * 32 * p.prefix.waves : rows * p.prefix.splits;
  p.sums = p.prefix_sums + (p.rest.splits > 1 ? p.rest.cells : rows);
  p.sums += p.sums & 1;   // (what lies behind float2s is 16-byte aligned)
  // one launch after the other: the same room for the parts of few rows that share out their keys
  p.own = std::max(p.prefix.stream ? p.prefix.work : 0, p.rest.stream ? p.rest.work : 0);
  p.own = (p.own + 15) / 16 * 16;
  p.work = p.sums * (c.hd * sizeof(float) + sizeof(float2)) + p.own + 64 * sizeof(int4);
  return p;
}

static bool picks_fit(const bfp_kv4 &c, int n) { return n >= 1 && (long long)n * c.page <= KV4_MAX_POS; }

// Rows that see the pages a list names: few rows to a list, one token's query
// heads, so always k_kv4_rows, its keys those of the list.
static Kv4Plan plan_picks(const bfp_kv4 &c, const bfp_kv4_batch &b, const bfp_rows &q, const bfp_rows &out, int n, int &token_tiles) {
  Kv4Plan p{};
  const int group = q.heads / c.heads, tiles = c.hd / 16;
  p.terms = terms_of(q, out, group);
  const int R = 16 / p.terms;
  token_tiles = (group + R - 1) / R;
  p.row_tiles = b.max_q * token_tiles;
  p.splits = 1;
  const long long key_tiles = ((long long)n * c.page + KEYS - 1) / KEYS;
  p.chunk = (int)key_tiles;
  const long long rows = b.n_rows < (long long)b.n_seq * b.max_q ? b.n_rows : (long long)b.n_seq * b.max_q;
  const long long groups = rows * token_tiles * c.heads, most_groups = (long long)p.row_tiles * c.heads * b.n_seq;
  p.waves = rows_waves(tiles);
  if (key_tiles > 4 * p.waves || most_groups * p.waves > 0x3ffffff || groups > 256) {
    p.waves = groups > 1536 ? 2 : 4;
    if (groups <= 256 && key_tiles > 16 && b.n_seq <= 256 && most_groups * (key_tiles + ROWS_EXTRA) < 0x7fffffffLL) {
      const long long most = groups * (key_tiles + ROWS_EXTRA) / 4 + 1, slots = tiles <= 4 ? 768 : tiles <= 8 ? 512 : 256;
      p.stream = (int)(most < slots ? most : slots);
      p.cells = 2 * (size_t)p.stream * R;
    }
  }
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

// The arguments that follow from a call's; the scale's checks.
static int attn_args(const char *op, Kv4AttnArgs &a, const bfp_kv4 &cache, const bfp_kv4_batch &batch, const bfp_rows &q,
                     const bfp_rows &out, double scale, int window) {
  const float scale2 = (float)(fabs(scale) * 1.44269504088896340736);
  if (!isfinite(scale2)) return set_err(BFP_EINVAL, "%s: scale=%g is not float32's", op, scale);
  a = Kv4AttnArgs{};
  a.c = cache;
  a.b = batch;
  a.q = q;
  a.out = out;
  a.tiles = cache.hd / 16;
  a.group = q.heads / cache.heads;
  a.page_shift = __builtin_ctz((unsigned)cache.page);
  a.window = window;
  // a scale of zero, or too small for float32: all scores alike, from queries of zeros
  a.scale2 = scale2 == 0.0f ? 1.0f : scale2;
  a.q_sign = scale2 == 0.0f ? 0.0f : scale < 0 ? -1.0f : 1.0f;
  // (kept finite, and so that no score below 2^126 passes float32 with it)
  a.slack = fminf(M_SLACK / a.scale2, 0x1p125f);
  a.by_head = FastDiv(cache.heads);
  a.by_group = FastDiv((uint32_t)a.group);
  a.out_wide = rows_aligned(out, 8, batch.n_rows);
  return BFP_OK;
}

static int check_work(const char *op, size_t need, const void *work, size_t work_bytes) {
  if (need && (!work || (uintptr_t)work % 16 || work_bytes < need))
    return set_err(BFP_EINVAL, "%s: needs %zu bytes of 16-byte-aligned scratch, got %zu", op, need, work ? work_bytes : (size_t)0);
  return BFP_OK;
}

// The arguments that follow from a plan, and how many workgroups it has.
static int plan_args(const char *op, Kv4AttnArgs &a, const Kv4Plan &p, long long &blocks) {
  a.splits = p.splits;
  a.chunk = p.chunk;
  a.stream = p.stream;
  a.row_tiles = p.row_tiles;
  a.by_split = FastDiv(p.splits);
  const long long each = (long long)p.row_tiles * p.splits * a.c.heads;
  if (!blocks) blocks = p.stream ? p.stream : each * a.b.n_seq;
  if (blocks > 0x3ffffff / p.waves || each > 0x7fffffff)   // 2^32 threads
    return set_err(BFP_EINVAL, "%s: n_seq=%d of max_q=%d rows are too many for one call", op, a.b.n_seq, a.b.max_q);
  a.by_seq = FastDiv((uint32_t)each);
  return BFP_OK;
}
template <typename Fn>
static int lds_limit(Fn fn, int lds) {
  if (lds > 65536)   // one limit for a kernel, whatever the call
    HIP_TRY(hipFuncSetAttribute((const void *)fn, hipFuncAttributeMaxDynamicSharedMemorySize, 158 * 1024));
  return BFP_OK;
}

static int launch_plan(const char *op, Kv4AttnArgs &a, const Kv4Plan &p, const AttnKernel &k, hipStream_t s, long long blocks = 0) {
  BFP_TRY(plan_args(op, a, p, blocks));
  BFP_TRY(lds_limit(k.fn, k.lds));
  hipLaunchKernelGGL(k.fn, dim3((unsigned)blocks), dim3(64 * p.waves), k.lds, s, a);
  return launch_status(op);
}

static int launch_attn(const char *op, Kv4AttnArgs &a, const Kv4Plan &p, const AttnKernel &k, void *work, size_t work_bytes, hipStream_t s) {
  BFP_TRY(check_work(op, p.work, work, work_bytes));
  if (p.work) {
    a.part_o = (float *)work;
    a.part_ml = (float2 *)((float *)work + p.cells * 16 * a.tiles);
    a.there = (unsigned long long *)(a.part_ml + p.cells);
    a.number = call_number();
  }
  return launch_plan(op, a, p, k, s);
}

// One of the two parts, with its own workspace.
static int launch_part(const char *op, Kv4AttnArgs a, const Kv4Plan &p, const AttnKernel &k, void *own, hipStream_t s,
                       long long blocks = 0) {
  if (p.stream) {
    a.slot_o = (float *)own;
    a.slot_ml = (float2 *)((float *)own + p.cells * 16 * a.tiles);
    a.there = (unsigned long long *)(a.slot_ml + p.cells);
    a.number = call_number();
  }
  return launch_plan(op, a, p, k, s, blocks);
}

static int check_shared(const char *op, const bfp_kv4_batch *b, const bfp_kv4_shared *sh, const bfp_kv4 *c, const bfp_rows *q) {
  if (!sh || !sh->pages || !sh->start || !sh->len) return set_err(BFP_EINVAL, "%s: no groups", op);
  if (((uintptr_t)sh->pages | (uintptr_t)sh->start | (uintptr_t)sh->len) % 4)
    return set_err(BFP_EINVAL, "%s: the groups' arrays are not aligned", op);
  if (sh->n_groups < 1 || sh->n_groups > 65535 || sh->width < 1 || sh->max_rows < 0 || sh->max_len < 0)
    return set_err(BFP_EINVAL, "%s: n_groups=%d (1 to 65535), width=%d, max_rows=%d, max_len=%d", op, sh->n_groups, sh->width,
                   sh->max_rows, sh->max_len);
  if ((long long)sh->width * c->page > KV4_MAX_POS)
    return set_err(BFP_EINVAL, "%s: width=%d pages of %d are more than %d positions", op, sh->width, c->page, KV4_MAX_POS);
  if ((long long)b->n_rows * (q->heads / c->heads) > 0x3fffffffLL && (sh->max_rows == 0 || (long long)sh->max_rows * (q->heads / c->heads) > 0x3fffffffLL))
    return set_err(BFP_EINVAL, "%s: groups of max_rows=%d rows of %d heads are too many", op, sh->max_rows, q->heads);
  if ((long long)(b->max_q < b->n_rows ? b->max_q : b->n_rows) * q->heads > 0x3fffff0LL)   // the join: 2^32 threads
    return set_err(BFP_EINVAL, "%s: max_q=%d rows of %d heads are too many", op, b->max_q, q->heads);
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
  Kv4AttnArgs a;
  BFP_TRY(attn_args(op, a, *cache, *batch, *q, *out, scale, window));
  if (batch->n_seq == 0 || batch->max_q == 0 || batch->n_rows == 0) return BFP_OK;
  const Kv4Plan p = plan_attn(*cache, *batch, *q, *out, window);
  BFP_TRY(launch_attn(op, a, p, p.prompt ? prompt_kernel(a.tiles, p.terms) : rows_kernel(a.tiles, p.terms, p.waves), work, work_bytes,
                      (hipStream_t)stream));
  if (p.splits == 1) return BFP_OK;
  launch_join_prompt(a, (hipStream_t)stream);
  return launch_status(op);
}

size_t bfp_kv4_attn_shared_work(const bfp_kv4 *cache, const bfp_kv4_batch *batch, const bfp_kv4_shared *shared, const bfp_rows *q,
                                const bfp_rows *out, int window) {
  const char *op = "kv4_attn_shared_work";
  if (check_attn(op, cache, batch, q, out, window, false) || check_shared(op, batch, shared, cache, q)) return 0;
  if (batch->n_seq == 0 || batch->max_q == 0 || batch->n_rows == 0) return 0;
  return plan_shared(*cache, *batch, *shared, *q, *out, window).work;
}

int bfp_kv4_attn_shared_d(const bfp_kv4 *cache, const bfp_kv4_batch *batch, const bfp_kv4_shared *shared, const bfp_rows *q,
                          const bfp_rows *out, double scale, int window, void *work, size_t work_bytes, void *stream) {
  const char *op = "kv4_attn_shared";
  BFP_TRY(check_attn(op, cache, batch, q, out, window, true));
  BFP_TRY(check_shared(op, batch, shared, cache, q));
  Kv4AttnArgs a;
  BFP_TRY(attn_args(op, a, *cache, *batch, *q, *out, scale, window));
  if (batch->n_seq == 0 || batch->max_q == 0 || batch->n_rows == 0) return BFP_OK;
  const SharedPlan p = plan_shared(*cache, *batch, *shared, *q, *out, window);
  BFP_TRY(check_work(op, p.work, work, work_bytes));
  hipStream_t s = (hipStream_t)stream;
  // Few tiles a workgroup, whose first one sets the maximum: it is raised less
  // often.  Not for rows in float32: exponents down to -32 are rounded to 2^-20, those
  // to -16 to 2^-21, which is what probabilities are off there (2^-16 in two terms).
  if (p.prefix.terms < 3) a.slack = fminf(2 * M_SLACK / a.scale2, 0x1p125f);
  a.sh = *shared;
  a.sh_seqs = batch->n_seq;
  a.prefix_splits = p.prefix.splits;
  a.rest_splits = p.rest.splits;
  a.rest_first = (long long)p.prefix_sums;
  a.part_o = (float *)work;
  a.part_ml = (float2 *)(a.part_o + p.sums * cache->hd);
  void *own = a.part_ml + p.sums;
  a.pieces = p.pieces;
  a.piece_shift = __builtin_ctz((unsigned)(32 * p.prefix.waves));
  a.piece_blocks = (int)p.blocks;
  a.piece_of = (int4 *)((char *)own + p.own);
  Kv4AttnArgs g = a;
  g.b = p.groups;
  const Kv4Plan &one = p.prefix, &two = p.rest;
  if (p.joined) {
    long long n1 = 0, n2 = 0;
    BFP_TRY(plan_args(op, g, one, n1));
    BFP_TRY(plan_args(op, a, two, n2));
    if (n1 + n2 > 0x3ffffff / one.waves)
      return set_err(BFP_EINVAL, "%s: n_groups=%d and n_seq=%d are too many for one call", op, shared->n_groups, batch->n_seq);
    const PartsKernel k = parts_kernel(a.tiles, one.terms, one.waves);
    BFP_TRY(lds_limit(k.fn, k.lds));
    hipLaunchKernelGGL(k.fn, dim3((unsigned)(n1 + n2)), dim3(64 * one.waves), k.lds, s, g, a, (uint32_t)n1);
    BFP_TRY(launch_status(op));
    launch_join_shared(a, s);
    return launch_status(op);
  }
  BFP_TRY(launch_part(op, g, one, one.prompt ? prefix_prompt_kernel(a.tiles, one.terms, p.pairs) : prefix_rows_kernel(a.tiles, one.terms, one.waves, one.stream > 0),
                      own, s, p.blocks));
  BFP_TRY(launch_part(op, a, two, two.prompt ? rest_prompt_kernel(a.tiles, two.terms) : rest_rows_kernel(a.tiles, two.terms, two.waves, two.stream > 0),
                      own, s));
  launch_join_shared(a, s);
  return launch_status(op);
}

size_t bfp_kv4_attn_picks_work(const bfp_kv4 *cache, const bfp_kv4_batch *batch, int n_picks, const bfp_rows *q, const bfp_rows *out) {
  int token_tiles;
  if (check_attn("kv4_attn_picks_work", cache, batch, q, out, 0, false) || !picks_fit(*cache, n_picks)) return 0;
  return plan_picks(*cache, *batch, *q, *out, n_picks, token_tiles).work;
}

int bfp_kv4_attn_picks_d(const bfp_kv4 *cache, const bfp_kv4_batch *batch, const int32_t *picks, int n_picks, const bfp_rows *q,
                         const bfp_rows *out, double scale, void *work, size_t work_bytes, void *stream) {
  const char *op = "kv4_attn_picks";
  BFP_TRY(check_attn(op, cache, batch, q, out, 0, true));
  if (!picks_fit(*cache, n_picks)) return set_err(BFP_EINVAL, "%s: n_picks=%d", op, n_picks);
  Kv4AttnArgs a;
  BFP_TRY(attn_args(op, a, *cache, *batch, *q, *out, scale, 0));
  if (batch->n_seq == 0 || batch->max_q == 0 || batch->n_rows == 0) return BFP_OK;
  if (!picks || (uintptr_t)picks % 4) return set_err(BFP_EINVAL, "%s: picks are null or not aligned", op);
  const Kv4Plan p = plan_picks(*cache, *batch, *q, *out, n_picks, a.token_tiles);
  a.picks = picks;
  a.n_picks = n_picks;
  return launch_attn(op, a, p, picks_kernel(a.tiles, p.terms, p.waves, p.stream > 0), work, work_bytes, (hipStream_t)stream);
}

}  // extern "C"
