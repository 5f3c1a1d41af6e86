// Which pages of a paged cache are held, how often, and their copies: pages
// given to new tokens, branches that share whole pages, pages given up, and a
// pool made compact.
//
// refs[p] counts the table entries that hold page p; a page is free where it
// is 0.  Whoever asks for pages gets the free ones with the lowest numbers, in
// the order of the tables' entries, so what a program's tables hold does not
// depend on how its threads ran.  The bookkeeping is one workgroup's (a few
// thousand counts a step, the whole pool's at worst: 16384 pages a round of
// 16-byte loads); what moves bytes is a launch of its own over all arrays.  The
// bookkeeping is bound by its chain of loads and barriers (1.8 to 6.6 us a launch),
// the moves by HBM: 4096 pages of 74 KB in two layers, 604 MB in 98-115 us, 5.3-6.2
// TB/s; 256 branches' last pages in eight layers, four of a source, in 34 us.
#include <string.h>

#include "bfp.h"
#include "bfp_internal.h"
#include "bfp_kv4.h"
#include "bfp_rows.h"

namespace bfp {

constexpr int POOL_T = 1024;        // threads of the bookkeeping's workgroup
constexpr int POOL_U = 4;           // 16-byte words of counts a thread has under way
constexpr int POOL_CHUNK = 4096;    // counts a workgroup of the compaction looks at
constexpr int POOL_MAX = 1 << 28;   // pages of a pool
constexpr int COPY_ARRAYS = 192;    // arrays of a copying launch: its arguments are 4 KB at most
constexpr int COPY_T = 256;
constexpr int COPY_UNIT = 4096;     // bytes a wave moves at a time: 4 words of 16 bytes a lane
constexpr int POOL_TABLES = 16;

struct CopyArgs {
  bfp_page_array array[COPY_ARRAYS];
  int n_arrays, n_pages, blocks;
  const int32_t *src, *dst, *count;   // count: how many moves there are (null: n)
  int n;
};

// Sums over the workgroup's threads before this one; total: over all.
template <int T, typename I>
__device__ __forceinline__ I block_scan(I v, I *waves, I &total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  I up = v;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const I x = __shfl_up(up, d, 64);
    up += lane >= d ? x : 0;
  }
  __syncthreads();   // the last call's sums have been read
  if (lane == 63) waves[w] = up;
  __syncthreads();
  I before = 0;
  total = 0;
#pragma unroll
  for (int k = 0; k < T / 64; ++k) {
    before += k < w ? waves[k] : 0;
    total += waves[k];
  }
  return before + up - v;
}

// Four counts from 4 * i on, and 1 behind the last page.
__device__ __forceinline__ int4 counts4(const int32_t *refs, int n_pages, long long i) {
  if (4 * i + 4 <= n_pages) return ((const int4 *)refs)[i];
  int4 c = make_int4(1, 1, 1, 1);
  if (4 * i < n_pages) c.x = refs[4 * i];
  if (4 * i + 1 < n_pages) c.y = refs[4 * i + 1];
  if (4 * i + 2 < n_pages) c.z = refs[4 * i + 2];
  return c;
}

// The `want` lowest free pages into give, all threads of a workgroup; returns
// how many there were.
__device__ int find_free(const int32_t *refs, int n_pages, int want, int32_t *give) {
  __shared__ unsigned long long waves[POOL_T / 64];
  int have = 0;
  for (long long base = 0; 4 * base < n_pages && have < want; base += POOL_T * POOL_U) {
    int4 c[POOL_U];
#pragma unroll
    for (int u = 0; u < POOL_U; ++u) c[u] = counts4(refs, n_pages, base + u * POOL_T + threadIdx.x);
    unsigned long long mine = 0, all;   // of each word 16 bits: at most 4096 a workgroup
#pragma unroll
    for (int u = 0; u < POOL_U; ++u)
      mine |= (unsigned long long)((c[u].x <= 0) + (c[u].y <= 0) + (c[u].z <= 0) + (c[u].w <= 0)) << (16 * u);
    const unsigned long long before = block_scan<POOL_T>(mine, waves, all);
#pragma unroll
    for (int u = 0; u < POOL_U; ++u) {
      int r = have + (int)((before >> (16 * u)) & 0xffff);
      const int id = (int)(4 * (base + u * POOL_T + threadIdx.x));
      const int free[4] = {c[u].x <= 0, c[u].y <= 0, c[u].z <= 0, c[u].w <= 0};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (free[k] && r < want) give[r] = id + k;
        r += free[k];
      }
      have += (int)((all >> (16 * u)) & 0xffff);
    }
  }
  __syncthreads();
  return have < want ? have : want;
}

// A free page of its own for whoever asks; those that are not there are
// counted.
__device__ __forceinline__ void count_short(int32_t *n_short, int want, int have) {
  if (threadIdx.x == 0 && n_short && want > have) atomicAdd(n_short, want - have);
}

struct ReserveArgs {
  int32_t *refs, *n_short, *pages, *give;
  bfp_kv4_batch b;
  int n_pages, page, touched;   // pages that a sequence's new rows can lie in, at most
};

// The entry (b, j) of the batch's touched pages that holds no page, or -1.
__device__ __forceinline__ long long wanting(const ReserveArgs &a, long long f) {
  const int seq = (int)(f / a.touched), j = (int)(f % a.touched);
  if (seq >= a.b.n_seq) return -1;
  const Kv4Span s = kv4_span(a.b.start[seq], a.b.start[seq + 1], a.b.len[seq], a.b.n_rows, a.b.max_q);
  const int stop = s.at + s.n, first = s.at > 0 ? s.at : 0;   // positions of its rows
  if (s.n == 0 || stop <= first) return -1;
  const int p = first / a.page + j;
  if (p > (stop - 1) / a.page || p >= a.b.width) return -1;
  const long long e = (long long)seq * a.b.width + p;
  return (unsigned)a.pages[e] < (unsigned)a.n_pages ? -1 : e;
}

__global__ __launch_bounds__(POOL_T) void k_pool_reserve(ReserveArgs a) {
  __shared__ int waves[POOL_T / 64];
  const long long all = (long long)a.b.n_seq * a.touched;
  int want = 0;
  for (long long f = threadIdx.x; f < all; f += POOL_T) want += wanting(a, f) >= 0;
  int total;
  block_scan<POOL_T>(want, waves, total);
  if (total == 0) return;
  const int have = find_free(a.refs, a.n_pages, total, a.give);
  count_short(a.n_short, total, have);
  int base = 0;
  for (long long f0 = 0; f0 < all; f0 += POOL_T) {
    const long long e = wanting(a, f0 + threadIdx.x);
    int n;
    const int r = base + block_scan<POOL_T>(e >= 0 ? 1 : 0, waves, n);
    if (e >= 0) {
      const int id = r < have ? a.give[r] : -1;
      a.pages[e] = id;
      if (id >= 0) a.refs[id] = 1;
    }
    base += n;
  }
}

struct ForkArgs {
  int32_t *refs, *n_short;
  const int32_t *pages, *len, *parents;
  int32_t *out_pages, *out_len, *give, *src, *dst;
  int n_pages, page, n_seq, width, out_width, n;
};

// How many tokens child i goes on from, and its parent's row.
__device__ __forceinline__ int child_len(const ForkArgs &a, int i, const int32_t *&row) {
  const int j = a.parents[i];
  if ((unsigned)j >= (unsigned)a.n_seq) return 0;
  row = a.pages + (long long)j * a.width;
  const int most = a.width * a.page, n = a.len[j];
  return n < 0 ? 0 : n < most ? n : most;
}

// The copies that the children need: src[i], dst[i] (-1: none; dst alone: no page
// was left).
__global__ __launch_bounds__(POOL_T) void k_pool_fork_plan(ForkArgs a) {
  __shared__ int waves[POOL_T / 64];
  int total = 0;
  for (int i0 = 0; i0 < a.n; i0 += POOL_T) {
    const int i = i0 + threadIdx.x;
    int id = -1;
    if (i < a.n) {
      const int32_t *row;
      const int n = child_len(a, i, row);
      if (n % a.page && n / a.page < a.out_width) id = row[n / a.page];
      if ((unsigned)id >= (unsigned)a.n_pages) id = -1;
    }
    int all;
    const int r = total + block_scan<POOL_T>(id >= 0 ? 1 : 0, waves, all);
    if (i < a.n) {
      a.src[i] = id;
      a.dst[i] = id >= 0 ? r : -1;
    }
    total += all;
  }
  if (total == 0) return;
  const int have = find_free(a.refs, a.n_pages, total, a.give);
  count_short(a.n_short, total, have);
  for (int i = threadIdx.x; i < a.n; i += POOL_T) {
    const int r = a.dst[i];
    if (r < 0) continue;
    const int id = r < have ? a.give[r] : -1;
    a.dst[i] = id;
    if (id >= 0) a.refs[id] = 1;
  }
}

// 4 KB of a page of one array, a wave.
__device__ __forceinline__ void copy_unit(const uint8_t *from, uint8_t *to, long long bytes, long long at) {
  const int lane = threadIdx.x & 63;
  uint4 v[COPY_UNIT / 1024];
#pragma unroll
  for (int u = 0; u < COPY_UNIT / 1024; ++u) {
    const long long o = at + 1024 * u + 16 * lane;
    if (o < bytes) v[u] = *(const uint4 *)(from + o);
  }
#pragma unroll
  for (int u = 0; u < COPY_UNIT / 1024; ++u) {
    const long long o = at + 1024 * u + 16 * lane;
    if (o < bytes) st_nt((uint4 *)(to + o), v[u]);
  }
}

// Workgroup `block` of a copying launch: every array has a.blocks of them,
// whose waves take 4 KB units of all moves in turn.
__device__ __forceinline__ void copy_pages(const CopyArgs &a, int block) {
  const int of = block / a.blocks;
  const bfp_page_array d = a.array[of];
  const long long per = (d.bytes + COPY_UNIT - 1) / COPY_UNIT;
  const int n = a.count ? *a.count : a.n;
  const long long waves = (long long)a.blocks * (COPY_T / 64);
  for (long long u = (block - of * a.blocks) * (COPY_T / 64) + (threadIdx.x >> 6); u < per * n; u += waves) {
    const long long k = u / per;
    const int src = a.src[k], dst = a.dst[k];
    if ((unsigned)src >= (unsigned)a.n_pages || (unsigned)dst >= (unsigned)a.n_pages || src == dst) continue;
    copy_unit(d.p + src * d.bytes, d.p + dst * d.bytes, d.bytes, (u - k * per) * COPY_UNIT);
  }
}

__global__ __launch_bounds__(COPY_T) void k_pool_copy(CopyArgs c) { copy_pages(c, blockIdx.x); }

// The children's tables, and the counts of what they share.
__device__ __forceinline__ void fork_tables(const ForkArgs &a, int blocks) {
  const long long all = (long long)a.n * a.out_width, step = (long long)blocks * COPY_T;
  for (long long e = (long long)blockIdx.x * COPY_T + threadIdx.x; e < all; e += step) {
    const int i = (int)(e / a.out_width), p = (int)(e - (long long)i * a.out_width);
    const int32_t *row;
    const int n = child_len(a, i, row), whole = n / a.page;
    int id = -1;
    if (p < whole) {
      id = row[p];
      id = (unsigned)id < (unsigned)a.n_pages ? id : -1;
      if (id >= 0) atomicAdd(a.refs + id, 1);
    } else if (p == whole) {
      id = a.dst[i];
    }
    a.out_pages[e] = id;
    // without the copy it wanted, a child ends at its whole pages: a page that
    // it is given later would hold another's tokens where its own are missing
    if (p == 0) a.out_len[i] = a.src[i] >= 0 && a.dst[i] < 0 ? whole * a.page : n;
  }
}

__global__ __launch_bounds__(COPY_T) void k_pool_fork(ForkArgs a, CopyArgs c, int tables) {
  if ((int)blockIdx.x < tables)
    fork_tables(a, tables);
  else
    copy_pages(c, blockIdx.x - tables);
}

// Entries that are given up.  A page's count never falls below 0.
__global__ __launch_bounds__(COPY_T) void k_pool_free(int32_t *refs, int n_pages, int32_t *pages, long long n) {
  for (long long e = (long long)blockIdx.x * COPY_T + threadIdx.x; e < n; e += (long long)gridDim.x * COPY_T) {
    const int id = pages[e];
    if (id == -1) continue;
    pages[e] = -1;
    if ((unsigned)id >= (unsigned)n_pages) continue;
    if (atomicSub(refs + id, 1) <= 0) atomicAdd(refs + id, 1);
  }
}

struct PoolTable {
  int32_t *p;
  long long n;
};
struct CompactArgs {
  // rank: of each page, -1 if it is free, and of those from L on which move is its; held: live pages of each chunk
  int32_t *refs, *live, *moves, *src, *dst, *rank, *held;
  int n_pages, chunks;
  PoolTable table[POOL_TABLES];
  int n_tables;
};

constexpr int CHUNK_T = 256, CHUNK_EACH = POOL_CHUNK / CHUNK_T / 4;   // words of four counts a thread looks at

// Which of a thread's counts are live, a bit each; its counts are neighbours,
// from base on.
__device__ __forceinline__ uint32_t chunk_live(const CompactArgs &a, int chunk, long long &base) {
  base = (long long)chunk * POOL_CHUNK + threadIdx.x * (4 * CHUNK_EACH);
  uint32_t m = 0;
#pragma unroll
  for (int k = 0; k < CHUNK_EACH; ++k) {
    if (base + 4 * k >= a.n_pages) break;
    const int4 c = counts4(a.refs, a.n_pages, base / 4 + k);
    m |= (uint32_t)((c.x > 0) | (c.y > 0) << 1 | (c.z > 0) << 2 | (c.w > 0) << 3) << (4 * k);
  }
  const long long left = a.n_pages - base;   // what lies behind the last page is neither
  return left <= 0 ? 0 : left < 16 ? m & ((1u << left) - 1) : m;
}

__global__ __launch_bounds__(CHUNK_T) void k_pool_held(CompactArgs a) {
  __shared__ int waves[CHUNK_T / 64];
  long long base;
  const int n = __popc(chunk_live(a, blockIdx.x, base));
  int all;
  block_scan<CHUNK_T>(n, waves, all);
  if (threadIdx.x == 0) a.held[blockIdx.x] = all;
}

// L pages are live.  The k-th live page from L on goes to the k-th free one
// below L: there are as many of the one as of the other.
__global__ __launch_bounds__(CHUNK_T) void k_pool_plan(CompactArgs a) {
  __shared__ int waves[CHUNK_T / 64];
  __shared__ int below;   // live pages below L
  int mine = 0, all, before = 0;   // live pages of all chunks, and of those before this one
  for (int c = threadIdx.x; c < a.chunks; c += CHUNK_T) {
    const int n = a.held[c];
    mine += n;
    before += c < (int)blockIdx.x ? n : 0;
  }
  block_scan<CHUNK_T>(mine, waves, all);
  const int L = all, edge = L / POOL_CHUNK;   // the chunk in which L lies (past the last: nothing is live from L on)
  block_scan<CHUNK_T>(before, waves, all);
  before = all;
  mine = 0;
  for (int c = threadIdx.x; c < a.chunks && c < edge; c += CHUNK_T) mine += a.held[c];
  long long base;
  if (edge < a.chunks) {
    const uint32_t m = chunk_live(a, edge, base);
    const long long n = L - base;
    mine += __popc(n <= 0 ? 0u : n < 16 ? m & ((1u << n) - 1) : m);
  }
  block_scan<CHUNK_T>(mine, waves, all);
  if (threadIdx.x == 0) below = all;
  __syncthreads();
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    *a.live = L;
    *a.moves = L - below;
  }
  const uint32_t m = chunk_live(a, blockIdx.x, base);
  int r = before + block_scan<CHUNK_T>((int)__popc(m), waves, all);   // live pages before this one
#pragma unroll 1
  for (int k = 0; k < 16; ++k) {
    const long long id = base + k;
    if (id >= a.n_pages) break;
    const bool is = (m >> k) & 1;
    if (id >= L) {
      if (is) a.src[r - below] = (int)id;
    } else if (!is) {
      a.dst[id - r] = (int)id;
    }
    a.rank[id] = !is ? -1 : id < L ? 0 : r - below;
    r += is;
  }
}

__device__ __forceinline__ void compact_tables(const CompactArgs &a, int blocks) {
  const long long step = (long long)blocks * CHUNK_T, first = (long long)blockIdx.x * CHUNK_T + threadIdx.x;
  const int n = *a.moves, L = *a.live;
  for (int t = 0; t < a.n_tables; ++t)
    for (long long e = first; e < a.table[t].n; e += step) {
      const int id = a.table[t].p[e];
      if ((unsigned)id >= (unsigned)a.n_pages) continue;
      const int k = a.rank[id];   // (the counts change in this launch)
      if (k < 0)
        a.table[t].p[e] = -1;   // free: another sequence's page lies there now, or none
      else if (id >= L)
        a.table[t].p[e] = a.dst[k];
    }
  for (long long k = first; k < n; k += step) {
    const int s = a.src[k];
    a.refs[a.dst[k]] = a.refs[s];
    a.refs[s] = 0;
  }
}

__global__ __launch_bounds__(COPY_T) void k_pool_compact(CompactArgs a, CopyArgs c, int tables) {
  if ((int)blockIdx.x < tables)
    compact_tables(a, tables);
  else
    copy_pages(c, blockIdx.x - tables);
}

// ---------------------------------------------------------------------- host
static int check_pool(const char *op, const bfp_pages *p) {
  if (!p || !p->refs) return set_err(BFP_EINVAL, "%s: no pool", op);
  if (p->n_pages < 1 || p->n_pages > POOL_MAX) return set_err(BFP_EINVAL, "%s: n_pages=%d", op, p->n_pages);
  if (p->page < 16 || p->page > 256 || (p->page & (p->page - 1)))
    return set_err(BFP_EINVAL, "%s: page=%d must be 16, 32, 64, 128 or 256", op, p->page);
  if ((uintptr_t)p->refs % 16 || (uintptr_t)p->n_short % 4)
    return set_err(BFP_EINVAL, "%s: refs must be 16-byte aligned, n_short 4", op);
  if (p->n_arrays < 0 || p->n_arrays > 65536 || (p->n_arrays && !p->arrays))
    return set_err(BFP_EINVAL, "%s: n_arrays=%d", op, p->n_arrays);
  for (int i = 0; i < p->n_arrays; ++i) {
    const bfp_page_array &a = p->arrays[i];
    if (!a.p || (uintptr_t)a.p % 16 || a.bytes < 16 || a.bytes % 16 || a.bytes > (1LL << 32))
      return set_err(BFP_EINVAL, "%s: array %d (%p, %lld bytes a page) must be 16-byte aligned, in multiples of 16 bytes", op, i,
                     (void *)a.p, a.bytes);
  }
  return BFP_OK;
}

// Memory of the calls' ints: no two of them may share any.
struct Ints {
  const char *what;
  const void *p;
  long long n;
};
static int check_ints(const char *op, const Ints *x, int n) {
  for (int i = 0; i < n; ++i) {
    if (!x[i].n) continue;
    if (!x[i].p || (uintptr_t)x[i].p % 4) return set_err(BFP_EINVAL, "%s: %s is null or not aligned", op, x[i].what);
    for (int j = 0; j < i; ++j) {
      if (!x[j].n || !x[j].p) continue;
      const uintptr_t a = (uintptr_t)x[i].p, b = (uintptr_t)x[j].p;
      if (a < b + 4 * (uintptr_t)x[j].n && b < a + 4 * (uintptr_t)x[i].n)
        return set_err(BFP_EINVAL, "%s: %s lies on %s", op, x[i].what, x[j].what);
    }
  }
  return BFP_OK;
}

// The scratch's pieces, in ints: `a` for whoever asks for pages, then lists of
// n moves.
static size_t pool_ints(const bfp_pages &p, long long n) {
  const size_t chunks = (p.n_pages + POOL_CHUNK - 1) / POOL_CHUNK;
  return 2 * (size_t)p.n_pages + chunks + 16 + 2 * (size_t)n;
}

// The copying launch for arrays from `first` on.  Each has as many workgroups
// as take a unit a wave of the largest array, up to what fills the card.
static CopyArgs copy_args(const bfp_pages &p, int first, const int32_t *src, const int32_t *dst, const int32_t *count, int n) {
  CopyArgs c;
  c.n_arrays = p.n_arrays - first < COPY_ARRAYS ? p.n_arrays - first : COPY_ARRAYS;
  if (c.n_arrays < 0) c.n_arrays = 0;
  if (c.n_arrays > 0) memcpy(c.array, p.arrays + first, c.n_arrays * sizeof(bfp_page_array));
  c.n_pages = p.n_pages;
  c.src = src;
  c.dst = dst;
  c.count = count;
  c.n = n;
  long long most = 0;
  for (int i = 0; i < c.n_arrays; ++i) most = c.array[i].bytes > most ? c.array[i].bytes : most;
  const double units = (double)n * ((most + COPY_UNIT - 1) / COPY_UNIT);
  const int fill = 8192 / (c.n_arrays > 0 ? c.n_arrays : 1) + 1;
  c.blocks = units / 4 < fill ? (int)(units / 4) + 1 : fill;
  return c;
}

// The arrays that the first launch had no room for.
static int copy_rest(const char *op, const bfp_pages &p, const int32_t *src, const int32_t *dst, const int32_t *count, int n,
                     int first, hipStream_t s) {
  for (; first < p.n_arrays; first += COPY_ARRAYS) {
    const CopyArgs c = copy_args(p, first, src, dst, count, n);
    hipLaunchKernelGGL(k_pool_copy, dim3(c.blocks * c.n_arrays), dim3(COPY_T), 0, s, c);
    BFP_TRY(launch_status(op));
  }
  return BFP_OK;
}

static int check_work(const char *op, const bfp_pages *p, long long n, const void *work, size_t bytes) {
  const size_t need = pool_ints(*p, n) * 4;
  if (!work || (uintptr_t)work % 16 || bytes < need)
    return set_err(BFP_EINVAL, "%s: needs %zu bytes of 16-byte-aligned scratch, got %zu", op, need, work ? bytes : (size_t)0);
  return BFP_OK;
}

}  // namespace bfp

using namespace bfp;

extern "C" {

size_t bfp_pages_work(const bfp_pages *pool, int n) {
  if (check_pool("pages_work", pool) || n < 0) return 0;
  return pool_ints(*pool, n) * 4;
}

int bfp_pages_copy_d(const bfp_pages *pool, const int32_t *src, const int32_t *dst, int n, void *stream) {
  const char *op = "pages_copy";
  BFP_TRY(check_pool(op, pool));
  if (n < 0) return set_err(BFP_EINVAL, "%s: n=%d", op, n);
  if (n == 0) return BFP_OK;
  if (!src || !dst || ((uintptr_t)src | (uintptr_t)dst) % 4) return set_err(BFP_EINVAL, "%s: src or dst is null or not aligned", op);
  return copy_rest(op, *pool, src, dst, nullptr, n, 0, (hipStream_t)stream);
}

int bfp_pages_reserve_d(const bfp_pages *pool, const bfp_kv4_batch *batch, void *work, size_t work_bytes, void *stream) {
  const char *op = "pages_reserve";
  BFP_TRY(check_pool(op, pool));
  BFP_TRY(check_batch(op, batch, pool->page));
  const Ints x[] = {{"refs", pool->refs, pool->n_pages}, {"n_short", pool->n_short, pool->n_short ? 1 : 0},
                    {"pages", batch->pages, (long long)batch->n_seq * batch->width},
                    {"start", batch->start, batch->n_seq ? batch->n_seq + 1 : 0}, {"len", batch->len, batch->n_seq}};
  BFP_TRY(check_ints(op, x, 5));
  if (batch->n_seq == 0 || batch->max_q == 0 || batch->n_rows == 0) return BFP_OK;
  BFP_TRY(check_work(op, pool, 0, work, work_bytes));
  ReserveArgs a{};
  a.refs = pool->refs;
  a.n_short = pool->n_short;
  a.pages = (int32_t *)batch->pages;   // the one call that writes a batch's table
  a.give = (int32_t *)work;
  a.b = *batch;
  a.n_pages = pool->n_pages;
  a.page = pool->page;
  const int rows = batch->max_q < batch->n_rows ? batch->max_q : batch->n_rows;
  a.touched = (int)(((long long)rows + pool->page - 2) / pool->page + 1);
  a.touched = a.touched < batch->width ? a.touched : batch->width;
  hipLaunchKernelGGL(k_pool_reserve, dim3(1), dim3(POOL_T), 0, (hipStream_t)stream, a);
  return launch_status(op);
}

int bfp_pages_fork_d(const bfp_pages *pool, const int32_t *pages, const int32_t *len, int n_seq, int width,
                     const int32_t *parents, int n, int32_t *out_pages, int32_t *out_len, int out_width, void *work,
                     size_t work_bytes, void *stream) {
  const char *op = "pages_fork";
  BFP_TRY(check_pool(op, pool));
  if (n_seq < 0 || n < 0 || width < 1 || out_width < 1 || (long long)width * pool->page > KV4_MAX_POS)
    return set_err(BFP_EINVAL, "%s: n_seq=%d, width=%d, n=%d, out_width=%d", op, n_seq, width, n, out_width);
  const Ints x[] = {{"refs", pool->refs, pool->n_pages}, {"n_short", pool->n_short, pool->n_short ? 1 : 0},
                    {"out_pages", out_pages, (long long)n * out_width}, {"out_len", out_len, n},
                    {"pages", pages, (long long)n_seq * width}, {"len", len, n_seq}, {"parents", parents, n}};
  BFP_TRY(check_ints(op, x, 7));
  if (n == 0) return BFP_OK;
  BFP_TRY(check_work(op, pool, n, work, work_bytes));
  ForkArgs a{};
  a.refs = pool->refs;
  a.n_short = pool->n_short;
  a.pages = pages, a.len = len, a.parents = parents;
  a.out_pages = out_pages, a.out_len = out_len;
  a.give = (int32_t *)work;
  a.src = a.give + pool->n_pages;
  a.dst = a.src + n;
  a.n_pages = pool->n_pages, a.page = pool->page;
  a.n_seq = n_seq, a.width = width, a.out_width = out_width, a.n = n;
  hipStream_t s = (hipStream_t)stream;
  hipLaunchKernelGGL(k_pool_fork_plan, dim3(1), dim3(POOL_T), 0, s, a);
  BFP_TRY(launch_status(op));
  const CopyArgs c = copy_args(*pool, 0, a.src, a.dst, nullptr, n);
  const long long rows = ((long long)n * out_width + COPY_T - 1) / COPY_T;
  const int tables = rows < 512 ? (int)rows : 512;
  hipLaunchKernelGGL(k_pool_fork, dim3(tables + c.blocks * c.n_arrays), dim3(COPY_T), 0, s, a, c, tables);
  BFP_TRY(launch_status(op));
  return copy_rest(op, *pool, a.src, a.dst, nullptr, n, COPY_ARRAYS, s);
}

int bfp_pages_free_d(const bfp_pages *pool, int32_t *pages, long long n, void *stream) {
  const char *op = "pages_free";
  BFP_TRY(check_pool(op, pool));
  if (n < 0 || n > (1LL << 40)) return set_err(BFP_EINVAL, "%s: n=%lld", op, n);
  const Ints x[] = {{"refs", pool->refs, pool->n_pages}, {"pages", pages, n}};
  BFP_TRY(check_ints(op, x, 2));
  if (n == 0) return BFP_OK;
  const long long blocks = (n + COPY_T - 1) / COPY_T;
  hipLaunchKernelGGL(k_pool_free, dim3((unsigned)(blocks < 2048 ? blocks : 2048)), dim3(COPY_T), 0, (hipStream_t)stream, pool->refs,
                     pool->n_pages, pages, n);
  return launch_status(op);
}

int bfp_pages_compact_d(const bfp_pages *pool, const bfp_page_table *tables, int n_tables, int32_t *live, void *work,
                        size_t work_bytes, void *stream) {
  const char *op = "pages_compact";
  BFP_TRY(check_pool(op, pool));
  if (n_tables < 0 || n_tables > POOL_TABLES || (n_tables && !tables))
    return set_err(BFP_EINVAL, "%s: n_tables=%d (at most %d)", op, n_tables, POOL_TABLES);
  Ints x[POOL_TABLES + 2] = {{"refs", pool->refs, pool->n_pages}, {"live", live, 1}};
  for (int t = 0; t < n_tables; ++t) {
    if (tables[t].n < 0 || tables[t].n > (1LL << 40)) return set_err(BFP_EINVAL, "%s: table %d has %lld entries", op, t, tables[t].n);
    x[2 + t] = {"a table", tables[t].pages, tables[t].n};
  }
  BFP_TRY(check_ints(op, x, 2 + n_tables));
  BFP_TRY(check_work(op, pool, 0, work, work_bytes));
  const int half = pool->n_pages / 2;   // no more than half of the pages can move
  CompactArgs a{};
  a.refs = pool->refs;
  a.live = live;
  a.moves = (int32_t *)work;
  a.src = a.moves + 16;
  a.dst = a.src + half;
  a.rank = a.dst + half;
  a.held = a.rank + pool->n_pages;
  a.n_pages = pool->n_pages;
  a.chunks = (pool->n_pages + POOL_CHUNK - 1) / POOL_CHUNK;
  a.n_tables = n_tables;
  for (int t = 0; t < n_tables; ++t) a.table[t] = {tables[t].pages, tables[t].n};
  hipStream_t s = (hipStream_t)stream;
  hipLaunchKernelGGL(k_pool_held, dim3(a.chunks), dim3(CHUNK_T), 0, s, a);
  BFP_TRY(launch_status(op));
  hipLaunchKernelGGL(k_pool_plan, dim3(a.chunks), dim3(CHUNK_T), 0, s, a);
  BFP_TRY(launch_status(op));
  const CopyArgs c = copy_args(*pool, 0, a.src, a.dst, a.moves, half);
  long long entries = half;
  for (int t = 0; t < n_tables; ++t) entries = tables[t].n > entries ? tables[t].n : entries;
  const int blocks = entries < 256 * CHUNK_T ? (int)(entries / CHUNK_T) + 1 : 256;
  hipLaunchKernelGGL(k_pool_compact, dim3(blocks + c.blocks * c.n_arrays), dim3(COPY_T), 0, s, a, c, blocks);
  BFP_TRY(launch_status(op));
  return copy_rest(op, *pool, a.src, a.dst, a.moves, half, COPY_ARRAYS, s);
}

}  // extern "C"
