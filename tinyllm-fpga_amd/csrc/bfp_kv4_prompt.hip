// Attention over the 4-bit cache for prompts, whole or in pieces
// (bfp_kv4_prompt.h), and the joining of its splits.
#include "bfp_kv4_prompt.h"

namespace bfp {

// Joins the splits: a wave takes one row and query head.
__global__ __launch_bounds__(256) void k_kv4_join_prompt(Kv4AttnArgs a) {
  const int seq = blockIdx.y;
  const Kv4Span sp = kv4_span(a.b.start[seq], a.b.start[seq + 1], a.b.len[seq], a.b.n_rows, a.b.max_q);
  const int u = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int i = u / a.q.heads, qh = u % a.q.heads;
  if (i >= sp.n) return;
  const long long tok = sp.row0 + i, at = (((long long)seq * a.b.max_q + i) * a.q.heads + qh) * a.splits;
  const int hd = 16 * a.tiles;
  // lane k holds split k's maximum and sum (at most 64 splits)
  const float2 ml = lane < a.splits ? a.part_ml[at + lane] : make_float2(-INFINITY, 0.0f);
  const float M = wave_max(ml.x);
  // a split that saw nothing (or NaN scores alone, whose sum is NaN): factor 0
  const float f = ml.x == -INFINITY ? 0.0f : exp2f(ml.x - M);
  const float L = wave_sum(f * ml.y);
  // four splits' loads under way together; past the last one: it again, with
  // the factor 0 (its NaN, if it has one, is the row's anyway)
  float acc[4] = {0, 0, 0, 0};
  for (int k0 = 0; k0 < a.splits; k0 += 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int k = k0 + e < a.splits ? k0 + e : a.splits - 1;
      const float fk = k0 + e < a.splits ? __shfl(f, k, 64) : 0.0f;
      const float *o = a.part_o + (at + k) * hd;
#pragma unroll
      for (int d = 0; d < 4; ++d)
        if (64 * d < hd) acc[d] += fk * o[64 * d + lane < hd ? 64 * d + lane : hd - 1];
    }
  }
#pragma unroll
  for (int d = 0; d < 4; ++d)
    if (64 * d + lane < hd)
      out_store(a.out, tok * a.out.row_stride + qh * a.out.head_stride + 64 * d + lane, L == 0.0f ? 0.0f : acc[d] / L);
}

// Joins the two parts of rows that share a prefix: the prefix's slots, which
// are not there outside every group, and those of the rest.  A wave takes one
// row and query head, 16 bytes a lane, so that several slots' values are
// loaded at once, and four such loads are under way.  Bound by the slots' bytes
// (64 rows of 32 heads of 128, 33 slots: 35 MB in 8.9 us).
__global__ __launch_bounds__(256) void k_kv4_join_shared(Kv4AttnArgs a) {
  __shared__ float rows[4][256];
  const int seq = blockIdx.y;
  const Kv4Span sp = kv4_span(a.b.start[seq], a.b.start[seq + 1], a.b.len[seq], a.b.n_rows, a.b.max_q);
  const int w = threadIdx.x >> 6, u = blockIdx.x * 4 + w, lane = threadIdx.x & 63;
  const int i = u / a.q.heads, qh = u % a.q.heads;
  if (i >= sp.n) return;   // (no barrier below)
  const long long tok = sp.row0 + i, rest = rest_place(a, seq, i, tok, qh, 0);
  const int hd = 16 * a.tiles;
  int g, before = 0;   // of its n parts the prefix's
  long long place = prefix_place(a, tok, qh, 0), step = 1;   // where the first lies, and how far apart they are
  if (kv4_shared_len(a, seq, g) > 0) {
    before = a.prefix_splits;
    if (a.pieces) {
      const int4 of = a.piece_of[g];
      uint32_t of_head;
      const int head = (int)a.by_group.div((uint32_t)qh, of_head), row = (int)(tok - of.w) * a.group + (int)of_head;
      const int rt = row >> a.piece_shift, tiles = of.z * a.c.heads, block = of.y + rt * a.c.heads + head;
      before = min(of.x, a.prefix_splits);
      place = ((long long)block << a.piece_shift) + (row & ((1 << a.piece_shift) - 1));
      step = (long long)tiles << a.piece_shift;
      // (rows past max_rows, groups that overlap: nobody took them)
      if (row < 0 || rt >= of.z || of.y < 0 || block < 0 || block + (before - 1LL) * tiles >= a.piece_blocks) before = 0;
    }
  }
  const int n = before + a.rest_splits;
  auto slot = [&](int k) { return k < before ? place + k * step : rest + k - before; };
  const float2 ml = lane < n ? a.part_ml[slot(lane)] : make_float2(-INFINITY, 0.0f);
  // lanes of a slot, slots at a time; this lane's
  const int lanes = hd / 4, each = 64 / lanes, mine = lane / lanes, d = 4 * (lane - mine * lanes);
  f32x4 acc = {0, 0, 0, 0}, x[4];
  float M, f, L;
  for (int k0 = 0; k0 < n; k0 += 4 * each) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {   // past the last slot: it again, with the factor 0 (its NaN, if it has one, is the row's anyway)
      const int k = k0 + e * each + mine;
      x[e] = *(const f32x4 *)(a.part_o + slot(k < n ? k : n - 1) * hd + d);
    }
    if (k0 == 0) {   // while the first ones are under way
      M = wave_max(ml.x);
      f = ml.x == -INFINITY ? 0.0f : exp2f(ml.x - M);
      L = wave_sum(f * ml.y);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int k = k0 + e * each + mine;
      const float fk = __shfl(f, k < n ? k : n - 1, 64);
      acc += (k < n && mine < each ? fk : 0.0f) * x[e];
    }
  }
  // the slots' sums, always in the same order
  float *row = rows[w];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float v = acc[e];
    for (int k = 1; k < each; ++k) v += __shfl(acc[e], (lane + k * lanes) & 63, 64);
    if (mine == 0) row[d + e] = v;
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
  for (int o = lane; o < hd; o += 64)   // whole groups of 16 lanes
    out_store(a.out, tok * a.out.row_stride + qh * a.out.head_stride + o, L == 0.0f ? 0.0f : row[o] / L);
}

AttnKernel prompt_kernel(int tiles, int terms) { return prompt_kernel_for<SEES_ALL>(tiles, terms); }

void launch_join_prompt(const Kv4AttnArgs &a, hipStream_t s) {
  const long long n = ((long long)a.b.max_q * a.q.heads + 3) / 4;
  hipLaunchKernelGGL(k_kv4_join_prompt, dim3((unsigned)n, a.b.n_seq), dim3(256), 0, s, a);
}

void launch_join_shared(const Kv4AttnArgs &a, hipStream_t s) {
  const long long n = ((long long)(a.b.max_q < a.b.n_rows ? a.b.max_q : a.b.n_rows) * a.q.heads + 3) / 4;
  hipLaunchKernelGGL(k_kv4_join_shared, dim3((unsigned)n, a.b.n_seq), dim3(256), 0, s, a);
}

}  // namespace bfp
