// leopard_b200 — attention of a tree of drafted tokens over a cache: what the kernels of lp_treeattn.cu and lp_treeattn_tc.cu share.
//
// The keys of an item (sequence, key head, block of rows) are cut into tiles; the tiles of all items stand in one line, of which every CTA takes an equal range: sequences
// of any lengths load all SMs alike.  Few items are dealt out whole, each with CTAs of its own, where the longest range is then little above an equal share: a range that goes on
// in another item costs the ends of two pieces, and a split item its join (26 nodes of 11 sequences of up to 5,000 rows 50.4 us and 60.3 without, 64 nodes of them 66 and 76; one
// node after 4,796 rows 16.2 and 22.3).  Where a CTA's range ends inside an item its rows' running maximum, sum and weighted values go to the workspace, to be joined.  Which CTAs
// an item has follows from the lengths alone, in every kernel.
#pragma once
#include "lp_common.cuh"
#include "lp_host.h"
#include "../../include/leopard_b200.h"

namespace lp {

struct TreeArgs {
  lp_tree_attn_desc d;
  int group, rows, row_bits, key_bits;    // query heads of a key head; rows of a block and their power of two; that of a tile's keys
  float scale_log2;
  float* part_o; float2* part_ml;         // [2 x CTAs][D / 4][rows][4] (a warp writes and reads 32 rows of 4 values side by side), [2 x CTAs][rows]: maximum (log2 units), sum
  int ctas;
};
// the tcgen05 kernel (lp_treeattn_tc.cu): whether it takes this cache, and its launch
bool tree_tc_takes(const lp_tree_attn_desc* d);
int launch_tree_tc(const TreeArgs& a, cudaStream_t stream);

#ifdef __CUDACC__
__device__ __forceinline__ float ta_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// a sequence's part of the line of tiles
struct TreeSeq {
  int len, n, tiles, blocks;              // cached rows that are there; nodes; tiles of an item; blocks of rows
  int keys;                               // rows that are there: cached and nodes', as far as the page table reaches (fewer than 2^31)
};
// what the line knows of a sequence: the tiles before it, its length and nodes, and its first CTA where items have CTAs of their own.
// line[B]: all tiles; how many an item's CTAs have at most (0: items have none of their own).
struct TreeLine {
  long long first;
  int len, n, cta;
};
__device__ __forceinline__ TreeSeq tree_seq(const TreeArgs& a, int len, int n) {
  TreeSeq s;
  const long long capacity = (long long)a.d.max_pages * a.d.page_size;
  s.n = n;
  s.len = (int)min((long long)len, capacity);      // (a sequence that says it is longer than its pages: no row behind them is a cached one)
  s.keys = (int)min((long long)len + n, capacity);
  s.tiles = n ? (int)(((unsigned)s.keys + (1u << a.key_bits) - 1) >> a.key_bits) : 0;
  s.blocks = (n * a.group + a.rows - 1) >> a.row_bits;
  return s;
}
// a / b of numbers that are seldom large: below 2^23 an approximate quotient is one off at most.  A kernel's first piece waits for about seven of these in a row, each
// of 0.1 us as a whole division and 0.3 in 64 bits.
__device__ __forceinline__ int tree_small(int a, int b) {
  int q = (int)__fdividef((float)a, (float)b);
  const int r = a - q * b;
  if (r < 0) --q;
  if (r >= b) ++q;
  return q;
}
__device__ __forceinline__ int tree_div32(int a, int b) { return ((a | b) >> 23) == 0 ? tree_small(a, b) : (int)((unsigned)a / (unsigned)b); }
__device__ __forceinline__ long long tree_div(long long a, long long b) {
  if (((a | b) >> 23) == 0) return tree_small((int)a, (int)b);
  return ((a | b) >> 32) == 0 ? (long long)((unsigned)a / (unsigned)b) : a / b;
}
__device__ __forceinline__ long long tree_cut(long long total, int cta, int ctas) {
  const long long each = tree_div(total, ctas);
  return each * cta + min((long long)cta, total - each * ctas);
}
__device__ __forceinline__ int tree_cta_of(long long total, long long unit, int ctas) {
  const long long each = tree_div(total, ctas), more = total - each * ctas;      // the first `more` CTAs have one tile more
  return unit < (each + 1) * more ? (int)tree_div(unit, each + 1) : (int)(more + tree_div(unit - (each + 1) * more, each));
}
// CTAs of an item of `tiles` tiles, where items have CTAs of their own: `most` tiles each
__device__ __forceinline__ int tree_own(int tiles, int most) { return tree_div32(tiles + most - 1, most); }
// For items to have CTAs of their own the longest range may have this many tiles above an equal share: of 64 and of 128 keys, the latter looked for in steps of two.  A tile is 1 to
// 2 us, the end of a piece and its join 6 to 12 (CTAs of their own, and as a line: 64 nodes of 14 sequences of 1,000 rows, 1.8 tiles above: 37.4 us and 56.1; of 12 of 3,000, 8.4 above: 75.4
// and 75.0; of 10 of 3,000, 11 above: 75.1 and 67.5).  The limits were found on such batches and are not the best for each: 26 nodes of 10 or 12 sequences of 3,000 rows stay a line, 53.1 and 56.6 us
// where own CTAs take 49.2 and 51.9; 8 nodes of 10 have their own, 43.7 where a line takes 43.0.
constexpr int TREE_SLACK = 3, TREE_SLACK_TC = 6;
__device__ __forceinline__ int tree_slack(const TreeArgs& a) { return a.key_bits == 7 ? TREE_SLACK_TC : TREE_SLACK; }
// by one warp, in shared memory.  Ends in the block's barrier.
__device__ __forceinline__ void tree_line(const TreeArgs& a, TreeLine* line) {
  if (a.d.B == 1) {                       // one sequence: nothing to add up
    if (threadIdx.x == 0) {
      const int len = max(a.d.lengths[0], 0), n = a.d.nodes ? min(max(a.d.nodes[0], 0), a.d.T) : a.d.T;
      const TreeSeq s = tree_seq(a, len, n);
      const int items = s.tiles ? a.d.KVH * s.blocks : 0;
      const long long all = (long long)items * s.tiles;
      int most = 0;
      // (of fewer tiles than CTAs each has its own in any case; of few of 128 keys the sums take longer than they give: 26 nodes after 4,796 rows 21.5 us and 22, after 20,000 34.4 and 27)
      if (items <= a.ctas && all > (a.key_bits == 7 ? 4LL : 1LL) * a.ctas) {
        most = tree_own(s.tiles, tree_div32(a.ctas, items));
        if (most > tree_div(all, a.ctas) + tree_slack(a)) most = 0;
      }
      line[0] = {0, len, n, 0};
      line[1] = {all, 0, most, most ? items * tree_own(s.tiles, most) : 0};
    }
  } else if (threadIdx.x < 32) {
    long long run = 0, items = 0;
    int my_items = 0, my_tiles = 0;       // of the first 32 sequences
    for (int b0 = 0; b0 < a.d.B; b0 += 32) {
      const int b = b0 + threadIdx.x;
      long long mine = 0, own = 0;
      if (b < a.d.B) {
        const int len = max(a.d.lengths[b], 0), n = a.d.nodes ? min(max(a.d.nodes[b], 0), a.d.T) : a.d.T;
        const TreeSeq s = tree_seq(a, len, n);
        line[b].len = len;
        line[b].n = n;
        own = s.tiles ? (long long)a.d.KVH * s.blocks : 0;
        mine = own * s.tiles;
        if (b0 == 0) my_items = (int)own, my_tiles = s.tiles;
      }
      long long sum = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, sum, o);
        if ((int)threadIdx.x >= o) sum += up;
      }
      if (b < a.d.B) line[b].first = run + sum - mine;
      run += __shfl_sync(0xffffffffu, sum, 31);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) own += __shfl_xor_sync(0xffffffffu, own, o);
      items += own;
    }
    int most = 0;
    if (items <= a.ctas && run > a.ctas && a.d.B <= 32) {        // (a lane a sequence) the least number of tiles for which the CTAs are enough
      const int share = (int)tree_div(run, a.ctas), step = a.key_bits == 7 ? 2 : 1;
#pragma unroll
      for (int k = 7; k >= 0; --k) {
        const int m = share + 1 + k * step;
        const int ctas = __reduce_add_sync(0xffffffffu, (unsigned)(my_items * tree_own(my_tiles, m)));
        if (ctas <= a.ctas && m <= share + tree_slack(a)) most = m;
      }
    }
    if (most) {
      int at = 0;
      for (int b0 = 0; b0 < a.d.B; b0 += 32) {
        const int b = b0 + threadIdx.x;
        int mine = 0;
        if (b < a.d.B) {
          const TreeSeq s = tree_seq(a, line[b].len, line[b].n);
          if (s.tiles) mine = a.d.KVH * s.blocks * tree_own(s.tiles, most);
        }
        int sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, sum, o);
          if ((int)threadIdx.x >= o) sum += up;
        }
        if (b < a.d.B) line[b].cta = at + sum - mine;
        at += __shfl_sync(0xffffffffu, sum, 31);
      }
      if (threadIdx.x == 0) line[a.d.B].cta = at;
    }
    if (threadIdx.x == 0) {
      line[a.d.B].first = run;
      line[a.d.B].n = most;
    }
  }
  __syncthreads();
}
// a CTA's range of the line
__device__ __forceinline__ void tree_range(const TreeArgs& a, const TreeLine* line, int cta, long long& from, long long& to) {
  const long long total = line[a.d.B].first;
  if (!line[a.d.B].n) {
    from = tree_cut(total, cta, a.ctas);
    to = tree_cut(total, cta + 1, a.ctas);
    return;
  }
  from = to = 0;
  if (cta >= line[a.d.B].cta) return;
  int b = a.d.B - 1;
  while (line[b].cta > cta) --b;          // (a sequence without tiles has no CTAs: its first one is the next sequence's)
  const TreeSeq s = tree_seq(a, line[b].len, line[b].n);
  const int own = tree_own(s.tiles, line[a.d.B].n), item = tree_div32(cta - line[b].cta, own), k = cta - line[b].cta - item * own;
  const long long first = line[b].first + (long long)item * s.tiles;
  from = first + tree_cut(s.tiles, k, own);
  to = first + tree_cut(s.tiles, k + 1, own);
}
// the CTAs that an item of sequence b (its item-th) lies in
__device__ __forceinline__ void tree_ctas_of(const TreeArgs& a, const TreeLine* line, int b, const TreeSeq& s, int item, int& c0, int& c1) {
  const TreeLine &its = line[b], &all = line[a.d.B];
  if (!all.n) {
    const long long at = its.first + (long long)item * s.tiles;
    c0 = tree_cta_of(all.first, at, a.ctas);
    c1 = tree_cta_of(all.first, at + s.tiles - 1, a.ctas);
    return;
  }
  const int own = tree_own(s.tiles, all.n);
  c0 = its.cta + item * own;
  c1 = c0 + own - 1;
}
__device__ __forceinline__ int tree_find(const TreeLine* line, int B, long long unit) {      // the sequence that `unit` belongs to
  int lo = 0, hi = B - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (line[mid].first <= unit) lo = mid; else hi = mid - 1;
  }
  return lo;
}

#endif

}  // namespace lp
