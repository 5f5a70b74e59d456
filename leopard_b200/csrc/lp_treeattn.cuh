// leopard_b200 — attention of a tree of drafted tokens over a cache: what the kernels of lp_treeattn.cu and lp_treeattn_tc.cu share.
//
// The keys of an item (sequence, key head, block of rows) are cut into tiles; the tiles of all items stand in one line, of which every CTA takes an equal range: sequences
// of any lengths load all SMs alike.  Few items are dealt out whole: each has CTAs of its own, as many as its tiles are a share of all, since a range that goes on in another
// item costs the ends of two pieces (6 us; 26 nodes after 4,796 rows, 8 items on 148 CTAs, 19.7 and TREEALIGNED).  Where a CTA's range ends inside an item its rows' running
// maximum, sum and weighted values go to the workspace, to be joined.  Which CTAs an item has follows from the lengths alone, in every kernel.
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
  int len, n, tiles, blocks;              // cached rows; nodes; tiles of an item; blocks of rows
  int keys;                               // rows that are there: cached and nodes', as far as the page table reaches (fewer than 2^31)
};
// what the line knows of a sequence: the tiles before it, its length and nodes, and its first CTA where items have CTAs of their own.
// line[B]: all tiles; whether items have.
struct TreeLine {
  long long first;
  int len, n, cta;
};
__device__ __forceinline__ TreeSeq tree_seq(const TreeArgs& a, int len, int n) {
  TreeSeq s;
  s.n = n;
  s.len = len;
  s.keys = (int)min((long long)len + n, (long long)a.d.max_pages * a.d.page_size);
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
// CTAs of an item of `tiles` tiles, where there are `items` of them: one, and of the others as many as its share
__device__ __forceinline__ int tree_own(int tiles, long long total, int items, int ctas) {
  return (int)min((long long)tiles, 1 + tree_div((long long)tiles * (ctas - items), total));
}
constexpr int TREE_OWN = 8;               // CTAs an item from which on each has its own
// by one warp, in shared memory.  Ends in the block's barrier.
__device__ __forceinline__ void tree_line(const TreeArgs& a, TreeLine* line) {
  if (a.d.B == 1) {                       // one sequence: nothing to add up
    if (threadIdx.x == 0) {
      const int len = max(a.d.lengths[0], 0), n = a.d.nodes ? min(max(a.d.nodes[0], 0), a.d.T) : a.d.T;
      const TreeSeq s = tree_seq(a, len, n);
      const int items = s.tiles ? a.d.KVH * s.blocks : 0;
      const long long all = (long long)items * s.tiles;
      const bool owned = items * TREE_OWN <= a.ctas;
      line[0] = {0, len, n, 0};
      line[1] = {all, items, owned, owned && items ? items * tree_own(s.tiles, all, items, a.ctas) : 0};
    }
  } else if (threadIdx.x < 32) {
    long long run = 0, items = 0;
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
    const bool owned = items * TREE_OWN <= a.ctas;
    if (owned) {                          // (then there are at most ctas / TREE_OWN sequences of any tiles)
      int at = 0;
      for (int b0 = 0; b0 < a.d.B; b0 += 32) {
        const int b = b0 + threadIdx.x;
        int mine = 0;
        if (b < a.d.B) {
          const TreeSeq s = tree_seq(a, line[b].len, line[b].n);
          if (s.tiles) mine = a.d.KVH * s.blocks * tree_own(s.tiles, run, (int)items, a.ctas);
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
      line[a.d.B].len = (int)min(items, (long long)a.ctas);
      line[a.d.B].n = owned;
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
  const int own = tree_own(s.tiles, total, line[a.d.B].len, a.ctas), item = tree_div32(cta - line[b].cta, own), k = cta - line[b].cta - item * own;
  const long long first = line[b].first + (long long)item * s.tiles;
  from = first + tree_cut(s.tiles, k, own);
  to = first + tree_cut(s.tiles, k + 1, own);
}
// the CTAs that an item of sequence b (its item-th) lies in
__device__ __forceinline__ void tree_ctas_of(const TreeArgs& a, const TreeLine* line, int b, const TreeSeq& s, int item, int& c0, int& c1) {
  const long long total = line[a.d.B].first;
  if (!line[a.d.B].n) {
    const long long at = line[b].first + (long long)item * s.tiles;
    c0 = tree_cta_of(total, at, a.ctas);
    c1 = tree_cta_of(total, at + s.tiles - 1, a.ctas);
    return;
  }
  const int own = tree_own(s.tiles, total, line[a.d.B].len, a.ctas);
  c0 = line[b].cta + item * own;
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
