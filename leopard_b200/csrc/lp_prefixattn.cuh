// leopard_b200 — attention of a batch over a prefix that it shares and over each request's own rows: what lp_prefixattn.cu and lp_prefixattn_tc.cu share.
//
// The tokens that the requests bring stand in one list (request after request); for a key head, row r = token * G + g of that list are the rows of one product with the prefix's keys, which are
// read once for all of them.  A request's own keys are read for its rows alone.  Keys are cut into pieces; each leaves its rows' maximum, sum and weighted values in the workspace, and a last
// kernel joins them.
#pragma once
#include "lp_common.cuh"
#include "lp_host.h"
#include "../../include/leopard_b200.h"

namespace lp {

constexpr int PA_MAX_BATCH = 2048;
constexpr int PA_KEYS = 64;               // keys of a tile of the requests' own rows (and of the prefix, where few rows look at it)

struct PrefixArgs {
  lp_prefix_attn_desc d;
  int group;
  float scale_log2;
  int own_block, own_blocks, own_splits, own_rows;      // rows of a block (8, 16), blocks of a request's rows, pieces of its keys (at most); keys that there may be
  int pre_rows, pre_tiles, pre_ctas;      // the prefix: rows of a block (8, 16; 128, 256: the tcgen05 kernel), tiles of its keys (of PA_KEYS, or 128), CTAs (0: there is none)
  long long pre_slots, own_slots;         // partial results' places
  // partial results of the prefix's pieces [item + CTA] and of the own rows' [request][key head][block][piece]: values [D / 4][rows of a block][4], maximum (log2 units) and sum [rows]
  float *pre_o, *own_o;
  float2 *pre_ml, *own_ml;
};
// the tcgen05 kernel for many rows: whether it takes this call, its blocks' rows, its pieces; its launch
bool prefix_tc_takes(const lp_prefix_attn_desc* d);
int launch_prefix_tc(const PrefixArgs& a, cudaStream_t stream);

#ifdef __CUDACC__
__device__ __forceinline__ float pa_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ int pa_new(const PrefixArgs& a, int b) { return a.d.fresh ? min(max(a.d.fresh[b], 0), a.d.T) : a.d.T; }
// first[b]: tokens of the requests before b; first[B]: of all.  By the whole block (a thread some neighbours), for every CTA of the join waits for it (1,000
// requests: 171 us a call by one warp, 116 so); ends in its barrier.
__device__ __forceinline__ void pa_tokens(const PrefixArgs& a, int* first) {
  __shared__ int warps[32];
  const int threads = blockDim.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (!a.d.fresh) {
    for (int b = threadIdx.x; b <= a.d.B; b += threads) first[b] = b * a.d.T;
    __syncthreads();
    return;
  }
  const int each = (a.d.B + threads - 1) / threads, b0 = min((int)threadIdx.x * each, a.d.B), b1 = min(b0 + each, a.d.B);
  int mine = 0;
#pragma unroll 4
  for (int b = b0; b < b1; ++b) mine += pa_new(a, b);
  int sum = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += up;
  }
  if (lane == 31) warps[warp] = sum;
  __syncthreads();
  const int n = (threads + 31) >> 5;
  int before = lane < n ? warps[lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += up;
  }
  const int all = __shfl_sync(0xffffffffu, before, 31);
  before = __shfl_sync(0xffffffffu, before, max(warp - 1, 0));
  int run = (warp ? before : 0) + sum - mine;
#pragma unroll 4
  for (int b = b0; b < b1; ++b) {
    first[b] = run;
    run += pa_new(a, b);
  }
  if (threadIdx.x == 0) first[a.d.B] = all;
  __syncthreads();
}
// the request that brings token i of the list
__device__ __forceinline__ int pa_find(const int* first, int B, int i) {
  int lo = 0, hi = B - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first[mid] <= i) lo = mid; else hi = mid - 1;
  }
  return lo;
}
// own rows of a request before its new tokens, and with them (as far as there is room for rows)
__device__ __forceinline__ void pa_own(const PrefixArgs& a, int length, int fresh, int& past, int& keys) {
  const int own = max(max(length, 0) - a.d.prefix, 0);
  past = min(own, a.own_rows);
  keys = (int)min((long long)own + fresh, (long long)a.own_rows);
}
// The prefix's tiles of all items (block of rows, key head) stand in one line, of which every CTA takes a range of equal cost; or each item has `own` CTAs, where the longest range is then little above an equal
// share: a range that goes on in another item costs another piece's start and end.  The last block of each key head comes last in the line; with 128 rows at most (one of the tcgen05 kernel's two
// streams) its tiles cost PA_HALF of PA_FULL (1.7 and 2.5 us).  How many rows there are, and so how many items, only the GPU knows.
constexpr int PA_SLACK = 4, PA_FULL = 10, PA_HALF = 7;
struct PrefixLine {
  int blocks, items, own, last_cost;      // last_cost: of a tile of the last blocks
  long long full, cost;                   // tiles of the other blocks; cost of the line
};
template <typename T>
__device__ __forceinline__ T pa_cut(T total, int k, int n) {      // the k-th of n equal ranges begins here
  const T each = total / n, more = total - each * n;
  return each * k + min((T)k, more);
}
__device__ __forceinline__ PrefixLine pa_line(const PrefixArgs& a, int rows) {
  PrefixLine l;
  l.blocks = (rows + a.pre_rows - 1) / a.pre_rows;
  l.items = a.d.KVH * l.blocks;
  l.own = 0;
  if (a.pre_rows <= 16) {                 // few rows: CTAs of their own
    if (l.items > 0) l.own = min(a.pre_ctas / l.items, a.pre_tiles);
    return l;
  }
  l.last_cost = a.pre_rows == 256 && rows - (l.blocks - 1) * 256 <= 128 ? PA_HALF : PA_FULL;
  l.full = (long long)(l.items - a.d.KVH) * a.pre_tiles;
  l.cost = l.full * PA_FULL + (long long)a.d.KVH * a.pre_tiles * l.last_cost;
  if (l.items > 0 && l.items <= a.pre_ctas) {
    l.own = min(a.pre_ctas / l.items, a.pre_tiles);
    if ((a.pre_tiles + l.own - 1) / l.own * (long long)(l.blocks > 1 ? PA_FULL : l.last_cost) > l.cost / a.pre_ctas + PA_SLACK * PA_FULL) l.own = 0;
  }
  return l;
}
__device__ __forceinline__ long long pa_begin(const PrefixArgs& a, const PrefixLine& l, int cta) {      // the first tile of a CTA's range of the line
  const long long c = pa_cut(l.cost, cta, a.pre_ctas), over = c - l.full * PA_FULL;
  return over <= 0 ? (c + PA_FULL - 1) / PA_FULL : l.full + (over + l.last_cost - 1) / l.last_cost;
}
__device__ __forceinline__ int pa_cta_of(const PrefixArgs& a, const PrefixLine& l, long long tile) {      // the CTA in whose range a tile is
  const long long c = tile <= l.full ? tile * PA_FULL : l.full * PA_FULL + (tile - l.full) * l.last_cost;
  int cta = (int)min((long long)a.pre_ctas - 1, c * a.pre_ctas / l.cost);
  while (pa_begin(a, l, cta) > tile) --cta;
  while (cta + 1 < a.pre_ctas && pa_begin(a, l, cta + 1) <= tile) ++cta;
  return cta;
}
__device__ __forceinline__ void pa_range(const PrefixArgs& a, const PrefixLine& l, int cta, long long& from, long long& to) {
  from = to = 0;
  if (!l.own) {
    if (l.items) from = pa_begin(a, l, cta), to = pa_begin(a, l, cta + 1);
  } else if (cta < l.items * l.own) {
    const int item = cta / l.own, k = cta - item * l.own;
    from = (long long)item * a.pre_tiles + pa_cut(a.pre_tiles, k, l.own);
    to = (long long)item * a.pre_tiles + pa_cut(a.pre_tiles, k + 1, l.own);
  }
}
// the CTAs that an item's pieces are in
__device__ __forceinline__ void pa_ctas_of(const PrefixArgs& a, const PrefixLine& l, int item, int& c0, int& c1) {
  if (l.own) {
    c0 = item * l.own;
    c1 = c0 + l.own - 1;
    return;
  }
  c0 = pa_cta_of(a, l, (long long)item * a.pre_tiles);
  c1 = pa_cta_of(a, l, (long long)(item + 1) * a.pre_tiles - 1);
}
__device__ __forceinline__ int pa_item(const PrefixArgs& a, int blk, int kvh) { return blk * a.d.KVH + kvh; }
// the prefix's pieces for row r of the list: how many, the first one's place, the row's in their block
__device__ __forceinline__ void pa_pieces_of(const PrefixArgs& a, int rows, int kvh, int r, int& n, long long& slot, int& in) {
  n = in = 0;
  slot = 0;
  if (!a.pre_ctas) return;
  const PrefixLine line = pa_line(a, rows);
  const int blk = r / a.pre_rows, item = pa_item(a, blk, kvh);
  int c0, c1;
  pa_ctas_of(a, line, item, c0, c1);
  in = r - blk * a.pre_rows;
  n = c1 - c0 + 1;
  slot = (long long)item + c0;
}
// a CTA's piece of an item
struct PrefixPiece { int item, kvh, r0, t0, n; };
__device__ __forceinline__ PrefixPiece pa_piece(const PrefixArgs& a, long long u, long long u_end) {
  PrefixPiece p;
  p.item = (int)(u / a.pre_tiles);
  p.t0 = (int)(u - (long long)p.item * a.pre_tiles);
  p.n = (int)min((long long)(a.pre_tiles - p.t0), u_end - u);
  const int blk = p.item / a.d.KVH;
  p.kvh = p.item - blk * a.d.KVH;
  p.r0 = blk * a.pre_rows;
  return p;
}
__device__ __forceinline__ int pa_own_pieces(const PrefixArgs& a, int keys) { return min(a.own_splits, (keys + PA_KEYS - 1) / PA_KEYS); }
#endif

}  // namespace lp
