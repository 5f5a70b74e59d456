// leopard_b200 — what drafting needs beside the attention of a tree (lp_treeattn.cu): which nodes of a tree see which, verification of the drafts against
// the target's probabilities, and rows and pages of a cache moved in all layers at once.
#include "lp_host.h"
#include <stdlib.h>
#include <algorithm>
#include "../../include/leopard_b200.h"

namespace lp {

// ---- trees ---------------------------------------------------------------------------------------------------------
// A node's word mask holds itself and its ancestors; its depth is the number of its ancestors.  A thread walks one node up to its root: parents lie before
// their children (an entry that does not ends the walk), so a walk takes at most T steps.
__global__ void __launch_bounds__(128)
tree_mask_kernel(const int* __restrict__ parents, long long ldp, int T, int words, unsigned long long* __restrict__ mask, int* __restrict__ depth) {
  const int b = blockIdx.y, i = blockIdx.x * 128 + threadIdx.x;
  if (i >= T) return;
  const int* p = parents + b * ldp;
  unsigned long long* m = mask + ((long long)b * T + i) * words;
  for (int w = 0; w < words; ++w) {
    unsigned long long bits = 0;
    for (int at = i; at >= 0;) {
      if ((at >> 6) == w) bits |= 1ull << (at & 63);
      const int up = p[at];
      at = up < at ? up : -1;
    }
    m[w] = bits;
  }
  if (depth) {
    int n = 0;
    for (int at = i; at >= 0; ++n) {
      const int up = p[at];
      at = up < at ? up : -1;
    }
    depth[(long long)b * T + i] = n - 1;
  }
}

// ---- verification --------------------------------------------------------------------------------------------------
constexpr int VERIFY_MAX_NODES = 1024;

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct VerifyArgs {
  const float* target; long long target_batch, target_row;
  const float* draft; long long draft_batch, draft_row;
  const long long* tokens; const int* parents; const float* uniform; const int* nodes;
  int T, V;
  int* path; int* count; long long* next;
};

// A cluster of up to 8 CTAs takes a sequence, a CTA an equal part of the vocabulary.  The walk over the nodes in their order is the walk down the tree, since children come after
// their parents: node c is tried when its parent is where the walk stands, and accepted when u[c] q(x) < P(x), P the target's distribution there less what was
// refused before.  A refusal takes P = max(P - q, 0) / sum.  What the tests need of a node, p and q at its token, is fetched for all nodes at once; the vocabulary is passed over
// once a refusal and once for the next token, and the CTAs add up their sums in the order of their ranks.  All CTAs go the same way.  Everything is computed in 64
// bits, so that the choices are those of the definition.
// HELD: vocabularies of up to 8 x 16,384 words stay in registers, 32 values of P (but for a factor) and q a thread, from a node's first pass to its last; of longer ones a value of P is taken
// again from p, q and the sums of the refusals (held and not: 8 nodes of 16 sequences, 32,000 words 16.8 and 21.5 us, 128,256 words 32.6 and 142; 5 nodes of one, 6.0 and 5.6, 6.1
// and 16.2).
// Bound by latency, not by the rows that are read: barriers of the cluster and dependent loads.  A chain of 6 nodes over 32,003 words takes 9.4 us (0.04 for its bytes), trees of 32
// nodes of 8 sequences over 128,256 words 22 (1.3).
constexpr int VERIFY_THREADS = 512;
constexpr int VERIFY_PART = 4096;                       // of the vocabulary, a CTA at least
constexpr int VERIFY_HELD = 32;                         // values of a thread

__device__ __forceinline__ void cluster_barrier() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ double cluster_read_f64(const double* p, int rank) {      // the same place of another CTA's shared memory
  uint32_t at = (uint32_t)__cvta_generic_to_shared(p);
  double v;
  asm volatile("mapa.shared::cluster.u32 %0, %0, %1;" : "+r"(at) : "r"(rank));
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(at) : "memory");
  return v;
}

template <bool HELD>
__global__ void __launch_bounds__(VERIFY_THREADS, 1)
verify_kernel(const __grid_constant__ VerifyArgs a, int ctas) {
  constexpr int WARPS = VERIFY_THREADS / 32;
  __shared__ double red[WARPS], sums[2], joined[2];     // by warp; this CTA's, of the passes in turn; all CTAs' and those of lower rank
  __shared__ double rows[32][33];                       // the part of the vocabulary that the next token lies in
  extern __shared__ double inv[];                       // [T] 1 / sum of each refusal at the node where the walk stands
  float* px = reinterpret_cast<float*>(inv + a.T);      // [T] p and q of a node's token, after its parent
  float* qx = px + a.T;
  float* us = qx + a.T;
  int* up = reinterpret_cast<int*>(us + a.T);           // [T] parents; -1 where the walk never comes
  int* tok = up + a.T;                                  // [T] tokens (-1: none of the vocabulary)
  int* gone = tok + a.T;                                // [T] the tokens that were refused at this node
  const int b = blockIdx.x / ctas, rank = blockIdx.x % ctas, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n = min(a.nodes ? a.nodes[b] : a.T, a.T);
  int* path = a.path + (long long)b * a.T;
  if (n <= 0) {
    if (rank == 0) {
      for (int i = tid; i < a.T; i += VERIFY_THREADS) path[i] = -1;
      if (tid == 0) { a.count[b] = 0; a.next[b] = -1; }
    }
    return;
  }
  const float* target = a.target + b * a.target_batch;
  const float* draft = a.draft ? a.draft + b * a.draft_batch : nullptr;
  for (int c = tid; c < n; c += VERIFY_THREADS) {
    const int at = a.parents[(long long)b * a.T + c];
    const long long x = a.tokens[(long long)b * a.T + c];
    const bool in = x >= 0 && x < a.V, comes = c > 0 && at >= 0 && at < c;
    up[c] = comes ? at : -1;
    tok[c] = in ? (int)x : -1;
    us[c] = a.uniform[(long long)b * a.T + c];
    px[c] = comes && in ? target[at * a.target_row + x] : 0.f;
    qx[c] = comes && in && draft ? draft[at * a.draft_row + x] : 1.f;
  }
  __syncthreads();
  const int part = (a.V + ctas - 1) / ctas, v0 = min(a.V, rank * part), v1 = min(a.V, v0 + part);
  const int each = ((v1 - v0 + WARPS - 1) / WARPS + 31) & ~31, w0 = min(v1, v0 + warp * each), w1 = min(v1, w0 + each);      // a warp's part, whole 32s
  int cur = 0, refused = 0, count = 1, passes = 0;
  const float* p = target;
  const float* q = draft;
  auto take = [&](double x, double d, int v) {          // P(v) of p(v), q(v)
    x = x > 0.0 ? x : 0.0;
    for (int k = 0; k < refused; ++k) {
      x -= draft ? d : (v == gone[k] ? 1.0 : 0.0);
      x = x > 0.0 ? x * inv[k] : 0.0;
    }
    return x;
  };
  const bool draws = draft != nullptr;
  double xs[HELD ? VERIFY_HELD : 1], unit = 1.0;        // P of this thread's words w0 + lane + 32 i is xs[i] x unit
  float ds[HELD ? VERIFY_HELD : 1];                     // q
  bool have_p = false, have_q = false;
  constexpr int DEEP = 8;                               // loads under way, of long vocabularies
  // sum of P, or of max(P - q, 0) when a token x has just been refused; red[] holds the warps' shares, `before` what the lower ranks have
  auto mass = [&](bool refusal, int x, double* before) {
    double s = 0.0;
    if (HELD) {
      if (!have_p) {
#pragma unroll
        for (int i = 0; i < VERIFY_HELD; ++i) ds[i] = w0 + lane + 32 * i < w1 ? p[w0 + lane + 32 * i] : 0.f;
#pragma unroll
        for (int i = 0; i < VERIFY_HELD; ++i) xs[i] = ds[i] > 0.f ? (double)ds[i] : 0.0;
        have_p = true;
        unit = 1.0;
      }
      if (refusal && draws && !have_q) {
#pragma unroll
        for (int i = 0; i < VERIFY_HELD; ++i) ds[i] = w0 + lane + 32 * i < w1 ? q[w0 + lane + 32 * i] : 0.f;
        have_q = true;
      }
      if (refusal) {
#pragma unroll
        for (int i = 0; i < VERIFY_HELD; ++i) {
          const float d = draws ? ds[i] : w0 + lane + 32 * i == x ? 1.f : 0.f;
          const double y = xs[i] * unit - (double)d;
          xs[i] = y > 0.0 ? y : 0.0;
        }
      }
#pragma unroll
      for (int i = 0; i < VERIFY_HELD; ++i) s += xs[i];
    } else {
      const bool less = draws && refused > 0;
      for (int v = w0 + lane; v < w1; v += 32 * DEEP) {
        float f[DEEP], d[DEEP];
#pragma unroll
        for (int k = 0; k < DEEP; ++k) f[k] = v + 32 * k < w1 ? p[v + 32 * k] : 0.f;
#pragma unroll
        for (int k = 0; k < DEEP; ++k) d[k] = less && v + 32 * k < w1 ? q[v + 32 * k] : 0.f;
#pragma unroll
        for (int k = 0; k < DEEP; ++k) s += take((double)f[k], (double)d[k], v + 32 * k);
      }
    }
    s = warp_sum_f64(s);
    if (lane == 0) red[warp] = s;
    __syncthreads();
    double mine = 0.0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) mine += red[w];
    *before = 0.0;
    if (ctas == 1) return mine;
    double* slot = &sums[passes & 1];                   // two in turn: who writes the first again has passed the barrier after its last reading
    ++passes;
    if (tid == 0) *slot = mine;
    cluster_barrier();
    if (warp == 0) {
      const double other = lane < ctas ? cluster_read_f64(slot, lane) : 0.0;
      double run = 0.0, mark = 0.0;
      for (int r = 0; r < ctas; ++r) {
        if (r == rank) mark = run;
        run += __shfl_sync(0xffffffffu, other, r);
      }
      if (lane == 0) { joined[0] = run; joined[1] = mark; }
    }
    __syncthreads();
    *before = joined[1];
    return joined[0];
  };
  double before;
  if (rank == 0 && tid == 0) path[0] = 0;
  for (int c = 1; c < n; ++c) {
    if (up[c] != cur || tok[c] < 0) continue;           // a token of no vocabulary takes nothing away
    if ((double)us[c] * (double)qx[c] < take((double)px[c], (double)qx[c], tok[c])) {
      cur = c;
      refused = 0;
      have_p = have_q = false;
      p = target + c * a.target_row;
      if (draws) q = draft + c * a.draft_row;
      if (rank == 0 && tid == 0) path[count] = c;
      ++count;
      continue;
    }
    __syncthreads();                                    // all have made the test
    if (tid == 0) { gone[refused] = tok[c]; inv[refused] = 1.0; }
    __syncthreads();
    ++refused;
    const double s = mass(true, tok[c], &before);
    if (s > 0.0) {
      const double f = 1.0 / s;
      if (tid == 0) inv[refused - 1] = f;               // (mass ends behind a barrier after its last look at it)
      unit = f;
    } else {                                            // nothing would be left: P stays
      --refused;
      if (HELD) {                                       // (rare: taken again from what came before)
        for (int i = 0; i < VERIFY_HELD; ++i) {
          const int v = w0 + lane + 32 * i;
          const double y = v < w1 ? take((double)p[v], draws && refused ? (double)q[v] : 0.0, v) : 0.0;
#pragma unroll
          for (int k = 0; k < VERIFY_HELD; ++k)
            if (k == i) xs[k] = y;
        }
        unit = 1.0;
      }
    }
    __syncthreads();
  }
  // the next token: the first whose running sum is above u[0] of the whole.  Its CTA, its warp there, its place in the warp's part.
  const double total = mass(false, -1, &before), goal = (double)us[0] * total;
  if (rank == 0) {
    for (int i = count + tid; i < a.T; i += VERIFY_THREADS) path[i] = -1;
    if (tid == 0) {
      a.count[b] = count;
      if (!(total > goal)) a.next[b] = -1;
    }
  }
  double mine = 0.0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) mine += red[w];
  if (before + mine > goal && !(before > goal)) {
    int w_of = -1, w_any = -1;
    double run = before, at = before;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      if (red[w] > 0.0 && w_of < 0) { w_any = w; at = run; }
      if (run + red[w] > goal && w_of < 0) w_of = w;
      run += red[w];
    }
    if (w_of < 0) w_of = w_any;                         // the sums' last bits: then the last warp that has any
    if (warp == w_of) {
      auto pick = [&](double x, double base, double* start) {      // the lane where base + the running sum passes the goal, else the last that has any
        double s = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double y = __shfl_up_sync(0xffffffffu, s, o);
          if (lane >= o) s += y;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, x > 0.0 && base + s > goal), any = __ballot_sync(0xffffffffu, x > 0.0);
        const int l = hit ? __ffs(hit) - 1 : 31 - __clz(any);
        *start = base + __shfl_sync(0xffffffffu, s - x, l);
        return l;
      };
      int found = -1;
      double start = at;
      if (HELD) {                                       // the 32s of the warp's part, then the words of one
#pragma unroll
        for (int i = 0; i < VERIFY_HELD; ++i) rows[i][lane] = xs[i];
        __syncwarp();
        double x = 0.0;
        for (int k = 0; k < 32; ++k) x += rows[lane][k];
        const int i = pick(x, at, &start);
        double end;
        found = w0 + 32 * i + pick(rows[i][lane], start, &end);
      } else {
        for (int from = w0; from < w1; from += 32) {
          const int v = from + lane;
          const double y = v < w1 ? take((double)p[v], draws && refused ? (double)q[v] : 0.0, v) : 0.0;
          if (!__any_sync(0xffffffffu, y > 0.0)) continue;
          double s = y, end;
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
          found = from + pick(y, start, &end);
          if (start + s > goal) break;
          start += s;
        }
      }
      if (lane == 0) a.next[b] = found;
    }
  }
  if (ctas > 1) cluster_barrier();                      // no CTA ends while another reads its sum
}

// ---- rows of a cache -----------------------------------------------------------------------------------------------
// where the pools of a call start, by value
constexpr int POOLS_MAX = 256;
struct Pools {
  unsigned long long base[POOLS_MAX];
};

// Accepted row path[j] of a sequence moves to place j behind its cached rows.  A thread takes one piece of the row through all moves in their order, ROWS_DEEP loads
// ahead of the stores: path rises, so path[j] >= j and a store never hits a row that a later move still has to read.  Bound by the latency of a launch and three loads that need one
// another (count, path and page, row) up to some MB: 32 layers of one sequence 3.4 us, 16 sequences of 32 layers, 64 nodes each, 6.1 (3.3 at a copy's rate).
constexpr int ROWS_DEEP = 8;
template <typename U>
__global__ void __launch_bounds__(128)
cache_compact_kernel(const __grid_constant__ Pools pools, long long page_stride, long long row_stride, int units, int n_pages, int page_size,
                     const int* __restrict__ table, long long ld_table, int max_pages, const int* __restrict__ lengths,
                     const int* __restrict__ path, long long ld_path, const int* __restrict__ count, int T) {
  const int b = blockIdx.z;
  const int n = min(count[b], T), len = lengths[b];
  if (len < 0) return;
  char* base = reinterpret_cast<char*>(pools.base[blockIdx.y]);
  const int c = blockIdx.x * 128 + threadIdx.x;
  if (c >= units) return;
  const int* order = path + b * ld_path;
  auto place = [&](int i) -> char* {
    const long long row = (long long)len + i;
    const long long logical = row / page_size;
    if (i < 0 || logical >= max_pages) return nullptr;
    const int page = table ? table[b * ld_table + logical] : b;
    if (page < 0 || page >= n_pages) return nullptr;
    return base + page * page_stride + (row - logical * page_size) * row_stride + (long long)c * sizeof(U);
  };
  for (int j0 = 0; j0 < n; j0 += ROWS_DEEP) {
    U held[ROWS_DEEP];
    char* to[ROWS_DEEP];
#pragma unroll
    for (int k = 0; k < ROWS_DEEP; ++k) {
      to[k] = nullptr;
      const int j = j0 + k;
      if (j >= n) continue;
      const int i = order[j];
      if (i == j || i < 0) continue;
      const char* from = place(i);
      to[k] = place(j);
      if (from == nullptr) to[k] = nullptr;
      if (to[k]) held[k] = *reinterpret_cast<const U*>(from);
    }
#pragma unroll
    for (int k = 0; k < ROWS_DEEP; ++k)
      if (to[k]) *reinterpret_cast<U*>(to[k]) = held[k];
  }
}

// Pages src[i] -> dst[i] of every pool: a CTA copies up to PAGE_PIECES pieces of one page, a thread four at once.  Bound by HBM: 40 pages of 128 KB in 64 pools 103 us, 6.5 TB/s.
constexpr int PAGE_PIECES = 1024;
template <typename U>
__global__ void __launch_bounds__(256)
cache_pages_kernel(const __grid_constant__ Pools pools, long long page_stride, long long units, int n_pages, const int* __restrict__ src,
                   const int* __restrict__ dst) {
  const int s = src[blockIdx.z], d = dst[blockIdx.z];
  if (s < 0 || s >= n_pages || d < 0 || d >= n_pages || s == d) return;
  char* base = reinterpret_cast<char*>(pools.base[blockIdx.y]);
  const U* from = reinterpret_cast<const U*>(base + s * page_stride);
  U* to = reinterpret_cast<U*>(base + d * page_stride);
  const long long at = (long long)blockIdx.x * PAGE_PIECES + threadIdx.x;
  U held[PAGE_PIECES / 256];
#pragma unroll
  for (int k = 0; k < PAGE_PIECES / 256; ++k)
    if (at + k * 256 < units) held[k] = from[at + k * 256];
#pragma unroll
  for (int k = 0; k < PAGE_PIECES / 256; ++k)
    if (at + k * 256 < units) to[at + k * 256] = held[k];
}

// the widest piece that a list of addresses and sizes is a multiple of
static int piece_bytes(const void* const* pools, long long step, int n, long long a, long long b, long long c) {
  unsigned long long all = (unsigned long long)a | (unsigned long long)b | (unsigned long long)c | (unsigned long long)step;
  for (int i = 0; i < (step ? 1 : n); ++i) all |= reinterpret_cast<unsigned long long>(pools[i]);
  return all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : all % 2 == 0 ? 2 : 1;
}

// Pools are moved by CTAs of their own, in no order: none may share memory with another, nor places within one.  1: apart, 0: not, -1: no memory to find out.
// `dims`, within a pool (nested afterwards: ascending); `inner`: bytes side by side.
static bool pools_meet(long long diff, const Dim* dims, const __int128* extent, int level) {      // a place of one pool and one of another `diff` bytes on
  if (level < 0) return diff < extent[0] && -diff < extent[0];
  if (dims[level].size <= 1) return pools_meet(diff, dims, extent, level - 1);
  // of the multiples of this stride only the two next to diff come nearer than what lies within it
  long long k = diff / dims[level].stride;
  if (diff % dims[level].stride < 0) --k;
  for (int i = 0; i < 2; ++i, ++k)
    if (k < dims[level].size && -k < dims[level].size && pools_meet(diff - k * dims[level].stride, dims, extent, level - 1)) return true;
  return false;
}
static int pools_apart(const void* const* pools, long long step, int n_pools, Dim* dims, int n_dims, long long inner) {
  if (step) {
    Dim all[4];
    for (int i = 0; i < n_dims; ++i) all[i] = dims[i];
    all[n_dims] = {n_pools, step};
    return strides_nest(all, n_dims + 1, inner);
  }
  if (!strides_nest(dims, n_dims, inner)) return 0;
  if (n_pools == 1) return 1;
  __int128 extent[4] = {inner};           // of a place, and with each dimension
  for (int i = 0; i < n_dims; ++i) extent[i + 1] = extent[i] + (dims[i].size > 1 ? (__int128)dims[i].stride * (dims[i].size - 1) : 0);
  unsigned long long* at = static_cast<unsigned long long*>(malloc(sizeof(unsigned long long) * (size_t)n_pools));
  if (!at) return -1;
  for (int i = 0; i < n_pools; ++i) at[i] = reinterpret_cast<unsigned long long>(pools[i]);
  std::sort(at, at + n_pools);
  unsigned long long least = ~0ull;
  for (int i = 1; i < n_pools; ++i) least = std::min(least, at[i] - at[i - 1]);
  bool apart = (__int128)least >= extent[n_dims];      // one behind the other
  bool within = true;                                  // or all of them within one stride, of this dimension and those above, as layers side by side in a page are
  for (int i = n_dims - 1; i >= 0 && !apart && within; --i) {
    if (dims[i].size <= 1) continue;
    within = (__int128)(at[n_pools - 1] - at[0]) + extent[i] <= dims[i].stride;
    apart = within && (__int128)least >= extent[i];
  }
  if (!apart) {
    apart = true;
    for (int i = 0; i < n_pools && apart; ++i)
      for (int j = i + 1; j < n_pools && apart && (__int128)(at[j] - at[i]) < extent[n_dims]; ++j) apart = !pools_meet((long long)(at[j] - at[i]), dims, extent, n_dims - 1);
  }
  free(at);
  return apart;
}

}  // namespace lp

extern "C" int lp_tree_mask(const int* parents, long long ld, int B, int T, unsigned long long* mask, int* depth, void* stream_) {
  using namespace lp;
  LP_REQUIRE(parents && mask && B > 0 && B <= 65535 && T > 0 && T <= LP_TREE_MAX_NODES && ld >= T,
             "lp_tree_mask: bad arguments B=%d T=%d (at most %d nodes) ld=%lld", B, T, LP_TREE_MAX_NODES, ld);
  note_launch();
  tree_mask_kernel<<<dim3((T + 127) / 128, B), 128, 0, reinterpret_cast<cudaStream_t>(stream_)>>>(parents, ld, T, (T + 63) / 64, mask, depth);
  LP_CHECK_CUDA(cudaGetLastError());
  return 0;
}

extern "C" int lp_verify_draft(const float* target, long long target_batch, long long target_row, const float* draft, long long draft_batch,
                               long long draft_row, const long long* tokens, const int* parents, const float* uniform, const int* nodes, int B, int T,
                               int V, int* path, int* count, long long* next, void* stream_) {
  using namespace lp;
  LP_REQUIRE(target && tokens && parents && uniform && path && count && next, "lp_verify_draft: null argument");
  LP_REQUIRE(B > 0 && T > 0 && T <= VERIFY_MAX_NODES && V > 0, "lp_verify_draft: bad sizes B=%d T=%d (at most %d nodes) V=%d", B, T, VERIFY_MAX_NODES, V);
  VerifyArgs a = {target, target_batch, target_row, draft, draft_batch, draft_row, tokens, parents, uniform, nodes, T, V, path, count, next};
  const int parts = (V + VERIFY_PART - 1) / VERIFY_PART, ctas = parts < 8 ? parts : 8;
  LP_REQUIRE(B <= (1 << 27), "lp_verify_draft: %d sequences are too many", B);
  note_launch();
  LP_CHECK_CUDA(launch_ex(V <= ctas * VERIFY_THREADS * VERIFY_HELD ? verify_kernel<true> : verify_kernel<false>, dim3((unsigned)B * ctas), dim3(VERIFY_THREADS), (size_t)T * 32, reinterpret_cast<cudaStream_t>(stream_), ctas, false, a, ctas));
  return 0;
}

extern "C" int lp_cache_compact(const void* const* pools, long long pool_step, int n_pools, long long page_stride, long long row_stride, long long row_bytes, int n_pages,
                                int page_size, const int* table, long long ld_table, int max_pages, const int* lengths, const int* path,
                                long long ld_path, const int* count, int B, int T, void* stream_) {
  using namespace lp;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  LP_REQUIRE(pools && lengths && path && count && n_pools > 0 && B > 0 && B <= 65535 && T > 0, "lp_cache_compact: bad arguments n_pools=%d B=%d T=%d", n_pools, B, T);
  LP_REQUIRE(n_pages > 0 && page_size > 0 && row_bytes > 0 && row_stride >= row_bytes && ld_path >= T && max_pages > 0 && (table == nullptr || ld_table >= max_pages),
             "lp_cache_compact: bad layout n_pages=%d page_size=%d row %lld of %lld bytes, %d pages a sequence", n_pages, page_size, row_bytes, row_stride, max_pages);
  LP_REQUIRE(table != nullptr || (max_pages == 1 && B <= n_pages), "lp_cache_compact: %d sequences without a page table need a page each, there are %d", B, n_pages);
  const int u = piece_bytes(pools, pool_step, n_pools, page_stride, row_stride, row_bytes);
  const long long units = row_bytes / u;
  Dim within[2] = {{n_pages, page_stride}, {page_size, row_stride}};
  const int apart = pools_apart(pools, pool_step, n_pools, within, 2, row_bytes);
  LP_REQUIRE(apart == 1, apart == 0 ? "lp_cache_compact: pools, pages or rows share their memory" : "lp_cache_compact: out of host memory");
  LP_REQUIRE(units < (1 << 30), "lp_cache_compact: rows of %lld bytes are too wide", row_bytes);
  for (int at = 0; at < n_pools; at += POOLS_MAX) {
    const int m = n_pools - at < POOLS_MAX ? n_pools - at : POOLS_MAX;
    Pools list;
    for (int i = 0; i < m; ++i)
      list.base[i] = pool_step ? reinterpret_cast<unsigned long long>(pools[0]) + (unsigned long long)pool_step * (at + i) : reinterpret_cast<unsigned long long>(pools[at + i]);
    const dim3 grid((unsigned)((units + 127) / 128), m, B);
    note_launch();
#define LP_COMPACT(U) cache_compact_kernel<U><<<grid, 128, 0, stream>>>(list, page_stride, row_stride, (int)units, n_pages, page_size, table, ld_table, max_pages, lengths, path, ld_path, count, T)
    if (u == 16) LP_COMPACT(uint4);
    else if (u == 4) LP_COMPACT(unsigned);
    else if (u == 2) LP_COMPACT(unsigned short);
    else LP_COMPACT(unsigned char);
#undef LP_COMPACT
    LP_CHECK_CUDA(cudaGetLastError());
  }
  return 0;
}

extern "C" int lp_cache_copy_pages(const void* const* pools, long long pool_step, int n_pools, long long page_stride, long long page_bytes, int n_pages, const int* src,
                                   const int* dst, int n, void* stream_) {
  using namespace lp;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  LP_REQUIRE(pools && src && dst && n_pools > 0 && n_pages > 0 && n >= 0 && n <= 65535, "lp_cache_copy_pages: bad arguments n_pools=%d n_pages=%d n=%d", n_pools, n_pages, n);
  LP_REQUIRE(page_bytes > 0 && page_stride >= page_bytes, "lp_cache_copy_pages: pages of %lld bytes, %lld apart", page_bytes, page_stride);
  if (n == 0) return 0;
  Dim within[1] = {{n_pages, page_stride}};
  const int apart = pools_apart(pools, pool_step, n_pools, within, 1, page_bytes);
  LP_REQUIRE(apart == 1, apart == 0 ? "lp_cache_copy_pages: pools or pages share their memory" : "lp_cache_copy_pages: out of host memory");
  const int u = piece_bytes(pools, pool_step, n_pools, page_stride, page_bytes, 0);
  const long long units = page_bytes / u, ctas = (units + PAGE_PIECES - 1) / PAGE_PIECES;
  LP_REQUIRE(ctas < (1LL << 31), "lp_cache_copy_pages: pages of %lld bytes are too large", page_bytes);
  for (int at = 0; at < n_pools; at += POOLS_MAX) {
    const int m = n_pools - at < POOLS_MAX ? n_pools - at : POOLS_MAX;
    Pools list;
    for (int i = 0; i < m; ++i)
      list.base[i] = pool_step ? reinterpret_cast<unsigned long long>(pools[0]) + (unsigned long long)pool_step * (at + i) : reinterpret_cast<unsigned long long>(pools[at + i]);
    const dim3 grid((unsigned)ctas, m, n);
    note_launch();
#define LP_PAGES(U) cache_pages_kernel<U><<<grid, 256, 0, stream>>>(list, page_stride, units, n_pages, src, dst)
    if (u == 16) LP_PAGES(uint4);
    else if (u == 4) LP_PAGES(unsigned);
    else if (u == 2) LP_PAGES(unsigned short);
    else LP_PAGES(unsigned char);
#undef LP_PAGES
    LP_CHECK_CUDA(cudaGetLastError());
  }
  return 0;
}
