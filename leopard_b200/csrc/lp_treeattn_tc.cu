// leopard_b200 — attention of a tree of drafted tokens over a cache, for many rows: tcgen05 products, keys and values by TMA from the cache's pages.
//
// One persistent CTA an SM takes its piece of the line of tiles (lp_treeattn.cuh), tile after tile of 128 keys.  Two 128-row streams, each with its own MMA issuer and softmax
// warps as in the prefill's kernel (lp_attn3.cu): S of a tile comes in two halves of 64 keys with their own TMEM columns, so that the product for the next half runs
// while the softmax is at this one.  Of up to 256 rows (node x query head of a key head) each stream has a half, on the same keys; up to 128 rows (SPLIT) are
// the rows of both streams, which take the tiles in turn and join their sums at the end of a piece: alone, a stream is bound by the latency of its chain
// S -> softmax -> P V (1.8 us a tile, where reading 64 KB at an SM's share of HBM takes 1.5; 8 sequences of 8,000 rows, 9 to 32 nodes,
// 67 to 77 us and 77 to 84 without; 24 of 4,000 90 to 99 and 99 to 108).
//   warp 0       TMA producer: K_j, V_j into rings of two (SPLIT: three), a box a page or part of one; pages that are not there come as zeros
//   warp 1 / 2   MMA issuer of stream 0 / 1:  S(j).h = Q K_j[h]^T,  O += P(j).h V_j[h] (P in TMEM)
//   warp 3       TMEM
//   warps 4-7, 8-11   softmax of stream 0 / 1: a thread a row; they also bring the rows' queries (rows of a product are G heads of each node) and take O out
// Bound by HBM for few rows of long caches (13 nodes of two sequences of 100,003 rows 143 us, 5.7 TB/s), by the softmax's exponentials for many (64 nodes of 8 of 8,191 rows, 32
// heads over 8, 103 us, 660 TFLOP/s); by the ends of pieces, 6 to 12 us each, in between (64 nodes of 8 sequences of 2,414 to 8,191 rows 72 us, where its bytes take 24).
// TMEM: S0 [0, 128) S1 [128, 256) O0 [256, 384) O1 [384, 512).
// Only the last tiles of an item, which hold nodes or reach past them, look at masks; there V is searched before its product: rows behind the keys become zeros (a
// cache's unwritten memory may hold anything), and values that are not finite are taken out and reach the rows that see them when O is taken out.
#include "lp_treeattn.cuh"

namespace lp {

constexpr int TT_BOX = 128 * 128;      // 128 rows x 64 bf16
constexpr int TT_THREADS = 384;
constexpr int TT_KEYS = 128;
constexpr int TT_MAX_BATCH = 1024;      // sequences whose line of tiles fits beside the tiles
constexpr int TT_SPLIT_BATCH = 24;      // sequences whose line of tiles leaves room for three stages (9 to 32 nodes of 24 of 4,000 rows 90 to 99 us, of 25 106 to 113)

#define LP_TT_TMEM_ST_16(regs, taddr)                                                                               \
  asm volatile(                                                                                                     \
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, " \
      "%15, %16};" ::"r"(taddr),                                                                                    \
      "r"(regs[0]), "r"(regs[1]), "r"(regs[2]), "r"(regs[3]), "r"(regs[4]), "r"(regs[5]), "r"(regs[6]),             \
      "r"(regs[7]), "r"(regs[8]), "r"(regs[9]), "r"(regs[10]), "r"(regs[11]), "r"(regs[12]), "r"(regs[13]),         \
      "r"(regs[14]), "r"(regs[15])                                                                                  \
      : "memory")

__device__ __forceinline__ uint64_t tt_pk2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void tt_upk2(uint64_t r, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r)); }
__device__ __forceinline__ uint64_t tt_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t tt_add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ void tt_bar_sync(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }
__device__ __forceinline__ void tt_bar_arrive(int id, int n) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(n) : "memory"); }

struct TreeTc {
  TreeArgs a;
  int box;                             // rows of a TMA box: of one page
};
constexpr int TT_BARS = 320;           // bytes of the barriers and what stands behind them

// a CTA's piece of an item
struct TreePiece {
  int b, kvh, r0, t0, n;               // sequence, key head, first row, first tile, tiles
  TreeSeq s;
};
__device__ __forceinline__ TreePiece tree_piece(const TreeArgs& a, const TreeLine* line, long long u, long long u_end) {
  TreePiece p;
  p.b = tree_find(line, a.d.B, u);
  p.s = tree_seq(a, line[p.b].len, line[p.b].n);
  const long long local = u - line[p.b].first;
  const int item = (int)tree_div(local, p.s.tiles);
  p.t0 = (int)(local - (long long)item * p.s.tiles);
  p.n = (int)min((long long)(p.s.tiles - p.t0), u_end - u);
  p.kvh = tree_div32(item, p.s.blocks);
  p.r0 = (item - p.kvh * p.s.blocks) * a.rows;
  return p;
}
// where row `key` of a sequence lies: its place in the page table and in the page.  A sequence's rows are fewer than 2^31 (the entry point sees to it).
struct TreePlace {
  int index, row;
  __device__ __forceinline__ TreePlace(const TreeArgs& a, int key) : index(tree_div32(key, a.d.page_size)), row(key - index * a.d.page_size) {}
  __device__ __forceinline__ void forward(const TreeArgs& a, int keys) {
    for (row += keys; row >= a.d.page_size; ++index) row -= a.d.page_size;
  }
  __device__ __forceinline__ int page(const TreeArgs& a, int b) const {      // -1: none
    if (index >= a.d.max_pages) return -1;
    const int page = a.d.page_table ? a.d.page_table[b * a.d.ld_table + index] : b;
    return page >= 0 && page < a.d.n_pages ? page : -1;
  }
};

template <int DH, bool SPLIT>
__global__ void __launch_bounds__(TT_THREADS, 1)
tree_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ TreeTc tc) {
  constexpr int NB = (DH + 63) / 64, KS_QK = DH / 16, HEAD_BYTES = NB * TT_BOX, STAGES = SPLIT ? 3 : 2;
  // A stage's loads have FULLS / STAGES barriers in turn.  SPLIT: three stages are dealt to two streams, and a stage's load before this one was the other stream's: a wait by parity for tile g on
  // one barrier a stage would pass while the load of g - 3 is still under way.  With six, the phase before is that of g - 6, which has been consumed when anybody waits for g: before
  // loads of g - 2, this stream's last tile, the producer sent those of g - 3, and for these it waited until g - 6 was free (a piece's first tiles: all before the piece has been consumed
  // when its queries are there).
  constexpr int FULLS = SPLIT ? 2 * STAGES : STAGES;
  constexpr int Q_OFF = 0, K_OFF = Q_OFF + (SPLIT ? 1 : 2) * HEAD_BYTES, V_OFF = K_OFF + STAGES * HEAD_BYTES, BAR_OFF = V_OFF + STAGES * HEAD_BYTES;
  constexpr int CH = DH / 8, MAX_WORDS = SPLIT ? 2 : LP_TREE_MAX_NODES / 64;
  constexpr uint32_t TM_S = 0, TM_O = 256;
  const TreeArgs& a = tc.a;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + BAR_OFF);      // [2] by stream, a phase a piece that the stream has tiles of
  uint64_t* k_full = q_full + 2;                                       // [FULLS] by tile
  uint64_t* v_full = k_full + FULLS;                                   // [FULLS]
  uint64_t* k_empty = v_full + FULLS;                                  // [3] by stage: both streams' issuers, or that of the tile's stream
  uint64_t* v_empty = k_empty + 3;                                     // [3]
  uint64_t* s_full = v_empty + 3;                                      // [4] stream x half
  uint64_t* p_full = s_full + 4;                                       // [4]
  uint64_t* pv_done = p_full + 4;                                      // [4]
  uint64_t* o_done = pv_done + 4;                                      // [2]
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(o_done + 2);
  int* odd = reinterpret_cast<int*>(tmem_at + 1);                      // [4] piece whose V had values that are not finite, by its number mod 4
  float2* other = reinterpret_cast<float2*>(smem + BAR_OFF + TT_BARS);     // [128] SPLIT: maximum and sum of stream 1's rows
  unsigned long long* mask_words = reinterpret_cast<unsigned long long*>(smem + BAR_OFF + TT_BARS);      // [256][MAX_WORDS] else: of this thread's row
  static_assert((2 + 2 * FULLS + 3 + 3 + 4 + 4 + 4 + 2) * 8 + 4 + 16 <= TT_BARS, "barriers");
  TreeLine* line = reinterpret_cast<TreeLine*>(smem + BAR_OFF + TT_BARS + (SPLIT ? 128 * 8 : 256 * MAX_WORDS * 8));

  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  pdl_launch_dependents();
  if (warp == 1 && lane == 0) {
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 128);
      mbar_init(&o_done[i], 1);
    }
    for (int i = 0; i < FULLS; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&v_full[i], 1);
    }
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&k_empty[i], SPLIT ? 1 : 2);
      mbar_init(&v_empty[i], SPLIT ? 1 : 2);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
      mbar_init(&pv_done[i], 1);
      odd[i] = -1;
    }
    fence_barrier_init();
  }
  if (warp == 3) {
    tmem_alloc(tmem_at, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  tree_line(a, line);                 // (ends in the block's barrier)
  tc_fence_after();
  long long u_begin, u_end;
  tree_range(a, line, blockIdx.x, u_begin, u_end);
  const uint32_t tmem_base = *tmem_at;

  if (warp == 0) {
    // ---------------------------------------------------------------- producer: the lanes know the pages of a tile's boxes, the first issues
    const int boxes = TT_KEYS / tc.box;
    int g = 0;
    for (long long u = u_begin; u < u_end;) {
      const TreePiece p = tree_piece(a, line, u, u_end);
      u += p.n;
      const int n_keys = p.s.keys;
      int key = lane < boxes ? p.t0 * TT_KEYS + lane * tc.box : 0;      // this lane's box of the tile
      TreePlace at(a, key);
      auto page_of = [&]() { return lane < boxes && key < n_keys ? at.page(a, p.b) : -1; };
      int page = page_of();
      for (int j = 0; j < p.n; ++j, ++g) {
        const int st = g % STAGES, row = at.row;
        int next = -1;
        if (j + 1 < p.n) {
          if (lane < boxes) {
            key += TT_KEYS;
            at.forward(a, TT_KEYS);
          }
          next = page_of();
        }
        const uint32_t ph = (g / STAGES) & 1;
        for (int kv = 0; kv < 2; ++kv) {
          uint64_t* full = kv ? &v_full[g % FULLS] : &k_full[g % FULLS];
          if (g >= STAGES) mbar_wait_warp(kv ? &v_empty[st] : &k_empty[st], ph ^ 1);
          if (lane == 0) mbar_arrive_expect_tx(full, HEAD_BYTES);
          uint8_t* to = smem + (kv ? V_OFF : K_OFF) + st * HEAD_BYTES;
          for (int i = 0; i < boxes; ++i) {
            const int pg = __shfl_sync(0xffffffffu, page, i), r = __shfl_sync(0xffffffffu, row, i);
            if (lane == 0) {
#pragma unroll
              for (int c = 0; c < NB; ++c) tma_load_4d(to + c * TT_BOX + i * tc.box * 128, kv ? &tmV : &tmK, full, c * 64, p.kvh, r, pg);
            }
          }
        }
        page = next;
      }
    }
  } else if (warp == 1 || warp == 2) {
    // ---------------------------------------------------------------- MMA issuer of a stream
    const int q = warp - 1;
    const bool issue = elect_one();
    constexpr uint32_t idesc_s = umma_idesc_bf16(128, 64, 0, 0), idesc_o = umma_idesc_bf16(128, DH, 0, 1);
    const uint32_t q_addr = smem_u32(smem + Q_OFF + (SPLIT ? 0 : q) * HEAD_BYTES), s_tm = tmem_base + TM_S + (uint32_t)q * 128, d_o = tmem_base + TM_O + (uint32_t)q * 128;
    constexpr int STEP = SPLIT ? 2 : 1;
    int g = 0, nt = 0, pieces = 0;      // tiles of the CTA so far; tiles of this stream; pieces whose queries it has waited for
    for (long long u = u_begin; u < u_end;) {
      const TreePiece p = tree_piece(a, line, u, u_end);
      u += p.n;
      const int j0 = SPLIT ? q : 0;
      if (SPLIT && j0 >= p.n) {         // one tile: the other stream's, with nothing to wait for here (a wait that the other stream does not wait for in turn may miss its phase)
        g += p.n;
        continue;
      }
      if (!SPLIT && p.r0 + q * 128 >= p.s.n * a.group) {      // no rows here: the stages are passed on
        for (int j = 0; j < p.n; ++j, ++g) {
          mbar_wait_warp(&k_full[g % FULLS], (g / FULLS) & 1);
          if (issue) mbar_arrive(&k_empty[g % STAGES]);
          mbar_wait_warp(&v_full[g % FULLS], (g / FULLS) & 1);
          if (issue) mbar_arrive(&v_empty[g % STAGES]);
        }
        continue;
      }
      auto issue_S = [&](int gt, int h) {
        const uint32_t k_addr = smem_u32(smem + K_OFF + (gt % STAGES) * HEAD_BYTES) + (uint32_t)h * 64 * 128;
        if (issue) {
#pragma unroll
          for (int ks = 0; ks < KS_QK; ++ks) {
            const uint32_t off = (ks >> 2) * TT_BOX + (ks & 3) * 32;
            umma_ss(s_tm + (uint32_t)h * 64, umma_desc_sw128(q_addr + off, 0, 1024), umma_desc_sw128(k_addr + off, 0, 1024), idesc_s, ks > 0 ? 1u : 0u);
          }
          umma_commit(&s_full[q * 2 + h]);
        }
      };
      auto issue_PV = [&](int gt, bool start, int h) {
        const uint32_t v_addr = smem_u32(smem + V_OFF + (gt % STAGES) * HEAD_BYTES);
        mbar_wait_warp(&p_full[q * 2 + h], nt & 1);
        tc_fence_after();
        if (issue) {
#pragma unroll
          for (int k4 = 0; k4 < 4; ++k4) {
            const int ks = h * 4 + k4;
            umma_ts(d_o, s_tm + (uint32_t)h * 64 + k4 * 8, umma_desc_sw128(v_addr + ks * 2048, TT_BOX, 1024), idesc_o, (!start || ks > 0) ? 1u : 0u);
          }
          umma_commit(&pv_done[q * 2 + h]);
        }
      };
      mbar_wait_warp(&q_full[q], pieces & 1);
      ++pieces;
      int gt = g + j0;
      mbar_wait_warp(&k_full[gt % FULLS], (gt / FULLS) & 1);
      tc_fence_after();
      issue_S(gt, 0);
      issue_S(gt, 1);
      if (issue) umma_commit(&k_empty[gt % STAGES]);
      for (int j = j0; j < p.n; j += STEP, gt += STEP, ++nt) {
        const bool more = j + STEP < p.n;
        const int gn = gt + STEP;
        mbar_wait_warp(&v_full[gt % FULLS], (gt / FULLS) & 1);
        issue_PV(gt, j == j0, 0);
        if (more) {
          mbar_wait_warp(&k_full[gn % FULLS], (gn / FULLS) & 1);
          tc_fence_after();
          issue_S(gn, 0);
        }
        issue_PV(gt, j == j0, 1);
        if (issue) umma_commit(&v_empty[gt % STAGES]);
        if (more) {
          issue_S(gn, 1);
          if (issue) umma_commit(&k_empty[gn % STAGES]);
        } else if (issue) {
          umma_commit(&o_done[q]);
        }
      }
      g += p.n;
    }
  } else if (warp >= 4) {
    // ---------------------------------------------------------------- softmax: thread = row
    const int q = (warp - 4) >> 2, lg = warp & 3, r = lg * 32 + lane;
    const uint32_t lane_addr = tmem_base + ((uint32_t)(lg * 32) << 16);
    const uint32_t s_addr = lane_addr + TM_S + (uint32_t)q * 128, o_addr = lane_addr + TM_O + (uint32_t)q * 128;
    constexpr int STEP = SPLIT ? 2 : 1;
    int g = 0, nt = 0, pieces = 0, joins = 0, seg = 0;      // tiles of the CTA and of this stream so far; pieces that it had tiles of; SPLIT: pieces of both streams
    for (long long u = u_begin; u < u_end; ++seg) {
      const TreePiece p = tree_piece(a, line, u, u_end);
      u += p.n;
      const int rows = p.s.n * a.group, row_base = p.r0 + (SPLIT ? 0 : q * 128), j0 = SPLIT ? q : 0;
      if (SPLIT ? j0 >= p.n : row_base >= rows) { g += p.n; continue; }
      const bool both = !SPLIT && p.r0 + 128 < rows;                   // the other stream is at the same tiles
      const int row = row_base + r;
      const bool row_ok = row < rows;
      const int node = row_ok ? tree_div32(row, a.group) : 0, head = p.kvh * a.group + (row_ok ? row - node * a.group : 0);
      // the warp's rows' queries, in the swizzled layout that TMA writes; 32 lanes take neighbouring pieces of 16 bytes
      if (!SPLIT || q == 0) {
        const long long from = p.b * a.d.q_batch + node * a.d.q_node + head * a.d.q_head;
        uint8_t* at = smem + Q_OFF + (SPLIT ? 0 : q) * HEAD_BYTES + lg * 32 * 128;
        uint4 x[CH];
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          const int rr = (i * 32 + lane) / CH, c = (i * 32 + lane) % CH;
          const long long src = __shfl_sync(0xffffffffu, from, rr);      // (of a row that is not there the first node's: loads without branches go out together)
          x[i] = *reinterpret_cast<const uint4*>(reinterpret_cast<const bf16*>(a.d.q) + src + c * 8);
        }
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          const int rr = (i * 32 + lane) / CH, c = (i * 32 + lane) % CH;
          sts_u4(at + (c >> 3) * TT_BOX + rr * 128 + (((c & 7) ^ (rr & 7)) << 4), row_base + lg * 32 + rr < rows ? x[i] : make_uint4(0, 0, 0, 0));
        }
        if (DH % 64 != 0)
          for (int c = CH; c < NB * 8; ++c) sts_u4(at + (c >> 3) * TT_BOX + lane * 128 + (((c & 7) ^ (lane & 7)) << 4), make_uint4(0, 0, 0, 0));
        fence_proxy_async_smem();
        mbar_arrive(&q_full[q]);
        if (SPLIT && p.n > 1) mbar_arrive(&q_full[1]);
      }
      // its node's mask, when this piece gets there
      const int nw = (a.d.T + 63) >> 6;
      unsigned long long word0 = 0, word1 = 0;                         // SPLIT: two at most
      unsigned long long* words = mask_words + (q * 128 + r) * MAX_WORDS;
      if ((p.t0 + p.n) * TT_KEYS > p.s.len) {
        const unsigned long long* src = a.d.mask + p.b * a.d.mask_batch + node * a.d.mask_node;
        if (SPLIT) {
          word0 = src[0];
          if (nw > 1) word1 = src[1];
        } else {
          for (int w = 0; w < nw; ++w) words[w] = src[w];
        }
      }
      auto word_at = [&](int w) -> unsigned long long { return w >= nw ? 0ull : SPLIT ? (w == 0 ? word0 : word1) : words[w]; };
      // which of a half's 64 keys there are, by their pages (known a step ahead)
      const int box = min(tc.box, 64), n_box = 64 / box;
      const int n_keys = p.s.keys, len = p.s.len;
      bool paged = a.d.page_table != nullptr;
      if (paged) {                                                     // (all of the piece's pages there: no more looks)
        const int from = tree_div32(p.t0 * TT_KEYS, a.d.page_size), to = tree_div32(min((p.t0 + p.n) * TT_KEYS, n_keys) - 1, a.d.page_size);
        bool there = true;
        for (int i = from + lane; i <= to; i += 32) {
          const int page = a.d.page_table[p.b * a.d.ld_table + i];
          there &= page >= 0 && page < a.d.n_pages;
        }
        paged = !__all_sync(0xffffffffu, there);
      }
      int box_key = lane < n_box ? (p.t0 + j0) * TT_KEYS + lane * box : 0;
      TreePlace box_at(a, paged && lane < n_box ? box_key : 0);
      auto page_there = [&]() { return !paged || lane >= n_box || box_key >= n_keys || box_at.page(a, p.b) >= 0; };
      bool there_next = page_there();
      if (SPLIT && q == 1 && joins > 0) tt_bar_sync(3, 256);           // stream 0 has taken out what this one had of its last piece
      float m_used = -INFINITY, l_sum = 0.f;
      uint32_t v[64];
      mbar_wait_warp(&s_full[q * 2], nt & 1);                          // (loads from and stores to TMEM are for whole warps, here and below)
      tc_fence_after();
      LP_TMEM_LD_32((v + 0), s_addr + 0);
      LP_TMEM_LD_32((v + 32), s_addr + 32);
      const int mine = (p.n - j0 + STEP - 1) / STEP;                   // tiles of this stream
#pragma unroll 1
      for (int t = 0; t < 2 * mine; ++t) {
        const int j = j0 + (t >> 1) * STEP, h = t & 1;
        const int key0 = (p.t0 + j) * TT_KEYS + h * 64;
        const bool tail = key0 - h * 64 + TT_KEYS > len;
        const unsigned pages = paged ? __ballot_sync(0xffffffffu, there_next) : 0xffffffffu;
        if (paged && t + 1 < 2 * mine) {
          const int on = h == 0 || STEP == 1 ? 64 : 64 + TT_KEYS;
          if (lane < n_box) {
            box_key += on;
            box_at.forward(a, on);
          }
          there_next = page_there();
        }
        if (tail && h == 0) {
          // V of this tile before its product: rows that are not keys, values that are not finite
          mbar_wait(&v_full[(g + j) % FULLS], ((g + j) / FULLS) & 1);
          const bool key_ok = key0 + r < n_keys;
          uint8_t* at = smem + V_OFF + ((g + j) % STAGES) * HEAD_BYTES + r * 128;
#pragma unroll 1
          for (int c = 0; c < NB; ++c) {
            if (both && NB == 2 && c != q) continue;                   // each stream searches its half of the columns
            if (both && NB == 1 && q == 1) continue;
            at += c * TT_BOX;
            if (!key_ok) {
#pragma unroll
              for (int i = 0; i < 8; ++i) sts_u4(at + (i << 4), make_uint4(0, 0, 0, 0));
              continue;
            }
            uint4 x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = lds_u4(at + ((i ^ (r & 7)) << 4));
            uint32_t any = 0;                                          // a carry into bit 15 (31): an exponent of all ones
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              auto look = [&](uint32_t w) { any |= ((w & 0x7fff7fffu) + 0x00800080u) & 0x80008000u; };
              look(x[i].x); look(x[i].y); look(x[i].z); look(x[i].w);
            }
            if (any) {
#pragma unroll 1
              for (int i = 0; i < 32; ++i) {
                uint32_t* w = reinterpret_cast<uint32_t*>(at) + i;
                const uint32_t b = ((*w & 0x7fff7fffu) + 0x00800080u) & 0x80008000u;
                if (b) *w &= (b & 0x8000u ? 0u : 0xffffu) | (b & 0x80000000u ? 0u : 0xffff0000u);
              }
              *reinterpret_cast<volatile int*>(&odd[seg & 3]) = seg;
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (both) tt_bar_sync(1, 256);
        }
        tmem_wait_ld();
        unsigned long long sees = ~0ull;
        if (pages != 0xffffffffu)
          for (int i = 0; i < n_box; ++i)
            if (!((pages >> i) & 1)) sees &= ~((box == 64 ? ~0ull : (1ull << box) - 1) << (i * box));
        if (key0 + 64 > len) {
          const int behind = n_keys - key0;                            // keys of this half
          if (behind < 64) sees &= behind <= 0 ? 0ull : (1ull << behind) - 1;
          const int first_node = key0 - len;
          unsigned long long bits;
          if (first_node < 0) bits = (word_at(0) << -first_node) | ((1ull << -first_node) - 1);
          else {
            const int w = first_node >> 6, sh = first_node & 63;
            bits = word_at(w) >> sh;
            if (sh) bits |= word_at(w + 1) << (64 - sh);
          }
          sees &= bits;
        }
        if (__any_sync(0xffffffffu, sees != ~0ull)) {
          const uint32_t lo = (uint32_t)sees, hi = (uint32_t)(sees >> 32);
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            if (!((lo >> i) & 1)) v[i] = 0xff800000u;
            if (!((hi >> i) & 1)) v[32 + i] = 0xff800000u;
          }
        }
        const uint64_t sc2 = tt_pk2(a.scale_log2, a.scale_log2);
        float mx;      // of scores, not scaled yet: scales are not negative here
        {
          float m0 = -INFINITY, m1 = -INFINITY, m2 = -INFINITY, m3 = -INFINITY;
#pragma unroll
          for (int i = 0; i < 64; i += 8) {
            m0 = fmaxf(m0, fmaxf(__uint_as_float(v[i]), __uint_as_float(v[i + 1])));
            m1 = fmaxf(m1, fmaxf(__uint_as_float(v[i + 2]), __uint_as_float(v[i + 3])));
            m2 = fmaxf(m2, fmaxf(__uint_as_float(v[i + 4]), __uint_as_float(v[i + 5])));
            m3 = fmaxf(m3, fmaxf(__uint_as_float(v[i + 6]), __uint_as_float(v[i + 7])));
          }
          mx = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3));
        }
        const float m_new = fmaxf(m_used, mx * a.scale_log2);
        const bool grow = (m_new - m_used) > 8.0f;
        if (t == 0) {
          m_used = m_new;
        } else if (__any_sync(0xffffffffu, grow)) {
          // every product issued so far has to be done before O is scaled in place
          mbar_wait_warp(&pv_done[q * 2 + (h ^ 1)], (nt + ((t - 1) >> 1)) & 1);
          tc_fence_after();
          float alpha = 1.0f;
          if (grow) {
            alpha = ta_ex2(m_used - m_new);
            m_used = m_new;
            l_sum *= alpha;
          }
          __syncwarp();
#pragma unroll 1
          for (int c = 0; c < DH / 16; ++c) {
            uint32_t o[16];
            LP_TMEM_LD_16(o, o_addr + c * 16);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            LP_TT_TMEM_ST_16(o, o_addr + c * 16);
          }
          tmem_wait_st();
        }
        const float neg_m = m_used == -INFINITY ? 0.f : -m_used;
        const uint64_t nm2 = tt_pk2(neg_m, neg_m);
        uint64_t acc2 = tt_pk2(0.f, 0.f);
        const int tn = (t + 1) >> 1, hn = (t + 1) & 1;
        const bool has_next = t + 1 < 2 * mine;
        const bool s_ready = has_next && mbar_test_wait(&s_full[q * 2 + hn], (nt + tn) & 1);
        if (both) {                                                    // the streams' exponentials in turns: one's loads and stores run beside the other's
          if (q == 1) tt_bar_sync(5, 256);
          else if (t > 0) tt_bar_sync(4, 256);
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float x0, x1;
            tt_upk2(tt_fma2(tt_pk2(__uint_as_float(v[c * 32 + i]), __uint_as_float(v[c * 32 + i + 1])), sc2, nm2), x0, x1);
            const float p0 = ta_ex2(x0), p1 = ta_ex2(x1);
            acc2 = tt_add2(acc2, tt_pk2(p0, p1));
            pk[i >> 1] = pack_bf16x2(p0, p1);      // half a step is 2^-8 of a weight; their sum is taken in fp32 before
          }
          LP_TT_TMEM_ST_16(pk, s_addr + h * 64 + c * 16);
        }
        if (both) {
          if (q == 0) tt_bar_arrive(5, 256);
          else if (has_next) tt_bar_arrive(4, 256);
        }
        bool loaded = false;
        if (has_next && __all_sync(0xffffffffu, s_ready || mbar_test_wait(&s_full[q * 2 + hn], (nt + tn) & 1))) {
          tc_fence_after();
          LP_TMEM_LD_32((v + 0), s_addr + hn * 64 + 0);
          LP_TMEM_LD_32((v + 32), s_addr + hn * 64 + 32);
          loaded = true;
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&p_full[q * 2 + h]);
        {
          float a0, a1;
          tt_upk2(acc2, a0, a1);
          l_sum += a0 + a1;
        }
        if (has_next && !loaded) {
          mbar_wait_warp(&s_full[q * 2 + hn], (nt + tn) & 1);
          tc_fence_after();
          LP_TMEM_LD_32((v + 0), s_addr + hn * 64 + 0);
          LP_TMEM_LD_32((v + 32), s_addr + hn * 64 + 32);
        }
      }
      g += p.n;
      nt += mine;
      // ---- O of this piece
      const bool two = SPLIT && p.n > 1;                               // both streams had tiles
      if (SPLIT && q == 1) {                                           // stream 0 takes it out
        other[r] = make_float2(m_used, l_sum);
        tt_bar_arrive(2, 256);
        ++pieces;
        ++joins;
        continue;
      }
      mbar_wait_warp(&o_done[q], pieces & 1);
      ++pieces;
      float f0 = 1.f, f1 = 0.f;
      if (two) {
        tt_bar_sync(2, 256);
        mbar_wait_warp(&o_done[1], joins & 1);
        ++joins;
        const float2 x = other[r];
        const float m = fmaxf(m_used, x.x);
        f0 = m_used == -INFINITY ? 1.f : ta_ex2(m_used - m);           // sums and values of a stream that saw nothing are zeros, or NaN
        f1 = x.x == -INFINITY ? 1.f : ta_ex2(x.x - m);
        l_sum = l_sum * f0 + x.y * f1;
        m_used = m;
      }
      tc_fence_after();
      const bool whole = p.t0 == 0 && p.n == p.s.tiles;
      const bool fix = *reinterpret_cast<volatile int*>(&odd[seg & 3]) == seg;
      const float inv_l = l_sum == 0.f ? 0.f : 1.0f / l_sum;
      const long long slot = 2LL * blockIdx.x + (p.t0 == 0 ? 1 : 0);
      const int in_block = (SPLIT ? 0 : q * 128) + r;
      float* part = a.part_o + (slot * (DH / 4) * a.rows + in_block) * 4;
      uint8_t* stage = smem + Q_OFF + (SPLIT ? 0 : q) * HEAD_BYTES + lg * 32 * 128;      // the queries are done with
      if (!whole && row_ok) a.part_ml[slot * a.rows + in_block] = make_float2(m_used, l_sum);
#pragma unroll 1
      for (int c = 0; c < DH / 32; ++c) {
        uint32_t o[32], y[32];
        __syncwarp();
        LP_TMEM_LD_32(o, o_addr + c * 32);
        if (two) LP_TMEM_LD_32(y, o_addr + 128 + c * 32);
        tmem_wait_ld();
        if (two)
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f0 + __uint_as_float(y[i]) * f1);
        if (fix) {
          const int k1 = min(n_keys, (p.t0 + p.n) * TT_KEYS);
          for (int key = max(p.t0, len / TT_KEYS) * TT_KEYS; key < k1; ++key) {
            const TreePlace at(a, key);
            const int page = at.page(a, p.b), nd = max(0, key - len);
            if (page < 0 || (key >= len && !((word_at(nd >> 6) >> (nd & 63)) & 1))) continue;
            const bf16* vr = reinterpret_cast<const bf16*>(a.d.v) + page * a.d.v_page + at.row * a.d.v_row + p.kvh * a.d.v_head + c * 32;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float x = __bfloat162float(vr[i]);
              if (not_finite(x)) o[i] = __float_as_uint(__uint_as_float(o[i]) + x);
            }
          }
        }
        if (whole) {
          uint8_t* at = stage + (c >> 1) * TT_BOX + lane * 128;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(__uint_as_float(o[k * 8 + 2 * i]) * inv_l, __uint_as_float(o[k * 8 + 2 * i + 1]) * inv_l);
            sts_u4(at + ((((c & 1) * 4 + k) ^ (lane & 7)) << 4), make_uint4(w[0], w[1], w[2], w[3]));
          }
        } else if (row_ok) {
#pragma unroll
          for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(part + (c * 8 + i) * a.rows * 4) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        }
      }
      tc_fence_before();
      if (two) tt_bar_arrive(3, 256);
      if (whole) {
        __syncwarp();
        const long long to = p.b * a.d.o_batch + node * a.d.o_node + head * a.d.o_head;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          const int rr = (i * 32 + lane) / CH, c = (i * 32 + lane) % CH;
          const long long dst = __shfl_sync(0xffffffffu, to, rr);
          const uint4 x = lds_u4(stage + (c >> 3) * TT_BOX + rr * 128 + (((c & 7) ^ (rr & 7)) << 4));
          if (row_base + lg * 32 + rr < rows) *reinterpret_cast<uint4*>(reinterpret_cast<bf16*>(a.d.out) + dst + c * 8) = x;
        }
        __syncwarp();
      }
    }
    if (SPLIT && q == 1 && joins > 0) tt_bar_sync(3, 256);             // (what stream 0 has arrived at)
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 3) {
    __syncwarp();
    tmem_dealloc(tmem_base, 512);
  }
}

// rows of a TMA box: a cache of one page a sequence takes whole tiles, else the largest part of a tile that pages are multiples of
static int tree_box(const lp_tree_attn_desc* d) {
  if (d->max_pages == 1) return 128;
  for (int box = 128; box >= 8; box /= 2)
    if (d->page_size % box == 0) return box;
  return 0;
}
bool tree_tc_takes(const lp_tree_attn_desc* d) {
  const bool strides = (d->n_pages == 1 || (d->k_page > 0 && d->v_page > 0)) && (d->page_size == 1 || (d->k_row > 0 && d->v_row > 0)) &&
                       (d->KVH == 1 || (d->k_head > 0 && d->v_head > 0));
  return tree_box(d) != 0 && strides && d->scale > 0.f && d->B <= TT_MAX_BATCH;      // (0 x -inf is not -inf)
}

template <int DH>
static int launch_tc(const TreeTc& tc, cudaStream_t stream) {
  constexpr int NB = (DH + 63) / 64;
  const lp_tree_attn_desc& d = tc.a.d;
  CUtensorMap tm[2];
  const void* base[2] = {d.k, d.v};
  const long long page[2] = {d.k_page, d.v_page}, row[2] = {d.k_row, d.v_row}, head[2] = {d.k_head, d.v_head};
  const uint32_t box[4] = {64, 1, (uint32_t)tc.box, 1};
  for (int i = 0; i < 2; ++i) {      // of a dimension of one the distance is any
    const uint64_t dims[4] = {(uint64_t)d.D, (uint64_t)d.KVH, (uint64_t)d.page_size, (uint64_t)d.n_pages};
    const uint64_t strides[3] = {d.KVH == 1 ? (uint64_t)d.D : (uint64_t)head[i], d.page_size == 1 ? (uint64_t)d.D : (uint64_t)row[i], d.n_pages == 1 ? (uint64_t)d.D : (uint64_t)page[i]};
    if (const int rc = make_tmap_bf16_4d(&tm[i], base[i], dims, strides, box)) return rc;
  }
  const bool split = d.B <= TT_SPLIT_BATCH && tc.a.rows <= 128;
  const size_t smem = (split ? 7 : 6) * NB * TT_BOX + TT_BARS + (split ? 128 * 8 : 256 * (LP_TREE_MAX_NODES / 64) * 8) + (size_t)(d.B + 1) * sizeof(TreeLine) + 1024;
  if (split) {
    LP_CHECK_CUDA((allow_smem<tree_tc_kernel<DH, true>>((int)smem)));
    tree_tc_kernel<DH, true><<<tc.a.ctas, TT_THREADS, smem, stream>>>(tm[0], tm[1], tc);
  } else {
    LP_CHECK_CUDA((allow_smem<tree_tc_kernel<DH, false>>((int)smem)));
    tree_tc_kernel<DH, false><<<tc.a.ctas, TT_THREADS, smem, stream>>>(tm[0], tm[1], tc);
  }
  LP_CHECK_CUDA(cudaGetLastError());
  return 0;
}

int launch_tree_tc(const TreeArgs& a, cudaStream_t stream) {
  TreeTc tc;
  tc.a = a;
  tc.box = tree_box(&a.d);
  if (a.d.D == 128) return launch_tc<128>(tc, stream);
  if (a.d.D == 96) return launch_tc<96>(tc, stream);
  return launch_tc<64>(tc, stream);
}

}  // namespace lp
