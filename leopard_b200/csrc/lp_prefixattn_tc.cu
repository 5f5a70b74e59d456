// leopard_b200 — attention over a shared prefix for many rows: tcgen05 products, keys and values by TMA from the prefix's pages.
//
// The pipeline of lp_treeattn_tc.cu with other rows and nothing hidden: one persistent CTA an SM takes a range of the line of tiles of 128 keys (lp_prefixattn.cuh).  Two 128-row streams, each with its own MMA
// issuer and softmax warps; S of a tile comes in two halves of 64 keys with their own TMEM columns, so that the product for the next half runs while the softmax is at this one.
// Of up to 256 rows (token x query head of a key head) each stream has a half, on the same keys; up to 128 rows in all (SPLIT) are the rows of both streams, which take the tiles in turn and join their
// sums at the end of a piece.
//   warp 0       TMA producer: K_j, V_j into rings of two (SPLIT: three), a box a page or part of one; pages that are not there come as zeros
//   warp 1 / 2   MMA issuer of stream 0 / 1:  S(j).h = Q K_j[h]^T,  O += P(j).h V_j[h] (P in TMEM)
//   warp 3       TMEM
//   warps 4-7, 8-11   softmax of stream 0 / 1: a thread a row; they also bring the rows' queries and take O out
// Bound by the softmax beside the products: 2.5 us a tile of 256 rows, where products alone take 1.5 and HBM's share 1.5 (276 tokens of 32 heads over 8 after 100,003 rows 508 us, 890 TFLOP/s; 57 after 32,771 37 us behind its
// start, and 4 for the pieces' way out).
// TMEM: S0 [0, 128) S1 [128, 256) O0 [256, 384) O1 [384, 512).
#include "lp_prefixattn.cuh"

namespace lp {

constexpr int PT_BOX = 128 * 128;      // 128 rows x 64 bf16
constexpr int PT_THREADS = 384;
constexpr int PT_KEYS = 128;
constexpr int PT_BARS = 320;           // bytes of the barriers and what stands behind them

#define LP_PT_TMEM_ST_16(regs, taddr)                                                                               \
  asm volatile(                                                                                                     \
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, " \
      "%15, %16};" ::"r"(taddr),                                                                                    \
      "r"(regs[0]), "r"(regs[1]), "r"(regs[2]), "r"(regs[3]), "r"(regs[4]), "r"(regs[5]), "r"(regs[6]),             \
      "r"(regs[7]), "r"(regs[8]), "r"(regs[9]), "r"(regs[10]), "r"(regs[11]), "r"(regs[12]), "r"(regs[13]),         \
      "r"(regs[14]), "r"(regs[15])                                                                                  \
      : "memory")

__device__ __forceinline__ uint64_t pt_pk2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void pt_upk2(uint64_t r, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r)); }
__device__ __forceinline__ uint64_t pt_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t pt_add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ void pt_bar_sync(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }
__device__ __forceinline__ void pt_bar_arrive(int id, int n) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(n) : "memory"); }

struct PrefixTc {
  PrefixArgs a;
  int box;                             // rows of a TMA box: of one page
};
// where a row of the prefix lies: its place in the page table and in the page
struct PrefixPlace {
  int index, row;
  __device__ __forceinline__ PrefixPlace(const PrefixArgs& a, int key) : index(a.d.page_table ? key / a.d.page_size : 0), row(a.d.page_table ? key - index * a.d.page_size : key) {}
  __device__ __forceinline__ void forward(const PrefixArgs& a, int keys) {
    row += keys;
    if (a.d.page_table)
      for (; row >= a.d.page_size; ++index) row -= a.d.page_size;
  }
  __device__ __forceinline__ int page(const PrefixArgs& a) const {      // -1: none
    if (!a.d.page_table) return 0;
    if (index >= a.d.max_pages) return -1;
    const int page = a.d.page_table[index];
    return page >= 0 && page < a.d.n_pages ? page : -1;
  }
};

template <int DH, bool SPLIT>
__global__ void __launch_bounds__(PT_THREADS, 1)
prefix_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ PrefixTc tc) {
  constexpr int NB = (DH + 63) / 64, KS_QK = DH / 16, HEAD_BYTES = NB * PT_BOX, STAGES = SPLIT ? 3 : 2;
  // A stage's loads have FULLS / STAGES barriers in turn.  SPLIT: three stages are dealt to two streams, and a stage's load before this one was the other stream's: a wait by parity for tile g on one barrier
  // a stage would pass while the load of g - 3 is still under way.  With six, the phase before is that of g - 6, which has been consumed when anybody waits for g.
  constexpr int FULLS = SPLIT ? 2 * STAGES : STAGES;
  constexpr int Q_OFF = 0, K_OFF = Q_OFF + (SPLIT ? 1 : 2) * HEAD_BYTES, V_OFF = K_OFF + STAGES * HEAD_BYTES, BAR_OFF = V_OFF + STAGES * HEAD_BYTES;
  constexpr int CH = DH / 8;
  constexpr uint32_t TM_S = 0, TM_O = 256;
  const PrefixArgs& a = tc.a;
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
  float2* other = reinterpret_cast<float2*>(smem + BAR_OFF + PT_BARS);     // [128] SPLIT: maximum and sum of stream 1's rows
  static_assert((2 + 2 * FULLS + 3 + 3 + 4 + 4 + 4 + 2) * 8 + 4 <= PT_BARS, "barriers");
  int* first = reinterpret_cast<int*>(smem + BAR_OFF + PT_BARS + (SPLIT ? 128 * 8 : 0));

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
    }
    fence_barrier_init();
  }
  if (warp == 3) {
    tmem_alloc(tmem_at, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  pa_tokens(a, first);                // (ends in the block's barrier)
  tc_fence_after();
  const int rows = first[a.d.B] * a.group, n_keys = a.d.prefix;
  const PrefixLine line = pa_line(a, rows);
  long long u_begin, u_end;
  pa_range(a, line, blockIdx.x, u_begin, u_end);
  const uint32_t tmem_base = *tmem_at;

  if (warp == 0) {
    // ---------------------------------------------------------------- producer: the lanes know the pages of a tile's boxes, the first issues
    const int boxes = PT_KEYS / tc.box;
    int g = 0;
    for (long long u = u_begin; u < u_end;) {
      const PrefixPiece p = pa_piece(a, u, u_end);
      u += p.n;
      int key = lane < boxes ? p.t0 * PT_KEYS + lane * tc.box : 0;      // this lane's box of the tile
      PrefixPlace at(a, key);
      auto page_of = [&]() { return lane < boxes && key < n_keys ? at.page(a) : -1; };
      int page = page_of();
      for (int j = 0; j < p.n; ++j, ++g) {
        const int st = g % STAGES, row = at.row;
        int next = -1;
        if (j + 1 < p.n) {
          if (lane < boxes) {
            key += PT_KEYS;
            at.forward(a, PT_KEYS);
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
              for (int c = 0; c < NB; ++c) tma_load_4d(to + c * PT_BOX + i * tc.box * 128, kv ? &tmV : &tmK, full, c * 64, p.kvh, r, pg);
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
      const PrefixPiece p = pa_piece(a, u, u_end);
      u += p.n;
      const int j0 = SPLIT ? q : 0;
      if (SPLIT && j0 >= p.n) {         // one tile: the other stream's, with nothing to wait for here (a wait that the other stream does not wait for in turn may miss its phase)
        g += p.n;
        continue;
      }
      if (!SPLIT && p.r0 + q * 128 >= rows) {      // no rows here: the stages are passed on
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
            const uint32_t off = (ks >> 2) * PT_BOX + (ks & 3) * 32;
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
            umma_ts(d_o, s_tm + (uint32_t)h * 64 + k4 * 8, umma_desc_sw128(v_addr + ks * 2048, PT_BOX, 1024), idesc_o, (!start || ks > 0) ? 1u : 0u);
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
    int g = 0, nt = 0, pieces = 0, joins = 0;      // tiles of the CTA and of this stream so far; pieces that it had tiles of; SPLIT: pieces of both streams
    for (long long u = u_begin; u < u_end;) {
      const PrefixPiece p = pa_piece(a, u, u_end);
      u += p.n;
      const int row_base = p.r0 + (SPLIT ? 0 : q * 128), j0 = SPLIT ? q : 0;
      if (SPLIT ? j0 >= p.n : row_base >= rows) { g += p.n; continue; }
      const bool both = !SPLIT && p.r0 + 128 < rows;                   // the other stream is at the same tiles
      const int row = row_base + r;
      const bool row_ok = row < rows;
      // the warp's rows' queries, in the swizzled layout that TMA writes; 32 lanes take neighbouring pieces of 16 bytes
      if (!SPLIT || q == 0) {
        const int token = row_ok ? row / a.group : 0, head = p.kvh * a.group + (row_ok ? row - token * a.group : 0), b = pa_find(first, a.d.B, token);
        const long long from = b * a.d.q_batch + (token - first[b]) * a.d.q_token + head * a.d.q_head;
        uint8_t* at = smem + Q_OFF + (SPLIT ? 0 : q) * HEAD_BYTES + lg * 32 * 128;
        uint4 x[CH];
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          const int rr = (i * 32 + lane) / CH, c = (i * 32 + lane) % CH;
          const long long src = __shfl_sync(0xffffffffu, from, rr);      // (of a row that is not there the first token's: loads without branches go out together)
          x[i] = *reinterpret_cast<const uint4*>(reinterpret_cast<const bf16*>(a.d.q) + src + c * 8);
        }
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          const int rr = (i * 32 + lane) / CH, c = (i * 32 + lane) % CH;
          sts_u4(at + (c >> 3) * PT_BOX + rr * 128 + (((c & 7) ^ (rr & 7)) << 4), row_base + lg * 32 + rr < rows ? x[i] : make_uint4(0, 0, 0, 0));
        }
        if (DH % 64 != 0)
          for (int c = CH; c < NB * 8; ++c) sts_u4(at + (c >> 3) * PT_BOX + lane * 128 + (((c & 7) ^ (lane & 7)) << 4), make_uint4(0, 0, 0, 0));
        fence_proxy_async_smem();
        mbar_arrive(&q_full[q]);
        if (SPLIT && p.n > 1) mbar_arrive(&q_full[1]);
      }
      // which of a half's 64 keys there are, by their pages (known a step ahead)
      const int box = min(tc.box, 64), n_box = 64 / box;
      bool paged = a.d.page_table != nullptr;
      if (paged) {                                                     // (all of the piece's pages there: no more looks)
        const int from = p.t0 * PT_KEYS / a.d.page_size, to = (min((p.t0 + p.n) * PT_KEYS, n_keys) - 1) / a.d.page_size;
        bool there = true;
        for (int i = from + lane; i <= to; i += 32) {
          const int page = a.d.page_table[i];
          there &= page >= 0 && page < a.d.n_pages;
        }
        paged = !__all_sync(0xffffffffu, there);
      }
      int box_key = lane < n_box ? (p.t0 + j0) * PT_KEYS + lane * box : 0;
      PrefixPlace box_at(a, paged && lane < n_box ? box_key : 0);
      auto page_there = [&]() { return !paged || lane >= n_box || box_key >= n_keys || box_at.page(a) >= 0; };
      bool there_next = page_there();
      if (SPLIT && q == 1 && joins > 0) pt_bar_sync(3, 256);           // stream 0 has taken out what this one had of its last piece
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
        const int key0 = (p.t0 + j) * PT_KEYS + h * 64;
        const bool tail = key0 - h * 64 + PT_KEYS > n_keys;
        const unsigned pages = paged ? __ballot_sync(0xffffffffu, there_next) : 0xffffffffu;
        if (paged && t + 1 < 2 * mine) {
          const int on = h == 0 || STEP == 1 ? 64 : 64 + PT_KEYS;
          if (lane < n_box) {
            box_key += on;
            box_at.forward(a, on);
          }
          there_next = page_there();
        }
        if (tail && h == 0) {
          // V of this tile before its product: rows of the last page that are not the prefix's become zeros
          mbar_wait_warp(&v_full[(g + j) % FULLS], ((g + j) / FULLS) & 1);
          if (key0 + r >= n_keys) {
            uint8_t* at = smem + V_OFF + ((g + j) % STAGES) * HEAD_BYTES + r * 128;
#pragma unroll
            for (int c = 0; c < NB; ++c)
              if (!(both && c % 2 != q))                               // each stream has its half of the columns
#pragma unroll
                for (int i = 0; i < 8; ++i) sts_u4(at + c * PT_BOX + (i << 4), make_uint4(0, 0, 0, 0));
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (both) pt_bar_sync(1, 256);
        }
        tmem_wait_ld();
        unsigned long long sees = ~0ull;
        if (pages != 0xffffffffu)
          for (int i = 0; i < n_box; ++i)
            if (!((pages >> i) & 1)) sees &= ~((box == 64 ? ~0ull : (1ull << box) - 1) << (i * box));
        if (key0 + 64 > n_keys) {
          const int left = n_keys - key0;                              // keys of this half
          sees &= left <= 0 ? 0ull : (1ull << left) - 1;
        }
        if (sees != ~0ull) {                                           // (the same for all rows)
          const uint32_t lo = (uint32_t)sees, hi = (uint32_t)(sees >> 32);
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            if (!((lo >> i) & 1)) v[i] = 0xff800000u;
            if (!((hi >> i) & 1)) v[32 + i] = 0xff800000u;
          }
        }
        const uint64_t sc2 = pt_pk2(a.scale_log2, a.scale_log2);
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
            alpha = pa_ex2(m_used - m_new);
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
            LP_PT_TMEM_ST_16(o, o_addr + c * 16);
          }
          tmem_wait_st();
        }
        const float neg_m = m_used == -INFINITY ? 0.f : -m_used;
        const uint64_t nm2 = pt_pk2(neg_m, neg_m);
        uint64_t acc2 = pt_pk2(0.f, 0.f);
        const int tn = (t + 1) >> 1, hn = (t + 1) & 1;
        const bool has_next = t + 1 < 2 * mine;
        const bool s_ready = has_next && mbar_test_wait(&s_full[q * 2 + hn], (nt + tn) & 1);
        if (both) {                                                    // the streams' exponentials in turns: one's loads and stores run beside the other's
          if (q == 1) pt_bar_sync(5, 256);
          else if (t > 0) pt_bar_sync(4, 256);
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float x0, x1;
            pt_upk2(pt_fma2(pt_pk2(__uint_as_float(v[c * 32 + i]), __uint_as_float(v[c * 32 + i + 1])), sc2, nm2), x0, x1);
            const float p0 = pa_ex2(x0), p1 = pa_ex2(x1);
            acc2 = pt_add2(acc2, pt_pk2(p0, p1));
            pk[i >> 1] = pack_bf16x2(p0, p1);      // half a step is 2^-8 of a weight; their sum is taken in fp32 before
          }
          LP_PT_TMEM_ST_16(pk, s_addr + h * 64 + c * 16);
        }
        if (both) {
          if (q == 0) pt_bar_arrive(5, 256);
          else if (has_next) pt_bar_arrive(4, 256);
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
          pt_upk2(acc2, a0, a1);
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
        pt_bar_arrive(2, 256);
        ++pieces;
        ++joins;
        continue;
      }
      mbar_wait_warp(&o_done[q], pieces & 1);
      ++pieces;
      float f0 = 1.f, f1 = 0.f;
      if (two) {
        pt_bar_sync(2, 256);
        mbar_wait_warp(&o_done[1], joins & 1);
        ++joins;
        const float2 x = other[r];
        const float m = fmaxf(m_used, x.x);
        f0 = m_used == -INFINITY ? 1.f : pa_ex2(m_used - m);           // sums and values of a stream that saw nothing are zeros, or NaN
        f1 = x.x == -INFINITY ? 1.f : pa_ex2(x.x - m);
        l_sum = l_sum * f0 + x.y * f1;
        m_used = m;
      }
      tc_fence_after();
      const int in_block = (SPLIT ? 0 : q * 128) + r;
      const long long slot = (long long)p.item + blockIdx.x;
      float* part = a.pre_o + (slot * (DH / 4) * a.pre_rows + in_block) * 4;
      if (row_ok) a.pre_ml[slot * a.pre_rows + in_block] = make_float2(m_used, l_sum);
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
        if (row_ok) {
#pragma unroll
          for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(part + (c * 8 + i) * a.pre_rows * 4) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        }
      }
      tc_fence_before();
      if (two) pt_bar_arrive(3, 256);
    }
    if (SPLIT && q == 1 && joins > 0) pt_bar_sync(3, 256);             // (what stream 0 has arrived at)
  }
  tc_fence_before();
  __syncthreads();
  pdl_wait();                           // (begun beside the own rows' kernel; the join, which waits for this one, needs that one to be over too)
  if (warp == 3) {
    __syncwarp();
    tmem_dealloc(tmem_base, 512);
  }
}

// rows of a TMA box: a prefix of its own takes whole tiles, else the largest part of a tile that pages are multiples of
static int prefix_box(const lp_prefix_attn_desc* d) {
  if (!d->page_table) return 128;
  for (int box = 128; box >= 8; box /= 2)
    if (d->page_size % box == 0) return box;
  return 0;
}
bool prefix_tc_takes(const lp_prefix_attn_desc* d) {
  bool strides;
  if (d->page_table)
    strides = (d->n_pages == 1 || (d->k_page > 0 && d->v_page > 0)) && (d->page_size == 1 || (d->k_row > 0 && d->v_row > 0)) && (d->KVH == 1 || (d->k_head > 0 && d->v_head > 0));
  else
    strides = d->prefix_k && (d->prefix == 1 || (d->pk_row > 0 && d->pv_row > 0)) && (d->KVH == 1 || (d->pk_head > 0 && d->pv_head > 0));
  return d->prefix > 0 && prefix_box(d) != 0 && strides && d->scale > 0.f;      // (0 x -inf is not -inf)
}

template <int DH>
static int launch_tc(const PrefixTc& tc, cudaStream_t stream) {
  constexpr int NB = (DH + 63) / 64;
  const lp_prefix_attn_desc& d = tc.a.d;
  CUtensorMap tm[2];
  const bool paged = d.page_table != nullptr;
  const void* base[2] = {paged ? d.k : d.prefix_k, paged ? d.v : d.prefix_v};
  const long long page[2] = {d.k_page, d.v_page}, row[2] = {paged ? d.k_row : d.pk_row, paged ? d.v_row : d.pv_row}, head[2] = {paged ? d.k_head : d.pk_head, paged ? d.v_head : d.pv_head};
  const uint32_t box[4] = {64, 1, (uint32_t)tc.box, 1};
  const int n_rows = paged ? d.page_size : d.prefix, n_pages = paged ? d.n_pages : 1;
  for (int i = 0; i < 2; ++i) {      // of a dimension of one the distance is any
    const uint64_t dims[4] = {(uint64_t)d.D, (uint64_t)d.KVH, (uint64_t)n_rows, (uint64_t)n_pages};
    const uint64_t strides[3] = {d.KVH == 1 ? (uint64_t)d.D : (uint64_t)head[i], n_rows == 1 ? (uint64_t)d.D : (uint64_t)row[i], n_pages == 1 ? (uint64_t)d.D : (uint64_t)page[i]};
    if (const int rc = make_tmap_bf16_4d(&tm[i], base[i], dims, strides, box)) return rc;
  }
  const bool split = tc.a.pre_rows == 128;
  const size_t smem = (split ? 7 : 6) * NB * PT_BOX + PT_BARS + (split ? 128 * 8 : 0) + (size_t)(d.B + 1) * 4 + 1024;
  if (split) {
    LP_CHECK_CUDA((allow_smem<prefix_tc_kernel<DH, true>>((int)smem)));
    LP_CHECK_CUDA(launch_ex(prefix_tc_kernel<DH, true>, dim3(tc.a.pre_ctas), dim3(PT_THREADS), smem, stream, 1, true, tm[0], tm[1], tc));
  } else {
    LP_CHECK_CUDA((allow_smem<prefix_tc_kernel<DH, false>>((int)smem)));
    LP_CHECK_CUDA(launch_ex(prefix_tc_kernel<DH, false>, dim3(tc.a.pre_ctas), dim3(PT_THREADS), smem, stream, 1, true, tm[0], tm[1], tc));
  }
  return 0;
}

int launch_prefix_tc(const PrefixArgs& a, cudaStream_t stream) {
  PrefixTc tc;
  tc.a = a;
  tc.box = prefix_box(&a.d);
  if (a.d.D == 128) return launch_tc<128>(tc, stream);
  if (a.d.D == 96) return launch_tc<96>(tc, stream);
  return launch_tc<64>(tc, stream);
}

}  // namespace lp
