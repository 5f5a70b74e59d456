// Test infrastructure: the tcgen05 kernel of the tree attention (leopard_b200/csrc/lp_treeattn_tc.cu, tree_tc_kernel: a persistent CTA that walks pieces of items, rings of
// keys and values by TMA from a cache's pages) run on the CPU under tests/emu/tc_emu.h.  `tree_shared.inc` (lp_treeattn.cuh) and `tree_tc_kernel.inc` are cut from the sources by
// the test; the file's inline-PTX helpers (tt_*) are restated here.
#include "tc_emu.h"
#include "emu_helpers.inc"
#include "leopard_b200.h"

namespace lp {
inline uint64_t warp_words[64][32];
template <typename T>
inline T emu_shuffle(T v, int from) {
  const unsigned t = emu::linear_tid(), w = t >> 5, l = t & 31;
  std::memcpy(&warp_words[w][l], &v, sizeof(T));
  __syncwarp();
  T r;
  std::memcpy(&r, &warp_words[w][from < 0 || from > 31 ? (int)l : from], sizeof(T));
  __syncwarp();
  return r;
}
template <typename T>
inline T emu_shfl(unsigned, T v, int lane) { return emu_shuffle(v, lane); }
template <typename T>
inline T __shfl_up_sync(unsigned, T v, int d) { return emu_shuffle(v, (int)(emu::linear_tid() & 31) - d); }
inline long long __shfl_xor_sync(unsigned, long long v, int m) { return emu_shuffle(v, (int)(emu::linear_tid() & 31) ^ m); }
inline unsigned __ballot_sync(unsigned, bool p) {
  unsigned bits = 0;
  const unsigned t = emu::linear_tid(), w = t >> 5, l = t & 31;
  warp_words[w][l] = p;
  __syncwarp();
  for (int i = 0; i < 32; ++i) bits |= (unsigned)(warp_words[w][i] != 0) << i;
  __syncwarp();
  return bits;
}
inline unsigned __reduce_add_sync(unsigned, unsigned v) {
  for (int m = 1; m < 32; m <<= 1) v += emu_shuffle(v, (int)(emu::linear_tid() & 31) ^ m);
  return v;
}
inline bool __all_sync(unsigned m, bool p) { return __ballot_sync(m, p) == 0xffffffffu; }
#define __shfl_sync emu_shfl
inline float __bfloat162float(bf16 v) { return (float)v; }
inline bool not_finite(float v) { return !(fabsf(v) <= 3.402823466e38f); }
inline float ta_ex2(float x) { return exp2f(x); }
struct Map4 : CUtensorMap { uint64_t d3, s3; };
inline const CUtensorMap* g_fourth[2];
inline void tma_load_4d(void* dst, const Map4* m, uint64_t* bar, int c0, int c1, int c2, int c3) {
  // (dims: column, head, row of a page, page); a box is 64 columns x box[2] rows
  for (uint32_t r = 0; r < m->box[2]; ++r)
    for (uint32_t e = 0; e < 64; ++e) {
      const long col = (long)c0 + e, row = (long)c2 + r;
      uint16_t v = 0;
      if (col >= 0 && (uint64_t)col < m->dims[0] && c1 >= 0 && (uint64_t)c1 < m->dims[1] && row >= 0 && (uint64_t)row < m->dims[2] && c3 >= 0 && (uint64_t)c3 < m->d3)
        std::memcpy(&v, m->base + col * 2 + (uint64_t)c1 * m->strides[0] + row * m->strides[1] + (uint64_t)c3 * m->s3, 2);
      std::memcpy(emu_tc::cta().smem + emu_tc::swz(smem_u32(dst) + r * 128 + e * 2, 128), &v, 2);
    }
  mbar_complete_tx_addr(smem_u32(bar), 64 * m->box[2] * 2);
}
#define __align__(n) alignas(n)
#include "tree_shared.inc"
constexpr int TT_BOX = 128 * 128, TT_THREADS = 384, TT_KEYS = 128;
inline uint64_t tt_pk2(float a, float b) { return (uint64_t)__float_as_uint(a) | ((uint64_t)__float_as_uint(b) << 32); }
inline void tt_upk2(uint64_t r, float& a, float& b) { a = __uint_as_float((uint32_t)r); b = __uint_as_float((uint32_t)(r >> 32)); }
inline uint64_t tt_fma2(uint64_t a, uint64_t b, uint64_t c) {
  float a0, a1, b0, b1, c0, c1;
  tt_upk2(a, a0, a1); tt_upk2(b, b0, b1); tt_upk2(c, c0, c1);
  return tt_pk2(fmaf(a0, b0, c0), fmaf(a1, b1, c1));
}
inline uint64_t tt_add2(uint64_t a, uint64_t b) {
  float a0, a1, b0, b1;
  tt_upk2(a, a0, a1); tt_upk2(b, b0, b1);
  return tt_pk2(a0 + b0, a1 + b1);
}
inline void tt_bar_sync(int id, int n) { named_bar(id, n, true); }
inline void tt_bar_arrive(int id, int n) { named_bar(id, n, false); }
#define LP_TT_TMEM_ST_16(regs, taddr) lp::tmem_st(regs, taddr, 16)
#define CUtensorMap Map4
#include "tree_tc_kernel.inc"
#undef CUtensorMap
}  // namespace lp

using namespace lp;

extern "C" void emu_tree_tc(const lp_tree_attn_desc* d, int ctas, int rows, int box, int split, float* part_o, float* part_ml) {
  TreeTc tc;
  tc.a.d = *d;
  tc.a.group = d->H / d->KVH;
  tc.a.rows = rows;
  for (tc.a.row_bits = 0; 1 << tc.a.row_bits < rows;) ++tc.a.row_bits;
  tc.a.key_bits = 7;
  tc.a.scale_log2 = d->scale * 1.4426950408889634f;
  tc.a.part_o = part_o;
  tc.a.part_ml = reinterpret_cast<float2*>(part_ml);
  tc.a.ctas = ctas;
  tc.box = box;
  Map4 tm[2];
  const void* base[2] = {d->k, d->v};
  const long long page[2] = {d->k_page, d->v_page}, row[2] = {d->k_row, d->v_row}, head[2] = {d->k_head, d->v_head};
  for (int i = 0; i < 2; ++i) {
    tm[i].base = reinterpret_cast<const uint8_t*>(base[i]);
    tm[i].dims[0] = d->D; tm[i].dims[1] = d->KVH; tm[i].dims[2] = d->page_size; tm[i].d3 = d->n_pages;
    tm[i].strides[0] = head[i] * 2; tm[i].strides[1] = row[i] * 2; tm[i].s3 = page[i] * 2;
    tm[i].box[0] = 64; tm[i].box[1] = 1; tm[i].box[2] = box;
  }
  emu::g_block_hook = [] { emu_tc::reset(); };
  emu::launch(dim3(ctas), dim3(TT_THREADS), [&] {
    if (split) {
      if (d->D == 128) tree_tc_kernel<128, true>(tm[0], tm[1], tc);
      else if (d->D == 96) tree_tc_kernel<96, true>(tm[0], tm[1], tc);
      else tree_tc_kernel<64, true>(tm[0], tm[1], tc);
    } else {
      if (d->D == 128) tree_tc_kernel<128, false>(tm[0], tm[1], tc);
      else if (d->D == 96) tree_tc_kernel<96, false>(tm[0], tm[1], tc);
      else tree_tc_kernel<64, false>(tm[0], tm[1], tc);
    }
  });
  emu::g_block_hook = nullptr;
}
