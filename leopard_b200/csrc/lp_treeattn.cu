// leopard_b200 — attention of a tree of drafted tokens over a cache (one step of speculative decoding; a single token is a tree of one node).
//
//   out[i, h] = sum_j softmax_j(scale q[i, h] . k[j, g]) v[j, g],   j < len (every cached row) or j = len + n with node n in node i's mask
//
// The T nodes and the G = H / KVH query heads of a key head are the rows of one product, row r = i G + g, so that a key is read once for all of them.  This file has the
// entry point, the kernel for few rows and any cache (mma.sync), and the one that joins the pieces; lp_treeattn_tc.cu has the kernel for many rows (tcgen05).
#include "lp_treeattn.cuh"

namespace lp {

constexpr int TA_KEYS = 64;               // keys of a tile
constexpr int TA_STAGES = 3;
constexpr int TA_RING = TA_STAGES + 1;    // tiles whose rows' places are known
constexpr int TA_MAX_BATCH = 2048;        // the line of the sequences is in shared memory

__device__ __forceinline__ void ta_ldmatrix(uint32_t* r, const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_u32(p)) : "memory");
}
__device__ __forceinline__ void ta_ldmatrix_t(uint32_t* r, const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_u32(p)) : "memory");
}
// 16 bytes into shared memory, zeros where the row is not there
__device__ __forceinline__ void ta_copy16(void* dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ta_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void ta_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// WM x WN warps: 16 WM rows, the 64 keys of a tile dealt to WN warps.  Two CTAs an SM, each with three stages of keys and values on their way.  Bound by HBM for long caches: one node
// of 64 sequences of 4,000 rows, 32 heads over 8, 188 us, 5.6 TB/s; of one after 100,000 rows 87, 4.7.  Short ones by latency: one node after 512 rows 9.3 us.  Many short ones by the ends
// of pieces: one node of 64 sequences of 512 rows, 512 items of 9 tiles on 296 CTAs, 44 us where their bytes take 21.
template <int D, int WM, int WN>
__global__ void __launch_bounds__(32 * WM * WN, 2)
tree_attn_kernel(const __grid_constant__ TreeArgs a) {
  constexpr int NT = 32 * WM * WN, R = 16 * WM, NK = TA_KEYS / WN, LD = D + 8;      // rows 16 bytes further apart than their length: no bank conflicts
  constexpr int CH = D / 8;                                                         // 16-byte pieces of a row
  extern __shared__ __align__(16) unsigned char ta_smem[];
  bf16* tiles = reinterpret_cast<bf16*>(ta_smem);                                   // [stage][K, V][64][LD]
  int2* place = reinterpret_cast<int2*>(tiles + TA_STAGES * 2 * TA_KEYS * LD);      // [ring][64]: page (-1: not there) and row in it
  uint32_t* present = reinterpret_cast<uint32_t*>(place + TA_RING * TA_KEYS);       // [ring][2]
  float2* ml = reinterpret_cast<float2*>(present + TA_RING * 2);                    // [WN][R]
  TreeLine* line = reinterpret_cast<TreeLine*>(ml + WN * R);                        // [B + 1]
  constexpr int LDO = D + 4;
  float* obuf = reinterpret_cast<float*>(ta_smem);                                  // [R][LDO], when the tiles are done with
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, wm = warp % WM, wn = warp / WM, g = lane >> 2, t4 = lane & 3;
  pdl_launch_dependents();
  tree_line(a, line);
  long long u, u_end;
  tree_range(a, line, blockIdx.x, u, u_end);

  while (u < u_end) {
    const int b = tree_find(line, a.d.B, u);
    const TreeSeq s = tree_seq(a, line[b].len, line[b].n);
    const long long local = u - line[b].first;
    const int item = (int)tree_div(local, s.tiles), t0 = (int)(local - (long long)item * s.tiles), t1 = (int)min((long long)s.tiles, t0 + (u_end - u));
    const int kvh = tree_div32(item, s.blocks), r0 = (item - kvh * s.blocks) * R;
    u += t1 - t0;
    const int n_rows = min(R, s.n * a.group - r0);
    const bf16* kb = reinterpret_cast<const bf16*>(a.d.k) + kvh * a.d.k_head;
    const bf16* vb = reinterpret_cast<const bf16*>(a.d.v) + kvh * a.d.v_head;
    const int* table = a.d.page_table ? a.d.page_table + b * a.d.ld_table : nullptr;

    auto locate = [&](int i) {                 // where the rows of the i-th tile of this piece lie
      if (tid < TA_KEYS) {
        const long long key = (long long)(t0 + i) * TA_KEYS + tid;
        int2 p = make_int2(-1, 0);
        if (key < s.keys) {
          const int logical = tree_div32((int)key, a.d.page_size);
          p.x = table ? table[logical] : b;
          p.y = (int)key - logical * a.d.page_size;
          if (p.x >= a.d.n_pages) p.x = -1;
        }
        place[(i % TA_RING) * TA_KEYS + tid] = p;
        const unsigned bits = __ballot_sync(0xffffffffu, p.x >= 0);
        if (lane == 0) present[(i % TA_RING) * 2 + warp] = bits;
      }
    };
    auto fetch = [&](int i) {
      bf16* kt = tiles + (i % TA_STAGES) * 2 * TA_KEYS * LD;
      bf16* vt = kt + TA_KEYS * LD;
#pragma unroll
      for (int c = tid; c < TA_KEYS * CH; c += NT) {
        const int row = c / CH, col = (c % CH) * 8;
        const int2 p = place[(i % TA_RING) * TA_KEYS + row];
        const bool there = p.x >= 0;
        const long long page = there ? p.x : 0, in = there ? p.y : 0;
        ta_copy16(kt + row * LD + col, kb + page * a.d.k_page + in * a.d.k_row + col, there);
        ta_copy16(vt + row * LD + col, vb + page * a.d.v_page + in * a.d.v_row + col, there);
      }
    };
    const int n = t1 - t0;
#pragma unroll
    for (int i = 0; i < TA_STAGES; ++i)
      if (i < n) locate(i);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TA_STAGES - 1; ++i) {
      if (i < n) fetch(i);
      ta_commit();
    }
    // this thread's two rows: their queries as the product's first operand, their nodes' masks
    uint32_t qa[D / 16][4];
    const unsigned long long* words[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = r0 + wm * 16 + g + 8 * h;
      const bool there = r < s.n * a.group;
      const int node = there ? tree_div32(r, a.group) : 0, head = kvh * a.group + (there ? r - node * a.group : 0);
      const bf16* q = reinterpret_cast<const bf16*>(a.d.q) + b * a.d.q_batch + node * a.d.q_node + head * a.d.q_head;
      words[h] = a.d.mask + b * a.d.mask_batch + node * a.d.mask_node;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        qa[k][h] = there ? *reinterpret_cast<const uint32_t*>(q + k * 16 + 2 * t4) : 0u;
        qa[k][2 + h] = there ? *reinterpret_cast<const uint32_t*>(q + k * 16 + 8 + 2 * t4) : 0u;
      }
    }
    float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) o[i][k] = 0.f;

    for (int i = 0; i < n; ++i) {
      ta_wait<TA_STAGES - 2>();
      __syncthreads();
      if (i + TA_STAGES - 1 < n) fetch(i + TA_STAGES - 1);
      ta_commit();
      if (i + TA_STAGES < n) locate(i + TA_STAGES);
      const bf16* kt = tiles + (i % TA_STAGES) * 2 * TA_KEYS * LD + wn * NK * LD;
      const bf16* vt = kt + TA_KEYS * LD;
      float sc[NK / 8][4];
#pragma unroll
      for (int j = 0; j < NK / 8; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) sc[j][k] = 0.f;
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
#pragma unroll
        for (int j = 0; j < NK / 16; ++j) {
          uint32_t f[4];
          ta_ldmatrix(f, kt + (j * 16 + (lane & 7) + (lane >> 4) * 8) * LD + k * 16 + ((lane >> 3) & 1) * 8);
          mma_bf16(sc[2 * j], qa[k][0], qa[k][1], qa[k][2], qa[k][3], f[0], f[1]);
          mma_bf16(sc[2 * j + 1], qa[k][0], qa[k][1], qa[k][2], qa[k][3], f[2], f[3]);
        }
#pragma unroll
      for (int j = 0; j < NK / 8; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) sc[j][k] *= a.scale_log2;
      // which keys a row sees; tiles of cached rows that are all there need no look
      const long long key0 = (long long)(t0 + i) * TA_KEYS;
      const unsigned long long there = present[(i % TA_RING) * 2] | ((unsigned long long)present[(i % TA_RING) * 2 + 1] << 32);
      const bool tail = key0 + TA_KEYS > s.len;
      unsigned long long sees[2] = {there, there};
      if (tail || there != ~0ull) {
        if (tail) {
          const long long j0 = key0 - s.len;             // the node of the tile's first key, negative while it is a cached row
          const int nw = (a.d.T + 63) >> 6;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            unsigned long long bits;
            if (j0 < 0) bits = (words[h][0] << (int)-j0) | ((1ull << (int)-j0) - 1);      // -64 < j0
            else {
              const int w = (int)(j0 >> 6), sh = (int)(j0 & 63);
              bits = w < nw ? words[h][w] >> sh : 0ull;
              if (sh && w + 1 < nw) bits |= words[h][w + 1] << (64 - sh);
            }
            sees[h] &= bits;
          }
        }
#pragma unroll
        for (int j = 0; j < NK / 8; ++j)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (!((sees[k >> 1] >> (wn * NK + j * 8 + 2 * t4 + (k & 1))) & 1)) sc[j][k] = -INFINITY;
      }
      float mx[2] = {m[0], m[1]};
#pragma unroll
      for (int j = 0; j < NK / 8; ++j) {
        mx[0] = fmaxf(mx[0], fmaxf(sc[j][0], sc[j][1]));
        mx[1] = fmaxf(mx[1], fmaxf(sc[j][2], sc[j][3]));
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
        const float ref = mx[h] == -INFINITY ? 0.f : mx[h], f = ta_ex2(m[h] - ref);
        m[h] = mx[h];
        l[h] *= f;
#pragma unroll
        for (int d = 0; d < D / 8; ++d) {
          o[d][2 * h] *= f;
          o[d][2 * h + 1] *= f;
        }
#pragma unroll
        for (int j = 0; j < NK / 8; ++j) {
          sc[j][2 * h] = ta_ex2(sc[j][2 * h] - ref);
          sc[j][2 * h + 1] = ta_ex2(sc[j][2 * h + 1] - ref);
          l[h] += sc[j][2 * h] + sc[j][2 * h + 1];
        }
      }
      // the weights go into the second product as bf16 (half a step is 2^-8 of a weight); their sum was taken before
      bool odd = false;
#pragma unroll
      for (int j = 0; j < NK / 16; ++j) {
        const uint32_t p0 = pack_bf16x2(sc[2 * j][0], sc[2 * j][1]), p1 = pack_bf16x2(sc[2 * j][2], sc[2 * j][3]);
        const uint32_t p2 = pack_bf16x2(sc[2 * j + 1][0], sc[2 * j + 1][1]), p3 = pack_bf16x2(sc[2 * j + 1][2], sc[2 * j + 1][3]);
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          uint32_t f[4];
          ta_ldmatrix_t(f, vt + (j * 16 + (lane & 15)) * LD + d * 16 + (lane >> 4) * 8);
          if (tail) {                                    // 0 x NaN: values that are not finite are left out of the product ...
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if ((f[k] & 0x7f80u) == 0x7f80u) { f[k] &= 0xffff0000u; odd = true; }
              if ((f[k] & 0x7f800000u) == 0x7f800000u) { f[k] &= 0xffffu; odd = true; }
            }
          }
          mma_bf16(o[2 * d], p0, p1, p2, p3, f[0], f[1]);
          mma_bf16(o[2 * d + 1], p0, p1, p2, p3, f[2], f[3]);
        }
      }
      if (tail && __any_sync(0xffffffffu, odd)) {        // ... and reach the rows that see them
        for (int key = 0; key < NK; ++key)
#pragma unroll
          for (int d = 0; d < D / 8; ++d)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const float v = __bfloat162float(vt[key * LD + d * 8 + 2 * t4 + k]);
              if (not_finite(v)) {
                if ((sees[0] >> (wn * NK + key)) & 1) o[d][k] += v;
                if ((sees[1] >> (wn * NK + key)) & 1) o[d][2 + k] += v;
              }
            }
      }
    }
    ta_wait<0>();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      if (t4 == 0) ml[wn * R + wm * 16 + g + 8 * h] = make_float2(m[h], l[h]);
    }
    __syncthreads();                                     // the tiles are done with: their place takes the rows' values
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = wm * 16 + g + 8 * h;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < WN; ++w) top = fmaxf(top, ml[w * R + r].x);
      const float f = m[h] == -INFINITY ? 1.f : ta_ex2(m[h] - top);
#pragma unroll
      for (int w = 0; w < WN; ++w) {
        if (w == wn)
#pragma unroll
          for (int d = 0; d < D / 8; ++d)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              float* at = obuf + r * LDO + d * 8 + 2 * t4 + k;
              *at = w == 0 ? o[d][2 * h + k] * f : *at + o[d][2 * h + k] * f;
            }
        if (WN > 1) __syncthreads();
      }
    }
    if (WN == 1) __syncthreads();
    const bool whole = t0 == 0 && t1 == s.tiles;
    const long long slot = 2LL * blockIdx.x + (t0 == 0 ? 1 : 0);
    auto row_ml = [&](int r) {                             // of all warps' keys
      float2 x = make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int w = 0; w < WN; ++w) x.x = fmaxf(x.x, ml[w * R + r].x);
#pragma unroll
      for (int w = 0; w < WN; ++w) x.y += ml[w * R + r].y * (ml[w * R + r].x == -INFINITY ? 1.f : ta_ex2(ml[w * R + r].x - x.x));
      return x;
    };
    if (whole) {
      for (int c = tid; c < n_rows * (D / 4); c += NT) {
        const int r = c / (D / 4), col = (c % (D / 4)) * 4;
        const float4 x = *reinterpret_cast<const float4*>(obuf + r * LDO + col);
        const float sum = row_ml(r).y, inv = sum == 0.f ? 0.f : 1.f / sum;
        bf16* out = reinterpret_cast<bf16*>(a.d.out) + b * a.d.o_batch + ((r0 + r) / a.group) * a.d.o_node + (kvh * a.group + (r0 + r) % a.group) * a.d.o_head;
        *reinterpret_cast<uint2*>(out + col) = make_uint2(pack_bf16x2(x.x * inv, x.y * inv), pack_bf16x2(x.z * inv, x.w * inv));
      }
    } else {
      for (int c = tid; c < R * (D / 4); c += NT) {
        const int r = c % R, c4 = c / R;
        if (r >= n_rows) continue;
        *reinterpret_cast<float4*>(a.part_o + ((slot * (D / 4) + c4) * R + r) * 4) = *reinterpret_cast<const float4*>(obuf + r * LDO + c4 * 4);
        if (c4 == 0) a.part_ml[slot * R + r] = row_ml(r);
      }
    }
    __syncthreads();
  }
}

// Rows whose tiles lie in several CTAs: a CTA joins groups of 8 rows of a key head, a thread four columns of a row over all pieces.  Bound by latency: ten pieces of a group, two
// of each of four or five of each of two are under way at once; weights follow a running maximum, so that each is read once.  A CTA takes 1 to 2 us for the line of tiles before it can
// join.  Few CTAs have done so when the pieces' kernel ends; of more than run at once (8 an SM) each takes four groups (64 nodes of 48 sequences of 1,000 rows 122 us in all, 161
// with one; 26 nodes of 6 sequences, 624 CTAs with one group, 44.8 with one and 50.9 with four).  Each CTA's line has all sequences, so the cost grows with the square of the batch: one
// node after 64 rows of 64 sequences 20 us, of 256 76, of 512 258, of 1,024 612, of 2,048 1,617 (their bytes take 3, 11, 22, 45 and 90).
constexpr int TA_JOIN_ROWS = 8, TA_JOIN_GROUPS = 4;
template <int N>
struct TreeN { static constexpr int value = N; };
struct TreeSum {
  float top = -INFINITY, sum = 0.f;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  template <int N>
  __device__ __forceinline__ void add(const float2* p, const float4* y) {
    float m = top;
#pragma unroll
    for (int k = 0; k < N; ++k) m = fmaxf(m, p[k].x);
    const float old = top == -INFINITY ? 1.f : ta_ex2(top - m);      // sums and values of pieces that saw nothing are zeros, or NaN
    top = m;
    sum *= old;
    x.x *= old; x.y *= old; x.z *= old; x.w *= old;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float f = p[k].x == -INFINITY ? 1.f : ta_ex2(p[k].x - m);
      sum += p[k].y * f;
      x.x += y[k].x * f; x.y += y[k].y * f; x.z += y[k].z * f; x.w += y[k].w * f;
    }
  }
  __device__ __forceinline__ uint2 result() const {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    return make_uint2(pack_bf16x2(x.x * inv, x.y * inv), pack_bf16x2(x.z * inv, x.w * inv));
  }
};
template <int D, int GROUPS>
__global__ void __launch_bounds__(TA_JOIN_ROWS * D / 4)
tree_join_kernel(const __grid_constant__ TreeArgs a) {
  extern __shared__ TreeLine join_line[];
  __shared__ __align__(16) bf16 done[GROUPS * TA_JOIN_ROWS][D + 8];
  const int b = blockIdx.z, kvh = blockIdx.y, row0 = blockIdx.x * TA_JOIN_ROWS * GROUPS, in = threadIdx.x % TA_JOIN_ROWS, c4 = threadIdx.x / TA_JOIN_ROWS;
  tree_line(a, join_line);
  const TreeSeq s = tree_seq(a, join_line[b].len, join_line[b].n);
  const int rows = min(s.n * a.group, row0 + TA_JOIN_ROWS * GROUPS);
  const int blk = row0 >> a.row_bits, r0 = row0 - (blk << a.row_bits) + in;      // (blocks are multiples of a CTA's rows, or there is one)
  int c0 = 0, c1 = 0;
  if (row0 < rows) tree_ctas_of(a, join_line, b, s, kvh * s.blocks + blk, c0, c1);
  if (c0 != c1 || blockIdx.x + blockIdx.y + blockIdx.z == 0) pdl_wait();      // (the first in any case: the join may not be over before the pieces' kernel is)
  if (c0 == c1) return;                                  // nothing, or written whole
  auto load = [&](int row, int c, float2& p, float4& y) {
    const bool on = row + in < rows && c <= c1;
    const long long slot = 2LL * c + (c == c0 ? 1 : 0);  // the first piece begins with the item, the others begin inside it
    const int r = r0 + row - row0;
    p = on ? a.part_ml[slot * a.rows + r] : make_float2(-INFINITY, 0.f);
    y = on ? *reinterpret_cast<const float4*>(a.part_o + ((slot * (D / 4) + c4) * a.rows + r) * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
  };
  auto join = [&](auto groups, auto pieces) {             // so many at once
    constexpr int NG = decltype(groups)::value, NP = decltype(pieces)::value;
    for (int row = row0; row < rows; row += NG * TA_JOIN_ROWS) {
      TreeSum t[NG];
      for (int c = c0; c <= c1; c += NP) {
        float2 p[NG][NP];
        float4 y[NG][NP];
#pragma unroll
        for (int i = 0; i < NG; ++i)
#pragma unroll
          for (int k = 0; k < NP; ++k) load(row + i * TA_JOIN_ROWS, c + k, p[i][k], y[i][k]);
#pragma unroll
        for (int i = 0; i < NG; ++i) t[i].template add<NP>(p[i], y[i]);
      }
#pragma unroll
      for (int i = 0; i < NG; ++i) *reinterpret_cast<uint2*>(&done[row - row0 + i * TA_JOIN_ROWS + in][c4 * 4]) = t[i].result();
    }
  };
  if constexpr (GROUPS == 1) join(TreeN<1>(), TreeN<10>());
  else if (c1 - c0 < 2) join(TreeN<4>(), TreeN<2>());
  else join(TreeN<2>(), TreeN<5>());
  __syncthreads();
  for (int i = threadIdx.x; i < (rows - row0) * (D / 8); i += TA_JOIN_ROWS * D / 4) {
    const int row = row0 + i / (D / 8), col = (i % (D / 8)) * 8;
    bf16* out = reinterpret_cast<bf16*>(a.d.out) + b * a.d.o_batch + (row / a.group) * a.d.o_node + (kvh * a.group + row % a.group) * a.d.o_head;
    *reinterpret_cast<uint4*>(out + col) = *reinterpret_cast<const uint4*>(&done[row - row0][col]);
  }
}

// ---- host ----------------------------------------------------------------------------------------------------------
// which kernel: tcgen05 for more rows than TREE_TC_ROWS where it takes the cache.  mma.sync and tcgen05 (us, 32 heads over 8, nodes x 4 rows), of one sequence of 512 rows, one of 20,000, 8 of
// 1,000, 8 of 4,000, 48 of 1,000, 48 of 4,000: 16 rows 9.3 and 12.6, 27.1 and 27.2, 18.5 and 21.4, 38 and 46, 57 and 74, 153 and 174; 32 rows 9.9 and 12.7, 34.2 and 27.7, 20.3 and 21.7,
// 44.5 and 45.5, 64 and 74, 184 and 175; 36 rows 11.3 and 12.9, 43.5 and 28.3, 25.9 and 22.0, 63 and 46, 96 and 76, 272 and 178; 128 rows 12.1 and 13.6, 67 and 29, 47 and 31, 110 and 55, 188 and
// 94, 525 and 189.  At 32 rows length decides as much as rows do: the rule loses a fifth after 20,000 rows and a twentieth at 48 of 4,000, and wins up to a seventh at the others.
constexpr int TREE_TC_ROWS = 32;
static bool tree_tc(const lp_tree_attn_desc* d) { return (long long)d->T * (d->H / d->KVH) > TREE_TC_ROWS && tree_tc_takes(d); }
// rows of a block: what the widest tree needs, 64 (256) at most
static int tree_rows(const lp_tree_attn_desc* d) {
  const long long rows = (long long)d->T * (d->H / d->KVH);
  if (tree_tc(d)) return rows <= 128 ? 128 : 256;
  return rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
}
static int tree_keys(const lp_tree_attn_desc* d) { return tree_tc(d) ? 128 : TA_KEYS; }
// two CTAs on each SM (tcgen05: one), no more than there can be tiles
static int tree_ctas(const lp_tree_attn_desc* d) {
  const int R = tree_rows(d), keys = tree_keys(d);
  const long long blocks = ((long long)d->T * (d->H / d->KVH) + R - 1) / R;
  const long long tiles = ((long long)d->max_pages * d->page_size + keys - 1) / keys;
  const long long most = (tree_tc(d) ? 1LL : 2LL) * sm_count();
  if (tiles > most || blocks > most) return (int)most;
  const long long all = tiles * blocks * d->KVH;
  return (int)(all > most / d->B ? most : all * d->B);
}
static size_t tree_smem(int D, int wm, int wn, int B) {
  return (size_t)TA_STAGES * 2 * TA_KEYS * (D + 8) * 2 + TA_RING * TA_KEYS * 8 + TA_RING * 8 + (size_t)wn * wm * 16 * 8 + (size_t)(B + 1) * sizeof(TreeLine);
}
static int tree_check(const lp_tree_attn_desc* d) {
  LP_REQUIRE(d != nullptr, "lp_tree_attention: null descriptor");
  LP_REQUIRE(d->B > 0 && d->B <= TA_MAX_BATCH && d->T > 0 && d->T <= LP_TREE_MAX_NODES, "lp_tree_attention: B=%d (1 to %d), T=%d (1 to %d)", d->B, TA_MAX_BATCH, d->T,
             LP_TREE_MAX_NODES);
  LP_REQUIRE(d->KVH > 0 && d->KVH <= 65535 && d->H >= d->KVH && d->H % d->KVH == 0 && d->H <= 65535, "lp_tree_attention: %d query heads over %d key heads", d->H, d->KVH);
  LP_REQUIRE(d->D == 64 || d->D == 96 || d->D == 128, "lp_tree_attention: heads of %d are not built (64, 96, 128)", d->D);
  LP_REQUIRE(d->n_pages > 0 && d->page_size > 0 && d->max_pages > 0, "lp_tree_attention: %d pages of %d rows, %d a sequence", d->n_pages, d->page_size, d->max_pages);
  LP_REQUIRE((long long)d->max_pages * d->page_size <= (1LL << 31) - 128 /* a row's place, and the end of its tile, in 32 bits */, "lp_tree_attention: %d pages of %d rows are too many", d->max_pages, d->page_size);
  return 0;
}

}  // namespace lp

extern "C" size_t lp_tree_attention_workspace_bytes(const lp_tree_attn_desc* d) {
  using namespace lp;
  if (tree_check(d) != 0) return 0;
  return (size_t)2 * tree_ctas(d) * tree_rows(d) * (d->D * 4 + 8);
}

extern "C" int lp_tree_attention(const lp_tree_attn_desc* d, void* workspace, size_t ws_bytes, void* stream_) {
  using namespace lp;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  if (const int rc = tree_check(d)) return rc;
  LP_REQUIRE(d->q && d->k && d->v && d->out && d->lengths && d->mask && workspace, "lp_tree_attention: null argument");
  LP_REQUIRE(d->page_table ? d->ld_table >= d->max_pages : (d->max_pages == 1 && d->B <= d->n_pages),
             "lp_tree_attention: %d sequences of %d pages: ld_table %lld, %d pages there", d->B, d->max_pages, d->ld_table, d->n_pages);
  TreeArgs a;
  a.d = *d;
  d = &a.d;                               // of a dimension of one any stride may have come
  if (d->B == 1) a.d.q_batch = a.d.o_batch = a.d.mask_batch = a.d.ld_table = 0;
  if (d->T == 1) a.d.q_node = a.d.o_node = a.d.mask_node = 0;
  if (d->H == 1) a.d.q_head = a.d.o_head = 0;
  if (d->n_pages == 1) a.d.k_page = a.d.v_page = 0;
  if (d->page_size == 1) a.d.k_row = a.d.v_row = 0;
  if (d->KVH == 1) a.d.k_head = a.d.v_head = 0;
  const long long strides = d->q_batch | d->q_node | d->q_head | d->k_page | d->k_row | d->k_head | d->v_page | d->v_row | d->v_head | d->o_batch | d->o_node | d->o_head;
  const uintptr_t bases = reinterpret_cast<uintptr_t>(d->q) | reinterpret_cast<uintptr_t>(d->k) | reinterpret_cast<uintptr_t>(d->v) |
                          reinterpret_cast<uintptr_t>(d->out) | reinterpret_cast<uintptr_t>(workspace);
  LP_REQUIRE(strides % 8 == 0 && bases % 16 == 0, "lp_tree_attention: strides in multiples of 8 elements, 16-byte aligned bases");
  Dim places[3] = {{d->B, d->o_batch}, {d->T, d->o_node}, {d->H, d->o_head}};
  LP_REQUIRE(strides_nest(places, 3, d->D), "lp_tree_attention: rows of out share their memory (strides %lld, %lld, %lld)", d->o_batch, d->o_node, d->o_head);
  LP_REQUIRE(ws_bytes >= lp_tree_attention_workspace_bytes(d), "lp_tree_attention: workspace too small");
  a.group = d->H / d->KVH;
  a.rows = tree_rows(d);
  for (a.row_bits = 0; 1 << a.row_bits < a.rows;) ++a.row_bits;
  a.key_bits = tree_keys(d) == 128 ? 7 : 6;
  a.scale_log2 = d->scale * 1.4426950408889634f;
  a.ctas = tree_ctas(d);
  a.part_o = reinterpret_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + (size_t)2 * a.ctas * a.rows * d->D);
  const bool tc = tree_tc(d);
  const int wm = tc ? 1 : a.rows / 16, wn = 4 / wm;
  const size_t smem = tree_smem(d->D, wm, wn, d->B), line = (size_t)(d->B + 1) * sizeof(TreeLine);
  dim3 join((unsigned)(((long long)d->T * a.group + TA_JOIN_ROWS - 1) / TA_JOIN_ROWS), d->KVH, d->B);
  const int groups = (long long)join.x * join.y * join.z <= 8LL * sm_count() ? 1 : TA_JOIN_GROUPS;
  join.x = (join.x + groups - 1) / groups;
  note_launch(2);
#define LP_TREE(DD, WM, WN)                                                                                                                    \
  {                                                                                                                                            \
    LP_CHECK_CUDA((allow_smem<tree_attn_kernel<DD, WM, WN>>((int)smem)));                                                                      \
    tree_attn_kernel<DD, WM, WN><<<a.ctas, 128, smem, stream>>>(a);                                                                            \
  }
#define LP_JOIN(DD, GG)                                                                                                                        \
  {                                                                                                                                            \
    LP_CHECK_CUDA((allow_smem<tree_join_kernel<DD, GG>>((int)line)));                                                                          \
    LP_CHECK_CUDA(launch_ex(tree_join_kernel<DD, GG>, join, dim3(TA_JOIN_ROWS * DD / 4), line, stream, 1, true, a));                           \
  }
#define LP_TREE_D(DD)                                                                                                                          \
  if (tc) { if (const int rc = launch_tree_tc(a, stream)) return rc; }                                                                          \
  else if (wm == 1) LP_TREE(DD, 1, 4) else if (wm == 2) LP_TREE(DD, 2, 2) else LP_TREE(DD, 4, 1)                                                    \
  LP_CHECK_CUDA(cudaGetLastError());                                                                                                           \
  if (groups == 1) LP_JOIN(DD, 1) else LP_JOIN(DD, TA_JOIN_GROUPS)
  if (d->D == 128) { LP_TREE_D(128) } else if (d->D == 96) { LP_TREE_D(96) } else { LP_TREE_D(64) }
#undef LP_TREE_D
#undef LP_JOIN
#undef LP_TREE
  return 0;
}
