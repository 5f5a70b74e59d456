// leopard_b200 — attention of a batch over a prefix that it shares (samples of one prompt, questions about one document).
//
//   out[b, t, h] = sum_j softmax_j(scale q[b, t, h] . k_j) v_j  over the prefix's rows j and the request's own rows up to its token t
//
// This file has the entry point, the kernel for the requests' own rows (and for a prefix that few rows look at), and the one that joins the pieces; lp_prefixattn_tc.cu has the prefix for
// many rows.
#include "lp_prefixattn.cuh"

namespace lp {

// A CTA takes 8 NT rows of a key head and a piece of the keys; its four warps take 16 keys of each tile of 64.  mma.sync, keys and values straight into registers: a lane loads 16 bytes of each of its keys'
// rows as they lie.  Keys are the products' 16 rows and the queries' rows their 8 columns, since few rows look at the same keys (four of a token with eight key heads of 32).  A product does not mind the order of
// what it sums over, so the dimensions of a head are dealt to the operands' places as the loads bring them: piece t + 4 c of a key's 16-byte pieces goes to places 2t, 2t + 1 and 2t + 8, 2t + 9 of steps
// 2c and 2c + 1.  In the second product the dimensions are the rows, values of two keys put side by side by byte permutations.
// Bound by HBM for many or long requests (300 own rows of 64, 32 heads over 8: 23 us, of which the tiles take 12, 6.6 TB/s, the first loads' latency 7), by latency else (4 rows a key head after 512 9 us).  Four CTAs an SM with
// 8 rows, three with 16.  At 128 dimensions the former spill 110 to 140 bytes (the join 100).  Fewer CTAs an SM and no spills, in both kernels: 64 samples after 32,771 rows 77 us a call and 76, 16 after 1,000 24.6 and
// 23.3, two after 4,796 22.5 and 24.6, four others the same.
template <int D>
constexpr int pa_ld() { return D / 4 + 1; }                       // 16-byte pieces from one row of a warp's sums to the next (eight rows' in eight different banks)
template <int D, int NT>
constexpr int pa_smem() { return 4 * 8 * NT * pa_ld<D>() * 16; }
template <int D, int NT, bool PRE>
__device__ __forceinline__ void prefix_rows(const PrefixArgs& a, int cta) {
  constexpr int KC = D / 32, VC = (D + 63) / 64, ROWS = 8 * NT;   // 16-byte pieces of a key's row a lane loads; of a value's
  constexpr int LD = pa_ld<D>();
  extern __shared__ float4 pa_sums[];                             // first, and behind it [warp][ROWS][LD]; before, the queries [KC][NT][32]
  int* first = reinterpret_cast<int*>(pa_sums);
  float4* sums = pa_sums + (a.d.B + 4) / 4;
  uint4* queries = reinterpret_cast<uint4*>(sums);
  __shared__ float2 ml[4][ROWS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;

  // ---- the piece
  int kvh, r0, rows, n_keys, past, t0, t1, owner = 0, slot;
  if (PRE) {
    pa_tokens(a, first);
    rows = first[a.d.B] * a.group;
    const PrefixLine line = pa_line(a, rows);
    const int item = line.own ? cta / line.own : 0;
    if (item >= line.items) return;
    const int piece = cta - item * line.own;                      // (of as many CTAs as items can be, each has at most one)
    const int blk = item / a.d.KVH;
    kvh = item - blk * a.d.KVH;
    r0 = blk * ROWS;
    t0 = pa_cut(a.pre_tiles, piece, line.own);
    t1 = pa_cut(a.pre_tiles, piece + 1, line.own);
    past = n_keys = a.d.prefix;
    slot = item + cta;
  } else {
    slot = cta;
    const int rest = cta / a.own_splits, piece = cta - rest * a.own_splits, i = rest / a.own_blocks;
    r0 = (rest - i * a.own_blocks) * ROWS;
    owner = i / a.d.KVH;
    kvh = i - owner * a.d.KVH;
    const int fresh = pa_new(a, owner);
    rows = fresh * a.group;
    pa_own(a, a.d.lengths[owner], fresh, past, n_keys);
    const int pieces = pa_own_pieces(a, n_keys);
    if (piece >= pieces) return;
    const int tiles = (n_keys + PA_KEYS - 1) / PA_KEYS;
    t0 = pa_cut(tiles, piece, pieces);
    t1 = pa_cut(tiles, piece + 1, pieces);
  }
  if (r0 >= rows) return;
  const bool apart = PRE && a.d.prefix_k;                         // the prefix has a cache of its own
  const bf16* kb = apart ? reinterpret_cast<const bf16*>(a.d.prefix_k) + kvh * a.d.pk_head : reinterpret_cast<const bf16*>(a.d.k) + kvh * a.d.k_head;
  const bf16* vb = apart ? reinterpret_cast<const bf16*>(a.d.prefix_v) + kvh * a.d.pv_head : reinterpret_cast<const bf16*>(a.d.v) + kvh * a.d.v_head;
  const int* table = a.d.page_table && !apart ? a.d.page_table + owner * a.d.ld_table : nullptr;
  const int page_of = apart ? 0 : owner, key_first = !PRE && table ? a.d.prefix : 0;
  auto key_at = [&](int page, int row) { return kb + (apart ? row * a.d.pk_row : page * a.d.k_page + row * a.d.k_row); };
  auto value_at = [&](int page, int row) { return vb + (apart ? row * a.d.pv_row : page * a.d.v_page + row * a.d.v_row); };

  // where the warp's 16 keys of a tile lie: lane i (and i + 16) knows key i's page and row
  int2 place;
  auto locate = [&](int tile) {
    const int key = tile * PA_KEYS + warp * 16 + (lane & 15);
    place = make_int2(-1, 0);
    if (tile < t1 && key < n_keys) {
      if (table) {
        const unsigned at = (unsigned)key + (unsigned)key_first, logical = at / (unsigned)a.d.page_size;
        const int page = table[logical];
        place = make_int2(page < a.d.n_pages ? page : -1, (int)(at - logical * a.d.page_size));
      } else {
        place = make_int2(page_of, key);
      }
    }
  };
  uint4 kr[2][KC], vr[4][VC];
  const uint4 none = make_uint4(0, 0, 0, 0);
  auto load_k = [&]() {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int page = __shfl_sync(0xffffffffu, place.x, j * 8 + g), row = __shfl_sync(0xffffffffu, place.y, j * 8 + g);
      const bf16* p = key_at(page, row) + t4 * 8;
#pragma unroll
      for (int c = 0; c < KC; ++c) kr[j][c] = page >= 0 ? ldg_once(p + c * 32) : none;
    }
  };
  auto load_v = [&](const int2& at) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int key = (j >> 1) * 8 + 2 * t4 + (j & 1);
      const int page = __shfl_sync(0xffffffffu, at.x, key), row = __shfl_sync(0xffffffffu, at.y, key);
      const bf16* p = value_at(page, row) + g * 8;
#pragma unroll
      for (int c = 0; c < VC; ++c) vr[j][c] = page >= 0 && c * 8 + g < D / 8 ? ldg_once(p + c * 64) : none;
    }
  };
  locate(t0);
  // ---- the queries, a piece a warp: row g (+ 8) as the first product's columns
  uint4 qx[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = r0 + 8 * n + g;
    const bool there = r < rows;
    const int i = there ? r / a.group : 0, head = kvh * a.group + (there ? r - i * a.group : 0);
    const int b = PRE ? pa_find(first, a.d.B, i) : owner, t = PRE ? i - first[b] : i;
    const bf16* q = reinterpret_cast<const bf16*>(a.d.q) + b * a.d.q_batch + t * a.d.q_token + head * a.d.q_head + t4 * 8 + warp * 32;
    qx[n] = there && warp < KC ? *reinterpret_cast<const uint4*>(q) : none;
  }
  load_k();
  load_v(place);
  int2 here = place;
  locate(t0 + 1);
  // keys that this lane's rows (two of each eight) see, and that all rows see
  int limit[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int h = 0; h < 2; ++h) limit[n][h] = PRE ? n_keys : min(n_keys, past + (r0 + 8 * n + 2 * t4 + h) / a.group + 1);
  const int sure = PRE ? n_keys : min(n_keys, past + 1);
  if (warp < KC)
#pragma unroll
    for (int n = 0; n < NT; ++n) queries[(warp * NT + n) * 32 + lane] = qx[n];
  __syncthreads();

  int odd = 0;                                                    // values that are not finite were left out
  float o[NT][VC][4][4], m[NT][2], l[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m[n][0] = m[n][1] = -INFINITY;
    l[n][0] = l[n][1] = 0.f;
#pragma unroll
    for (int c = 0; c < VC; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[n][c][j][k] = 0.f;
  }
  for (int tile = t0; tile < t1; ++tile) {
    float s[NT][4];                                               // keys g, g (row 2t4, 2t4 + 1), g + 8, g + 8
#pragma unroll
    for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int c = 0; c < KC; ++c)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint4 q = lds_u4(queries + (c * NT + n) * 32 + lane);
        mma_bf16(s[n], kr[0][c].x, kr[1][c].x, kr[0][c].y, kr[1][c].y, q.x, q.y);
        mma_bf16(s[n], kr[0][c].z, kr[1][c].z, kr[0][c].w, kr[1][c].w, q.z, q.w);
      }
    const int2 next = place;
    load_k();                                                     // (of the next tile)
    locate(tile + 2);
    const int key0 = tile * PA_KEYS + warp * 16;
    const unsigned there = __ballot_sync(0xffffffffu, here.x >= 0) & 0xffffu;
    const bool tail = key0 + 16 > sure;
    bool grow = tile == t0;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        s[n][k] *= a.scale_log2;
        if (tail || there != 0xffffu) {
          const int key = g + 8 * (k >> 1);
          if (!((there >> key) & 1) || key0 + key >= limit[n][k & 1]) s[n][k] = -INFINITY;
        }
        grow |= s[n][k] > m[n][k & 1] + 8.f;
      }
    // weights are taken to a maximum that is at most 2^8 too small: sums and values are scaled when one grows past that
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float mx = fmaxf(s[n][h], s[n][2 + h]);
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
          mx = fmaxf(mx, m[n][h]);
          const float f = m[n][h] == -INFINITY ? 0.f : pa_ex2(m[n][h] - mx);
          m[n][h] = mx;
          l[n][h] *= f;
#pragma unroll
          for (int c = 0; c < VC; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[n][c][j][h] *= f, o[n][c][j][2 + h] *= f;
        }
    }
    uint32_t p[NT][2];                                            // weights as the second product's columns: rows g, keys 2t4, 2t4 + 1 (+ 8)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        w[k] = pa_ex2(s[n][k] - (m[n][k & 1] == -INFINITY ? 0.f : m[n][k & 1]));
        l[n][k & 1] += w[k];
      }
      // as bf16 (half a step is 2^-8 of a weight); their sum was taken before
      asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(p[n][0]) : "r"(pack_bf16x2(w[0], w[1])));
      asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(p[n][1]) : "r"(pack_bf16x2(w[2], w[3])));
    }
    if (!PRE && tail && a.d.T > 1) {                              // 0 x NaN: values that are not finite are left out of the product, and reach the rows that see them at the end
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int c = 0; c < VC; ++c) {
          uint32_t* w = &vr[j][c].x;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if ((w[k] & 0x7f80u) == 0x7f80u) w[k] &= 0xffff0000u, odd = 1;
            if ((w[k] & 0x7f800000u) == 0x7f800000u) w[k] &= 0xffffu, odd = 1;
          }
        }
    }
#pragma unroll
    for (int c = 0; c < VC; ++c) {
      const uint32_t *x0 = &vr[0][c].x, *x1 = &vr[1][c].x, *y0 = &vr[2][c].x, *y1 = &vr[3][c].x;
#pragma unroll
      for (int j = 0; j < 4; ++j) {                               // rows g: dimension 8 (8 c + g) + 2 j, rows g + 8: the next one
        const uint32_t a0 = __byte_perm(x0[j], x1[j], 0x5410), a1 = __byte_perm(x0[j], x1[j], 0x7632), a2 = __byte_perm(y0[j], y1[j], 0x5410), a3 = __byte_perm(y0[j], y1[j], 0x7632);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_bf16(o[n][c][j], a0, a1, a2, a3, p[n][0], p[n][1]);
      }
    }
    load_v(next);
    here = next;
  }
  // ---- the warps' rows together.  Of a row's 16-byte pieces the even ones stand first, then the odd ones: eight lanes' stores find different banks.
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l[n][h] += __shfl_xor_sync(0xffffffffu, l[n][h], x);
      if (g == 0) ml[warp][8 * n + 2 * t4 + h] = make_float2(m[n][h], l[n][h]);
    }
  __syncthreads();                                                // (the queries are done with)
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = 8 * n + 2 * t4 + h;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < 4; ++w) top = fmaxf(top, ml[w][r].x);
      const float f = m[n][h] == -INFINITY ? 1.f : pa_ex2(m[n][h] - top);      // (sums and values of a warp that saw nothing are zeros, or NaN)
      float4* at = sums + (warp * ROWS + r) * LD;
#pragma unroll
      for (int c = 0; c < VC; ++c)
        if (c * 8 + g < D / 8) {
          const float(&x)[4][4] = o[n][c];
          at[c * 8 + g] = make_float4(x[0][h] * f, x[0][2 + h] * f, x[1][h] * f, x[1][2 + h] * f);
          at[D / 8 + c * 8 + g] = make_float4(x[2][h] * f, x[2][2 + h] * f, x[3][h] * f, x[3][2 + h] * f);
        }
    }
  if (__syncthreads_or(odd)) {      // (PRE: never)
    // the tiles that some rows do not see whole: a thread looks at one dimension of all their keys
    const int k0 = max(t0 * PA_KEYS, sure & ~15), k1 = min(t1 * PA_KEYS, n_keys);
    for (int d = threadIdx.x; d < D; d += 128) {
      float* to = reinterpret_cast<float*>(sums + (d >> 3) + ((d >> 2) & 1) * (D / 8)) + d % 4;
      for (int key = k0; key < k1; ++key) {
        const unsigned at = (unsigned)key + (unsigned)key_first, logical = table ? at / (unsigned)a.d.page_size : 0;
        const int page = table ? table[logical] : page_of;
        if (page < 0 || page >= a.d.n_pages) continue;
        const float v = __bfloat162float(value_at(page, table ? (int)(at - logical * a.d.page_size) : key)[d]);
        if (!not_finite(v)) continue;
        for (int r = 0; r < min(ROWS, rows - r0); ++r)
          if (key < past + (r0 + r) / a.group + 1) to[r * LD * 4] += v;
      }
    }
    __syncthreads();
  }
  const int mine = min(ROWS, rows - r0), r = threadIdx.x % ROWS;
  float* po = (PRE ? a.pre_o : a.own_o) + (long long)slot * (D * ROWS);
  float2* pm = (PRE ? a.pre_ml : a.own_ml) + (long long)slot * ROWS;
  if (r >= mine) return;
#pragma unroll
  for (int c4 = threadIdx.x / ROWS; c4 < D / 4; c4 += 128 / ROWS) {
    const int from = r * LD + (c4 >> 1) + (c4 & 1) * (D / 8);
    float4 x = sums[from];
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      const float4 y = sums[w * ROWS * LD + from];
      x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
    }
    *reinterpret_cast<float4*>(po + (c4 * ROWS + r) * 4) = x;
  }
  if (threadIdx.x < ROWS) {
    float2 x = make_float2(-INFINITY, 0.f);
#pragma unroll
    for (int w = 0; w < 4; ++w) x.x = fmaxf(x.x, ml[w][r].x);
#pragma unroll
    for (int w = 0; w < 4; ++w) x.y += ml[w][r].y * (ml[w][r].x == -INFINITY ? 1.f : pa_ex2(ml[w][r].x - x.x));
    pm[r] = x;
  }
}
// PRE: the prefix's pieces come first, of 8 PRE rows; then the own rows', of 8 OWN
template <int D, int PRE, int OWN>
__global__ void __launch_bounds__(128, PRE == 2 || OWN == 2 ? 3 : 4)
prefix_rows_kernel(const __grid_constant__ PrefixArgs a, int pre_ctas) {
  pdl_launch_dependents();
  if constexpr (PRE > 0) {
    if ((int)blockIdx.x < pre_ctas) {
      prefix_rows<D, PRE, true>(a, blockIdx.x);
      return;
    }
  }
  prefix_rows<D, OWN, false>(a, blockIdx.x - pre_ctas);
}

// The pieces of a row together: a CTA takes 8 rows of a key head, a thread four columns of one and, of GROUPS groups, every GROUPS-th eight pieces, which are under way at once; weights follow a running maximum, so
// that each piece is read once.  Bound by latency, and by the workspace's way through L2: 20 pieces of 228 rows x 8 heads 8 us, 5 of 1,104 x 8 7 behind the last piece.
constexpr int PJ_ROWS = 8, PJ_AT_ONCE = 8;
template <int D, int GROUPS>
__global__ void __launch_bounds__(PJ_ROWS * D / 4 * GROUPS, 1024 / (PJ_ROWS * D / 4 * GROUPS))
prefix_join_kernel(const __grid_constant__ PrefixArgs a) {
  constexpr int THREADS = PJ_ROWS * D / 4;
  extern __shared__ int pa_first[];
  __shared__ __align__(16) bf16 done[PJ_ROWS][D + 8];
  __shared__ long long to[PJ_ROWS];
  __shared__ float4 more_x[GROUPS > 1 ? GROUPS - 1 : 1][GROUPS > 1 ? THREADS : 1];
  __shared__ float2 more_ml[GROUPS > 1 ? GROUPS - 1 : 1][GROUPS > 1 ? THREADS : 1];
  const int group = GROUPS > 1 ? threadIdx.x / THREADS : 0, tid = GROUPS > 1 ? threadIdx.x - group * THREADS : threadIdx.x;
  const int kvh = blockIdx.y, in = tid % PJ_ROWS, c4 = tid / PJ_ROWS;
  pa_tokens(a, pa_first);
  const int rows = pa_first[a.d.B] * a.group, r0 = blockIdx.x * PJ_ROWS;
  if (r0 >= rows) {
    pdl_wait();
    return;
  }
  const int r = min(r0 + in, rows - 1), i = r / a.group, g = r - i * a.group, b = pa_find(pa_first, a.d.B, i), t = i - pa_first[b];
  int past, keys;
  pa_own(a, a.d.lengths[b], pa_first[b + 1] - pa_first[b], past, keys);
  int n_pre, pre_in;
  long long pre_slot;
  pa_pieces_of(a, rows, kvh, r, n_pre, pre_slot, pre_in);
  const int own = t * a.group + g, n = n_pre + pa_own_pieces(a, keys), own_blk = own / a.own_block, own_in = own - own_blk * a.own_block;
  const long long own_slot = (((long long)b * a.d.KVH + kvh) * a.own_blocks + own_blk) * a.own_splits;
  if (tid < PJ_ROWS && group == 0) to[tid] = r0 + tid < rows ? b * a.d.o_batch + t * a.d.o_token + (kvh * a.group + g) * a.d.o_head : -1;
  pdl_wait();
  float top = -INFINITY, sum = 0.f;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p0 = group * PJ_AT_ONCE; p0 < n; p0 += GROUPS * PJ_AT_ONCE) {
    float2 ml[PJ_AT_ONCE];
    float4 y[PJ_AT_ONCE];
#pragma unroll
    for (int k = 0; k < PJ_AT_ONCE; ++k) {
      const int p = p0 + k;
      ml[k] = make_float2(-INFINITY, 0.f);
      y[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (p < n_pre) {
        ml[k] = a.pre_ml[(pre_slot + p) * a.pre_rows + pre_in];
        y[k] = *reinterpret_cast<const float4*>(a.pre_o + (((pre_slot + p) * (D / 4) + c4) * a.pre_rows + pre_in) * 4);
      } else if (p < n) {
        const long long s = own_slot + p - n_pre;
        ml[k] = a.own_ml[s * a.own_block + own_in];
        y[k] = *reinterpret_cast<const float4*>(a.own_o + ((s * (D / 4) + c4) * a.own_block + own_in) * 4);
      }
    }
    float m = top;
#pragma unroll
    for (int k = 0; k < PJ_AT_ONCE; ++k) m = fmaxf(m, ml[k].x);
    const float old = top == -INFINITY ? 1.f : pa_ex2(top - m);      // sums and values of pieces that saw nothing are zeros, or NaN
    top = m;
    sum *= old;
    x.x *= old; x.y *= old; x.z *= old; x.w *= old;
#pragma unroll
    for (int k = 0; k < PJ_AT_ONCE; ++k) {
      const float f = ml[k].x == -INFINITY ? 1.f : pa_ex2(ml[k].x - m);
      sum += ml[k].y * f;
      x.x += y[k].x * f; x.y += y[k].y * f; x.z += y[k].z * f; x.w += y[k].w * f;
    }
  }
  if (GROUPS > 1) {
    if (group > 0) more_x[group - 1][tid] = x, more_ml[group - 1][tid] = make_float2(top, sum);
    __syncthreads();
    if (group == 0) {
      float m = top;
#pragma unroll
      for (int k = 0; k < GROUPS - 1; ++k) m = fmaxf(m, more_ml[k][tid].x);
      const float old = top == -INFINITY ? 1.f : pa_ex2(top - m);
      sum *= old;
      x.x *= old; x.y *= old; x.z *= old; x.w *= old;
#pragma unroll
      for (int k = 0; k < GROUPS - 1; ++k) {
        const float2 ml = more_ml[k][tid];
        const float4 y = more_x[k][tid];
        const float f = ml.x == -INFINITY ? 1.f : pa_ex2(ml.x - m);
        sum += ml.y * f;
        x.x += y.x * f; x.y += y.y * f; x.z += y.z * f; x.w += y.w * f;
      }
    }
  }
  if (group == 0) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    *reinterpret_cast<uint2*>(&done[in][c4 * 4]) = make_uint2(pack_bf16x2(x.x * inv, x.y * inv), pack_bf16x2(x.z * inv, x.w * inv));
  }
  __syncthreads();
  if (threadIdx.x < PJ_ROWS * (D / 8)) {
    const int row = threadIdx.x / (D / 8), col = (threadIdx.x % (D / 8)) * 8;
    if (to[row] >= 0) *reinterpret_cast<uint4*>(reinterpret_cast<bf16*>(a.d.out) + to[row] + col) = *reinterpret_cast<const uint4*>(&done[row][col]);
  }
}

// The same for many rows: a CTA takes 32 rows, a lane one of them and the warps its columns, so that where a row's pieces lie (some 64-bit divisions) is worked out by one warp for all
// columns: of 12,288 rows x 8 heads, two pieces each, 59 us less than by the kernel above.
constexpr int PW_ROWS = 32, PW_WARPS = 8, PW_AT_ONCE = 2;
struct PrefixJoinRow { long long pre_slot, own_slot, to; int n_pre, pre_in, n, own_in; };
template <int D>
__global__ void __launch_bounds__(PW_WARPS * 32, 3)
prefix_join_wide_kernel(const __grid_constant__ PrefixArgs a) {
  constexpr int K = D / 4 / PW_WARPS;     // columns (of four) of a thread
  extern __shared__ int pa_first[];
  __shared__ __align__(16) bf16 done[PW_ROWS][D + 8];
  __shared__ PrefixJoinRow info[PW_ROWS];
  const int kvh = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pa_tokens(a, pa_first);
  const int rows = pa_first[a.d.B] * a.group, r0 = blockIdx.x * PW_ROWS;
  if (r0 >= rows) {
    pdl_wait();
    return;
  }
  if (warp == 0) {
    const int r = min(r0 + lane, rows - 1), i = r / a.group, g = r - i * a.group, b = pa_find(pa_first, a.d.B, i), t = i - pa_first[b];
    int past, keys;
    pa_own(a, a.d.lengths[b], pa_first[b + 1] - pa_first[b], past, keys);
    PrefixJoinRow x;
    pa_pieces_of(a, rows, kvh, r, x.n_pre, x.pre_slot, x.pre_in);
    const int own = t * a.group + g, own_blk = own / a.own_block;
    x.n = x.n_pre + pa_own_pieces(a, keys);
    x.own_in = own - own_blk * a.own_block;
    x.own_slot = (((long long)b * a.d.KVH + kvh) * a.own_blocks + own_blk) * a.own_splits;
    x.to = r0 + lane < rows ? b * a.d.o_batch + t * a.d.o_token + (kvh * a.group + g) * a.d.o_head : -1;
    info[lane] = x;
  }
  __syncthreads();
  const PrefixJoinRow at = info[lane];
  pdl_wait();
  float top = -INFINITY, sum = 0.f;
  float4 x[K];
#pragma unroll
  for (int j = 0; j < K; ++j) x[j] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p0 = 0; p0 < at.n; p0 += PW_AT_ONCE) {
    float2 ml[PW_AT_ONCE];
    float4 y[PW_AT_ONCE][K];
#pragma unroll
    for (int k = 0; k < PW_AT_ONCE; ++k) {
      const int p = p0 + k;
      const bool pre = p < at.n_pre;
      const long long s = pre ? at.pre_slot + p : at.own_slot + p - at.n_pre;
      const int block = pre ? a.pre_rows : a.own_block, in = pre ? at.pre_in : at.own_in;
      ml[k] = p < at.n ? (pre ? a.pre_ml : a.own_ml)[s * block + in] : make_float2(-INFINITY, 0.f);
      const float* o = (pre ? a.pre_o : a.own_o) + ((s * (D / 4) + warp) * block + in) * 4;
#pragma unroll
      for (int j = 0; j < K; ++j) y[k][j] = p < at.n ? *reinterpret_cast<const float4*>(o + j * PW_WARPS * block * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float m = top;
#pragma unroll
    for (int k = 0; k < PW_AT_ONCE; ++k) m = fmaxf(m, ml[k].x);
    const float old = top == -INFINITY ? 1.f : pa_ex2(top - m);      // (as above)
    top = m;
    sum *= old;
#pragma unroll
    for (int j = 0; j < K; ++j) x[j].x *= old, x[j].y *= old, x[j].z *= old, x[j].w *= old;
#pragma unroll
    for (int k = 0; k < PW_AT_ONCE; ++k) {
      const float f = ml[k].x == -INFINITY ? 1.f : pa_ex2(ml[k].x - m);
      sum += ml[k].y * f;
#pragma unroll
      for (int j = 0; j < K; ++j) x[j].x += y[k][j].x * f, x[j].y += y[k][j].y * f, x[j].z += y[k][j].z * f, x[j].w += y[k][j].w * f;
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int j = 0; j < K; ++j)
    *reinterpret_cast<uint2*>(&done[lane][(warp + j * PW_WARPS) * 4]) = make_uint2(pack_bf16x2(x[j].x * inv, x[j].y * inv), pack_bf16x2(x[j].z * inv, x[j].w * inv));
  __syncthreads();
  for (int i = threadIdx.x; i < PW_ROWS * (D / 8); i += PW_WARPS * 32) {
    const int row = i / (D / 8), col = (i - row * (D / 8)) * 8;
    if (info[row].to >= 0) *reinterpret_cast<uint4*>(reinterpret_cast<bf16*>(a.d.out) + info[row].to + col) = *reinterpret_cast<const uint4*>(&done[row][col]);
  }
}

// ---- host ----------------------------------------------------------------------------------------------------------
static int prefix_check(const lp_prefix_attn_desc* d) {
  LP_REQUIRE(d != nullptr, "lp_prefix_attention: null descriptor");
  LP_REQUIRE(d->B > 0 && d->B <= PA_MAX_BATCH && d->T > 0 && d->T <= LP_PREFIX_MAX_NEW, "lp_prefix_attention: B=%d (1 to %d), T=%d (1 to %d)", d->B, PA_MAX_BATCH, d->T, LP_PREFIX_MAX_NEW);
  LP_REQUIRE(d->KVH > 0 && d->H >= d->KVH && d->H % d->KVH == 0 && d->H <= 1024, "lp_prefix_attention: %d query heads over %d key heads (1024 at most)", d->H, d->KVH);
  LP_REQUIRE(d->D == 64 || d->D == 96 || d->D == 128, "lp_prefix_attention: heads of %d are not built (64, 96, 128)", d->D);
  LP_REQUIRE((long long)d->B * d->T * d->H <= 1LL << 24, "lp_prefix_attention: %d requests of %d tokens and %d heads are too many", d->B, d->T, d->H);
  LP_REQUIRE(d->n_pages > 0 && d->page_size > 0 && d->max_pages > 0, "lp_prefix_attention: %d pages of %d rows, %d a request", d->n_pages, d->page_size, d->max_pages);
  LP_REQUIRE((long long)d->max_pages * d->page_size <= (1LL << 31) - 512, "lp_prefix_attention: %d pages of %d rows are too many", d->max_pages, d->page_size);
  LP_REQUIRE(d->B * (long long)d->KVH * ((d->T * (d->H / d->KVH) + 7) / 8) <= 1 << 24, "lp_prefix_attention: %d requests of %d tokens over %d key heads are too many", d->B, d->T, d->KVH);
  LP_REQUIRE(d->prefix >= 0 && d->prefix <= (1LL << 31) - 512, "lp_prefix_attention: prefix %d", d->prefix);
  if (d->prefix_k) LP_REQUIRE(!d->page_table && d->prefix_v, "lp_prefix_attention: a prefix of its own goes with a cache of its own each");
  else if (d->page_table) LP_REQUIRE(d->prefix <= (long long)d->max_pages * d->page_size, "lp_prefix_attention: a prefix of %d rows in %d pages of %d", d->prefix, d->max_pages, d->page_size);
  else LP_REQUIRE(d->prefix == 0, "lp_prefix_attention: a prefix of %d rows that is nowhere", d->prefix);
  return 0;
}
// Whether the prefix goes to the tcgen05 kernel: it costs a launch and 10 us of start and end, the other reads the prefix once for every 16 rows.  Decided by blocks of 16 rows x key heads x keys, of more than 8 rows.
// mma.sync and tcgen05, us a call, 60 own rows a request, at 180,000 of these: 32 rows of 32 heads over 8 after 11,250 34.8 and 32.8, 64 after 5,625 32.8 and 30.7, 256 after 1,406 32.8 and 28.7, 32 of 16 heads over 16 after
// 5,625 34.9 and 34.8, 256 of 8 over 1 after 5,625 26.6 and 24.6, 192 of 12 over 4 (64 dimensions) after 3,750 20.5 and 24.6; at 270,000 47 - 53 and 31 - 39 (the last one 30.7 and 27.5).  Below 8 x 10^4 tcgen05's is 4 - 6 us behind.
// Up to 8 rows read it once in any case: 8 after 100,003 84 and 84 (160, 154).
constexpr long long PA_TC_WORK = 160000;
static bool prefix_tc(const lp_prefix_attn_desc* d) {
  const long long rows = (long long)d->B * d->T * (d->H / d->KVH);
  return rows > 8 && (rows + 15) / 16 * d->KVH * d->prefix > PA_TC_WORK && prefix_tc_takes(d);
}
// how a call is cut: what the descriptor's numbers alone decide
static size_t prefix_plan(const lp_prefix_attn_desc* d, PrefixArgs& a) {
  a.d = *d;
  a.group = d->H / d->KVH;
  const long long own = (long long)d->max_pages * d->page_size - (d->page_table ? d->prefix : 0);
  a.own_rows = (int)own;
  a.own_block = d->T * a.group <= 8 ? 8 : 16;
  a.own_blocks = (d->T * a.group + a.own_block - 1) / a.own_block;
  const long long rows = (long long)d->B * d->T * a.group;
  const bool tc = prefix_tc(d);
  a.pre_rows = !tc ? (rows <= 8 ? 8 : 16) : rows <= 128 ? 128 : 256;
  const long long items = (long long)d->B * d->KVH * a.own_blocks, tiles = (own + PA_KEYS - 1) / PA_KEYS, room = ((a.own_block == 16 || (a.pre_rows == 16 && d->prefix > 0)) ? 3LL : 4LL) * sm_count();      // (as many CTAs as run at once)
  long long splits = items >= room ? 1 : room / items;
  a.own_splits = (int)(splits < tiles ? splits : tiles > 0 ? tiles : 1);
  a.own_slots = items * a.own_splits;
  const int keys = tc ? 128 : PA_KEYS;
  a.pre_tiles = (int)(((long long)d->prefix + keys - 1) / keys);
  a.pre_ctas = 0;
  a.pre_slots = 0;
  if (d->prefix > 0) {
    const long long pre_items = (rows + a.pre_rows - 1) / a.pre_rows * d->KVH;
    if (tc) {
      const long long most = pre_items * a.pre_tiles;
      a.pre_ctas = (int)(most < sm_count() ? most : sm_count());
    } else {
      const long long left = a.own_slots < room / 2 ? room - a.own_slots : room / 2;      // (at once with the own rows')
      splits = pre_items >= left ? 1 : left / pre_items;
      // pieces of more than 12 tiles become such of 8, as long as all of them are half as many again as the CTAs that run at once: the longest piece is what a call waits for (us a call, without and so: 64 samples after
      // 1,200 rows 45 and 31, two prompts of 32 after 1,000 37 and 25, 16 samples after 4,900 35 and 32; with 600 rows of their own 32 after 2,400 39 and 43, 64 after 1,200 47 both)
      if ((a.pre_tiles + splits - 1) / splits > 12) {
        const long long most = room * 3 / 2 / pre_items, fine = (a.pre_tiles + 7) / 8, more = fine < most ? fine : most;
        if (more > splits) splits = more;
      }
      a.pre_ctas = (int)((splits < a.pre_tiles ? splits : a.pre_tiles) * pre_items);
    }
    a.pre_slots = pre_items + a.pre_ctas;
  }
  return ((size_t)a.pre_slots * a.pre_rows + (size_t)a.own_slots * a.own_block) * (d->D * 4 + 8);
}

}  // namespace lp

extern "C" size_t lp_prefix_attention_workspace_bytes(const lp_prefix_attn_desc* d) {
  using namespace lp;
  if (prefix_check(d) != 0) return 0;
  PrefixArgs a;
  return prefix_plan(d, a);
}

extern "C" int lp_prefix_attention(const lp_prefix_attn_desc* desc, void* workspace, size_t ws_bytes, void* stream_) {
  using namespace lp;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  if (const int rc = prefix_check(desc)) return rc;
  PrefixArgs a;
  const size_t need = prefix_plan(desc, a);
  lp_prefix_attn_desc* d = &a.d;          // of a dimension of one any stride may have come
  LP_REQUIRE(d->q && d->k && d->v && d->out && d->lengths && workspace, "lp_prefix_attention: null argument");
  LP_REQUIRE(d->page_table ? d->B == 1 || d->ld_table >= d->max_pages : (d->max_pages == 1 && d->B <= d->n_pages), "lp_prefix_attention: %d requests of %d pages: ld_table %lld, %d pages there", d->B,
             d->max_pages, d->ld_table, d->n_pages);
  if (d->B == 1) d->q_batch = d->o_batch = d->ld_table = 0;
  if (d->T == 1) d->q_token = d->o_token = 0;
  if (d->H == 1) d->q_head = d->o_head = 0;
  if (d->n_pages == 1) d->k_page = d->v_page = 0;
  if (d->page_size == 1) d->k_row = d->v_row = 0;
  if (d->KVH == 1) d->k_head = d->v_head = d->pk_head = d->pv_head = 0;
  if (d->prefix <= 1) d->pk_row = d->pv_row = 0;
  if (!d->prefix_k) d->pk_row = d->pk_head = d->pv_row = d->pv_head = 0;
  const long long strides = d->q_batch | d->q_token | d->q_head | d->k_page | d->k_row | d->k_head | d->v_page | d->v_row | d->v_head | d->o_batch | d->o_token | d->o_head | d->pk_row | d->pk_head |
                            d->pv_row | d->pv_head;
  const uintptr_t bases = reinterpret_cast<uintptr_t>(d->q) | reinterpret_cast<uintptr_t>(d->k) | reinterpret_cast<uintptr_t>(d->v) | reinterpret_cast<uintptr_t>(d->out) |
                          reinterpret_cast<uintptr_t>(d->prefix_k) | reinterpret_cast<uintptr_t>(d->prefix_v) | reinterpret_cast<uintptr_t>(workspace);
  LP_REQUIRE(strides % 8 == 0 && bases % 16 == 0, "lp_prefix_attention: strides in multiples of 8 elements, 16-byte aligned bases");
  Dim places[3] = {{d->B, d->o_batch}, {d->T, d->o_token}, {d->H, d->o_head}};
  LP_REQUIRE(strides_nest(places, 3, d->D), "lp_prefix_attention: rows of out share their memory (strides %lld, %lld, %lld)", d->o_batch, d->o_token, d->o_head);
  const Span out = {d->out, 2, 4, {{d->B, d->o_batch}, {d->T, d->o_token}, {d->H, d->o_head}, {d->D, 1}}};
  const Span reads[8] = {{d->q, 2, 4, {{d->B, d->q_batch}, {d->T, d->q_token}, {d->H, d->q_head}, {d->D, 1}}}, {d->k, 2, 4, {{d->n_pages, d->k_page}, {d->page_size, d->k_row}, {d->KVH, d->k_head}, {d->D, 1}}},
                         {d->v, 2, 4, {{d->n_pages, d->v_page}, {d->page_size, d->v_row}, {d->KVH, d->v_head}, {d->D, 1}}}, {d->prefix_k, 2, 3, {{d->prefix, d->pk_row}, {d->KVH, d->pk_head}, {d->D, 1}}},
                         {d->prefix_v, 2, 3, {{d->prefix, d->pv_row}, {d->KVH, d->pv_head}, {d->D, 1}}}, {d->page_table, 4, 2, {{d->B, d->ld_table}, {d->max_pages, 1}}}, {d->lengths, 4, 1, {{d->B, 1}}},
                         {d->fresh, 4, 1, {{d->B, 1}}}};
  for (const Span& r : reads) LP_REQUIRE(!r.p || !spans_meet(out, r), "lp_prefix_attention: out must share no memory with the inputs");
  LP_REQUIRE(ws_bytes >= need, "lp_prefix_attention: workspace too small");
  a.scale_log2 = d->scale * 1.4426950408889634f;
  const size_t pre = (size_t)a.pre_slots * a.pre_rows, mine = (size_t)a.own_slots * a.own_block;
  a.pre_o = reinterpret_cast<float*>(workspace);
  a.own_o = a.pre_o + pre * d->D;
  a.pre_ml = reinterpret_cast<float2*>(a.own_o + mine * d->D);
  a.own_ml = a.pre_ml + pre;
  const bool tc = a.pre_rows > 16;
  const int pre_ctas = tc ? 0 : a.pre_ctas;
  const long long ctas = pre_ctas + a.own_slots;
  const size_t first = (size_t)(d->B + 1) * 4;
  const dim3 join((unsigned)(((long long)d->B * d->T * a.group + PJ_ROWS - 1) / PJ_ROWS), d->KVH);
  note_launch(tc ? 3 : 2);
  const long long pieces = a.pre_ctas ? a.pre_ctas / (a.pre_slots - a.pre_ctas) + a.own_splits : a.own_splits, joins = (long long)join.x * join.y;
  // 32 rows a CTA where that leaves work for all SMs: it takes few pieces at once, so where there are many of them from later on (us a call, 8 rows and 32: 96 requests of 32 tokens, two pieces, 272 and 213, of 8 70 and
  // 59; 60 of two and 12 heads over 4, 500 rows before, 180 CTAs of 8 rows 16.4 and 14.3, 4,000 before, 38 pieces, 26.7 and 34.8)
  const bool wide = joins > (pieces <= PJ_AT_ONCE ? 1 : 4) * (long long)sm_count();
  const int groups = pieces <= PJ_AT_ONCE ? 1 : joins > sm_count() ? 2 : 4;
  const size_t list = ((size_t)d->B + 4) / 4 * 16;
#define LP_ROWS(DD, PRE, OWN)                                                                                                       \
  {                                                                                                                                 \
    const size_t smem = list + pa_smem<DD, (PRE > OWN ? PRE : OWN)>();                                                              \
    LP_CHECK_CUDA((allow_smem<prefix_rows_kernel<DD, PRE, OWN>>((int)smem)));                                                       \
    prefix_rows_kernel<DD, PRE, OWN><<<(unsigned)ctas, 128, smem, stream>>>(a, pre_ctas);                                           \
  }
#define LP_PREFIX(DD)                                                                                                               \
  {                                                                                                                                 \
    if (tc || !pre_ctas) { if (a.own_block == 8) LP_ROWS(DD, 0, 1) else LP_ROWS(DD, 0, 2) }                                         \
    else if (a.pre_rows == 8) LP_ROWS(DD, 1, 1) else if (a.own_block == 8) LP_ROWS(DD, 2, 1) else LP_ROWS(DD, 2, 2)                 \
    LP_CHECK_CUDA(cudaGetLastError());                                                                                              \
    if (tc) { if (const int rc = launch_prefix_tc(a, stream)) return rc; }                                                          \
    if (wide) LP_CHECK_CUDA(launch_ex(prefix_join_wide_kernel<DD>, dim3((join.x + 3) / 4, join.y), dim3(PW_WARPS * 32), first, stream, 1, true, a)); \
    else if (groups == 4) LP_CHECK_CUDA(launch_ex(prefix_join_kernel<DD, 4>, join, dim3(PJ_ROWS * DD), first, stream, 1, true, a));      \
    else if (groups == 2) LP_CHECK_CUDA(launch_ex(prefix_join_kernel<DD, 2>, join, dim3(PJ_ROWS * DD / 2), first, stream, 1, true, a)); \
    else LP_CHECK_CUDA(launch_ex(prefix_join_kernel<DD, 1>, join, dim3(PJ_ROWS * DD / 4), first, stream, 1, true, a));              \
  }
  if (d->D == 128) LP_PREFIX(128) else if (d->D == 96) LP_PREFIX(96) else LP_PREFIX(64)
#undef LP_ROWS
#undef LP_PREFIX
  return 0;
}
