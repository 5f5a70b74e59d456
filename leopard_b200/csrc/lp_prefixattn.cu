// leopard_b200 — attention of a batch over a prefix that it shares (samples of one prompt, questions about one document).
//
//   out[b, t, h] = sum_j softmax_j(scale q[b, t, h] . k_j) v_j  over the prefix's rows j and the request's own rows up to its token t
//
// This file has the entry point, the kernel for the requests' own rows (and for a prefix that few rows look at), and the one that joins the pieces; lp_prefixattn_tc.cu has the prefix for
// many rows.
#include "lp_prefixattn.cuh"

namespace lp {

// A CTA takes 16 rows of a key head and a piece of the keys; its four warps take 16 keys of each tile of 64.  mma.sync, keys and values straight into registers: a lane loads 16 bytes of each of its keys'
// rows as they lie.  The products do not mind the order of what they sum over, so the dimensions of a head (and the columns of the values) are dealt to the operands' places as the loads bring them;
// values of two keys are put side by side by byte permutations.  The queries are in shared memory as the product's first operand takes them, so that four CTAs fit on an SM.
template <int D>
constexpr int pa_smem(int B) { return 4 * PA_ROWS * (D + 8) * 4 + (B + 1) * 4; }
template <int D>
__global__ void __launch_bounds__(128, 3)
prefix_rows_kernel(const __grid_constant__ PrefixArgs a, int pre_ctas) {
  constexpr int KC = D / 32, VC = (D + 63) / 64;                  // 16-byte pieces of a key's row a lane loads; of a value's
  constexpr int LD = D / 4 + 2;                                   // 16-byte pieces from one row of a warp's sums to the next
  extern __shared__ float4 pa_sums[];                             // [warp][PA_ROWS][LD]; before, the queries [KC][2][32]; then first
  int* first = reinterpret_cast<int*>(pa_sums + 4 * PA_ROWS * LD);
  uint4* queries = reinterpret_cast<uint4*>(pa_sums);
  __shared__ float2 ml[4][PA_ROWS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;
  const bool pre = (int)blockIdx.x < pre_ctas;
  pdl_launch_dependents();

  // ---- the piece
  int kvh, r0, rows, n_keys, past, t0, t1, owner = 0, slot, length = 0;
  if (!pre) {
    const int i = (int)(blockIdx.x - pre_ctas) / a.own_splits / a.own_blocks;
    owner = i / a.d.KVH;
    kvh = i - owner * a.d.KVH;
    length = a.d.lengths[owner];
  }
  pa_tokens(a, first);
  if (pre) {
    rows = first[a.d.B] * a.group;
    const PrefixLine line = pa_line(a, rows);
    const int item = line.own ? (int)blockIdx.x / line.own : 0;
    if (item >= line.items) return;
    const int piece = blockIdx.x - item * line.own;               // (of as many CTAs as items can be, each has at most one)
    kvh = item / line.blocks;
    r0 = (item - kvh * line.blocks) * PA_ROWS;
    t0 = pa_cut(a.pre_tiles, piece, line.own);
    t1 = pa_cut(a.pre_tiles, piece + 1, line.own);
    past = n_keys = a.d.prefix;
    slot = item + blockIdx.x;
  } else {
    slot = blockIdx.x - pre_ctas;
    const int rest = slot / a.own_splits, piece = slot - rest * a.own_splits;
    r0 = rest % a.own_blocks * PA_ROWS;
    const int fresh = first[owner + 1] - first[owner];
    rows = fresh * a.group;
    pa_own(a, length, fresh, past, n_keys);
    const int pieces = pa_own_pieces(a, n_keys);
    if (piece >= pieces) return;
    const int tiles = (n_keys + PA_KEYS - 1) / PA_KEYS;
    t0 = pa_cut(tiles, piece, pieces);
    t1 = pa_cut(tiles, piece + 1, pieces);
  }
  if (r0 >= rows) return;
  const bool apart = pre && a.d.prefix_k;                         // the prefix has a cache of its own
  const bf16* kb = apart ? reinterpret_cast<const bf16*>(a.d.prefix_k) + kvh * a.d.pk_head : reinterpret_cast<const bf16*>(a.d.k) + kvh * a.d.k_head;
  const bf16* vb = apart ? reinterpret_cast<const bf16*>(a.d.prefix_v) + kvh * a.d.pv_head : reinterpret_cast<const bf16*>(a.d.v) + kvh * a.d.v_head;
  const long long k_row = apart ? a.d.pk_row : a.d.k_row, v_row = apart ? a.d.pv_row : a.d.v_row, k_page = a.d.k_page, v_page = a.d.v_page;
  const int* table = a.d.page_table && !apart ? a.d.page_table + owner * a.d.ld_table : nullptr;
  const int page_of = apart ? 0 : owner, key_first = table && !pre ? a.d.prefix : 0;

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
      const bf16* p = kb + (apart ? 0 : page * k_page) + row * k_row + t4 * 8;
#pragma unroll
      for (int c = 0; c < KC; ++c) kr[j][c] = page >= 0 ? ldg_once(p + c * 32) : none;
    }
  };
  auto load_v = [&](const int2& at) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int key = (j >> 1) * 8 + 2 * t4 + (j & 1);
      const int page = __shfl_sync(0xffffffffu, at.x, key), row = __shfl_sync(0xffffffffu, at.y, key);
      const bf16* p = vb + (apart ? 0 : page * v_page) + row * v_row + g * 8;
#pragma unroll
      for (int c = 0; c < VC; ++c) vr[j][c] = page >= 0 && c * 8 + g < D / 8 ? ldg_once(p + c * 64) : none;
    }
  };
  locate(t0);
  // ---- this lane's two rows: how many keys they see; their queries
  int limit[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = r0 + g + 8 * h;
    const bool there = r < rows;
    const int i = there ? r / a.group : 0, head = kvh * a.group + (there ? r - i * a.group : 0);
    const int b = pre ? pa_find(first, a.d.B, i) : owner, t = pre ? i - first[b] : i;
    limit[h] = pre ? n_keys : min(n_keys, past + t + 1);
    for (int c = warp; c < KC; c += 4) {
      const bf16* q = reinterpret_cast<const bf16*>(a.d.q) + b * a.d.q_batch + t * a.d.q_token + head * a.d.q_head + t4 * 8 + c * 32;
      queries[(c * 2 + h) * 32 + lane] = there ? *reinterpret_cast<const uint4*>(q) : none;
    }
  }
  const int sure = pre ? n_keys : min(n_keys, past + 1);          // keys that all rows see
  float o[VC][8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int c = 0; c < VC; ++c)
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k) o[c][j][k] = 0.f;
  load_k();
  load_v(place);
  int2 here = place;
  locate(t0 + 1);
  __syncthreads();                                                // the queries are there
  for (int tile = t0; tile < t1; ++tile) {
    float s[2][4] = {};
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      const uint4 qa = lds_u4(queries + c * 64 + lane), qb = lds_u4(queries + c * 64 + 32 + lane);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        mma_bf16(s[j], qa.x, qb.x, qa.y, qb.y, kr[j][c].x, kr[j][c].y);
        mma_bf16(s[j], qa.z, qb.z, qa.w, qb.w, kr[j][c].z, kr[j][c].w);
      }
    }
    const int2 next = place;
    load_k();                                                     // (of the next tile)
    locate(tile + 2);
    const int key0 = tile * PA_KEYS + warp * 16;
    const unsigned there = __ballot_sync(0xffffffffu, here.x >= 0) & 0xffffu;
    const bool tail = key0 + 16 > sure;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k) s[j][k] *= a.scale_log2;
    if (tail || there != 0xffffu) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int key = j * 8 + 2 * t4 + (k & 1);
          if (!((there >> key) & 1) || key0 + key >= limit[k >> 1]) s[j][k] = -INFINITY;
        }
    }
    float mx[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      mx[h] = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
      mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
      mx[h] = fmaxf(m[h], fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2)));
    }
    if (__any_sync(0xffffffffu, mx[0] > m[0] || mx[1] > m[1])) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float f = m[h] == -INFINITY ? 0.f : pa_ex2(m[h] - mx[h]);
        m[h] = mx[h];
        l[h] *= f;
#pragma unroll
        for (int c = 0; c < VC; ++c)
#pragma unroll
          for (int j = 0; j < 8; ++j) o[c][j][2 * h] *= f, o[c][j][2 * h + 1] *= f;
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float ref = m[h] == -INFINITY ? 0.f : m[h];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          s[j][2 * h + k] = pa_ex2(s[j][2 * h + k] - ref);
          l[h] += s[j][2 * h + k];
        }
    }
    // weights go into the second product as bf16 (half a step is 2^-8 of a weight); their sum was taken before
    const uint32_t p0 = pack_bf16x2(s[0][0], s[0][1]), p1 = pack_bf16x2(s[0][2], s[0][3]), p2 = pack_bf16x2(s[1][0], s[1][1]), p3 = pack_bf16x2(s[1][2], s[1][3]);
    if (tail && a.d.T > 1) {                                      // 0 x NaN: values that are not finite are left out of the product, and reach the rows that see them
      bool odd = false;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int c = 0; c < VC; ++c) {
          uint32_t* w = &vr[j][c].x;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if ((w[k] & 0x7f80u) == 0x7f80u) w[k] &= 0xffff0000u, odd = true;
            if ((w[k] & 0x7f800000u) == 0x7f800000u) w[k] &= 0xffffu, odd = true;
          }
        }
      if (__any_sync(0xffffffffu, odd)) {
        for (int key = 0; key < 16; ++key) {
          const int page = __shfl_sync(0xffffffffu, here.x, key), row = __shfl_sync(0xffffffffu, here.y, key);
          if (page < 0) continue;
          const bf16* p = vb + (apart ? 0 : page * v_page) + row * v_row;
#pragma unroll
          for (int c = 0; c < VC; ++c)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int piece = c * 8 + 2 * t4 + x;
              if (piece >= D / 8) continue;
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const float v = __bfloat162float(p[piece * 8 + j]);
                if (not_finite(v)) {
                  if (key0 + key < limit[0]) o[c][j][x] += v;
                  if (key0 + key < limit[1]) o[c][j][2 + x] += v;
                }
              }
            }
        }
      }
    }
#pragma unroll
    for (int c = 0; c < VC; ++c) {
      const uint32_t* x0 = &vr[0][c].x;
      const uint32_t* x1 = &vr[1][c].x;
      const uint32_t* y0 = &vr[2][c].x;
      const uint32_t* y1 = &vr[3][c].x;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t sel = j & 1 ? 0x7632 : 0x5410;
        mma_bf16(o[c][j], p0, p1, p2, p3, __byte_perm(x0[j >> 1], x1[j >> 1], sel), __byte_perm(y0[j >> 1], y1[j >> 1], sel));
      }
    }
    load_v(next);
    here = next;
  }
  // ---- the warps' rows together: 16-byte pieces, of which eights change places so that the eight lanes that one access serves find them in different banks
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    if (t4 == 0) ml[warp][g + 8 * h] = make_float2(m[h], l[h]);
  }
  __syncthreads();                                                // (the queries are done with)
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) top = fmaxf(top, ml[w][g + 8 * h].x);
    const float f = m[h] == -INFINITY ? 1.f : pa_ex2(m[h] - top);      // (sums and values of a warp that saw nothing are zeros, or NaN)
    float4* at = pa_sums + (warp * PA_ROWS + g + 8 * h) * LD;
#pragma unroll
    for (int c = 0; c < VC; ++c)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int piece = c * 8 + 2 * t4 + x;
        if (piece < D / 8)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int p4 = piece * 2 + j;
            at[p4 ^ ((p4 >> 3) & 1)] = make_float4(o[c][4 * j][2 * h + x] * f, o[c][4 * j + 1][2 * h + x] * f, o[c][4 * j + 2][2 * h + x] * f, o[c][4 * j + 3][2 * h + x] * f);
          }
      }
  }
  __syncthreads();
  const int mine = min(PA_ROWS, rows - r0);
  float* po = (pre ? a.pre_o : a.own_o) + (long long)slot * (D * PA_ROWS);
  float2* pm = (pre ? a.pre_ml : a.own_ml) + (long long)slot * PA_ROWS;
  const int r = threadIdx.x % PA_ROWS;
  if (r >= mine) return;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    const int c4 = i * 8 + threadIdx.x / PA_ROWS, from = r * LD + (c4 ^ ((c4 >> 3) & 1));
    float4 x = pa_sums[from];
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      const float4 y = pa_sums[w * PA_ROWS * LD + from];
      x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
    }
    *reinterpret_cast<float4*>(po + (c4 * PA_ROWS + r) * 4) = x;
  }
  if (threadIdx.x < PA_ROWS) {
    float2 x = make_float2(-INFINITY, 0.f);
#pragma unroll
    for (int w = 0; w < 4; ++w) x.x = fmaxf(x.x, ml[w][r].x);
#pragma unroll
    for (int w = 0; w < 4; ++w) x.y += ml[w][r].y * (ml[w][r].x == -INFINITY ? 1.f : pa_ex2(ml[w][r].x - x.x));
    pm[r] = x;
  }
}

// The pieces of a row together: a CTA takes 8 rows of a key head, a thread four columns of one; weights follow a running maximum, so that each piece is read once, eight at a time.
constexpr int PJ_ROWS = 8, PJ_AT_ONCE = 8;
template <int D>
__global__ void __launch_bounds__(PJ_ROWS * D / 4)
prefix_join_kernel(const __grid_constant__ PrefixArgs a) {
  extern __shared__ int pa_first[];
  __shared__ __align__(16) bf16 done[PJ_ROWS][D + 8];
  __shared__ long long to[PJ_ROWS];
  const int kvh = blockIdx.y, in = threadIdx.x % PJ_ROWS, c4 = threadIdx.x / PJ_ROWS;
  pa_tokens(a, pa_first);
  const int rows = pa_first[a.d.B] * a.group, r0 = blockIdx.x * PJ_ROWS;
  pdl_wait();
  if (r0 >= rows) return;
  const int r = min(r0 + in, rows - 1), i = r / a.group, g = r - i * a.group, b = pa_find(pa_first, a.d.B, i), t = i - pa_first[b];
  int past, keys;
  pa_own(a, a.d.lengths[b], pa_first[b + 1] - pa_first[b], past, keys);
  int n_pre = 0, pre_in = 0;
  long long pre_slot = 0;
  if (a.pre_ctas) {
    const PrefixLine line = pa_line(a, rows);
    const int blk = r / a.pre_rows, item = kvh * line.blocks + blk;
    int c0, c1;
    pa_ctas_of(a, line, item, c0, c1);
    pre_in = r - blk * a.pre_rows;
    n_pre = c1 - c0 + 1;
    pre_slot = (long long)item + c0;
  }
  const int own = t * a.group + g, n = n_pre + pa_own_pieces(a, keys), own_blk = own / PA_ROWS, own_in = own - own_blk * PA_ROWS;
  const long long own_slot = (((long long)b * a.d.KVH + kvh) * a.own_blocks + own_blk) * a.own_splits;
  if (c4 == 0) to[in] = r0 + in < rows ? b * a.d.o_batch + t * a.d.o_token + (kvh * a.group + g) * a.d.o_head : -1;
  float top = -INFINITY, sum = 0.f;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p0 = 0; p0 < n; p0 += PJ_AT_ONCE) {
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
        ml[k] = a.own_ml[s * PA_ROWS + own_in];
        y[k] = *reinterpret_cast<const float4*>(a.own_o + ((s * (D / 4) + c4) * PA_ROWS + own_in) * 4);
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
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  *reinterpret_cast<uint2*>(&done[in][c4 * 4]) = make_uint2(pack_bf16x2(x.x * inv, x.y * inv), pack_bf16x2(x.z * inv, x.w * inv));
  __syncthreads();
  if (threadIdx.x < PJ_ROWS * (D / 8)) {
    const int row = threadIdx.x / (D / 8), col = (threadIdx.x % (D / 8)) * 8;
    if (to[row] >= 0) *reinterpret_cast<uint4*>(reinterpret_cast<bf16*>(a.d.out) + to[row] + col) = *reinterpret_cast<const uint4*>(&done[row][col]);
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
  LP_REQUIRE((long long)d->max_pages * d->page_size <= (1LL << 31) - 256, "lp_prefix_attention: %d pages of %d rows are too many", d->max_pages, d->page_size);
  LP_REQUIRE(d->B * (long long)d->KVH * ((d->T * (d->H / d->KVH) + PA_ROWS - 1) / PA_ROWS) <= 1 << 24, "lp_prefix_attention: %d requests of %d tokens over %d key heads are too many", d->B, d->T, d->KVH);
  LP_REQUIRE(d->prefix >= 0 && d->prefix <= (1LL << 31) - 256, "lp_prefix_attention: prefix %d", d->prefix);
  if (d->prefix_k) LP_REQUIRE(!d->page_table && d->prefix_v, "lp_prefix_attention: a prefix of its own goes with a cache of its own each");
  else if (d->page_table) LP_REQUIRE(d->prefix <= (long long)d->max_pages * d->page_size, "lp_prefix_attention: a prefix of %d rows in %d pages of %d", d->prefix, d->max_pages, d->page_size);
  else LP_REQUIRE(d->prefix == 0, "lp_prefix_attention: a prefix of %d rows that is nowhere", d->prefix);
  return 0;
}
// whether the prefix goes to the tcgen05 kernel
constexpr int PA_TC_ROWS = 16;
static bool prefix_tc(const lp_prefix_attn_desc* d) { return (long long)d->B * d->T * (d->H / d->KVH) > PA_TC_ROWS && prefix_tc_takes(d); }
// how a call is cut: what the descriptor's numbers alone decide
static size_t prefix_plan(const lp_prefix_attn_desc* d, PrefixArgs& a) {
  a.d = *d;
  a.group = d->H / d->KVH;
  const long long own = (long long)d->max_pages * d->page_size - (d->page_table ? d->prefix : 0);
  a.own_rows = (int)own;
  a.own_blocks = (d->T * a.group + PA_ROWS - 1) / PA_ROWS;
  const long long items = (long long)d->B * d->KVH * a.own_blocks, tiles = (own + PA_KEYS - 1) / PA_KEYS, room = 4LL * sm_count();
  long long splits = items >= room ? 1 : room / items;
  a.own_splits = (int)(splits < tiles ? splits : tiles > 0 ? tiles : 1);
  const long long rows = (long long)d->B * d->T * a.group;
  const bool tc = prefix_tc(d);
  const int keys = tc ? 128 : PA_KEYS;
  a.pre_rows = !tc ? PA_ROWS : rows <= 128 ? 128 : 256;
  a.pre_tiles = (int)(((long long)d->prefix + keys - 1) / keys);
  a.pre_ctas = 0;
  a.pre_slots = 0;
  if (d->prefix > 0) {
    const long long pre_items = (rows + a.pre_rows - 1) / a.pre_rows * d->KVH;
    if (tc) {
      const long long most = pre_items * a.pre_tiles;
      a.pre_ctas = (int)(most < sm_count() ? most : sm_count());
    } else {
      splits = pre_items >= room ? 1 : room / pre_items;
      a.pre_ctas = (int)((splits < a.pre_tiles ? splits : a.pre_tiles) * pre_items);
    }
    a.pre_slots = pre_items + a.pre_ctas;
  }
  a.own_slots = items * a.own_splits;
  return ((size_t)a.pre_slots * a.pre_rows + (size_t)a.own_slots * PA_ROWS) * (d->D * 4 + 8);
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
  LP_REQUIRE(ws_bytes >= need, "lp_prefix_attention: workspace too small");
  a.scale_log2 = d->scale * 1.4426950408889634f;
  const size_t pre = (size_t)a.pre_slots * a.pre_rows, mine = (size_t)a.own_slots * PA_ROWS;
  a.pre_o = reinterpret_cast<float*>(workspace);
  a.own_o = a.pre_o + pre * d->D;
  a.pre_ml = reinterpret_cast<float2*>(a.own_o + mine * d->D);
  a.own_ml = a.pre_ml + pre;
  const bool tc = a.pre_ctas && a.pre_rows != PA_ROWS;
  const int pre_ctas = tc ? 0 : a.pre_ctas;
  const long long ctas = pre_ctas + a.own_slots;
  const size_t first = (size_t)(d->B + 1) * 4;
  const dim3 join((unsigned)(((long long)d->B * d->T * a.group + PJ_ROWS - 1) / PJ_ROWS), d->KVH);
  note_launch(tc ? 3 : 2);
#define LP_PREFIX(DD)                                                                                             \
  {                                                                                                               \
    LP_CHECK_CUDA((allow_smem<prefix_rows_kernel<DD>>(pa_smem<DD>(d->B))));                                       \
    prefix_rows_kernel<DD><<<(unsigned)ctas, 128, pa_smem<DD>(d->B), stream>>>(a, pre_ctas);                      \
    LP_CHECK_CUDA(cudaGetLastError());                                                                            \
    if (tc) { if (const int rc = launch_prefix_tc(a, stream)) return rc; }                                        \
    LP_CHECK_CUDA(launch_ex(prefix_join_kernel<DD>, join, dim3(PJ_ROWS * DD / 4), first, stream, 1, true, a));    \
  }
  if (d->D == 128) LP_PREFIX(128) else if (d->D == 96) LP_PREFIX(96) else LP_PREFIX(64)
#undef LP_PREFIX
  return 0;
}
