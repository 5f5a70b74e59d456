// leopard_b200 — around a serving step's products: which rows belong to whom and where their keys and values go (tables and cache pages from the requests' lengths), and rotary
// positions, with the rows that they turn written to the cache in the same pass.
#include "lp_common.cuh"
#include "lp_host.h"
#include "../../include/leopard_b200.h"

namespace lp {

// ---- step tables ---------------------------------------------------------------------------------------------------
//   row0[b] = sum of new[0 .. b),  row r of request b:  position lengths[b] + r - row0[b],  slot = page_table[b][position / size] size + position % size
// Entries of the new rows' pages that are negative get the next pages of the free list, request after request and page after page.
// One cluster does it all.  Its CTAs share the requests, count their rows and missing pages and tell one another; every CTA adds up all of them, gives its requests their pages and, when all have, writes its
// share of the rows.  Bound by latency: the chain lengths -> table -> sums -> free list -> table -> slot, two barriers of the
// cluster: one token of 64 requests 4 us,
// 6 where all of them begin a page; 63,897 rows of 256 prompts 9.3 and 5 for the rows, 2 more where 4,385 pages are given out.
constexpr int ST_MAX_BATCH = 8192, ST_FEW = 4;      // a span of more pages than ST_FEW is looked at by a whole warp

struct StepTablesArgs {
  const int* lengths; const int* fresh;
  int* table; long long ld; int max_pages, size;
  const int* pages; int n_pages; int* used;
  int B, rows, each;                      // `each` requests a CTA
  bool wide_stores;                       // the row tables begin on 16 bytes
  int *row_seq, *row_pos; long long* slots; int* row0;
};
// the pages that a request's new rows lie in: [first, last), none where it brings nothing
__device__ __forceinline__ void st_span(const StepTablesArgs& a, int len, int fresh, int& first, int& last) {
  first = (int)min((unsigned)len / (unsigned)a.size, (unsigned)a.max_pages);
  last = fresh > 0 ? (int)min(((unsigned)len + (unsigned)fresh - 1) / (unsigned)a.size + 1, (unsigned)a.max_pages) : first;
}
// rows: a thread takes PER neighbours
template <int PER>
__device__ __forceinline__ void st_rows(const StepTablesArgs& a, const int* row0, const int* past, int thread, int threads) {
  const int steps = 32 - __clz(a.B), there = min(a.rows, row0[a.B]);
  for (int r0 = thread * PER; r0 < a.rows; r0 += threads * PER) {
    int seq[PER], pos[PER], b = -1, end = 0, page = -1;
    long long slot[PER];
    unsigned at = 0, logical = 0, in = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int r = r0 + k;
      seq[k] = pos[k] = -1;
      slot[k] = -1;
      if (r >= there) continue;
      bool look = true;
      if (b < 0 || r >= end) {            // the last request that begins at the row or before it (those that bring nothing begin where the next one does)
        b = 0;
        for (int i = steps - 1; i >= 0; --i) {
          const int next = b + (1 << i);
          if (next < a.B && row0[next] <= r) b = next;
        }
        end = row0[b + 1];
        at = (unsigned)max(past[b], 0) + (unsigned)(r - row0[b]);
        logical = at / (unsigned)a.size;
        in = at - logical * a.size;
      } else {
        ++at;
        look = ++in == (unsigned)a.size;
        if (look) ++logical, in = 0;
      }
      if (look) page = logical < (unsigned)a.max_pages ? __ldcg(a.table + b * a.ld + logical) : -1;
      seq[k] = b;
      pos[k] = (int)min(at, 2147483647u);
      if (page >= 0) slot[k] = (long long)page * a.size + in;
    }
    if (PER % 4 == 0 && a.wide_stores && r0 + PER <= a.rows) {
#pragma unroll
      for (int k = 0; k + 3 < PER; k += 4) {
        *reinterpret_cast<int4*>(a.row_seq + r0 + k) = make_int4(seq[k], seq[k + 1], seq[k + 2], seq[k + 3]);
        *reinterpret_cast<int4*>(a.row_pos + r0 + k) = make_int4(pos[k], pos[k + 1], pos[k + 2], pos[k + 3]);
        *reinterpret_cast<longlong2*>(a.slots + r0 + k) = make_longlong2(slot[k], slot[k + 1]);
        *reinterpret_cast<longlong2*>(a.slots + r0 + k + 2) = make_longlong2(slot[k + 2], slot[k + 3]);
      }
      continue;
    }
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      if (r0 + k >= a.rows) break;
      a.row_seq[r0 + k] = seq[k];
      a.row_pos[r0 + k] = pos[k];
      a.slots[r0 + k] = slot[k];
    }
  }
}
template <int THREADS, int PER>
__global__ void __launch_bounds__(THREADS)
step_tables_kernel(const __grid_constant__ StepTablesArgs a) {
  constexpr int WARPS = THREADS / 32;
  extern __shared__ int st_smem[];
  int* row0 = st_smem;                    // [B + 1]: tokens, then their sums
  int* given = row0 + a.B + 1;            // [B]: missing pages, then those given to the requests before
  int* past = given + a.B;                // [B]
  int* wide = past + a.B;                 // [each]: requests of this CTA that want many pages
  __shared__ long long warps[2][WARPS];
  __shared__ int n_wide;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, cta = blockIdx.x, ctas = gridDim.x;
  pdl_launch_dependents();
  const int base = min(max(a.used[0], 0), a.n_pages);
  if (threadIdx.x == 0) n_wide = 0;
  if (ctas > 1) cluster_sync_all();       // (no CTA is written to before it has begun)
  else __syncthreads();
  auto tell = [&](int* place, int v) {
    const uint32_t at = smem_u32(place);
    if (ctas == 1) *place = v;
    else
      for (int c = 0; c < ctas; ++c) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(mapa_u32(at, c)), "r"(v) : "memory");
  };
  const int b0 = cta * a.each, b1 = min(a.B, b0 + a.each);
  for (int b = b0 + threadIdx.x; b < b1; b += THREADS) {
    const int fresh = max(a.fresh[b], 0), len = max(a.lengths[b], 0);
    int first, last, missing = 0;
    st_span(a, len, fresh, first, last);
    if (last - first <= ST_FEW) {
#pragma unroll
      for (int i = 0; i < ST_FEW; ++i)
        if (first + i < last) missing += a.table[b * a.ld + first + i] < 0;
      tell(&given[b], missing);
    } else {
      wide[atomicAdd(&n_wide, 1)] = b;
    }
    tell(&row0[b], fresh);
    tell(&past[b], len);
  }
  __syncthreads();
  for (int i = warp; i < n_wide; i += WARPS) {
    const int b = wide[i];
    int first, last, n = 0;
    st_span(a, max(a.lengths[b], 0), max(a.fresh[b], 0), first, last);
#pragma unroll 4
    for (int k = first + lane; k < last; k += 32) n += a.table[b * a.ld + k] < 0;
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) tell(&given[b], n);
  }
  if (ctas > 1) cluster_sync_all();       // all counts are here
  else __syncthreads();
  // their sums, in place
  long long rows = 0, need = 0;
  for (int s0 = 0; s0 < a.B; s0 += THREADS) {
    const int b = s0 + threadIdx.x;
    const int fresh = b < a.B ? row0[b] : 0, missing = b < a.B ? given[b] : 0;
    long long r = fresh, m = missing;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long up_r = __shfl_up_sync(0xffffffffu, r, o), up_m = __shfl_up_sync(0xffffffffu, m, o);
      if (lane >= o) r += up_r, m += up_m;
    }
    if (lane == 31) warps[0][warp] = r, warps[1][warp] = m;
    __syncthreads();
    long long wr = lane < WARPS ? warps[0][lane] : 0, wm = lane < WARPS ? warps[1][lane] : 0;
#pragma unroll
    for (int o = 1; o < WARPS; o <<= 1) {
      const long long up_r = __shfl_up_sync(0xffffffffu, wr, o), up_m = __shfl_up_sync(0xffffffffu, wm, o);
      if (lane >= o) wr += up_r, wm += up_m;
    }
    const long long all_r = __shfl_sync(0xffffffffu, wr, WARPS - 1), all_m = __shfl_sync(0xffffffffu, wm, WARPS - 1);
    wr = __shfl_sync(0xffffffffu, wr, max(warp - 1, 0));
    wm = __shfl_sync(0xffffffffu, wm, max(warp - 1, 0));
    if (b < a.B) {
      row0[b] = (int)min(rows + r - fresh + (warp ? wr : 0), 2147483647LL);
      given[b] = (int)min(need + m - missing + (warp ? wm : 0), 2147483647LL);
    }
    rows += all_r;
    need += all_m;
    __syncthreads();
  }
  if (threadIdx.x == 0) row0[a.B] = (int)min(rows, 2147483647LL);
  __syncthreads();
  if (cta == 0 && threadIdx.x == 0) a.used[0] = (int)min((long long)a.n_pages, base + need);
  for (int b = cta * THREADS + threadIdx.x; b <= a.B; b += ctas * THREADS) a.row0[b] = row0[b];
  // pages
  for (int b = b0 + threadIdx.x; b < b1; b += THREADS) {
    int first, last;
    st_span(a, past[b], max(a.fresh[b], 0), first, last);
    if (last - first > ST_FEW) continue;
    long long at = (long long)base + given[b];
#pragma unroll
    for (int i = 0; i < ST_FEW; ++i)
      if (first + i < last && a.table[b * a.ld + first + i] < 0) {
        if (at < a.n_pages) a.table[b * a.ld + first + i] = a.pages[at];
        ++at;
      }
  }
  for (int i = warp; i < n_wide; i += WARPS) {
    const int b = wide[i];
    int first, last;
    st_span(a, past[b], max(a.fresh[b], 0), first, last);
    int* entries = a.table + b * a.ld;
    long long at = (long long)base + given[b];
    for (int k = first; k < last; k += 32) {
      const bool gap = k + lane < last && entries[k + lane] < 0;
      const unsigned gaps = __ballot_sync(0xffffffffu, gap);
      const long long mine = at + __popc(gaps & ((1u << lane) - 1));
      if (gap && mine < a.n_pages) entries[k + lane] = a.pages[mine];
      at += __popc(gaps);
    }
  }
  __threadfence();
  if (ctas > 1) cluster_sync_all();       // the table is as it will be
  else __syncthreads();
  if (PER > 0) st_rows<(PER > 0 ? PER : 1)>(a, row0, past, cta * THREADS + threadIdx.x, ctas * THREADS);
}
// many rows: all SMs write them (63,897 of 256 prompts: 7.5 us by the cluster's eight)
__global__ void __launch_bounds__(256)
step_rows_kernel(const __grid_constant__ StepTablesArgs a) {
  extern __shared__ int st_smem[];
  pdl_wait();
  for (int b = threadIdx.x; b <= a.B; b += 256) st_smem[b] = __ldcg(a.row0 + b);
  __syncthreads();
  st_rows<4>(a, st_smem, a.lengths, blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
}

// ---- rotary positions ----------------------------------------------------------------------------------------------
//   y[i], y[i'] = s (x[i] cos a - x[i'] sin a),  s (x[i'] cos a + x[i] sin a),   a = position f[i],  i' = i + n ("half") or the pairs (2i, 2i + 1) ("interleaved")
// The inverse (the gradient) turns by -a.  The angle is formed in 64 bits, in turns, of which whole ones are dropped: at position 10^6 a 32-bit angle is off by 0.03.  A CTA knows the angles of a few rows
// (shared memory) and turns all heads of them, 16 bytes and their partners a thread.  Bound by HBM: 16,384 rows of 32 heads of 128, bf16, 40 us, 6.7 TB/s; 4,796 of fp32 26.4, 5.9; 4,796 rows of 32 + 8 + 8 heads into
// a cache 22.9, 5.2.  64 such rows 3 us.
constexpr int RO_MAX_FREQ = 256;

struct RotarySeg {                        // heads of one tensor: x -> y
  const void* x; long long x_row, x_head;
  void* y; long long y_row, y_head, y_page;      // y_page: of a cache, whose rows are slots
  int heads;
  bool turned, paged;
};
struct RotaryArgs {
  RotarySeg seg[3];
  int segs, rows, D, n;                   // n frequencies: 2 n leading dimensions are turned
  const void* pos; int pos64;
  const float* freq;
  float scale, sign;
  const long long* slots; int page_size; long long n_slots;
  bool copy;                              // dimensions that are not turned are copied (not in place)
};
template <typename T> struct RotaryVec;   // 16 bytes of T
template <> struct RotaryVec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void get(const uint4& u, float* f) { f[0] = __uint_as_float(u.x), f[1] = __uint_as_float(u.y), f[2] = __uint_as_float(u.z), f[3] = __uint_as_float(u.w); }
  static __device__ __forceinline__ uint4 put(const float* f) { return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])); }
};
template <> struct RotaryVec<bf16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(const uint4& u, float* f) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
  static __device__ __forceinline__ uint4 put(const float* f) { return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])); }
};
template <typename T, bool VEC> struct RotaryRaw { typedef uint4 type; };
template <typename T> struct RotaryRaw<T, false> { typedef T type; };
template <typename T> __device__ __forceinline__ void rotary_get(const uint4& x, float* f) { RotaryVec<T>::get(x, f); }
template <typename T> __device__ __forceinline__ void rotary_put(uint4& x, const float* f) { x = RotaryVec<T>::put(f); }
template <typename T> __device__ __forceinline__ void rotary_get(const T& x, float* f) { f[0] = (float)x; }
template <typename T> __device__ __forceinline__ void rotary_put(float& x, const float* f) { x = f[0]; }
template <typename T> __device__ __forceinline__ void rotary_put(bf16& x, const float* f) { x = __float2bfloat16_rn(f[0]); }

// Cosine and sine of frequency f stand at place ro_at(f): 16-byte pieces (two frequencies) change places within fours, so that the eight lanes that one shared-memory access serves, which take pieces
// 1, 2 or 4 apart, find them in different banks (16,384 rows of 32 heads of 128, bf16: 53.6 us without, 46.4 with).
__device__ __forceinline__ int ro_piece(int p) { return p ^ ((p >> 3) & 3); }
__device__ __forceinline__ int ro_at(int f) { return 2 * ro_piece(f >> 1) + (f & 1); }
__host__ __device__ __forceinline__ int ro_row(int n) { return (n + 7) & ~7; }
// the angles' cosines and sines of `rows` rows from row0 on
template <int THREADS>
__device__ __forceinline__ void rotary_angles(const RotaryArgs& a, int row0, int rows, float2* cs) {
  for (int i = threadIdx.x; i < rows * a.n; i += THREADS) {
    const int r = i / a.n, f = i - r * a.n;
    const long long pos = a.pos64 ? reinterpret_cast<const long long*>(a.pos)[row0 + r] : reinterpret_cast<const int*>(a.pos)[row0 + r];
    double turns = (double)pos * (double)a.freq[f] * 0.15915494309189533577;      // / 2 pi
    turns -= rint(turns);
    float s, c;
    sincospif(2.f * (float)turns, &s, &c);
    cs[r * ro_row(a.n) + ro_at(f)] = make_float2(c * a.scale, s * a.sign * a.scale);
  }
}
// What a thread does of a row: a place of N dimensions and, "half", its partner; or (plain) a place that is copied.
template <typename T, bool VEC>
struct RotaryPlace {
  typedef typename RotaryRaw<T, VEC>::type Raw;
  static constexpr int N = VEC ? RotaryVec<T>::N : 1;
  const RotarySeg* g;
  int h, d, e, c;                         // head, its first dimension, its partner's (-1: none), its first angle (-1: plain)
};
// VEC: 16 bytes at a time (strides, bases and the turned dimensions are multiples of them); else single values.  A CTA takes ROWS rows; a thread the same places of all of them, the first ones' loads under
// way while the angles are formed.
template <typename T, bool HALF, bool VEC, int ROWS, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)
rotary_kernel(const __grid_constant__ RotaryArgs a) {
  typedef RotaryPlace<T, VEC> Place;
  typedef typename Place::Raw Raw;
  constexpr int N = Place::N;
  constexpr bool PAIRS = VEC && !HALF;    // a place holds its pairs
  extern __shared__ float4 ro_smem[];     // [ROWS][n, rounded up]
  __shared__ long2 where[ROWS];           // page and row of a slot (page -1: none)
  float2* cs = reinterpret_cast<float2*>(ro_smem);
  const int row0 = blockIdx.x * ROWS, rows = min(ROWS, a.rows - row0);
  const int turned = PAIRS ? 2 * a.n / N : a.n / N, plain = (a.D - 2 * a.n) / N, whole = a.D / N;
  int items[3], all = 0;
#pragma unroll
  for (int s = 0; s < 3; ++s) {
    items[s] = s < a.segs ? a.seg[s].heads * (a.seg[s].turned ? turned + (a.copy || a.seg[s].paged ? plain : 0) : whole) : 0;
    all += items[s];
  }
  if (all == 0) return;
  auto place = [&](int i) {
    Place p;
    const int s = i < items[0] ? 0 : i < items[0] + items[1] ? 1 : 2;
    p.g = &a.seg[s];
    i -= s > 0 ? items[0] : 0;
    i -= s > 1 ? items[1] : 0;
    const int units = items[s] / p.g->heads;
    p.h = i / units;
    const int u = i - p.h * units;
    p.c = p.e = -1;
    if (p.g->turned && u < turned) {
      p.c = PAIRS ? u * (N / 2) : u * N;
      p.d = VEC || HALF ? u * N : 2 * u;
      if (!PAIRS) p.e = HALF ? p.d + a.n : p.d + 1;
    } else {
      p.d = p.g->turned ? 2 * a.n + (u - turned) * N : u * N;
    }
    return p;
  };
  Raw x[ROWS], w[ROWS];
  auto load = [&](const Place& p) {
    const T* at = reinterpret_cast<const T*>(p.g->x) + row0 * p.g->x_row + p.h * p.g->x_head;
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
      if (r < rows) {
        x[r] = *reinterpret_cast<const Raw*>(at + r * p.g->x_row + p.d);
        if (!PAIRS && p.e >= 0) w[r] = *reinterpret_cast<const Raw*>(at + r * p.g->x_row + p.e);
      }
  };
  auto finish = [&](const Place& p) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      if (r >= rows) break;
      T* y = reinterpret_cast<T*>(p.g->y) + p.h * p.g->y_head;
      if (p.g->paged) {
        const long2 at = where[r];
        if (at.x < 0) continue;
        y += at.x * p.g->y_page + at.y * p.g->y_row;
      } else {
        y += (row0 + r) * p.g->y_row;
      }
      if (p.c >= 0) {
        float v[N], q[N];
        float2 m[PAIRS ? N / 2 : N];
        constexpr int ANGLES = PAIRS ? N / 2 : N;
        if constexpr (ANGLES >= 2) {
#pragma unroll
          for (int k = 0; k < ANGLES / 2; ++k) {
            const float4 two = ro_smem[r * (ro_row(a.n) / 2) + ro_piece(p.c / 2 + k)];
            m[2 * k] = make_float2(two.x, two.y);
            m[2 * k + 1] = make_float2(two.z, two.w);
          }
        } else {
          m[0] = cs[r * ro_row(a.n) + ro_at(p.c)];
        }
        rotary_get<T>(x[r], v);
        if constexpr (PAIRS) {
#pragma unroll
          for (int k = 0; k < N / 2; ++k) {
            const float v0 = v[2 * k], v1 = v[2 * k + 1];
            v[2 * k] = v0 * m[k].x - v1 * m[k].y;
            v[2 * k + 1] = v1 * m[k].x + v0 * m[k].y;
          }
        } else {
          rotary_get<T>(w[r], q);
#pragma unroll
          for (int k = 0; k < N; ++k) {
            const float v0 = v[k], q0 = q[k];
            v[k] = v0 * m[k].x - q0 * m[k].y;
            q[k] = q0 * m[k].x + v0 * m[k].y;
          }
          rotary_put<T>(w[r], q);
          *reinterpret_cast<Raw*>(y + p.e) = w[r];
        }
        rotary_put<T>(x[r], v);
      }
      *reinterpret_cast<Raw*>(y + p.d) = x[r];
    }
  };
  Place p = place(min((int)threadIdx.x, all - 1));
  if ((int)threadIdx.x < all) load(p);
  if (a.slots && (int)threadIdx.x < rows) {
    const long long slot = a.slots[row0 + threadIdx.x], page = slot / a.page_size;
    where[threadIdx.x] = make_long2(slot >= 0 && slot < a.n_slots ? page : -1, slot - page * a.page_size);
  }
  rotary_angles<THREADS>(a, row0, rows, cs);
  __syncthreads();
  for (int i = threadIdx.x; i < all;) {
    finish(p);
    i += THREADS;
    if (i < all) {
      p = place(i);
      load(p);
    }
  }
}

// ---- host ----------------------------------------------------------------------------------------------------------
template <typename T, bool HALF, bool VEC>
static int launch_rotary_rows(const RotaryArgs& a, cudaStream_t stream) {
  // four rows a CTA where there are enough of them to fill the GPU (16,384 rows 40 us, two a CTA 48; 64 registers a thread, so that four CTAs run on an SM: 43 with three), else one, by more threads (64 rows 3.5, by 256 4.4)
  const bool four = a.rows >= 8 * sm_count();
  const unsigned ctas = four ? (unsigned)((a.rows + 3) / 4) : (unsigned)a.rows;
  note_launch(1);
  if (four) rotary_kernel<T, HALF, VEC, 4, 256><<<ctas, 256, 4 * ro_row(a.n) * sizeof(float2), stream>>>(a);
  else rotary_kernel<T, HALF, VEC, 1, 512><<<ctas, 512, ro_row(a.n) * sizeof(float2), stream>>>(a);
  LP_CHECK_CUDA(cudaGetLastError());
  return 0;
}
template <typename T, bool HALF>
static int launch_rotary_as(const RotaryArgs& a, bool vec, cudaStream_t stream) {
  return vec ? launch_rotary_rows<T, HALF, true>(a, stream) : launch_rotary_rows<T, HALF, false>(a, stream);
}
static int launch_rotary(RotaryArgs& a, int fp32, int interleaved, cudaStream_t stream) {
  const long long N = fp32 ? 4 : 8;
  long long odd = a.D | (interleaved ? 2 * a.n : a.n);
  uintptr_t at = 0;
  for (int i = 0; i < a.segs; ++i) {
    const RotarySeg& g = a.seg[i];
    odd |= (a.rows > 1 ? g.x_row : 0) | (g.heads > 1 ? g.x_head | g.y_head : 0) | (a.rows > 1 || g.paged ? g.y_row : 0) | g.y_page;
    at |= reinterpret_cast<uintptr_t>(g.x) | reinterpret_cast<uintptr_t>(g.y);
  }
  const bool vec = odd % N == 0 && at % 16 == 0;
  if (fp32) return interleaved ? launch_rotary_as<float, false>(a, vec, stream) : launch_rotary_as<float, true>(a, vec, stream);
  return interleaved ? launch_rotary_as<bf16, false>(a, vec, stream) : launch_rotary_as<bf16, true>(a, vec, stream);
}

}  // namespace lp

extern "C" int lp_step_tables(const int* lengths, const int* fresh, int* page_table, long long ld_table, int max_pages, int page_size, const int* free_pages, int n_free,
                              int* used, int B, int rows, int* row_seq, int* row_pos, long long* slots, int* row0, void* stream_) {
  using namespace lp;
  LP_REQUIRE(lengths && fresh && page_table && used && row0 && (n_free == 0 || free_pages) && (rows == 0 || (row_seq && row_pos && slots)), "lp_step_tables: null argument");
  LP_REQUIRE(B > 0 && B <= ST_MAX_BATCH, "lp_step_tables: B=%d (1 to %d)", B, ST_MAX_BATCH);
  LP_REQUIRE(page_size > 0 && max_pages > 0 && (B == 1 || ld_table >= max_pages), "lp_step_tables: %d pages of %d rows, ld_table %lld", max_pages, page_size, ld_table);
  LP_REQUIRE((long long)max_pages * page_size <= 1LL << 31, "lp_step_tables: %d pages of %d rows are too many", max_pages, page_size);
  LP_REQUIRE(rows >= 0 && rows <= 1 << 30 && n_free >= 0, "lp_step_tables: rows=%d, %d free pages", rows, n_free);
  const Span table = {page_table, 4, 2, {{B, ld_table}, {max_pages, 1}}}, count = {used, 4, 1, {{1, 1}}};
  const Span reads[3] = {{lengths, 4, 1, {{B, 1}}}, {fresh, 4, 1, {{B, 1}}}, {free_pages, 4, 1, {{n_free, 1}}}};
  LP_REQUIRE(!spans_meet(table, count), "lp_step_tables: page_table and used share their memory");
  for (const Span& r : reads) LP_REQUIRE(!spans_meet(table, r) && !spans_meet(count, r), "lp_step_tables: page_table and used must share no memory with what the call reads");
  // one CTA while a thread has a row or two, then eight; above 16,384 rows they are a kernel of their own
  const bool one = rows <= 2048 && B <= 1024, small = rows <= 512 && B <= 256;
  const int ctas = one ? 1 : 8, each = (B + ctas - 1) / ctas;
  const bool wide = (reinterpret_cast<uintptr_t>(row_seq) | reinterpret_cast<uintptr_t>(row_pos) | reinterpret_cast<uintptr_t>(slots)) % 16 == 0;
  StepTablesArgs a = {lengths, fresh, page_table, B == 1 ? 0 : ld_table, max_pages, page_size, free_pages, n_free, used, B, rows, each, wide, row_seq, row_pos, slots, row0};
  const size_t smem = (size_t)(3 * B + 1 + each) * 4;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  note_launch(rows <= 16384 ? 1 : 2);
#define LP_TABLES(THREADS, PER)                                                                                                        \
  {                                                                                                                                    \
    LP_CHECK_CUDA((allow_smem<step_tables_kernel<THREADS, PER>>((int)smem)));                                                          \
    LP_CHECK_CUDA(launch_ex(step_tables_kernel<THREADS, PER>, dim3(ctas), dim3(THREADS), smem, stream, ctas, false, a));               \
  }
  if (small) LP_TABLES(256, 1) else if (rows <= 16384) LP_TABLES(1024, 1) else LP_TABLES(1024, 0)
#undef LP_TABLES
  if (rows > 16384) {
    const int blocks = (rows + 1023) / 1024;
    LP_CHECK_CUDA(launch_ex(step_rows_kernel, dim3(blocks < 2 * sm_count() ? blocks : 2 * sm_count()), dim3(256), (size_t)(B + 1) * 4, stream, 1, true, a));
  }
  return 0;
}

extern "C" int lp_rotary(const void* x, long long x_row, long long x_head, void* y, long long y_row, long long y_head, int fp32, int rows, int heads, int D, const void* positions,
                         int positions_64, const float* inv_freq, int n_freq, int interleaved, float scale, int inverse, void* stream) {
  using namespace lp;
  LP_REQUIRE(x && y && positions && (n_freq == 0 || inv_freq), "lp_rotary: null argument");
  LP_REQUIRE(rows >= 0 && heads > 0 && D > 0 && D <= 4096, "lp_rotary: %d rows of %d heads of %d (4096 at most)", rows, heads, D);
  LP_REQUIRE(n_freq >= 0 && n_freq <= RO_MAX_FREQ && 2 * n_freq <= D, "lp_rotary: %d frequencies (%d at most) for heads of %d", n_freq, RO_MAX_FREQ, D);
  LP_REQUIRE((long long)heads * D <= 1 << 20, "lp_rotary: %d heads of %d", heads, D);
  Dim places[2] = {{rows, y_row}, {heads, y_head}};
  LP_REQUIRE(strides_nest(places, 2, D), "lp_rotary: rows of the output share their memory (strides %lld, %lld)", y_row, y_head);
  if (rows == 0) return 0;
  const int elem = fp32 ? 4 : 2;
  const Span in = {x, elem, 3, {{rows, x_row}, {heads, x_head}, {D, 1}}}, out = {y, elem, 3, {{rows, y_row}, {heads, y_head}, {D, 1}}};
  const Span at = {positions, positions_64 ? 8 : 4, 1, {{rows, 1}}}, freq = {inv_freq, 4, 1, {{n_freq, 1}}};
  LP_REQUIRE((x == y && (rows == 1 || x_row == y_row) && (heads == 1 || x_head == y_head)) || !spans_meet(in, out), "lp_rotary: the output must be the input or share no memory with it");
  LP_REQUIRE(!spans_meet(out, at) && !spans_meet(out, freq), "lp_rotary: the output must share no memory with positions and inv_freq");
  RotaryArgs a = {};
  a.seg[0] = {x, x_row, x_head, y, y_row, y_head, 0, heads, true, false};
  a.segs = 1, a.rows = rows, a.D = D, a.n = n_freq;
  a.pos = positions, a.pos64 = positions_64, a.freq = inv_freq, a.scale = scale, a.sign = inverse ? -1.f : 1.f;
  a.copy = x != y;
  return launch_rotary(a, fp32, interleaved, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int lp_rotary_append(const lp_rotary_append_desc* d, void* stream) {
  using namespace lp;
  LP_REQUIRE(d != nullptr, "lp_rotary_append: null descriptor");
  LP_REQUIRE(d->q && d->q_out && d->k && d->v && d->k_pool && d->v_pool && d->positions && d->slots && (d->n_freq == 0 || d->inv_freq), "lp_rotary_append: null argument");
  LP_REQUIRE(d->rows >= 0 && d->H > 0 && d->KVH > 0 && d->D > 0 && d->D <= 4096, "lp_rotary_append: %d rows of %d and %d heads of %d (4096 at most)", d->rows, d->H, d->KVH, d->D);
  LP_REQUIRE(d->n_freq >= 0 && d->n_freq <= RO_MAX_FREQ && 2 * d->n_freq <= d->D, "lp_rotary_append: %d frequencies (%d at most) for heads of %d", d->n_freq, RO_MAX_FREQ, d->D);
  LP_REQUIRE((long long)d->H * d->D <= 1 << 20 && (long long)d->KVH * d->D <= 1 << 20, "lp_rotary_append: %d and %d heads of %d", d->H, d->KVH, d->D);
  LP_REQUIRE(d->n_pages > 0 && d->page_size > 0, "lp_rotary_append: %d pages of %d rows", d->n_pages, d->page_size);
  Dim out[2] = {{d->rows, d->o_row}, {d->H, d->o_head}};
  LP_REQUIRE(strides_nest(out, 2, d->D), "lp_rotary_append: rows of q_out share their memory (strides %lld, %lld)", d->o_row, d->o_head);
  Dim kp[3] = {{d->n_pages, d->kp_page}, {d->page_size, d->kp_row}, {d->KVH, d->kp_head}}, vp[3] = {{d->n_pages, d->vp_page}, {d->page_size, d->vp_row}, {d->KVH, d->vp_head}};
  LP_REQUIRE(strides_nest(kp, 3, d->D) && strides_nest(vp, 3, d->D), "lp_rotary_append: rows of a pool share their memory");
  if (d->rows == 0) return 0;
  const int elem = d->fp32 ? 4 : 2;
  auto heads = [&](const void* p, long long row, long long head, int n) { return Span{p, elem, 3, {{d->rows, row}, {n, head}, {d->D, 1}}}; };
  auto pool = [&](const void* p, long long page, long long row, long long head) { return Span{p, elem, 4, {{d->n_pages, page}, {d->page_size, row}, {d->KVH, head}, {d->D, 1}}}; };
  const Span writes[3] = {pool(d->k_pool, d->kp_page, d->kp_row, d->kp_head), pool(d->v_pool, d->vp_page, d->vp_row, d->vp_head), heads(d->q_out, d->o_row, d->o_head, d->H)};
  const Span reads[6] = {heads(d->q, d->q_row, d->q_head, d->H), heads(d->k, d->k_row, d->k_head, d->KVH), heads(d->v, d->v_row, d->v_head, d->KVH),
                         {d->positions, d->positions_64 ? 8 : 4, 1, {{d->rows, 1}}}, {d->inv_freq, 4, 1, {{d->n_freq, 1}}}, {d->slots, 8, 1, {{d->rows, 1}}}};
  const bool in_place = d->q == d->q_out && (d->rows == 1 || d->q_row == d->o_row) && (d->H == 1 || d->q_head == d->o_head);
  for (int w = 0; w < 3; ++w) {
    for (int r = 0; r < 6; ++r)
      LP_REQUIRE((w == 2 && r == 0 && in_place) || !spans_meet(writes[w], reads[r]), "lp_rotary_append: the pools and q_out must share no memory with what the call reads (q_out may be q)");
    for (int o = 0; o < w; ++o) LP_REQUIRE(!spans_meet(writes[w], writes[o]), "lp_rotary_append: the pools and q_out must share no memory with one another");
  }
  RotaryArgs a = {};
  a.seg[0] = {d->q, d->q_row, d->q_head, d->q_out, d->o_row, d->o_head, 0, d->H, true, false};
  a.seg[1] = {d->k, d->k_row, d->k_head, d->k_pool, d->kp_row, d->kp_head, d->n_pages > 1 ? d->kp_page : 0, d->KVH, true, true};
  a.seg[2] = {d->v, d->v_row, d->v_head, d->v_pool, d->vp_row, d->vp_head, d->n_pages > 1 ? d->vp_page : 0, d->KVH, false, true};
  a.segs = 3, a.rows = d->rows, a.D = d->D, a.n = d->n_freq;
  a.pos = d->positions, a.pos64 = d->positions_64, a.freq = d->inv_freq, a.scale = d->scale, a.sign = 1.f;
  a.slots = d->slots, a.page_size = d->page_size, a.n_slots = (long long)d->n_pages * d->page_size;
  a.copy = d->q != d->q_out;
  return launch_rotary(a, d->fp32, d->interleaved, reinterpret_cast<cudaStream_t>(stream));
}
