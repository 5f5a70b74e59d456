// leopard_b200 — around a serving step's products: which rows belong to whom and where their keys and values go (tables and cache pages from the requests' lengths), and rotary
// positions, with the rows that they turn written to the cache in the same pass.
#include "lp_common.cuh"
#include "lp_host.h"
#include "../../include/leopard_b200.h"

namespace lp {

// ---- step tables ---------------------------------------------------------------------------------------------------
//   row0[b] = sum of new[0 .. b),  row r of request b:  position lengths[b] + r - row0[b],  slot = page_table[b][position / size] size + position % size
// Entries of the new rows' pages that are negative get the next pages of the free list, request after request and page after page.
// One cluster does it all: every CTA adds up rows and missing pages of all requests (a few KB), then each gives pages to its share of them and, when all have, writes its share of
// the rows.  Bound by latency: the chain lengths -> table -> free list -> table -> slot, two barriers of the cluster.
constexpr int ST_THREADS = 1024, ST_MAX_BATCH = 8192, ST_FEW = 4;      // a span of more pages than ST_FEW is looked at by a whole warp

struct StepTablesArgs {
  const int* lengths; const int* fresh;
  int* table; long long ld; int max_pages, size;
  const int* pages; int n_pages; int* used;
  int B, rows;
  int *row_seq, *row_pos; long long* slots; int* row0;
};
// the pages that a request's new rows lie in: [first, last), none where it brings nothing
__device__ __forceinline__ void st_span(const StepTablesArgs& a, int len, int fresh, int& first, int& last) {
  first = (int)min((unsigned)len / (unsigned)a.size, (unsigned)a.max_pages);
  last = fresh > 0 ? (int)min(((long long)len + fresh + a.size - 1) / a.size, (long long)a.max_pages) : first;
}
// inclusive sum over the block's threads; `total`: of all of them
__device__ __forceinline__ long long st_scan(long long v, long long* warps, long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += up;
  }
  if (lane == 31) warps[warp] = v;
  __syncthreads();
  long long w = warps[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += up;
  }
  total = __shfl_sync(0xffffffffu, w, 31);
  const long long before = __shfl_sync(0xffffffffu, w, max(warp - 1, 0));
  __syncthreads();
  return v + (warp ? before : 0);
}
__global__ void __launch_bounds__(ST_THREADS)
step_tables_kernel(const __grid_constant__ StepTablesArgs a) {
  extern __shared__ int st_smem[];
  int* row0 = st_smem;                    // [B + 1]
  int* given = st_smem + a.B + 1;         // [B] pages given to the requests before
  __shared__ long long warps[32];
  const int lane = threadIdx.x & 31, cta = blockIdx.x, ctas = gridDim.x;
  const int base = min(max(a.used[0], 0), a.n_pages);
  long long rows = 0, need = 0;
  for (int b0 = 0; b0 < a.B; b0 += ST_THREADS) {
    const int b = b0 + threadIdx.x;
    int fresh = 0, first = 0, last = 0, missing = 0;
    if (b < a.B) {
      fresh = max(a.fresh[b], 0);
      st_span(a, max(a.lengths[b], 0), fresh, first, last);
      if (last - first <= ST_FEW)
#pragma unroll
        for (int i = 0; i < ST_FEW; ++i)
          if (first + i < last) missing += __ldcg(a.table + b * a.ld + first + i) < 0;
    }
    for (unsigned todo = __ballot_sync(0xffffffffu, last - first > ST_FEW); todo; todo &= todo - 1) {
      const int src = __ffs(todo) - 1, f = __shfl_sync(0xffffffffu, first, src), l = __shfl_sync(0xffffffffu, last, src);
      const int* entries = a.table + (long long)__shfl_sync(0xffffffffu, b, src) * a.ld;
      int n = 0;
      for (int i = f + lane; i < l; i += 32) n += __ldcg(entries + i) < 0;
      n = __reduce_add_sync(0xffffffffu, n);
      if (lane == src) missing = n;
    }
    long long all_rows, all_need;
    const long long r = st_scan(fresh, warps, all_rows), p = st_scan(missing, warps, all_need);
    if (b < a.B) {
      row0[b] = (int)min(rows + r - fresh, 2147483647LL);
      given[b] = (int)min(need + p - missing, 2147483647LL);
    }
    rows += all_rows;
    need += all_need;
  }
  if (threadIdx.x == 0) row0[a.B] = (int)min(rows, 2147483647LL);
  __syncthreads();
  cluster_sync_all();                     // everybody knows the table as it was
  if (cta == 0 && threadIdx.x == 0) a.used[0] = (int)min((long long)a.n_pages, base + need);
  for (int b = cta * ST_THREADS + threadIdx.x; b <= a.B; b += ctas * ST_THREADS) a.row0[b] = row0[b];
  // pages: a warp takes 32 requests
  const int per = (a.B + ctas * ST_THREADS - 1) / (ctas * ST_THREADS) * ST_THREADS;
  for (int b0 = cta * per; b0 < min(a.B, (cta + 1) * per); b0 += ST_THREADS) {
    const int b = b0 + threadIdx.x;
    int first = 0, last = 0;
    if (b < a.B) {
      st_span(a, max(a.lengths[b], 0), max(a.fresh[b], 0), first, last);
      if (last - first <= ST_FEW) {
        long long at = (long long)base + given[b];
        for (int i = first; i < last; ++i)
          if (__ldcg(a.table + b * a.ld + i) < 0) {
            if (at < a.n_pages) a.table[b * a.ld + i] = a.pages[at];
            ++at;
          }
      }
    }
    for (unsigned todo = __ballot_sync(0xffffffffu, last - first > ST_FEW); todo; todo &= todo - 1) {
      const int src = __ffs(todo) - 1, f = __shfl_sync(0xffffffffu, first, src), l = __shfl_sync(0xffffffffu, last, src), owner = __shfl_sync(0xffffffffu, b, src);
      int* entries = a.table + (long long)owner * a.ld;
      long long at = (long long)base + given[owner];
      for (int i0 = f; i0 < l; i0 += 32) {
        const bool gap = i0 + lane < l && __ldcg(entries + i0 + lane) < 0;
        const unsigned gaps = __ballot_sync(0xffffffffu, gap);
        const long long mine = at + __popc(gaps & ((1u << lane) - 1));
        if (gap && mine < a.n_pages) entries[i0 + lane] = a.pages[mine];
        at += __popc(gaps);
      }
    }
  }
  __syncthreads();
  cluster_sync_all();                     // ... and as it is now
  for (int r = cta * ST_THREADS + threadIdx.x; r < a.rows; r += ctas * ST_THREADS) {
    int seq = -1, pos = -1;
    long long slot = -1;
    if (r < row0[a.B]) {
      int lo = 0, hi = a.B - 1;           // the last request that begins at r or before it (those that bring nothing begin where the next one does)
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (row0[mid] <= r) lo = mid; else hi = mid - 1;
      }
      seq = lo;
      const long long at = (long long)max(a.lengths[lo], 0) + r - row0[lo];
      pos = (int)min(at, 2147483647LL);
      const long long logical = at / a.size;
      if (logical < a.max_pages) {
        const int page = __ldcg(a.table + lo * a.ld + logical);
        if (page >= 0) slot = (long long)page * a.size + (at - logical * a.size);
      }
    }
    a.row_seq[r] = seq;
    a.row_pos[r] = pos;
    a.slots[r] = slot;
  }
}

// ---- rotary positions ----------------------------------------------------------------------------------------------
//   y[i], y[i'] = s (x[i] cos a - x[i'] sin a),  s (x[i'] cos a + x[i] sin a),   a = position f[i],  i' = i + n ("half") or the pairs (2i, 2i + 1) ("interleaved")
// The inverse (the gradient) turns by -a.  The angle is formed in 64 bits, in turns, of which whole ones are dropped: at position 10^6 a 32-bit angle is off by 0.03.  A CTA knows the angles of a few rows
// (shared memory) and turns all heads of them, 16 bytes and their partners a thread.  Bound by HBM.
constexpr int RO_THREADS = 256, RO_MAX_ROWS = 4, RO_MAX_FREQ = 256;

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
template <typename T> __device__ __forceinline__ T rotary_as(float x);
template <> __device__ __forceinline__ float rotary_as<float>(float x) { return x; }
template <> __device__ __forceinline__ bf16 rotary_as<bf16>(float x) { return __float2bfloat16_rn(x); }

// the angles' cosines and sines of `rows` rows from row0 on
__device__ __forceinline__ void rotary_angles(const RotaryArgs& a, int row0, int rows, float2* cs) {
  for (int i = threadIdx.x; i < rows * a.n; i += RO_THREADS) {
    const int r = i / a.n, f = i - r * a.n;
    const long long pos = a.pos64 ? reinterpret_cast<const long long*>(a.pos)[row0 + r] : reinterpret_cast<const int*>(a.pos)[row0 + r];
    double turns = (double)pos * (double)a.freq[f] * 0.15915494309189533577;      // / 2 pi
    turns -= rint(turns);
    float s, c;
    sincospif(2.f * (float)turns, &s, &c);
    cs[i] = make_float2(c * a.scale, s * a.sign * a.scale);
  }
}
// VEC: 16 bytes at a time (strides, bases and the turned dimensions are multiples of them); else single values
template <typename T, bool HALF, bool VEC>
__global__ void __launch_bounds__(RO_THREADS)
rotary_kernel(const __grid_constant__ RotaryArgs a, int rows_each) {
  __shared__ float2 cs[RO_MAX_ROWS * RO_MAX_FREQ];
  constexpr int N = VEC ? RotaryVec<T>::N : 1;
  const int row0 = blockIdx.x * rows_each, rows = min(rows_each, a.rows - row0);
  rotary_angles(a, row0, rows, cs);
  __syncthreads();
  // units of a head: pairs (two places of N, or one place of N whose neighbours are pairs), then what is not turned
  const int turned = VEC && !HALF ? 2 * a.n / N : a.n / N, plain = (a.D - 2 * a.n) / N, whole = a.D / N;
  for (int s = 0; s < a.segs; ++s) {
    const RotarySeg& g = a.seg[s];
    const int units = g.turned ? turned + (a.copy || g.paged ? plain : 0) : whole;
    const int per_row = g.heads * units;
    for (int i = threadIdx.x; i < rows * per_row; i += RO_THREADS) {
      const int r = i / per_row, in = i - r * per_row, h = in / units, u = in - h * units;
      const T* x = reinterpret_cast<const T*>(g.x) + (row0 + r) * g.x_row + h * g.x_head;
      T* y = reinterpret_cast<T*>(g.y) + h * g.y_head;
      if (g.paged) {
        const long long slot = a.slots[row0 + r];
        if (slot < 0 || slot >= a.n_slots) continue;
        const long long page = slot / a.page_size;
        y += page * g.y_page + (slot - page * a.page_size) * g.y_row;
      } else {
        y += (row0 + r) * g.y_row;
      }
      if (!g.turned || u >= turned) {
        const int d = g.turned ? 2 * a.n + (u - turned) * N : u * N;
        if (VEC) *reinterpret_cast<uint4*>(y + d) = *reinterpret_cast<const uint4*>(x + d);
        else y[d] = x[d];
        continue;
      }
      const float2* c = cs + r * a.n;
      if (VEC && !HALF) {
        float v[N];
        RotaryVec<T>::get(*reinterpret_cast<const uint4*>(x + u * N), v);
#pragma unroll
        for (int k = 0; k < N; k += 2) {
          const float2 w = c[(u * N + k) >> 1];
          const float p = v[k] * w.x - v[k + 1] * w.y, q = v[k + 1] * w.x + v[k] * w.y;
          v[k] = p;
          v[k + 1] = q;
        }
        *reinterpret_cast<uint4*>(y + u * N) = RotaryVec<T>::put(v);
      } else if (VEC) {
        float p[N], q[N];
        RotaryVec<T>::get(*reinterpret_cast<const uint4*>(x + u * N), p);
        RotaryVec<T>::get(*reinterpret_cast<const uint4*>(x + a.n + u * N), q);
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const float2 w = c[u * N + k];
          const float p0 = p[k] * w.x - q[k] * w.y, q0 = q[k] * w.x + p[k] * w.y;
          p[k] = p0;
          q[k] = q0;
        }
        *reinterpret_cast<uint4*>(y + u * N) = RotaryVec<T>::put(p);
        *reinterpret_cast<uint4*>(y + a.n + u * N) = RotaryVec<T>::put(q);
      } else {
        const int i0 = HALF ? u : 2 * u, i1 = HALF ? u + a.n : 2 * u + 1;
        const float p = (float)x[i0], q = (float)x[i1];
        const float2 w = c[u];
        y[i0] = rotary_as<T>(p * w.x - q * w.y);
        y[i1] = rotary_as<T>(q * w.x + p * w.y);
      }
    }
  }
}

// ---- host ----------------------------------------------------------------------------------------------------------
template <typename T, bool HALF>
static int launch_rotary_as(const RotaryArgs& a, bool vec, cudaStream_t stream) {
  const int rows = a.rows >= 8 * sm_count() && a.n * RO_MAX_ROWS <= RO_MAX_ROWS * RO_MAX_FREQ ? RO_MAX_ROWS : 1;
  const dim3 grid((unsigned)((a.rows + rows - 1) / rows));
  note_launch(1);
  if (vec) rotary_kernel<T, HALF, true><<<grid, RO_THREADS, 0, stream>>>(a, rows);
  else rotary_kernel<T, HALF, false><<<grid, RO_THREADS, 0, stream>>>(a, rows);
  LP_CHECK_CUDA(cudaGetLastError());
  return 0;
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
  LP_REQUIRE(rows >= 0 && n_free >= 0, "lp_step_tables: rows=%d, %d free pages", rows, n_free);
  StepTablesArgs a = {lengths, fresh, page_table, B == 1 ? 0 : ld_table, max_pages, page_size, free_pages, n_free, used, B, rows, row_seq, row_pos, slots, row0};
  const int ctas = rows <= 4 * ST_THREADS && B <= ST_THREADS ? 1 : 8;
  const size_t smem = (size_t)(2 * B + 1) * 4;
  note_launch(1);
  LP_CHECK_CUDA((allow_smem<step_tables_kernel>((int)smem)));
  LP_CHECK_CUDA(launch_ex(step_tables_kernel, dim3(ctas), dim3(ST_THREADS), smem, reinterpret_cast<cudaStream_t>(stream_), ctas, false, a));
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
