// leopard_b200 — distillation from a teacher's top logits: the loss of a row of student logits and its gradient, beside the masked LM loss of lp_train.cu.
//
// Row r with weight w != 0, teacher entries (id_k, T_k) of which those with 0 <= id_k < V count, temperature tau, hard share h:
//   t = softmax over k of T_k / tau,  p = softmax(z / tau),  p1 = softmax(z)
//   loss = (1 - h) tau^2 sum_k t_k (log t_k - log p[id_k]) + h (-log p1[y])
//   dz   = w ((1 - h) tau (p - t) + h (p1 - onehot(y)))
// A row without teacher entries has no first term, one whose y lies outside [0, V) no second.  Rows of weight 0 are zeros and their logits are not read.
#include "lp_common.cuh"
#include "lp_host.h"
#include "../../include/leopard_b200.h"

namespace lp {

constexpr int DISTILL_MAX_TOP = 1024;

struct DistillArgs {
  const void* logits; long long ld;
  const void* ids; int ids_64; long long ld_ids;
  const void* teacher; int teacher_fp32; long long ld_teacher;
  int K;
  const float* weight;
  const long long* target;
  float inv_tau, tau, hard;
  float* loss;
  bf16* dlogits; long long ldd;
  int V, Vp;
};

__device__ __forceinline__ float block_sum_f32(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) t += red[w];
  __syncthreads();
  return t;
}
__device__ __forceinline__ float block_max_f32(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = red[0];
#pragma unroll
  for (int w = 1; w < 8; ++w) t = fmaxf(t, red[w]);
  __syncthreads();
  return t;
}

// ---- pieces that the kernels share ---------------------------------------------------------------------------------
// The teacher's entries of a row into shared memory: top[k] = t_k (0 where there is none), lt[k] = log t_k, id[k] (-1).  Returns whether there are any; the whole block.
__device__ __forceinline__ bool teacher_side(const DistillArgs& a, int r, float* top, float* lt, int* id, float* red) {
  const int tid = threadIdx.x;
  float tm = -INFINITY;
  for (int k = tid; k < a.K; k += 256) {
    const long long at = (long long)r * a.ld_ids + k, at_t = (long long)r * a.ld_teacher + k;
    const long long i = a.ids_64 ? reinterpret_cast<const long long*>(a.ids)[at] : reinterpret_cast<const int*>(a.ids)[at];
    const bool in = i >= 0 && i < a.V;
    id[k] = in ? (int)i : -1;
    lt[k] = !in ? -INFINITY : a.teacher_fp32 ? reinterpret_cast<const float*>(a.teacher)[at_t] : (float)reinterpret_cast<const bf16*>(a.teacher)[at_t];
    if (in) tm = fmaxf(tm, lt[k]);
  }
  tm = block_max_f32(tm, red);
  float ts = 0.f;
  for (int k = tid; k < a.K; k += 256)
    if (lt[k] != -INFINITY) ts += expf((lt[k] - tm) * a.inv_tau);
  ts = block_sum_f32(ts, red);
  const float log_ts = logf(ts);
  for (int k = tid; k < a.K; k += 256) {
    const bool in = lt[k] != -INFINITY;
    lt[k] = in ? (lt[k] - tm) * a.inv_tau - log_ts : 0.f;
    top[k] = in ? expf(lt[k]) : 0.f;
  }
  return !(ts == 0.f);                      // a NaN stays one
}
// 2^x in one instruction (2^-22 of the value)
__device__ __forceinline__ float di_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// the largest of a warp's values (one that is not a number does not count)
__device__ __forceinline__ float warp_top(float v) {
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
// Exponents in the exponent's own units: z c - m c in one fma, where m c is rounded once and cancels out of every quotient: its rounding shifts the exponents by 2^-25 |m c|, 64 at most
// up to 2^31.  Beyond that (a mask of -1e10, say) unequal logits are 64 apart at least after a factor c, and only those equal to the maximum count: a factor of a power of two above c
// (far below it where the product would overflow) says as much, and its product is exact.
__device__ __forceinline__ float factor_at(float m, float c) {
  return fabsf(m * c) <= 2147483648.f || m == -INFINITY ? c : fabsf(m) > 1e30f ? 0x1p-40f : __uint_as_float((__float_as_uint(c) & 0x7f800000u) + 0x00800000u);
}
// minus a maximum in those units; 0 of nothing
__device__ __forceinline__ float in_units(float m, float c) { return m == -INFINITY ? 0.f : -__fmul_rn(m, c); }      // (not to be contracted: all uses have one rounding)
// what a row's gradient is made of, once its maximum and sums are known
struct RowGrad {
  float m, c, ks, kh;                       // maximum; log2(e) / tau; w (1 - h) tau / sum, w h / sum1
  float cs, ch;                             // the same without the sums: what the named entries lose of each t, and the label
  __device__ __forceinline__ float at(float z) const {
    const float d = z - m;
    float g = 0.f;
    if (ks != 0.f) g = di_ex2(d * c) * ks;
    if (kh != 0.f) g += di_ex2(d * 1.4426950408889634f) * kh;
    return g;
  }
};
// The places of [v0, v1) that the teacher or the label names are written again with their whole value: by the first entry of each id, the sum of its entries taken off.
// For after a barrier behind the row's other stores.
template <typename T>
__device__ __forceinline__ void named_places(const DistillArgs& a, const RowGrad& g, const T* row, bf16* drow, const float* top, const int* id, long long y, int v0, int v1) {
  const bool label = y >= v0 && y < v1 && g.ch != 0.f;
  for (int k = threadIdx.x; k < a.K; k += 256) {
    if (id[k] < v0 || id[k] >= v1) continue;
    float t = 0.f;
    bool first = true;
    for (int o = 0; o < a.K; ++o)
      if (id[o] == id[k]) {
        if (o < k) first = false;
        t += top[o];
      }
    if (first) drow[id[k]] = __float2bfloat16_rn(g.at((float)row[id[k]]) - g.cs * t - (label && y == id[k] ? g.ch : 0.f));
  }
  if (label && threadIdx.x == 0) {
    bool named = false;
    for (int o = 0; o < a.K; ++o) named |= id[o] == y;
    if (!named) drow[y] = __float2bfloat16_rn(g.at((float)row[y]) - g.ch);
  }
}
// loss of a row (thread 0 writes it); the whole block
template <typename T>
__device__ __forceinline__ void row_loss(const DistillArgs& a, int r, bool soft, float m, float s, float s1, const T* row, const float* top, const float* lt, const int* id,
                                         long long y, float* red) {
  const float log_s = logf(s);
  float kl = 0.f;
  if (soft)
    for (int k = threadIdx.x; k < a.K; k += 256)
      if (id[k] >= 0 && top[k] != 0.f) kl += top[k] * (lt[k] - ((float)row[id[k]] - m) * a.inv_tau + log_s);
  kl = block_sum_f32(kl, red);
  if (threadIdx.x == 0) {
    float l = soft ? (1.f - a.hard) * a.tau * a.tau * kl : 0.f;
    if (y >= 0 && y < a.V && a.hard != 0.f) l += a.hard * (logf(s1) - ((float)row[y] - m));
    a.loss[r] = l;
  }
}
__device__ __forceinline__ RowGrad row_grad(const DistillArgs& a, float w, bool soft, long long y, float m, float s, float s1) {
  RowGrad g;
  g.m = m;
  g.c = a.inv_tau * 1.4426950408889634f;
  g.cs = soft ? w * (1.f - a.hard) * a.tau : 0.f;
  g.ch = y >= 0 && y < a.V ? w * a.hard : 0.f;
  g.ks = g.cs == 0.f ? 0.f : g.cs / s;      // (a term that is not there has no part, whatever the sum is)
  g.kh = g.ch == 0.f ? 0.f : g.ch / s1;
  return g;
}

// ---- rows that fit the registers of a cluster ------------------------------------------------------------------------
// Bound by HBM: logits in, gradient out, once each.  A row is held by the registers of up to 8 CTAs (a cluster), 64 values a thread, between the sums and the gradient
// that needs them; the CTAs tell one another their maximum and sums through their shared memory.  All loads of a row are in flight at once.
// VEC values a load: 16 bytes where all rows start on 16 (and the gradient's on 8), else single values.  BOTH: a temperature and labels, two exponentials a value.
// For rows that do not start on 16 bytes (2,048 x 32,003 fp32 194 us, 2 TB/s; bf16 295) and more than 255 entries (2,048 x 32,000 with 300 280 us, of bf16 318): the next kernel takes what it can.
constexpr int DISTILL_HELD = 64;
template <typename T, int VEC, bool BOTH>
__global__ void __launch_bounds__(256, 2)
distill_held_kernel(const __grid_constant__ DistillArgs a, int ctas) {
  constexpr int N = DISTILL_HELD / VEC;
  extern __shared__ float top[];
  __shared__ float red[8];
  __shared__ float3 shared_sums;
  float* lt = top + a.K;
  int* id = reinterpret_cast<int*>(lt + a.K);
  const int r = blockIdx.x / ctas, rank = blockIdx.x % ctas, tid = threadIdx.x;
  const T* row = reinterpret_cast<const T*>(a.logits) + (long long)r * a.ld;
  bf16* drow = a.dlogits + (long long)r * a.ldd;
  const int all = (a.V + VEC - 1) / VEC, each = (all + ctas - 1) / ctas;
  const int i0 = min(all, rank * each), i1 = min(all, i0 + each);
  const int v0 = min(a.V, i0 * VEC), v1 = min(a.V, i1 * VEC);
  const float w = a.weight[r];
  if (rank == ctas - 1)
    for (int i = a.V + tid; i < a.Vp; i += 256) drow[i] = __float2bfloat16_rn(0.f);
  if (w == 0.f) {
    for (int i = i0 + tid; i < i1; i += 256) {
      if (VEC > 1 && (i + 1) * VEC <= a.V) {
        if (VEC == 8) *reinterpret_cast<uint4*>(drow + i * VEC) = make_uint4(0, 0, 0, 0);
        else *reinterpret_cast<uint2*>(drow + i * VEC) = make_uint2(0, 0);
      } else {
        for (int e = i * VEC; e < min(a.V, (i + 1) * VEC); ++e) drow[e] = __float2bfloat16_rn(0.f);
      }
    }
    if (tid == 0 && rank == 0) a.loss[r] = 0.f;
    return;
  }
  float x[DISTILL_HELD];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int i = i0 + k * 256 + tid;
    if (VEC > 1 && i < i1 && (i + 1) * VEC <= a.V) {
      const uint4 u = ldg_once(row + (long long)i * VEC);
      if (sizeof(T) == 4) {
        x[k * VEC] = __uint_as_float(u.x); x[k * VEC + 1] = __uint_as_float(u.y); x[k * VEC + 2] = __uint_as_float(u.z); x[k * VEC + 3] = __uint_as_float(u.w);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t h = e == 0 ? u.x : e == 1 ? u.y : e == 2 ? u.z : u.w;
          x[k * VEC + (2 * e) % VEC] = __uint_as_float(h << 16);
          x[k * VEC + (2 * e + 1) % VEC] = __uint_as_float(h & 0xffff0000u);
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[k * VEC + e] = i < i1 && i * VEC + e < a.V ? (float)row[(long long)i * VEC + e] : -INFINITY;
    }
  }
  const bool soft = teacher_side(a, r, top, lt, id, red);
  const long long y = a.target ? a.target[r] : -1;
  float m = x[0];
#pragma unroll
  for (int k = 1; k < DISTILL_HELD; ++k) m = fmaxf(m, x[k]);
  m = block_max_f32(m, red);
  const float ref = m == -INFINITY ? 0.f : m, c = a.inv_tau * 1.4426950408889634f;
  float s = 0.f, s1 = 0.f;
#pragma unroll
  for (int k = 0; k < DISTILL_HELD; ++k) {
    const float d = x[k] - ref, e = di_ex2(d * c);
    s += e;
    if (BOTH) s1 += di_ex2(d * 1.4426950408889634f);
    else x[k] = e;                          // the gradient is this, scaled
  }
  s = block_sum_f32(s, red);
  if (BOTH) s1 = block_sum_f32(s1, red);
  float top_m = m;
  if (ctas > 1) {
    if (tid == 0) shared_sums = make_float3(m, s, s1);
    __syncwarp();                           // (the cluster's barrier is for whole warps)
    cluster_sync_all();
    float3 part[8];
    const uint32_t here = smem_u32(&shared_sums);
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      part[q] = make_float3(-INFINITY, 0.f, 0.f);
      if (q < ctas) {
        const uint32_t there = mapa_u32(here, q);
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(part[q].x) : "r"(there) : "memory");
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(part[q].y) : "r"(there + 4) : "memory");
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(part[q].z) : "r"(there + 8) : "memory");
      }
      top_m = fmaxf(top_m, part[q].x);
    }
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");      // this CTA has read; it stays until the others have (below)
    s = s1 = 0.f;
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (q < ctas) {
        const float d = part[q].x == -INFINITY ? 0.f : part[q].x - top_m;      // sums of nothing are 0, or NaN
        s += part[q].y * di_ex2(d * c);
        if (BOTH) s1 += part[q].z * di_ex2(d * 1.4426950408889634f);
      }
  }
  if (!BOTH) s1 = s;                        // no label, or no temperature: one sum does
  const RowGrad g = row_grad(a, w, soft, y, top_m, s, s1);
  const bool some = g.ks != 0.f || g.kh != 0.f;      // (a row without terms is zeros, whatever its logits are)
  const float down = !BOTH ? (g.ks + g.kh) * (ctas > 1 && m != -INFINITY ? di_ex2((m - top_m) * c) : 1.f) : 0.f;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int i = i0 + k * 256 + tid;
#pragma unroll
    for (int e = 0; e < VEC; ++e) x[k * VEC + e] = BOTH ? g.at(x[k * VEC + e]) : some ? x[k * VEC + e] * down : 0.f;
    if (VEC > 1 && i < i1 && (i + 1) * VEC <= a.V) {
      if (VEC == 8)
        *reinterpret_cast<uint4*>(drow + (long long)i * VEC) =
            make_uint4(pack_bf16x2(x[k * VEC], x[k * VEC + 1 % VEC]), pack_bf16x2(x[k * VEC + 2 % VEC], x[k * VEC + 3 % VEC]),
                       pack_bf16x2(x[k * VEC + 4 % VEC], x[k * VEC + 5 % VEC]), pack_bf16x2(x[k * VEC + 6 % VEC], x[k * VEC + 7 % VEC]));
      else
        *reinterpret_cast<uint2*>(drow + (long long)i * VEC) = make_uint2(pack_bf16x2(x[k * VEC], x[k * VEC + 1 % VEC]), pack_bf16x2(x[k * VEC + 2 % VEC], x[k * VEC + 3 % VEC]));
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (i < i1 && i * VEC + e < a.V) drow[(long long)i * VEC + e] = __float2bfloat16_rn(x[k * VEC + e]);
    }
  }
  __syncthreads();
  named_places(a, g, row, drow, top, id, y, v0, v1);
  if (rank == 0) row_loss(a, r, soft, top_m, s, s1, row, top, lt, id, y, red);
  __syncwarp();
  if (ctas > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ---- the same, persistent: while a row is worked on, the next one's values are on their way into shared memory ----------------
// A cluster takes every n-th row that has a weight (and zeroes every n-th that has none): in a batch where the answers alone count it matters that all have as many.
// A CTA's part of the next row (64 KB of fp32) comes by one bulk copy, the next row's teacher entries into registers, a thread an entry and
// the label as one more (K <= 255), for rows that start on 16 bytes.  What is left is the chain of a row: values -> maximum -> exponentials -> sums -> gradient.
// It has one wait: every WARP sends its maximum and sums, against its own maximum, to all CTAs of the cluster (st.async on a barrier of the receiver), and takes the
// row's from the 8 x CTAs entries that arrive.  (Block sums, a barrier of the cluster and sums of sums took 4 of 7 us a row; the barrier alone 0.7, since it waits for the
// row before to be stored.)  A warp's part of the row's loss, which needs the row's sums, goes along with the next row's.
// This kernel and the one above (us, 64 entries): 300 rows of 32,000 fp32 15.3 and 22.8, 2,048 68.8 and 142, of bf16 62.6 and 177; 4,096 of 1,000 37 and 104; 512 of 128,256 73 and
// 149; one of 32,000 7.4 and 7.6.
// Measured: 4,096 rows of 128,256 fp32 logits, 64 entries, 519 us, 6.1 TB/s of logits read and gradient written (a copy's rate would be 489); 2,048 x 32,000, the label too, 69.0
// (60.9), at another temperature and 60 % of the rows 71 (45), of all rows 99 (61); of bf16 logits 4,096 x 32,000 in 119 (81), where the exponentials and the chain of a row are longer than its bytes.
constexpr int RING_TOP = 255;
constexpr int RING_LIST = 1536, RING_LOOK = 1024;      // rows that a cluster knows to be its own; weights that are looked at at once
struct __align__(16) RingEntry {             // of a warp: maximum and sums of the row; the teacher's maximum
  float m, s, s1, tm;
  float ts, loss, x, y;                      // sum over the teacher's entries of e^((T - tm) / tau); the warp's part of the loss of the row before
};
__device__ __forceinline__ void ring_send(uint32_t at, uint32_t bar, float a, float b, float c, float d) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(at), "r"(__float_as_uint(a)), "r"(__float_as_uint(b)),
               "r"(__float_as_uint(c)), "r"(__float_as_uint(d)), "r"(bar)
               : "memory");
}
template <typename T, bool BOTH, int HELD>
__global__ void __launch_bounds__(256, HELD >= 64 ? 2 : HELD >= 32 ? 3 : 5)
distill_ring_kernel(const __grid_constant__ DistillArgs a, int ctas, int rows) {
  constexpr int VEC = 16 / sizeof(T), N = HELD / VEC;
  constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
  extern __shared__ __align__(128) unsigned char ring_smem[];
  T* part = reinterpret_cast<T*>(ring_smem);                                       // [256 x HELD]
  // (what the rows write in turn: a warp that is at the next row but one has seen that all have sent for the next one, and so are done with this one)
  __shared__ RingEntry all[2][64];                                                 // [rank x 8 + warp]
  __shared__ __align__(8) uint64_t full, got[2];
  __shared__ int ids_of[2][256];
  __shared__ float es_of[2][256];
  __shared__ uint32_t bits_of[3][256 * HELD / 32];                          // the places of this part that an entry names (three: cleared while the next row is done) ...
  __shared__ uint32_t twice[2];                                                     // ... and the last row that named one twice
  __shared__ int list[RING_LIST], empty_rows[RING_LIST];                            // this cluster's rows of a weight, and of none
  __shared__ float list_weight[RING_LIST];
  __shared__ int counts[8];
  // what a thread or warp needs between rows: not in registers, which the row's values take
  __shared__ int late_id[256], state[4];                                            // a named place of the row before, for after that row's other stores; the list's numbers
  __shared__ float late_value[256], warp_loss[8];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = blockIdx.x % ctas;
  const int n_clusters = gridDim.x / ctas;
  const int vecs = (a.V + VEC - 1) / VEC, each = (vecs + ctas - 1) / ctas, i0 = min(vecs, rank * each), i1 = min(vecs, i0 + each);
  const int v0 = min(a.V, i0 * VEC), v1 = min(a.V, i1 * VEC), whole = max(0, min(i1, a.V / VEC) - i0);      // (whole: pieces of 16 bytes that the row has)
  const float c = a.inv_tau * LOG2E;
  auto row_of = [&](int r) { return reinterpret_cast<const T*>(a.logits) + (long long)r * a.ld; };
  auto fetch = [&](int r) {                                                         // one thread
    mbar_arrive_expect_tx(&full, (uint32_t)whole * 16);
    if (whole) bulk_load(part, row_of(r) + (long long)i0 * VEC, (uint32_t)whole * 16, &full);
  };
  // an entry of a row: its id (-1: none), the teacher's value; the label is entry K
  auto entry_id = [&](int r) {
    long long i = -1;
    if (r < rows && tid < a.K) {
      const long long at = (long long)r * a.ld_ids + tid;
      i = a.ids_64 ? reinterpret_cast<const long long*>(a.ids)[at] : reinterpret_cast<const int*>(a.ids)[at];
    } else if (r < rows && tid == a.K && a.target) {
      i = a.target[r];
    }
    return i;
  };
  auto entry_value = [&](int r) {
    if (r >= rows || tid >= a.K) return -INFINITY;
    const long long at = (long long)r * a.ld_teacher + tid;
    return a.teacher_fp32 ? reinterpret_cast<const float*>(a.teacher)[at] : (float)reinterpret_cast<const bf16*>(a.teacher)[at];
  };
  for (int i = tid; i < 3 * 256 * HELD / 32; i += 256) (&bits_of[0][0])[i] = 0;
  for (int v = whole * VEC + tid; v < 256 * HELD; v += 256) part[v] = (T)-INFINITY;      // copies never reach there
  // the row's last values, where they are fewer than 16 bytes, are brought by the thread that their piece falls to
  const int tail = v1 - min(v1, (i0 + whole) * VEC);
  const bool tail_here = tail > 0 && tid == whole % 256;
  if (tid == 0) {
    twice[0] = twice[1] = 0;
    mbar_init(&full, 1);
    mbar_init(&got[0], 8);
    mbar_init(&got[1], 8);
    fence_barrier_init();
  }
  __syncthreads();
  // which rows: of those of a weight the cluster's is every n_clusters-th, likewise of the others; the block looks at RING_LOOK weights at a time
  const int cluster = blockIdx.x / ctas;
  if (tid < 4) state[tid] = 0;                                                      // rows looked at, those of a weight among them, list, empty_rows
  auto look = [&]() {
    __syncthreads();
    int looked = state[0], some_before = state[1], n_list = 0, n_empty = 0;
    int list_from = (some_before - cluster + n_clusters - 1) / n_clusters, empty_from = (looked - some_before - cluster + n_clusters - 1) / n_clusters;      // (what came before)
    list_from = max(list_from, 0), empty_from = max(empty_from, 0);
    const int most = RING_LOOK / n_clusters + 2;
    while (looked < rows && n_list + most <= RING_LIST && n_empty + most <= RING_LIST) {
      float w[4];
      int mine = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = looked + tid * 4 + k;
        w[k] = i < rows ? a.weight[i] : 0.f;
        mine += w[k] != 0.f;
      }
      int before = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += up;
      }
      __syncthreads();                                                              // (counts of the last round, and the lists, have been read)
      if (lane == 31) counts[warp] = before;
      __syncthreads();
      int some = 0;
      before -= mine;
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        if (q < warp) before += counts[q];
        some += counts[q];
      }
      const int here = min(RING_LOOK, rows - looked);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const bool on = w[k] != 0.f;
        const int i = tid * 4 + k, nth = on ? some_before + before : looked - some_before + i - before;
        if (i < here && nth % n_clusters == cluster) {
          if (on) {
            list[nth / n_clusters - list_from] = looked + i;
            list_weight[nth / n_clusters - list_from] = w[k];
          } else empty_rows[nth / n_clusters - empty_from] = looked + i;
        }
        before += on;
      }
      looked += here;
      some_before += some;
      n_list = max(0, (some_before - cluster + n_clusters - 1) / n_clusters - list_from);
      n_empty = max(0, (looked - some_before - cluster + n_clusters - 1) / n_clusters - empty_from);
    }
    __syncthreads();
    if (tid == 0) { state[0] = looked; state[1] = some_before; state[2] = n_list; state[3] = n_empty; }
    __syncthreads();
    return n_list + n_empty > 0;
  };
  uint32_t steps = 0;                                                               // rows of a weight so far
  late_id[tid] = -1;
  if (lane == 0) warp_loss[warp] = 0.f;
  int row_before = -1;
  auto store_late = [&]() {
    if (late_id[tid] >= 0) a.dlogits[(long long)row_before * a.ldd + late_id[tid]] = __float2bfloat16_rn(late_value[tid]);
    late_id[tid] = -1;
  };
  __syncwarp();
  if (ctas > 1) cluster_sync_all();                                                 // no CTA sends to one that has not started
  auto send = [&](uint32_t turn, float m, float s, float s1, float tm, float ts) {
    __syncwarp();
    if (ctas == 1) {                                                                // (not launched as a cluster: st.async is for clusters)
      if (lane == 0) {
        all[turn][warp] = {m, s, s1, tm, ts, warp_loss[warp], 0.f, 0.f};
        mbar_arrive(&got[turn]);
      }
    } else {
      if (lane == 0) mbar_arrive_expect_tx(&got[turn], (uint32_t)ctas * sizeof(RingEntry));
      if (lane < ctas) {
        const uint32_t at = mapa_u32(smem_u32(&all[turn][rank * 8 + warp]), lane), bar = mapa_u32(smem_u32(&got[turn]), lane);
        ring_send(at, bar, m, s, s1, tm);
        ring_send(at + 16, bar, ts, warp_loss[warp], 0.f, 0.f);
      }
    }
  };
  auto write_loss = [&](const RingEntry* from) {                                    // of the row before, by one warp: in the order of the warps
    float l = (lane < 8 * ctas ? from[lane].loss : 0.f) + (lane + 32 < 8 * ctas ? from[lane + 32].loss : 0.f);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (lane == 0) a.loss[row_before] = l;
  };
  while (look()) {
  long long id_now = -1;
  float value = -INFINITY;
  if (state[2] > 0) {
    if (tid == 0) fetch(list[0]);      // (the part is free: thread 0 has waited for the row before)
    id_now = entry_id(list[0]);
    value = entry_value(list[0]);
  }
  for (int k = 0; k < state[3]; ++k) {
    const int r = empty_rows[k];
    bf16* drow = a.dlogits + (long long)r * a.ldd;
    for (int i = i0 + tid; i < i0 + whole; i += 256) {
      if (VEC == 8) *reinterpret_cast<uint4*>(drow + (long long)i * VEC) = make_uint4(0, 0, 0, 0);
      else *reinterpret_cast<uint2*>(drow + (long long)i * VEC) = make_uint2(0, 0);
    }
    for (int i = max(v0, (i0 + whole) * VEC) + tid; i < (rank == ctas - 1 ? a.Vp : v1); i += 256) drow[i] = __float2bfloat16_rn(0.f);
    if (tid == 0 && rank == 0) a.loss[r] = 0.f;
  }
  for (int at_row = 0; at_row < state[2]; ++at_row) {
    const int r = list[at_row];
    bf16* drow = a.dlogits + (long long)r * a.ldd;
    if (rank == ctas - 1)
      for (int i = a.V + tid; i < a.Vp; i += 256) drow[i] = __float2bfloat16_rn(0.f);
    const T* row = row_of(r);
    const uint32_t turn = steps & 1, phase = (steps >> 1) & 1;
    mbar_wait(&full, steps & 1);
    uint32_t* bits = bits_of[steps % 3];
    uint32_t* bits_before = bits_of[(steps + 2) % 3];
    ++steps;
    if (tail_here)
      for (int e = 0; e < tail; ++e) part[whole * VEC + e] = row[(i0 + whole) * VEC + e];
    // pairs of values, in two-wide arithmetic, loads and stores at fixed offsets: what bounds a row is the instructions of its 64 values a thread (1,180 a warp and row with single
    // values, a branch a load and z - max taken before the factor: 699 us instead of 519 for 4,096 x 128,256 of fp32)
    uint4 raw[N];                                                                   // (as they come: bf16 pairs are taken apart where they are used)
    constexpr int HELD_PAIRS = !BOTH && sizeof(T) == 2 ? HELD / 2 : 1;
    float2 held[HELD_PAIRS];
#pragma unroll
    for (int k = 0; k < N; ++k) raw[k] = lds_u4(part + (k * 256 + tid) * VEC);
    auto pair = [&](int k) {                                                        // two neighbouring values
      const uint4& u = raw[k * 2 / VEC];
      const int e = k % (VEC / 2);
      if (sizeof(T) == 4) return e == 0 ? make_float2(__uint_as_float(u.x), __uint_as_float(u.y)) : make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
      const uint32_t h = e == 0 ? u.x : e == 1 ? u.y : e == 2 ? u.z : u.w;
      return make_float2(__uint_as_float(h << 16), __uint_as_float(h & 0xffff0000u));
    };
    const int id = id_now >= 0 && id_now < a.V ? (int)id_now : -1;
    const bool here = id >= v0 && id < v1;
    const float z = !here ? 0.f : id < (i0 + whole) * VEC ? (float)part[id - v0] : (float)row[id];
    float m4[4] = {pair(0).x, pair(0).y, pair(1).x, pair(1).y};
#pragma unroll
    for (int k = 2; k < HELD / 2; ++k) {
      m4[(k & 1) * 2] = fmaxf(m4[(k & 1) * 2], pair(k).x);
      m4[(k & 1) * 2 + 1] = fmaxf(m4[(k & 1) * 2 + 1], pair(k).y);
    }
    float m = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
    const float mine = id >= 0 && tid < a.K ? value : -INFINITY;
    float tm = mine;
    m = warp_top(m);
    tm = warp * 32 < a.K ? warp_top(tm) : -INFINITY;
    // exponents against the maximum in the exponent's own units, rounded once: c m here and wherever the warp's sums are used
    const float cm = factor_at(m, c), lm = factor_at(m, LOG2E), ref = in_units(m, cm), lref = in_units(m, lm);
    const float2 cm2 = make_float2(cm, cm), ref2 = make_float2(ref, ref), one = make_float2(1.f, 1.f), lm2 = make_float2(lm, lm), lref2 = make_float2(lref, lref);
    float2 s2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)}, t2 = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < HELD / 2; ++k) {
      const float2 x = pair(k), y = fma2(x, cm2, ref2), e = make_float2(di_ex2(y.x), di_ex2(y.y));
      s2[k & 1] = fma2(e, one, s2[k & 1]);
      if (BOTH) {
        const float2 y1 = fma2(x, lm2, lref2);
        t2 = fma2(make_float2(di_ex2(y1.x), di_ex2(y1.y)), one, t2);
      } else if (sizeof(T) == 2) {                                                  // the gradient is this, scaled
        held[k % HELD_PAIRS] = e;
      } else {
        uint4& u = raw[k * 2 / VEC];
        if (k % 2 == 0) u.x = __float_as_uint(e.x), u.y = __float_as_uint(e.y);
        else u.z = __float_as_uint(e.x), u.w = __float_as_uint(e.y);
      }
    }
    // this thread's entry; a NaN stays one
    const float e = mine == -INFINITY ? 0.f : expf((mine - tm) * a.inv_tau);
    ids_of[turn][tid] = id;
    es_of[turn][tid] = e;
    if (here && tid < a.K) {
      const uint32_t bit = 1u << ((id - v0) & 31);
      if (atomicOr(&bits[(id - v0) >> 5], bit) & bit) twice[turn] = steps;
    }
    float s = (s2[0].x + s2[0].y) + (s2[1].x + s2[1].y), s1 = t2.x + t2.y, ts_mine = e;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, o);
      if (BOTH) s1 += __shfl_xor_sync(0xffffffffu, s1, o);
    }
    if (warp * 32 < a.K)
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) ts_mine += __shfl_xor_sync(0xffffffffu, ts_mine, o);
    send(turn, m, s, s1, tm, ts_mine);
    const int next = at_row + 1 < state[2] ? list[at_row + 1] : rows;
    const long long id_next = entry_id(next);
    const float value_next = entry_value(next);
    mbar_wait(&got[turn], phase);
    if (next < rows && tid == 0) fetch(next);                                       // all warps have read the part
    store_late();                                                                   // ... and stored the row before
    if (steps > 1 && tid < a.K) {
      const int old = ids_of[turn ^ 1][tid];
      if (old >= v0 && old < v1) bits_before[(old - v0) >> 5] = 0;
    }
    // the row's maximum and sums, from all warps of the cluster: two entries a lane
    const RingEntry* from = all[turn];
    const int n_from = 8 * ctas;
    if (rank == 0 && warp == 7 && row_before >= 0) write_loss(from);
    row_before = r;
    float4 f0 = make_float4(-INFINITY, 0.f, 0.f, 0.f), f1 = f0;
    if (lane < n_from) f0 = *reinterpret_cast<const float4*>(from + lane);
    if (lane + 32 < n_from) f1 = *reinterpret_cast<const float4*>(from + lane + 32);
    const float top = warp_top(fmaxf(f0.x, f1.x));
    const float ct = factor_at(top, c), lt = factor_at(top, LOG2E), up = in_units(top, ct), lup = in_units(top, lt);
    auto against = [&](float mw, float f, float u) { return mw == -INFINITY ? 1.f : di_ex2(u - in_units(mw, f)); };      // (sums of a warp that has nothing are 0, or NaN)
    float S = f0.y * against(f0.x, ct, up) + f1.y * against(f1.x, ct, up), S1 = BOTH ? f0.z * against(f0.x, lt, lup) + f1.z * against(f1.x, lt, lup) : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      S += __shfl_xor_sync(0xffffffffu, S, o);
      if (BOTH) S1 += __shfl_xor_sync(0xffffffffu, S1, o);
    }
    if (!BOTH) S1 = S;
    const int* ids = ids_of[turn];
    const bool has_label = ids[a.K] >= 0;
    // the teacher's: of this CTA's warps, all of which have all entries' sums between them
    float t_top = -INFINITY, ts = 0.f;
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (q * 32 < a.K) t_top = fmaxf(t_top, from[rank * 8 + q].tm);
    auto teacher_scale = [&](float tmw) { return tmw == -INFINITY ? 1.f : di_ex2((tmw - t_top) * c); };
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (q * 32 < a.K) ts += from[rank * 8 + q].ts * teacher_scale(from[rank * 8 + q].tm);
    const bool soft = !(ts == 0.f);
    const float w = list_weight[at_row];
    const float cs = soft ? w * (1.f - a.hard) * a.tau : 0.f, ch = has_label ? w * a.hard : 0.f;
    const float ks = __fdividef(cs, S), kh = __fdividef(ch, S1);                    // (2^-22 of the value; S lies in [1, V])
    auto grad = [&](float z) {
      float g = ks != 0.f ? di_ex2(fmaf(z, ct, up)) * ks : 0.f;
      if (kh != 0.f) g += di_ex2(fmaf(z, lt, lup)) * kh;
      return g;
    };
    float down = !BOTH ? (ks + kh) * against(m, ct, up) : 0.f;
    // a row without terms is zeros, whatever its logits are (0 x NaN otherwise; BOTH: the stores' bits, since values set to zero cost every row 5 %, these 3)
    const bool none = cs == 0.f && ch == 0.f;
    const uint32_t keep = BOTH && none ? 0u : ~0u;
    if (!BOTH && none) {
      down = 0.f;
#pragma unroll
      for (int k = 0; k < N; ++k) raw[k] = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int k = 0; k < HELD_PAIRS; ++k) held[k] = make_float2(0.f, 0.f);
    }
    const float2 down2 = make_float2(down, down), c2 = make_float2(ct, ct), l2 = make_float2(lt, lt), up2 = make_float2(up, up), lup2 = make_float2(lup, lup);
    const float2 ks2 = make_float2(ks, ks), kh2 = make_float2(kh, kh);
    bf16* out = drow + (long long)(i0 + tid) * VEC;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      uint32_t p[VEC / 2];
#pragma unroll
      for (int q = 0; q < VEC / 2; ++q) {
        float2 y = !BOTH && sizeof(T) == 2 ? held[(k * VEC / 2 + q) % HELD_PAIRS] : pair(k * VEC / 2 + q);
        if (BOTH) {
          const float2 e = fma2(y, c2, up2), e1 = fma2(y, l2, lup2);
          y = fma2(make_float2(di_ex2(e.x), di_ex2(e.y)), ks2, mul2(make_float2(di_ex2(e1.x), di_ex2(e1.y)), kh2));
        } else {
          y = mul2(y, down2);
        }
        p[q] = pack_bf16x2(y.x, y.y) & keep;
      }
      if (k * 256 + tid < whole) {
        if (VEC == 8) *reinterpret_cast<uint4*>(out + k * 256 * VEC) = make_uint4(p[0], p[1], p[2 % (VEC / 2)], p[3 % (VEC / 2)]);
        else *reinterpret_cast<uint2*>(out + k * 256 * VEC) = make_uint2(p[0], p[1]);
      }
    }
    if (tail_here)
      for (int e = 0; e < tail; ++e) drow[(i0 + whole) * VEC + e] = __float2bfloat16_rn(none ? 0.f : grad((float)part[whole * VEC + e]));
    // the places that entries name lose the teacher's share, the label's its own.  Of entries with one id the first writes, of the label and entries these.
    if (here) {
      const uint32_t word = (id - v0) >> 5, bit = 1u << ((id - v0) & 31);
      const bool label = ids[a.K] == id;
      float share = es_of[turn][tid] * teacher_scale(from[rank * 8 + warp].tm);
      bool writes = tid < a.K || !(bits[word] & bit);
      if (writes && tid < a.K && twice[turn] == steps) {
        share = 0.f;
        for (int o = 0; o < a.K; ++o)
          if (ids[o] == id) {
            if (o < tid) writes = false;
            share += es_of[turn][o] * teacher_scale(from[rank * 8 + (o >> 5)].tm);
          }
      }
      if (writes && ((share != 0.f && cs != 0.f) || (label && ch != 0.f))) {
        late_id[tid] = id;
        late_value[tid] = grad(z) - (soft ? cs * (share / ts) : 0.f) - (label ? ch : 0.f);
      }
    }
    if (warp * 32 <= a.K) {
      float loss = 0.f;
      if (here && tid < a.K && soft) {
        const float log_t = (value - t_top) * a.inv_tau - logf(ts), t = es_of[turn][tid] * teacher_scale(from[rank * 8 + warp].tm) / ts;
        if (t != 0.f) loss = (1.f - a.hard) * a.tau * a.tau * t * (log_t - (ct == c ? fmaf(z, c, up) * LN2 : (z - top) * a.inv_tau) + logf(S));
      }
      if (here && tid == a.K && a.hard != 0.f) loss = a.hard * (logf(S1) - (lt == LOG2E ? fmaf(z, lt, lup) * LN2 : z - top));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) loss += __shfl_xor_sync(0xffffffffu, loss, o);
      if (lane == 0) warp_loss[warp] = loss;
    }
    id_now = id_next, value = value_next;
  }
  }
  if (row_before >= 0) {                                                            // the last row's loss
    const uint32_t turn = steps & 1;
    send(turn, 0.f, 0.f, 0.f, 0.f, 0.f);
    mbar_wait(&got[turn], (steps >> 1) & 1);
    if (rank == 0 && warp == 7) write_loss(all[turn]);
  }
  __syncthreads();
  store_late();
}

// ---- longer rows: a CTA reads its row three times, mostly from the L2 (512 x 300,000 fp32 710 - 725 us, 1.3 TB/s of what has to be read and written) ---------------
template <typename T>
__global__ void __launch_bounds__(256)
distill_long_kernel(const __grid_constant__ DistillArgs a) {
  extern __shared__ float top[];
  __shared__ float red[8];
  float* lt = top + a.K;
  int* id = reinterpret_cast<int*>(lt + a.K);
  const int r = blockIdx.x, tid = threadIdx.x;
  const T* row = reinterpret_cast<const T*>(a.logits) + (long long)r * a.ld;
  bf16* drow = a.dlogits + (long long)r * a.ldd;
  const float w = a.weight[r];
  if (w == 0.f) {
    for (int i = tid * 2; i < a.Vp; i += 512) *reinterpret_cast<uint32_t*>(drow + i) = 0u;
    if (tid == 0) a.loss[r] = 0.f;
    return;
  }
  const bool soft = teacher_side(a, r, top, lt, id, red);
  const long long y = a.target ? a.target[r] : -1;
  float m = -INFINITY;
  for (int i = tid; i < a.V; i += 256) m = fmaxf(m, (float)row[i]);
  m = block_max_f32(m, red);
  const float c = a.inv_tau * 1.4426950408889634f;
  float s = 0.f, s1 = 0.f;
  for (int i = tid; i < a.V; i += 256) {
    const float d = (float)row[i] - m;
    s += di_ex2(d * c);
    s1 += di_ex2(d * 1.4426950408889634f);
  }
  s = block_sum_f32(s, red);
  s1 = block_sum_f32(s1, red);
  const RowGrad g = row_grad(a, w, soft, y, m, s, s1);
  for (int i = tid * 2; i < a.Vp; i += 512) {
    const float e = i < a.V ? g.at((float)row[i]) : 0.f, o = i + 1 < a.V ? g.at((float)row[i + 1]) : 0.f;
    *reinterpret_cast<uint32_t*>(drow + i) = pack_bf16x2(e, o);
  }
  __syncthreads();
  named_places(a, g, row, drow, top, id, y, 0, a.V);
  row_loss(a, r, soft, m, s, s1, row, top, lt, id, y, red);
}

// clusters that run at once: two CTAs an SM, as far as clusters fit the GPU's groups of SMs (asked once a kernel, device and size of cluster: 7 us)
template <auto Kernel>
static cudaError_t launch_ring(const DistillArgs& a, int rows, int ctas, size_t smem, cudaStream_t stream) {
  static std::atomic<int> fit[64][9];
  int dev = 0, n = 0;
  if (const cudaError_t rc = cudaGetDevice(&dev)) return rc;
  if (const cudaError_t rc = allow_smem<Kernel>((int)smem)) return rc;
  if (dev < 64) n = fit[dev][ctas].load(std::memory_order_relaxed);
  if (n == 0) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = ctas;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = smem;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (const cudaError_t rc = cudaOccupancyMaxActiveClusters(&n, Kernel, &cfg)) return rc;
    if (n < 1) n = 1;
    if (dev < 64) fit[dev][ctas].store(n, std::memory_order_relaxed);
  }
  if (n > rows) n = rows;
  return launch_ex(Kernel, dim3((unsigned)(n * ctas)), dim3(256), smem, stream, ctas, false, a, ctas, rows);
}

}  // namespace lp

extern "C" int lp_distill_fwd_bwd(const void* logits, int logits_fp32, long long ld, const void* ids, int ids_64, long long ld_ids,
                                  const void* teacher, int teacher_fp32, long long ld_teacher, int K, const float* weight, const long long* target, float temperature, float hard, float* loss,
                                  void* dlogits, long long ldd, int rows, int V, int Vp, void* stream_) {
  using namespace lp;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  LP_REQUIRE(logits && ids && teacher && weight && loss && dlogits && rows > 0 && V > 0, "lp_distill_fwd_bwd: bad arguments rows=%d V=%d", rows, V);
  LP_REQUIRE(K > 0 && K <= DISTILL_MAX_TOP && ld_ids >= K && ld_teacher >= K, "lp_distill_fwd_bwd: %d teacher entries a row (1 to %d), ld %lld, %lld", K,
             DISTILL_MAX_TOP, ld_ids, ld_teacher);
  LP_REQUIRE(Vp >= V && Vp % 2 == 0 && ldd % 2 == 0 && ldd >= Vp && ld >= V && (reinterpret_cast<uintptr_t>(dlogits) & 3) == 0,
             "lp_distill_fwd_bwd: Vp=%d must be even and >= V=%d, ldd=%lld even and >= Vp", Vp, V, ldd);
  // (the product of a maximum up to 1e30 and its factor, up to 2 log2(e) / temperature, is finite, and so is the square)
  LP_REQUIRE(temperature >= 1e-6f && temperature <= 1e6f, "lp_distill_fwd_bwd: temperature %g must lie in [1e-6, 1e6]", (double)temperature);
  LP_REQUIRE(hard >= 0.f && hard <= 1.f && (hard == 0.f || target), "lp_distill_fwd_bwd: a hard share of %g needs labels and lies in [0, 1]", (double)hard);
  DistillArgs a = {logits, ld, ids, ids_64, ld_ids, teacher, teacher_fp32, ld_teacher, K, weight, target, 1.f / temperature, temperature, hard, loss, reinterpret_cast<bf16*>(dlogits), ldd, V, Vp};
  note_launch();
  const size_t smem = (size_t)K * 12;
  const int ctas = (V + 256 * DISTILL_HELD - 1) / (256 * DISTILL_HELD);
  const int size = logits_fp32 ? 4 : 2;
  const bool wide = reinterpret_cast<uintptr_t>(logits) % 16 == 0 && ld * size % 16 == 0 && reinterpret_cast<uintptr_t>(dlogits) % 16 == 0 && ldd * 2 % (logits_fp32 ? 8 : 16) == 0;
  const bool both = hard != 0.f && temperature != 1.f;
  if (ctas > 8) {                           // more than a cluster holds
    if (logits_fp32) distill_long_kernel<float><<<rows, 256, smem, stream>>>(a);
    else distill_long_kernel<bf16><<<rows, 256, smem, stream>>>(a);
  } else {
    LP_REQUIRE((long long)rows * ctas < (1LL << 31), "lp_distill_fwd_bwd: %d rows of %d columns are too many", rows, V);
    cudaError_t rc;
    if (wide && K <= RING_TOP) {
#define LP_RING(T, HELD)                                                                                    \
  rc = both ? launch_ring<distill_ring_kernel<T, true, HELD>>(a, rows, ctas, (size_t)256 * HELD * size, stream) \
            : launch_ring<distill_ring_kernel<T, false, HELD>>(a, rows, ctas, (size_t)256 * HELD * size, stream)
      // few values a thread leave registers for more CTAs an SM, five and three: 4,096 rows of 1,000 fp32 37.5 us (57.9 with 64), 3,000 of 8,000 39 (50), of 4,000 with a
      // temperature and labels 49.5 (71), of 2,048 bf16 35 (72); where a row has several CTAs either way their messages cost more (1,000 of 60,000 fp32 89 us with 32, 68 with 64)
      if (V <= 256 * 8) { if (logits_fp32) LP_RING(float, 8); else LP_RING(bf16, 8); }
      else if (V <= 256 * 32) { if (logits_fp32) LP_RING(float, 32); else LP_RING(bf16, 32); }
      else { if (logits_fp32) LP_RING(float, DISTILL_HELD); else LP_RING(bf16, DISTILL_HELD); }
#undef LP_RING
      LP_CHECK_CUDA(rc);
      return 0;
    }
#define LP_HELD(T, VEC) \
  rc = both ? launch_ex(distill_held_kernel<T, VEC, true>, dim3((unsigned)rows * ctas), dim3(256), smem, stream, ctas, false, a, ctas) \
            : launch_ex(distill_held_kernel<T, VEC, false>, dim3((unsigned)rows * ctas), dim3(256), smem, stream, ctas, false, a, ctas)
    if (logits_fp32) { if (wide) LP_HELD(float, 4); else LP_HELD(float, 1); }
    else { if (wide) LP_HELD(bf16, 8); else LP_HELD(bf16, 1); }
#undef LP_HELD
    LP_CHECK_CUDA(rc);
  }
  LP_CHECK_CUDA(cudaGetLastError());
  return 0;
}
