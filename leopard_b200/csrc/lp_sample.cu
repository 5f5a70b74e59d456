// leopard_b200 — the next tokens from a step's logits, by given random numbers.
//
// Row r at temperature t > 0:  w_v = exp((z_v - max z) / t).  Words stand in the order of their logits, the largest first, equal ones by their index.  Of these are kept
//   the first top_k (0: all),  of them those before which less than top_p of their mass lies (the first in any case),  of them those with w >= min_p,
// and drawn is the first kept word, by index, up to which more than u of the kept mass lies.  t = 0 takes the largest.
//
// Weights are integers in units of 2^-43 (from a 64-bit exponential): their sums do not depend on the order in which they are taken, and the draw is the one that 64 bits give.
// A cluster of CTAs holds a row in shared memory, read once.  Nothing is sorted: what top_k and top_p keep ends at one word, which is found by counts and masses of 512 ranges of
// logits, first of all of the row, then of the range where the limit lies, until the few words left in it are put in order one by one.
#include "lp_common.cuh"
#include "lp_host.h"
#include "../../include/leopard_b200.h"

namespace lp {

constexpr int SA_THREADS = 512, SA_WARPS = SA_THREADS / 32, SA_BINS = SA_THREADS, SA_LIST = 256, SA_MAX_CTAS = 8;
constexpr int SA_MAX_SLICE = 48 * 1024;      // words that a CTA can hold
typedef unsigned long long u64;

struct SampleArgs {
  const void* logits; long long ld;
  const float* uniform;
  const float *temperature, *top_p, *min_p; const int* top_k;      // NULL: the value
  float temperature_all, top_p_all, min_p_all; int top_k_all;
  int V, slice;                           // words of a CTA
  bool vec;
  long long* out;
};
struct SaHist { unsigned n[SA_BINS]; u64 w[SA_BINS]; };
struct SaList { unsigned key[SA_LIST]; int at[SA_LIST]; u64 w[SA_LIST]; int n; };
struct alignas(16) SaShared {
  SaHist all, part[2];
  SaList list[2];
  SaList gathered;
  u64 total[2][SA_MAX_CTAS];              // of each CTA of the cluster, written by it; in turns
  float2 top[SA_MAX_CTAS];                // largest and least logit of each CTA
  int best[SA_MAX_CTAS];
  int tie;                                // a word's index, from the CTA that has it
  u64 warp_w[SA_WARPS];
  unsigned warp_n[SA_WARPS];
  float2 warp_top[SA_WARPS];
  // what all threads are told
  int bin; unsigned bin_n; u64 bin_w, above_n, above_w;
  unsigned last_rank; unsigned last_key; int last_at; u64 last_mass;
};

// a number whose order is that of the floats
__device__ __forceinline__ unsigned sa_key(float z) {
  const unsigned b = __float_as_uint(z);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float sa_of_key(unsigned k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
// 2^x for x <= 0 in units of 2^-43, rounded to nearest: 2^x = 2^n e^(f ln 2), |f| <= 1/2, the series of e^y to y^11 (the next term is below 2^-46)
__device__ __forceinline__ u64 sa_weight(double x) {
  if (!(x > -45.0)) return 0;
  const double n = rint(x), y = (x - n) * 0.69314718055994530942;
  double p = 1.0 / 39916800.0;
  p = fma(p, y, 1.0 / 3628800.0);
  p = fma(p, y, 1.0 / 362880.0);
  p = fma(p, y, 1.0 / 40320.0);
  p = fma(p, y, 1.0 / 5040.0);
  p = fma(p, y, 1.0 / 720.0);
  p = fma(p, y, 1.0 / 120.0);
  p = fma(p, y, 1.0 / 24.0);
  p = fma(p, y, 1.0 / 6.0);
  p = fma(p, y, 0.5);
  p = fma(p, y, 1.0);
  p = fma(p, y, 1.0);
  p = __longlong_as_double(__double_as_longlong(p) + ((long long)(int)n << 52));
  return (u64)__double_as_longlong(p + 512.0) - 0x4080000000000000ULL;      // (at 512 a step is 2^-43)
}
__device__ __forceinline__ u64 sa_warp_sum(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// the same place of another CTA of the cluster
template <typename T>
__device__ __forceinline__ T* sa_at(T* mine, int rank) {
  u64 to;
  asm("mapa.u64 %0, %1, %2;" : "=l"(to) : "l"(mine), "r"(rank));
  return reinterpret_cast<T*>(to);
}
__device__ __forceinline__ void sa_cluster(int ctas) {
  if (ctas > 1) cluster_sync_all();
  else __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(SA_THREADS)
sample_kernel(const __grid_constant__ SampleArgs a, int ctas) {
  extern __shared__ __align__(16) unsigned char sa_smem[];
  SaShared& s = *reinterpret_cast<SaShared*>(sa_smem);
  float* z = reinterpret_cast<float*>(sa_smem + sizeof(SaShared));
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / ctas, rank = blockIdx.x - row * ctas;
  const int v0 = rank * a.slice, count = max(0, min(a.slice, a.V - v0));
  const int part = a.slice / SA_WARPS, from = warp * part, to = min(from + part, count);      // a warp's words lie side by side

  if (ctas > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");      // (no CTA is written to before it has begun)
  const float t = a.temperature ? a.temperature[row] : a.temperature_all;
  const int top_k = a.top_k ? a.top_k[row] : a.top_k_all;
  const float top_p = a.top_p ? a.top_p[row] : a.top_p_all, min_p = a.min_p ? a.min_p[row] : a.min_p_all, u01 = a.uniform[row];

  // ---- the row, its largest and least logit
  const T* src = reinterpret_cast<const T*>(a.logits) + row * a.ld + v0;
  float hi = -INFINITY, lo = INFINITY;
  auto take = [&](int i, float x) {
    x = x > -INFINITY ? x + 0.f : -INFINITY;              // (what is not a number is never drawn; the two zeros are equal)
    z[i] = x;
    hi = fmaxf(hi, x);
    if (x > -INFINITY) lo = fminf(lo, x);
  };
  if (a.vec) {
    constexpr int N = 16 / (int)sizeof(T);
    for (int i = tid * N; i < count; i += SA_THREADS * N) {
      if (i + N <= count) {
        const uint4 u = *reinterpret_cast<const uint4*>(src + i);
        const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (N == 4) take(i + k, __uint_as_float(w[k]));
          else {
            take(i + 2 * k, __uint_as_float(w[k] << 16));
            take(i + 2 * k + 1, __uint_as_float(w[k] & 0xffff0000u));
          }
        }
      } else {
        for (int k = i; k < count; ++k) take(k, (float)src[k]);
      }
    }
  } else {
    for (int i = tid; i < count; i += SA_THREADS) take(i, (float)src[i]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
  }
  if (lane == 0) s.warp_top[warp] = make_float2(hi, lo);
  for (int i = tid; i < SA_BINS; i += SA_THREADS) s.all.n[i] = 0, s.all.w[i] = 0;
  if (tid < 2) s.list[tid].n = 0;
  __syncthreads();
  if (ctas > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (tid < ctas) {
    for (int w = 0; w < SA_WARPS; ++w) hi = fmaxf(hi, s.warp_top[w].x), lo = fminf(lo, s.warp_top[w].y);
    *sa_at(&s.top[rank], tid) = make_float2(hi, lo);
  }
  sa_cluster(ctas);
  hi = -INFINITY, lo = INFINITY;
  for (int c = 0; c < ctas; ++c) hi = fmaxf(hi, s.top[c].x), lo = fminf(lo, s.top[c].y);

  // ---- nothing to draw; the largest
  if (hi == -INFINITY || !(t > 0.f)) {                    // (the same in all CTAs of the cluster)
    int best = 0x7fffffff;
    if (hi > -INFINITY)
      for (int i = tid; i < count; i += SA_THREADS)
        if (z[i] == hi) { best = v0 + i; break; }
    best = __reduce_min_sync(0xffffffffu, best);
    if (lane == 0) s.warp_n[warp] = best;
    __syncthreads();
    if (tid == 0) {
      for (int w = 0; w < SA_WARPS; ++w) best = min(best, (int)s.warp_n[w]);
      *sa_at(&s.best[rank], 0) = best;
    }
    sa_cluster(ctas);
    if (rank == 0 && tid == 0) {
      for (int c = 0; c < ctas; ++c) best = min(best, s.best[c]);
      a.out[row] = best == 0x7fffffff ? -1 : best;
    }
    return;
  }
  if (hi == INFINITY) {                                   // only these count, and alike
    for (int i = tid; i < count; i += SA_THREADS) z[i] = z[i] == INFINITY ? 0.f : -INFINITY;
    hi = lo = 0.f;
    __syncthreads();
  }
  const double unit = 1.4426950408889634074 / (double)t, top = (double)hi;
  auto weight = [&](float x) { return sa_weight(((double)x - top) * unit); };

  // ---- what is kept: keys above last_key, and of those equal to it the ones up to last_at
  unsigned last_key = 0;
  int last_at = 0x7fffffff;
  const bool by_count = top_k > 0 && top_k < a.V, by_mass = top_p < 1.f;
  int turn = 0;                                           // of s.total
  // The word (by index) up to which more than `limit` of value(i) lies, by all CTAs; every CTA's sum is known to all when it returns.  `all`: of the sums, limit = choose(all).
  // Returns its index in the one CTA that has it, -1 in the others.
  auto locate = [&](auto value, auto choose) -> int {
    u64 sum = 0;
    for (int i = from + lane; i < to; i += 32) sum += value(i);
    sum = sa_warp_sum(sum);
    if (lane == 0) s.warp_w[warp] = sum;
    __syncthreads();
    u64 mine = 0;
    for (int w = 0; w < SA_WARPS; ++w) mine += s.warp_w[w];
    if (tid < ctas) *sa_at(&s.total[turn][rank], tid) = mine;
    sa_cluster(ctas);
    u64 all = 0, before = 0;
    for (int c = 0; c < ctas; ++c) {
      if (c == rank) before = all;
      all += s.total[turn][c];
    }
    turn ^= 1;
    const u64 limit = choose(all);
    if (limit < before || limit >= before + mine) return -1;
    u64 at = before;
    int w = 0;
    while (at + s.warp_w[w] <= limit) at += s.warp_w[w++];
    // that warp's words, a thread some of them side by side
    const int each = (part + SA_THREADS - 1) / SA_THREADS, i0 = w * part + tid * each, i1 = min(min(i0 + each, (w + 1) * part), count);
    u64 own = 0;
    for (int i = i0; i < i1; ++i) own += value(i);
    u64 run = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 up = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += up;
    }
    __syncthreads();                                      // (warp_w has been read)
    if (lane == 31) s.warp_w[warp] = run;
    __syncthreads();
    at += run - own;
    for (int k = 0; k < warp; ++k) at += s.warp_w[k];
    if (limit >= at && limit < at + own)
      for (int i = i0; i < i1; ++i) {
        const u64 v = value(i);
        if (limit < at + v) { s.tie = i; break; }
        at += v;
      }
    __syncthreads();
    return s.tie;
  };

  if (by_count || by_mass) {
    // ranges of equal width below the largest logit, as far as weights reach (30 t) or a top_k may look
    const float reach = fminf(fmaxf(30.f * t, 24.f), hi - lo), fine = reach > 0.f ? (float)SA_BINS / reach : 0.f;
    auto bin_of = [&](float x) { return (int)fminf((hi - x) * fine, (float)(SA_BINS - 1)); };
    for (int i = from + lane; i < to; i += 32)
      if (z[i] > -INFINITY) {
        const int b = bin_of(z[i]);
        const u64 w = weight(z[i]);
        atomicAdd(&s.all.n[b], 1u);
        if (w) atomicAdd(&s.all.w[b], w);
      }
    sa_cluster(ctas);
    u64 mass = 0;                                         // of what top_k has kept
    int lists = 0, parts = 0;
    // the last word before which fewer than k words or less than `limit` mass lies
    auto cut = [&](bool count_them, u64 limit, auto limit_of_mass) {
      unsigned key_lo = 0, key_hi = 0xffffffffu;
      u64 above_n = 0, above_w = 0;
      SaHist* h = &s.all;
      unsigned shift = 0;
      for (bool first = true;; first = false) {
        // every CTA adds up all CTAs' ranges, a thread one, and finds the one where the limit lies
        unsigned n = 0;
        u64 w = 0;
        for (int c = 0; c < ctas; ++c) {
          const SaHist* o = sa_at(h, c);
          n += o->n[tid];
          w += o->w[tid];
        }
        u64 run_n = n, run_w = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const u64 up_n = __shfl_up_sync(0xffffffffu, run_n, o), up_w = __shfl_up_sync(0xffffffffu, run_w, o);
          if (lane >= o) run_n += up_n, run_w += up_w;
        }
        __syncthreads();
        if (lane == 31) s.warp_n[warp] = (unsigned)run_n, s.warp_w[warp] = run_w;
        if (tid == 0) s.bin = -1;
        __syncthreads();
        u64 all_w = 0, all_n = 0;
        for (int k = 0; k < SA_WARPS; ++k) {
          if (k < warp) run_n += s.warp_n[k], run_w += s.warp_w[k];
          all_n += s.warp_n[k];
          all_w += s.warp_w[k];
        }
        if (first && !count_them) limit = limit_of_mass(all_w);
        run_n += above_n;
        run_w += above_w;
        const u64 upto = count_them ? run_n : run_w, before = upto - (count_them ? (u64)n : w);
        if (before < limit && upto >= limit) {
          s.bin = tid;
          s.bin_n = n;
          s.bin_w = w;
          s.above_n = run_n - n;
          s.above_w = run_w - w;
        }
        __syncthreads();
        const int bin = s.bin;
        if (bin < 0) {                                    // the limit is not reached: everything stays
          mass = all_w;
          return;
        }
        above_n = s.above_n;
        above_w = s.above_w;
        const unsigned in_bin = s.bin_n;
        // its keys
        if (first) {
          auto edge = [&](int b) {                        // the least key whose range is b or one above it
            unsigned l = sa_key(lo), r = sa_key(hi);
            while (l < r) {
              const unsigned m = l + ((r - l) >> 1);
              if (bin_of(sa_of_key(m)) <= b) r = m; else l = m + 1;
            }
            return l;
          };
          key_lo = edge(bin);
          key_hi = bin ? edge(bin - 1) - 1 : sa_key(hi);
        } else {
          const u64 top_of = (u64)key_hi - ((u64)bin << shift), low_of = top_of - ((1ULL << shift) - 1);
          key_lo = (long long)low_of < (long long)key_lo ? key_lo : (unsigned)low_of;
          key_hi = (unsigned)top_of;
        }
        if (in_bin <= SA_LIST) {
          // few words: each counts those before it
          SaList& mine = s.list[lists & 1];
          for (int i = from + lane; i < to; i += 32) {
            const unsigned k = sa_key(z[i]);
            if (z[i] > -INFINITY && k >= key_lo && k <= key_hi) {
              const int at = atomicAdd(&mine.n, 1);       // (below SA_LIST: the range holds in_bin words)
              mine.key[at] = k;
              mine.at[at] = v0 + i;
              mine.w[at] = weight(z[i]);
            }
          }
          if (tid == 0) s.last_rank = 0;
          sa_cluster(ctas);
          int base = 0;
          for (int c = 0; c < ctas; ++c) {
            const SaList* o = sa_at(&mine, c);
            const int m = o->n;
            if (tid < m) {
              s.gathered.key[base + tid] = o->key[tid];
              s.gathered.at[base + tid] = o->at[tid];
              s.gathered.w[base + tid] = o->w[tid];
            }
            base += m;
          }
          ++lists;
          __syncthreads();
          unsigned before_n = 0, key = 0;
          u64 before_w = 0, w_own = 0;
          int at = 0;
          bool keep = false;
          if (tid < base) {
            key = s.gathered.key[tid];
            at = s.gathered.at[tid];
            w_own = s.gathered.w[tid];
            for (int j = 0; j < base; ++j) {
              const unsigned k = s.gathered.key[j];
              if (k > key || (k == key && s.gathered.at[j] < at)) {
                ++before_n;
                before_w += s.gathered.w[j];
              }
            }
            keep = (count_them ? above_n + before_n : above_w + before_w) < limit;
            if (keep) atomicMax(&s.last_rank, before_n);
          }
          __syncthreads();
          if (keep && before_n == s.last_rank) {
            s.last_key = key;
            s.last_at = at;
            s.last_mass = above_w + before_w + w_own;
          }
          __syncthreads();
          last_key = s.last_key;
          last_at = s.last_at;
          mass = s.last_mass;
          return;
        }
        if (key_lo == key_hi) {
          // equal logits: as many as the limit allows, by their index
          const u64 w_each = weight(sa_of_key(key_lo));
          const u64 left = limit - (count_them ? above_n : above_w);      // > 0
          const u64 take_n = count_them ? left : w_each ? min((left + w_each - 1) / w_each, (u64)in_bin) : (u64)in_bin;
          const float same = sa_of_key(key_lo);
          const int i = locate([&](int k) -> u64 { return z[k] == same ? 1 : 0; }, [&](u64) { return take_n - 1; });
          if (i >= 0 && tid < ctas) *sa_at(&s.last_at, tid) = v0 + i;
          sa_cluster(ctas);
          last_key = key_lo;
          last_at = s.last_at;
          mass = above_w + take_n * w_each;
          return;
        }
        // the range in 512 parts again
        SaHist& p = s.part[parts & 1];
        ++parts;
        p.n[tid] = 0;
        p.w[tid] = 0;
        __syncthreads();
        const unsigned span = key_hi - key_lo;
        shift = 0;
        while (span >> shift >= SA_BINS) ++shift;
        for (int i = from + lane; i < to; i += 32) {
          const unsigned k = sa_key(z[i]);
          if (z[i] > -INFINITY && k >= key_lo && k <= key_hi) {
            const int b = (key_hi - k) >> shift;
            const u64 w = weight(z[i]);
            atomicAdd(&p.n[b], 1u);
            if (w) atomicAdd(&p.w[b], w);
          }
        }
        sa_cluster(ctas);
        h = &p;
      }
    };
    auto nothing = [](u64) { return (u64)0; };
    if (by_count) cut(true, (u64)top_k, nothing);
    if (by_mass) {
      auto of = [&](u64 m) -> u64 {
        const double x = ceil((double)top_p * (double)m);
        return top_p > 0.f && x >= 1.0 ? (u64)x : 1ULL;
      };
      // (the first level has the whole row's mass: what top_k has kept takes its place)
      const u64 kept = mass;
      cut(false, 0, [&](u64 m) { return of(by_count ? kept : m); });
    }
  }
  // ---- the draw
  const float least = min_p > 0.f ? fminf(min_p, 1.f) : 0.f;
  const u64 w_min = least > 0.f ? (u64)ceil((double)least * 8796093022208.0) : 0;
  const double u = (double)u01;
  const int i = locate(
      [&](int k) -> u64 {
        const float x = z[k];
        const unsigned key = sa_key(x);
        if (!(x > -INFINITY) || key < last_key || (key == last_key && v0 + k > last_at)) return 0;
        const u64 w = weight(x);
        return w >= w_min ? w : 0;
      },
      [&](u64 all) -> u64 {
        const double x = u > 0.0 ? floor(u * (double)all) : 0.0;
        return x < (double)all ? min((u64)x, all - 1) : all - 1;
      });
  if (i >= 0 && tid == 0) a.out[row] = v0 + i;
  sa_cluster(ctas);                                       // nobody leaves while others may read here
}

}  // namespace lp

extern "C" int lp_sample_tokens(const void* logits, int logits_fp32, long long ld, const float* uniform, const float* temperature, float temperature_all, const int* top_k,
                                int top_k_all, const float* top_p, float top_p_all, const float* min_p, float min_p_all, int rows, int V, long long* out, void* stream_) {
  using namespace lp;
  LP_REQUIRE(rows >= 0 && V > 0 && V <= SA_MAX_CTAS * SA_MAX_SLICE, "lp_sample_tokens: %d rows of %d words (%d at most)", rows, V, SA_MAX_CTAS * SA_MAX_SLICE);
  if (rows == 0) return 0;
  LP_REQUIRE(logits && uniform && out, "lp_sample_tokens: null argument");
  LP_REQUIRE(ld >= V || rows == 1, "lp_sample_tokens: ld %lld below %d words", ld, V);
  LP_REQUIRE(temperature || temperature_all >= 0.f, "lp_sample_tokens: temperature %g", temperature_all);
  LP_REQUIRE(top_k || top_k_all >= 0, "lp_sample_tokens: top_k %d", top_k_all);
  LP_REQUIRE(top_p || (top_p_all > 0.f && top_p_all <= 1.f), "lp_sample_tokens: top_p %g (above 0, 1 at most)", top_p_all);
  LP_REQUIRE(min_p || (min_p_all >= 0.f && min_p_all <= 1.f), "lp_sample_tokens: min_p %g (0 to 1)", min_p_all);
  // CTAs of a row: so that each has 16,384 words at most, and few rows more of them
  int ctas = 1;
  while (ctas < SA_MAX_CTAS && ((V + ctas - 1) / ctas > 16384 || ((long long)rows * ctas < sm_count() && V / ctas > 4096))) ctas *= 2;
  const int unit = SA_WARPS * 8;
  SampleArgs a = {logits, rows > 1 ? ld : 0, uniform, temperature, top_p, min_p, top_k, temperature_all, top_p_all, min_p_all, top_k_all, V, ((V + ctas - 1) / ctas + unit - 1) / unit * unit, false, out};
  const long long size = logits_fp32 ? 4 : 2;
  a.vec = reinterpret_cast<uintptr_t>(logits) % 16 == 0 && a.ld * size % 16 == 0;
  const size_t smem = sizeof(SaShared) + (size_t)a.slice * 4;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  LP_REQUIRE((long long)rows * ctas <= 2147483647LL, "lp_sample_tokens: %d rows", rows);
  note_launch(1);
  if (logits_fp32) {
    LP_CHECK_CUDA((allow_smem<sample_kernel<float>>((int)smem)));
    LP_CHECK_CUDA(launch_ex(sample_kernel<float>, dim3(rows * ctas), dim3(SA_THREADS), smem, stream, ctas, false, a, ctas));
  } else {
    LP_CHECK_CUDA((allow_smem<sample_kernel<bf16>>((int)smem)));
    LP_CHECK_CUDA(launch_ex(sample_kernel<bf16>, dim3(rows * ctas), dim3(SA_THREADS), smem, stream, ctas, false, a, ctas));
  }
  return 0;
}
