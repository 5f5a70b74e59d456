// leopard_b200 — the next tokens from a step's logits, by given random numbers.
//
// Row r at temperature t > 0:  w_v = exp((z_v - max z) / t).  Words stand in the order of their logits, the largest first, equal ones by their index.  Of these are kept
//   the first top_k (0: all),  of them those before which less than top_p of their mass lies (the first in any case),  of them those with w >= min_p,
// and drawn is the first kept word, by index, up to which more than u of the kept mass lies.  t = 0 takes the largest.
//
// Weights are integers in units of 2^-43 (from a 64-bit exponential), each less than one unit off: their sums do not depend on the order in which they are taken and are less than V units off, 4 x 10^-8 of the
// largest weight for the largest vocabulary.  The draw is the one that 64 bits give, but where a sum lies that near a border.  What top_p sums up is in units of 2^-35 (vocabularies above 131,072:
// 2^-32): of two equal words and others below 2^-36 it takes the first alone at top_p 0.5, where the others' share would let the second in.
// A cluster of CTAs holds a row in shared memory, read once.  Nothing is sorted: what top_k and top_p keep ends at one word, which is found by counts and masses of 1,024 ranges of
// logits, first of all of the row, then of the range where the limit lies, until the few words left in it are put in order one by one.  Where the words down to the limit are few altogether (a top_k of
// 50 or 200, a sure model's top_p), one CTA takes them all and the others leave.
// Bound by latency and by passes over shared memory, at two CTAs an SM: one row of 128,256 18 us (a barrier of the cluster takes 0.5 to 1, a load 2.5, counts 2, the few words 5), 64 rows of 128,256 28 (no limit), 36
// (top_k 40) to 85 (top_p 0.9, when thousands of words are kept), 256 of 32,003 30, their logits not in L2; the bytes take 5.
#include "lp_common.cuh"
#include "lp_host.h"
#include "../../include/leopard_b200.h"

namespace lp {

constexpr int SA_THREADS = 512, SA_WARPS = SA_THREADS / 32, SA_BINS = 2 * SA_THREADS, SA_LIST = 256, SA_MAX_CTAS = 8;
constexpr int SA_MORE = SA_THREADS;          // words that one CTA finishes with (a list of them takes the place of a SaHist)
constexpr int SA_MAX_SLICE = 46 * 1024;      // words that a CTA can hold
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
// of a range of logits: words, and their mass in two parts, since 64-bit sums in shared memory are ten times slower than 32-bit ones
struct SaHist { unsigned n[SA_BINS], lo[SA_BINS], hi[SA_BINS]; };
struct alignas(16) SaList { u64 word[SA_LIST]; };      // key and, below it, what is left of 2^32 - 1 behind the index: larger numbers stand before
struct alignas(16) SaShared {
  SaHist hist[2];                         // in turns: others may read the one before until the next barrier
  SaList list[2], gathered;
  u64 sorted[SA_LIST], by_index[SA_LIST];      // masses or weights of what is gathered, in two orders
  double root[64];                        // 2^(i / 64)
  u64 total[2][SA_MAX_CTAS];              // of each CTA of the cluster, written by it; in turns
  float2 top[SA_MAX_CTAS];                // largest and least logit of each CTA
  int best[SA_MAX_CTAS], n_list[2];
  int tie;                                // a word's index, from the CTA that has it
  u64 warp_w[SA_WARPS];
  unsigned warp_n[SA_WARPS];
  float2 warp_top[SA_WARPS];
  // what all threads are told
  int bin; unsigned bin_n; u64 above_n, above_w;
  unsigned last_rank; unsigned last_key; int last_at;
};

// a number whose order is that of the floats
__device__ __forceinline__ unsigned sa_key(float z) {
  const unsigned b = __float_as_uint(z);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float sa_of_key(unsigned k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
__device__ const double SA_ROOT[64] = {      // 2^(i / 64)
    1.0, 1.0108892860517005, 1.0218971486541166, 1.0330248790212284, 1.0442737824274138, 1.0556451783605572, 1.0671404006768237, 1.0787607977571199,
    1.0905077326652577, 1.102382583307841, 1.1143867425958924, 1.1265216186082418, 1.1387886347566916, 1.1511892299529827, 1.1637248587775775, 1.1763969916502812,
    1.189207115002721, 1.202156731452703, 1.215247359980469, 1.22848053610687, 1.241857812073484, 1.255380757024691, 1.2690509571917332, 1.2828700160787783,
    1.2968395546510096, 1.3109612115247644, 1.3252366431597413, 1.339667524053303, 1.3542555469368927, 1.3690024229745905, 1.383909881963832, 1.3989796725383112,
    1.4142135623730951, 1.42961333839197, 1.4451808069770467, 1.460917794180647, 1.4768261459394993, 1.4929077282912648, 1.5091644275934228, 1.5255981507445384,
    1.5422108254079407, 1.559004400237837, 1.5759808451078865, 1.593142151342267, 1.6104903319492543, 1.6280274218573478, 1.645755478153965, 1.6636765803267364,
    1.681792830507429, 1.7001063537185235, 1.718619298122478, 1.7373338352737062, 1.7562521603732995, 1.7753764925265212, 1.7947090750031072, 1.8142521755003989,
    1.8340080864093424, 1.8539791250833855, 1.8741676341103, 1.8945759815869656, 1.9152065613971474, 1.9360617934922943, 1.9571441241754002, 1.978456026387951};
// 2^(x / 64), x <= 0: x = 64 e + i + r, |r| <= 1/2; 2^(i / 64) from the table, e^y, y = r ln 2 / 64, by its series to y^4 (the next term is 2^-44.6).  Added to a power of two, it is a whole number
// in the sum's low bits: 512 makes units of 2^-43 (off by 0.83 of one at most:
// half for the whole number, a third for the series; 2 % are not the nearest), 131072 of 2^-35, 2^20 of 2^-32 (the nearest); that power's own bits are left in.  Below x = -2944 (-inf among it) the result is that of about there, less than half a unit.
__device__ __forceinline__ u64 sa_weight_bits(double x, double power, const double* root) {
  x = __hiloint2double((int)min((unsigned)__double2hiint(x), 0xc0a70000u), __double2loint(x));
  const double m = x + 6755399441055744.0;                // 1.5 2^52: the whole number is in the low bits
  const int n = __double2loint(m);
  const double r = x - (m - 6755399441055744.0), c = 0.010830424696249145260;
  double p = fma(r, c * c * c * c / 24.0, c * c * c / 6.0);
  p = fma(p, r, c * c / 2.0);
  p = fma(p, r, c) * r;
  const double t = root[n & 63], w = fma(t, p, t);
  return (u64)__double_as_longlong(__hiloint2double(__double2hiint(w) + ((n >> 6) << 20), __double2loint(w)) + power);
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
// A few hundred words (key and index, as in SaList) of which all that can be kept are: top_k (limit, by_count) or the mass that top_p leaves (limit, if not by_count), top_p, min_p and the draw, by one CTA.  They are sorted
// by their order, cut by sums over it, sorted by their index and drawn by sums over that.  words: SA_MORE (0 behind the last), and behind them room for as many.
struct SaDraw {
  double top, unit, power, u;
  u64 power_bits, w_min;
  float top_p;
};
constexpr u64 SA_AT_512 = 0x4080000000000000ULL;
__device__ __forceinline__ u64 sa_drawn(double u, u64 all) {      // the word up to which more than this lies
  const double x = u > 0.0 ? floor(u * (double)all) : 0.0;
  return x < (double)all ? min((u64)x, all - 1) : all - 1;
}
__device__ __forceinline__ u64 sa_mass_limit(float top_p, u64 m) {
  const double x = ceil((double)top_p * (double)m);
  return top_p > 0.f && x >= 1.0 ? (u64)x : 1ULL;
}
__device__ __forceinline__ u64 sa_upto_lanes(u64 v) {             // the sum of v up to this lane
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 up = __shfl_up_sync(0xffffffffu, v, o);
    if ((int)(threadIdx.x & 31) >= o) v += up;
  }
  return v;
}
// (a warp's pairs up to 32 apart are its own 64 words)
__device__ __forceinline__ void sa_sort(u64* a, bool down) {
  for (int k = 2; k <= SA_MORE; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      if (threadIdx.x < SA_MORE / 2) {
        const int i = 2 * threadIdx.x - (threadIdx.x & (j - 1));
        const u64 x = a[i], y = a[i + j];
        if ((x > y) == (((i & k) == 0) != down)) a[i] = y, a[i + j] = x;
      }
      if (j > 32 || (j > 1 ? j >> 1 : k) > 32) __syncthreads();
      else __syncwarp();
    }
  __syncthreads();
}
// sum up to this thread, and of all
__device__ __forceinline__ u64 sa_upto_threads(SaShared& s, u64 v, u64& all) {
  v = sa_upto_lanes(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 31) s.warp_w[threadIdx.x >> 5] = v;
  __syncthreads();
  all = 0;
#pragma unroll
  for (int k = 0; k < SA_WARPS; ++k) {
    if (k < (int)(threadIdx.x >> 5)) v += s.warp_w[k];
    all += s.warp_w[k];
  }
  return v;
}
__device__ __noinline__ void sa_finish(SaShared& s, u64* words, int n, bool by_count, u64 limit, bool by_mass, const SaDraw& d, long long* out) {
  u64* values = words + SA_MORE;
  const int tid = threadIdx.x;
  sa_sort(words, true);
  int stay = by_count ? (int)min(limit, (u64)n) : n;
  u64 word = words[tid], all;
  const double x = ((double)sa_of_key((unsigned)(word >> 32)) - d.top) * d.unit;
  if (by_mass) {
    const u64 v = tid < stay ? sa_weight_bits(x, d.power, s.root) - d.power_bits : 0, before = sa_upto_threads(s, v, all) - v;
    if (by_count) limit = sa_mass_limit(d.top_p, all);            // (of what top_k has kept)
    stay = __syncthreads_count(tid < stay && before < limit);
  }
  if (tid < stay) {
    const u64 w = sa_weight_bits(x, 512.0, s.root) - SA_AT_512;
    values[tid] = w >= d.w_min ? w : 0;
  }
  words[tid] = tid < stay ? (u64)(unsigned)~(unsigned)word << 32 | (unsigned)tid : ~0ULL;
  __syncthreads();
  sa_sort(words, false);
  word = words[tid];
  const u64 w = word != ~0ULL ? values[(unsigned)word] : 0, end = sa_upto_threads(s, w, all), lies = sa_drawn(d.u, all);
  if (lies >= end - w && lies < end) *out = (long long)(word >> 32);
}
struct SaByCount { static constexpr bool value = false; };
struct SaByMass { static constexpr bool value = true; };
template <int CTAS>
__device__ __forceinline__ void sa_cluster() {
  if (CTAS > 1) cluster_sync_all();
  else __syncthreads();
}

template <typename T, int CTAS>
__global__ void __launch_bounds__(SA_THREADS, 2)
sample_kernel(const __grid_constant__ SampleArgs a) {
  extern __shared__ __align__(16) unsigned char sa_smem[];
  SaShared& s = *reinterpret_cast<SaShared*>(sa_smem);
  float* z = reinterpret_cast<float*>(sa_smem + sizeof(SaShared));
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / CTAS, rank = blockIdx.x % CTAS;
  const int v0 = rank * a.slice, count = max(0, min(a.slice, a.V - v0));
  const int part = a.slice / SA_WARPS, from = warp * part;      // a warp's words lie side by side
  if (CTAS > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");         // (no CTA is written to before it has begun)
  const float t = a.temperature ? a.temperature[row] : a.temperature_all;
  const int top_k = a.top_k ? a.top_k[row] : a.top_k_all;
  const float top_p = a.top_p ? a.top_p[row] : a.top_p_all, min_p = a.min_p ? a.min_p[row] : a.min_p_all, u01 = a.uniform[row];

  const double root = tid < 64 ? SA_ROOT[tid] : 0.0;

  // ---- the row (-inf behind its end), its largest and least logit
  const T* src = reinterpret_cast<const T*>(a.logits) + row * a.ld + v0;
  float hi = -INFINITY, lo = INFINITY;
  auto take = [&](float x) {
    x = x > -INFINITY ? x + 0.f : -INFINITY;              // (what is not a number is never drawn; the two zeros are equal)
    hi = fmaxf(hi, x);
    if (x > -INFINITY) lo = fminf(lo, x);
    return x;
  };
  int done = 0;
  if (a.vec) {
    constexpr int N = 16 / (int)sizeof(T), AT_ONCE = 4;
    const int whole = count / N;
    done = whole * N;
    for (int i0 = tid; i0 < whole; i0 += SA_THREADS * AT_ONCE) {
      uint4 u[AT_ONCE];
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k)
        if (i0 + k * SA_THREADS < whole) u[k] = ldg_once(src + (long long)(i0 + k * SA_THREADS) * N);
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) {
        const int i = i0 + k * SA_THREADS;
        if (i >= whole) continue;
        if (N == 4) {
          *reinterpret_cast<float4*>(z + i * 4) = make_float4(take(__uint_as_float(u[k].x)), take(__uint_as_float(u[k].y)), take(__uint_as_float(u[k].z)), take(__uint_as_float(u[k].w)));
        } else {
          const float2 a0 = unpack_bf16x2(u[k].x), a1 = unpack_bf16x2(u[k].y), a2 = unpack_bf16x2(u[k].z), a3 = unpack_bf16x2(u[k].w);
          *reinterpret_cast<float4*>(z + i * 8) = make_float4(take(a0.x), take(a0.y), take(a1.x), take(a1.y));
          *reinterpret_cast<float4*>(z + i * 8 + 4) = make_float4(take(a2.x), take(a2.y), take(a3.x), take(a3.y));
        }
      }
    }
  } else {
    constexpr int AT_ONCE = 8;
    done = count;
    for (int i0 = tid; i0 < count; i0 += SA_THREADS * AT_ONCE) {
      float x[AT_ONCE];
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k)
        if (i0 + k * SA_THREADS < count) x[k] = (float)src[i0 + k * SA_THREADS];
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k)
        if (i0 + k * SA_THREADS < count) z[i0 + k * SA_THREADS] = take(x[k]);
    }
  }
  for (int i = done + tid; i < a.slice; i += SA_THREADS) z[i] = i < count ? take((float)src[i]) : -INFINITY;
  auto top_of_warp = [&]() {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    }
  };
  top_of_warp();
  if (lane == 0) s.warp_top[warp] = make_float2(hi, lo);
  for (int i = tid; i < (int)(sizeof(s.hist) / 4); i += SA_THREADS) reinterpret_cast<unsigned*>(s.hist)[i] = 0;
  if (tid < 2) s.n_list[tid] = 0;
  if (tid < 64) s.root[tid] = root;
  __syncthreads();
  if (CTAS > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (warp == 0) {
    hi = s.warp_top[lane % SA_WARPS].x, lo = s.warp_top[lane % SA_WARPS].y;
    top_of_warp();
    if (lane < CTAS) *sa_at(&s.top[rank], lane) = make_float2(hi, lo);
  }
  sa_cluster<CTAS>();
  hi = -INFINITY, lo = INFINITY;
#pragma unroll
  for (int c = 0; c < CTAS; ++c) hi = fmaxf(hi, s.top[c].x), lo = fminf(lo, s.top[c].y);

  // ---- nothing to draw; the largest
  if (hi == -INFINITY || !(t > 0.f) || top_k == 1) {      // (the same in all CTAs of the cluster)
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
    sa_cluster<CTAS>();
    if (rank == 0 && tid == 0) {
      for (int c = 0; c < CTAS; ++c) best = min(best, s.best[c]);
      a.out[row] = best == 0x7fffffff ? -1 : best;
    }
    return;
  }
  if (hi == INFINITY) {                                   // only these count, and alike
    for (int i = tid; i < count; i += SA_THREADS) z[i] = z[i] == INFINITY ? 0.f : -INFINITY;
    hi = lo = 0.f;
    __syncthreads();
  }
  const double unit = fmax(1.4426950408889634074 * 64.0 / (double)t, 1e-300), top = (double)hi;
  constexpr u64 AT_512 = SA_AT_512, AT_2_17 = 0x4100000000000000ULL, AT_2_20 = 0x4130000000000000ULL;      // 512, 2^17, 2^20
  auto weight_bits = [&](float x) { return sa_weight_bits(((double)x - top) * unit, 512.0, s.root); };
  auto weight = [&](float x) { return weight_bits(x) - AT_512; };
  // four of the warp's words a lane, at a time
  auto each = [&](auto f) {
#pragma unroll 2
    for (int i = from + lane * 4; i < from + part; i += 128) f(i, *reinterpret_cast<const float4*>(z + i));
  };

  // ---- what is kept: logits above `last`, and of those equal to it the ones up to last_at
  float last = -INFINITY;
  int last_at = -1;
  auto kept = [&](float x, int i) { return x > last || (x == last && v0 + i <= last_at); };
  const bool by_count = top_k > 0 && top_k < a.V, by_mass = top_p < 1.f;
  const float least = min_p > 0.f ? fminf(min_p, 1.f) : 0.f;
  const u64 w_min = least > 0.f ? (u64)ceil((double)least * 8796093022208.0) : 0;
  const double u = (double)u01;
  auto drawn = [&](u64 all) { return sa_drawn(u, all); };
  int turn = 0;                                           // of s.total
  // The word (by index) up to which more than `limit` of value(i, z_i) lies, by all CTAs; limit = choose(the sum of all).  Returns its index in the one CTA that has it, -1 in the others.
  // value(...) is `base` too large.
  // on(i, z_i): whether a word counts at all.
  auto locate = [&](auto on, auto value_of, u64 base, auto choose) -> int {
    u64 sum = 0;
    each([&](int i, const float4& x) {
      const bool a0 = on(i, x.x), a1 = on(i + 1, x.y), a2 = on(i + 2, x.z), a3 = on(i + 3, x.w);
      if (__any_sync(0xffffffffu, a0 || a1 || a2 || a3)) {
        const u64 w0 = value_of(x.x), w1 = value_of(x.y), w2 = value_of(x.z), w3 = value_of(x.w);
        sum += ((a0 ? w0 : base) + (a1 ? w1 : base)) + ((a2 ? w2 : base) + (a3 ? w3 : base));
      }
    });
    sum = sa_warp_sum(sum) - base * part;
    auto value = [&](int i, float x) { return on(i, x) ? value_of(x) : base; };
    if (lane == 0) s.warp_w[warp] = sum;
    __syncthreads();
    const u64 w_upto = sa_upto_lanes(lane < SA_WARPS ? s.warp_w[lane] : 0), mine = __shfl_sync(0xffffffffu, w_upto, 31);
    if (tid < CTAS) *sa_at(&s.total[turn][rank], tid) = mine;
    sa_cluster<CTAS>();
    u64 all = 0, before = 0;
#pragma unroll
    for (int c = 0; c < CTAS; ++c) {
      if (c == rank) before = all;
      all += s.total[turn][c];
    }
    turn ^= 1;
    const u64 limit = choose(all);
    if (limit < before || limit >= before + mine) return -1;
    const int w = __popc(__ballot_sync(0xffffffffu, before + w_upto <= limit));      // the warp in whose words it lies
    u64 at = before + (w ? __shfl_sync(0xffffffffu, w_upto, max(w - 1, 0)) : 0);
    // that warp's words, a thread some of them side by side
    const int some = (part + SA_THREADS - 1) / SA_THREADS, i0 = min(tid * some, part) + w * part, i1 = min((tid + 1) * some, part) + w * part;
    u64 own = 0;
#pragma unroll 2
    for (int i = i0; i < i1; ++i) own += value(i, z[i]) - base;
    const u64 run = sa_upto_lanes(own);
    __syncthreads();                                      // (warp_w has been read)
    if (lane == 31) s.warp_w[warp] = run;
    __syncthreads();
    const u64 upto = sa_upto_lanes(lane < SA_WARPS ? s.warp_w[lane] : 0);
    at += run - own + (warp ? __shfl_sync(0xffffffffu, upto, max(warp - 1, 0)) : 0);
    if (limit >= at && limit < at + own)
      for (int i = i0; i < i1; ++i) {
        const u64 v = value(i, z[i]) - base;
        if (limit < at + v) { s.tie = i; break; }
        at += v;
      }
    __syncthreads();
    return s.tie;
  };

  if (by_count || by_mass) {
    // masses are in units of 2^-35 (2^-32) here, so that the sums of their two parts over a CTA's words fit into 32 bits
    const int low = a.slice <= 16384 ? 18 : 16;
    const double power = a.slice <= 16384 ? 131072.0 : 1048576.0;
    const u64 power_bits = a.slice <= 16384 ? AT_2_17 : AT_2_20;
    auto mass = [&](float x) { return sa_weight_bits(((double)x - top) * unit, power, s.root) - power_bits; };
    // ranges of equal width below the largest logit, as far as weights reach (30 t) or a top_k may look
    const float reach = fminf(fmaxf(30.f * t, 24.f), hi - lo), fine = reach > 1e-30f ? (float)(SA_BINS - 1) / reach : 0.f;
    constexpr float WHOLE = 12582912.f;                   // 1.5 2^23: the whole number is in the low bits
    auto depth = [&](float x) { return fminf(__fmaf_rn(hi - x, fine, WHOLE), WHOLE + (SA_BINS - 1)); };
    auto bin_of = [&](float x) { return __float_as_int(depth(x)) - 0x4b400000; };
    int hists = 0;
    // The last word before which fewer than `limit` words lie (MASS: less than top_p of the mass): `last` and last_at.  True: the word has been drawn.
    auto cut = [&](auto by, u64 limit) -> bool {
      constexpr bool MASS = decltype(by)::value;
      SaHist* h;
      auto count_in = [&](int b, u64 w) {
        atomicAdd(&h->n[b], 1u);
        if (MASS) {
          const unsigned w_hi = (unsigned)(w >> low);
          atomicAdd(&h->lo[b], (unsigned)w & ((1u << low) - 1));
          if (w_hi) atomicAdd(&h->hi[b], w_hi);
        }
      };
      auto next_hist = [&]() {
        h = &s.hist[hists & 1];
        if (hists++ > 1) {                                // (the first two are empty)
          for (int i = tid; i < (int)(sizeof(SaHist) / 4); i += SA_THREADS) reinterpret_cast<unsigned*>(h)[i] = 0;
          __syncthreads();
        }
      };
      next_hist();
      each([&](int i, const float4& x) {
        const float v[4] = {x.x, x.y, x.z, x.w};
        bool on[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) on[k] = MASS && by_count ? kept(v[k], i + k) : v[k] > -INFINITY;      // (of the mass what top_k has kept)
        if (__any_sync(0xffffffffu, on[0] || on[1] || on[2] || on[3])) {
          u64 w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] = MASS ? mass(v[k]) : 0;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (on[k]) count_in(bin_of(v[k]), w[k]);
        }
      });
      sa_cluster<CTAS>();
      u64 above_n = 0, above_w = 0;
      unsigned key_lo = 0, key_hi = 0;                    // of the range, from the second level on
      int shift = 0;
      for (bool first = true;; first = false) {
        // every CTA adds up all CTAs' ranges, a thread two, and finds the one where the limit lies
        uint2 n = make_uint2(0, 0);
        u64 w0 = 0, w1 = 0;
#pragma unroll
        for (int c = 0; c < CTAS; ++c) {
          const SaHist* o = sa_at(h, c);
          const uint2 x = *reinterpret_cast<const uint2*>(&o->n[2 * tid]);
          n.x += x.x, n.y += x.y;
          if (MASS) {
            const uint2 l = *reinterpret_cast<const uint2*>(&o->lo[2 * tid]), m = *reinterpret_cast<const uint2*>(&o->hi[2 * tid]);
            w0 += ((u64)m.x << low) + l.x;
            w1 += ((u64)m.y << low) + l.y;
          }
        }
        unsigned run_n = n.x + n.y;
        u64 run_w = w0 + w1;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const unsigned up_n = __shfl_up_sync(0xffffffffu, run_n, o);
          if (lane >= o) run_n += up_n;
          if (MASS) {
            const u64 up_w = __shfl_up_sync(0xffffffffu, run_w, o);
            if (lane >= o) run_w += up_w;
          }
        }
        if (lane == 31) s.warp_n[warp] = run_n, s.warp_w[warp] = run_w;      // (the last reads of these lie before a barrier)
        if (tid == 0) s.bin = -1;
        __syncthreads();
        u64 all_w = 0, upto_n = above_n + run_n, upto_w = above_w + run_w;
#pragma unroll
        for (int k = 0; k < SA_WARPS; ++k) {
          if (k < warp) upto_n += s.warp_n[k], upto_w += s.warp_w[k];
          all_w += s.warp_w[k];
        }
        if (first && MASS) limit = sa_mass_limit(top_p, all_w);
        auto look = [&](int b, unsigned in, u64 mass, u64 n_end, u64 w_end) {
          const u64 end = MASS ? w_end : n_end, begin = end - (MASS ? mass : in);
          if (begin < limit && end >= limit) s.bin = b, s.bin_n = in, s.above_n = n_end - in, s.above_w = w_end - mass;
        };
        look(2 * tid, n.x, w0, upto_n - n.y, upto_w - w1);
        look(2 * tid + 1, n.y, w1, upto_n, upto_w);
        __syncthreads();
        const int bin = s.bin;
        if (bin < 0) return false;                        // fewer words than the limit: all stay
        above_n = s.above_n;
        above_w = s.above_w;
        const unsigned in_bin = s.bin_n;
        if (!first) {
          const unsigned lo_of = key_hi - ((unsigned)bin << shift), width = (1u << shift) - 1;
          key_hi = lo_of;
          key_lo = lo_of - key_lo > width ? lo_of - width : key_lo;
        }
        const bool finish = first && !(MASS && by_count) && above_n + in_bin <= SA_MORE;      // few words down to the limit: all of them are listed
        const float from_depth = finish ? 0.f : WHOLE + (float)bin, to_depth = WHOLE + (float)bin;
        auto on = [&](float x, int i) { return MASS && by_count ? kept(x, i) : x > -INFINITY; };
        auto inside = [&](float x, int i) {               // of the range (finish: of it and of those above)
          const float d = depth(x);
          const unsigned k = sa_key(x);
          return on(x, i) && (first ? d >= from_depth && d <= to_depth : k >= key_lo && k <= key_hi);
        };
        if (finish || in_bin <= SA_LIST) {
          u64* list_at = finish ? reinterpret_cast<u64*>(&s.hist[1]) : s.list[MASS].word;      // (of the first cut's first level the other counts are not in use)
          auto list = [&](int i, float x) {
            const int at = atomicAdd(&s.n_list[MASS], 1);      // (below SA_LIST, SA_MORE: there are no more words)
            list_at[at] = (u64)sa_key(x) << 32 | ~(unsigned)(v0 + i);
          };
          auto look_through = [&](auto in) {
            each([&](int i, const float4& x) {
              const bool a0 = in(x.x, i), a1 = in(x.y, i + 1), a2 = in(x.z, i + 2), a3 = in(x.w, i + 3);
              if (__any_sync(0xffffffffu, a0 || a1 || a2 || a3)) {
                if (a0) list(i, x.x);
                if (a1) list(i + 1, x.y);
                if (a2) list(i + 2, x.z);
                if (a3) list(i + 3, x.w);
              }
            });
          };
          if (first && !(MASS && by_count)) look_through([&](float x, int) { const float d = depth(x); return d >= from_depth && d <= to_depth && x > -INFINITY; });
          else look_through(inside);
          sa_cluster<CTAS>();
          if (finish && rank != 0) {
            sa_cluster<CTAS>();                           // (its list has been read)
            return true;
          }
          int n_all = 0, sizes[CTAS];
          u64 word = 0;
#pragma unroll
          for (int c = 0; c < CTAS; ++c) sizes[c] = *sa_at(&s.n_list[MASS], c);
#pragma unroll
          for (int c = 0; c < CTAS; ++c) {
            if (tid >= n_all && tid < n_all + sizes[c]) word = sa_at(list_at, c)[tid - n_all];
            n_all += sizes[c];
          }
          if (finish && n_all > SA_LIST) {
            u64* words = reinterpret_cast<u64*>(z);       // (the logits are done with)
            words[tid] = word;                            // (0 stands behind all words)
            sa_cluster<CTAS>();
            sa_finish(s, words, n_all, !MASS, limit, by_mass, SaDraw{top, unit, power, u, power_bits, w_min, top_p}, a.out + row);
            return true;
          }
          if (tid < SA_LIST) s.gathered.word[tid] = word;
          if (finish) sa_cluster<CTAS>();
          __syncthreads();
          // each word counts those before it: by two threads, half of the words each
          const int mine = tid >> 1, half = tid & 1;
          word = s.gathered.word[mine];
          unsigned before = 0;                            // those before it in order, and (upper half: where all is drawn from the list) by index
          if (warp * 16 < n_all) {
            if (finish)
#pragma unroll 2
              for (int j = half * 2; j < n_all; j += 4) {
                const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(&s.gathered.word[j]);
                before += (o.x > word ? 1u : 0u) + (o.y > word ? 1u : 0u) + ((unsigned)o.x > (unsigned)word ? 0x10000u : 0u) + ((unsigned)o.y > (unsigned)word ? 0x10000u : 0u);
              }
            else
#pragma unroll 2
              for (int j = half * 2; j < n_all; j += 4) {
                const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(&s.gathered.word[j]);
                before += (o.x > word ? 1u : 0u) + (o.y > word ? 1u : 0u);
              }
          }
          before += __shfl_xor_sync(0xffffffffu, before, 1);
          const unsigned before_n = before & 0xffffu, before_at = before >> 16;
          const bool is = mine < n_all && half == 0;
          const float x = sa_of_key((unsigned)(word >> 32));
          // of the first SA_LIST threads: the sum of v up to this one
          auto upto = [&](u64 v) {
            v = sa_upto_lanes(v);
            __syncthreads();
            if (lane == 31) s.warp_w[warp] = v;
            __syncthreads();
#pragma unroll
            for (int k = 0; k < SA_LIST / 32; ++k)
              if (k < warp) v += s.warp_w[k];
            return v;
          };
          // how many of the words in order stay
          unsigned stay = MASS ? n_all : (unsigned)min(limit - (finish ? 0 : above_n), (u64)n_all);
          if (MASS || (finish && by_mass)) {
            if (tid < SA_LIST) s.sorted[tid] = 0;
            if (tid == 0) s.last_rank = 0;
            __syncthreads();
            if (is && before_n < stay) s.sorted[before_n] = mass(x);
            __syncthreads();
            const u64 v = tid < SA_LIST ? s.sorted[tid] : 0, end = upto(v);
            if (!MASS) limit = sa_mass_limit(top_p, [&] {           // of the mass that top_k has kept
              u64 all = 0;
#pragma unroll
              for (int k = 0; k < SA_LIST / 32; ++k) all += s.warp_w[k];
              return all;
            }());
            const unsigned in = __ballot_sync(0xffffffffu, tid < (int)stay && (finish ? 0 : above_w) + end - v < limit);      // (`end` of a warp's words is that of all)
            if (lane == 0 && in) atomicAdd(&s.last_rank, __popc(in));
            __syncthreads();
            stay = s.last_rank;
          }
          if (!finish) {
            __syncthreads();
            if (is && before_n == stay - 1) {
              s.last_key = (unsigned)(word >> 32);
              s.last_at = (int)~(unsigned)word;
            }
            __syncthreads();
            last = sa_of_key(s.last_key);
            last_at = s.last_at;
            return false;
          }
          // all that can be kept is here: the draw
          if (tid < SA_LIST) s.by_index[tid] = 0;
          __syncthreads();
          if (is && before_n < stay) {
            const u64 w = weight(x);
            s.by_index[before_at] = w >= w_min ? w : 0;
            s.sorted[before_at] = ~(unsigned)word;
          }
          __syncthreads();
          const u64 w = tid < SA_LIST ? s.by_index[tid] : 0, end = upto(w);
          u64 all = 0;
#pragma unroll
          for (int k = 0; k < SA_LIST / 32; ++k) all += s.warp_w[k];
          const u64 d = drawn(all);
          if (w && d >= end - w && d < end) a.out[row] = (long long)s.sorted[tid];
          return true;
        }
        if (first) {                                      // the range's keys
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
        }
        if (key_lo == key_hi) {
          // equal logits: as many as the limit allows, by their index
          const float same = sa_of_key(key_lo);
          const u64 w_each = MASS ? mass(same) : 1, left = limit - (MASS ? above_w : above_n);      // > 0
          const u64 n_left = w_each ? min((left + w_each - 1) / w_each, (u64)in_bin) : (u64)in_bin;
          const int i = locate([&](int k, float x) { return x == same && (!(MASS && by_count) || kept(x, k)); }, [](float) -> u64 { return 1; }, 0, [&](u64) { return n_left - 1; });
          if (i >= 0 && tid < CTAS) *sa_at(&s.last_at, tid) = v0 + i;
          sa_cluster<CTAS>();
          last = same;
          last_at = s.last_at;
          return false;
        }
        // the range in parts again
        next_hist();
        const unsigned span = key_hi - key_lo;
        shift = 0;
        while (span >> shift >= SA_BINS) ++shift;
        each([&](int i, const float4& x) {
          const bool a0 = inside(x.x, i), a1 = inside(x.y, i + 1), a2 = inside(x.z, i + 2), a3 = inside(x.w, i + 3);
          if (!__any_sync(0xffffffffu, a0 || a1 || a2 || a3)) return;
          if (a0) count_in((key_hi - sa_key(x.x)) >> shift, MASS ? mass(x.x) : 0);
          if (a1) count_in((key_hi - sa_key(x.y)) >> shift, MASS ? mass(x.y) : 0);
          if (a2) count_in((key_hi - sa_key(x.z)) >> shift, MASS ? mass(x.z) : 0);
          if (a3) count_in((key_hi - sa_key(x.w)) >> shift, MASS ? mass(x.w) : 0);
        });
        sa_cluster<CTAS>();
      }
    };
    if ((by_count && cut(SaByCount(), (u64)top_k)) || (by_mass && cut(SaByMass(), 0))) return;
  }
  // ---- the draw
  const bool whole = !by_count && !by_mass && w_min == 0;
  const int i = whole ? locate([](int, float) { return true; }, weight_bits, AT_512, drawn)
                      : locate([&](int k, float x) { return kept(x, k); },
                               [&](float x) {
                                 const u64 w = weight(x);
                                 return w >= w_min ? w : 0;
                               },
                               0, drawn);
  if (i >= 0 && tid == 0) a.out[row] = v0 + i;            // (since the last barrier nobody reads or writes in another CTA)
}

template <typename T, int CTAS>
static int launch_sample(const SampleArgs& a, int rows, cudaStream_t stream) {
  static_assert(SA_WARPS * 128 * 4 >= 2 * SA_MORE * (int)sizeof(u64), "the few words' place is that of the least slice");
  const size_t smem = sizeof(SaShared) + (size_t)a.slice * 4;
  LP_CHECK_CUDA((allow_smem<sample_kernel<T, CTAS>>((int)smem)));
  LP_CHECK_CUDA(launch_ex(sample_kernel<T, CTAS>, dim3(rows * CTAS), dim3(SA_THREADS), smem, stream, CTAS, false, a));
  return 0;
}
template <typename T>
static int launch_sample_at(const SampleArgs& a, int rows, int ctas, cudaStream_t stream) {
  if (ctas == 1) return launch_sample<T, 1>(a, rows, stream);
  if (ctas == 2) return launch_sample<T, 2>(a, rows, stream);
  if (ctas == 4) return launch_sample<T, 4>(a, rows, stream);
  return launch_sample<T, 8>(a, rows, stream);
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
  // CTAs of a row: so that each has 16,384 words at most (two run on an SM then), and few rows more of them
  int ctas = 1;
  while (ctas < SA_MAX_CTAS && ((V + ctas - 1) / ctas > 16384 || ((long long)rows * ctas < sm_count() && V / ctas > 4096))) ctas *= 2;
  const int unit = SA_WARPS * 128;
  SampleArgs a = {logits, rows > 1 ? ld : 0, uniform, temperature, top_p, min_p, top_k, temperature_all, top_p_all, min_p_all, top_k_all, V, ((V + ctas - 1) / ctas + unit - 1) / unit * unit, false, out};
  const long long size = logits_fp32 ? 4 : 2;
  a.vec = reinterpret_cast<uintptr_t>(logits) % 16 == 0 && a.ld * size % 16 == 0;
  LP_REQUIRE((long long)rows * ctas <= 2147483647LL, "lp_sample_tokens: %d rows", rows);
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  note_launch(1);
  return logits_fp32 ? launch_sample_at<float>(a, rows, ctas, stream) : launch_sample_at<bf16>(a, rows, ctas, stream);
}
