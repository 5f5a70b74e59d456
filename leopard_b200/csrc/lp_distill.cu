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

template <typename T>
__global__ void __launch_bounds__(256)
distill_kernel(const DistillArgs a) {
  extern __shared__ float top[];            // t_k of the row's entries, then their ids
  __shared__ float red[8];
  int* id = reinterpret_cast<int*>(top + a.K);
  const int r = blockIdx.x, tid = threadIdx.x;
  const T* row = reinterpret_cast<const T*>(a.logits) + (long long)r * a.ld;
  bf16* drow = a.dlogits + (long long)r * a.ldd;
  const float w = a.weight[r];
  if (w == 0.f) {
    for (int i = tid * 2; i < a.Vp; i += 512) *reinterpret_cast<uint32_t*>(drow + i) = 0u;
    if (tid == 0) a.loss[r] = 0.f;
    return;
  }
  // the teacher's side
  float tm = -INFINITY;
  for (int k = tid; k < a.K; k += 256) {
    const long long at = (long long)r * a.ld_ids + k, at_t = (long long)r * a.ld_teacher + k;
    const long long i = a.ids_64 ? reinterpret_cast<const long long*>(a.ids)[at] : reinterpret_cast<const int*>(a.ids)[at];
    const bool in = i >= 0 && i < a.V;
    id[k] = in ? (int)i : -1;
    top[k] = !in ? -INFINITY : a.teacher_fp32 ? reinterpret_cast<const float*>(a.teacher)[at_t] : (float)reinterpret_cast<const bf16*>(a.teacher)[at_t];
    if (in) tm = fmaxf(tm, top[k]);
  }
  tm = block_max_f32(tm, red);
  float ts = 0.f;
  for (int k = tid; k < a.K; k += 256)
    if (top[k] != -INFINITY) ts += expf((top[k] - tm) * a.inv_tau);
  ts = block_sum_f32(ts, red);
  const bool soft = !(ts == 0.f);           // a NaN stays one
  // the student's
  float m = -INFINITY;
  for (int i = tid; i < a.V; i += 256) m = fmaxf(m, (float)row[i]);
  m = block_max_f32(m, red);
  float s = 0.f, s1 = 0.f;
  for (int i = tid; i < a.V; i += 256) {
    const float d = (float)row[i] - m;
    s += __expf(d * a.inv_tau);
    s1 += __expf(d);
  }
  s = block_sum_f32(s, red);
  s1 = block_sum_f32(s1, red);
  const float log_s = logf(s), log_ts = logf(ts);
  float kl = 0.f;
  for (int k = tid; k < a.K; k += 256) {
    float t = 0.f;
    if (id[k] >= 0 && soft) {
      const float lt = (top[k] - tm) * a.inv_tau - log_ts;
      t = expf(lt);
      if (t != 0.f) kl += t * (lt - ((float)row[id[k]] - m) * a.inv_tau + log_s);
    }
    top[k] = t;
  }
  kl = block_sum_f32(kl, red);              // ... and top[] is written
  const long long y = a.target ? a.target[r] : -1;
  const bool has_y = y >= 0 && y < a.V;
  const float cs = soft ? w * (1.f - a.hard) * a.tau : 0.f, ch = has_y ? w * a.hard : 0.f;
  if (tid == 0) {
    float l = soft ? (1.f - a.hard) * a.tau * a.tau * kl : 0.f;
    if (has_y && a.hard != 0.f) l += a.hard * (logf(s1) - ((float)row[y] - m));
    a.loss[r] = l;
  }
  const float ks = cs / s, kh = ch / s1;
  auto grad = [&](int i) {
    const float d = (float)row[i] - m;
    float g = 0.f;
    if (cs != 0.f) g = __expf(d * a.inv_tau) * ks;
    if (ch != 0.f) g += __expf(d) * kh;
    return g;
  };
  for (int i = tid * 2; i < a.Vp; i += 512) {
    const float x = i < a.V ? grad(i) : 0.f, z = i + 1 < a.V ? grad(i + 1) : 0.f;
    *reinterpret_cast<uint32_t*>(drow + i) = pack_bf16x2(x, z);
  }
  __syncthreads();
  // the places that the teacher or the label names are written again with their whole value: by the first entry of each id, the sum of its entries taken off
  for (int k = tid; k < a.K; k += 256) {
    if (id[k] < 0) continue;
    float t = 0.f;
    bool first = true;
    for (int o = 0; o < a.K; ++o)
      if (id[o] == id[k]) {
        if (o < k) first = false;
        t += top[o];
      }
    if (first) drow[id[k]] = __float2bfloat16_rn(grad(id[k]) - cs * t - (has_y && y == id[k] ? ch : 0.f));
  }
  if (has_y && tid == 0 && ch != 0.f) {
    bool named = false;
    for (int o = 0; o < a.K; ++o) named |= id[o] == y;
    if (!named) drow[y] = __float2bfloat16_rn(grad((int)y) - ch);
  }
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
  LP_REQUIRE(temperature > 0.f && temperature <= 3.0e38f, "lp_distill_fwd_bwd: temperature %g must be positive", (double)temperature);
  LP_REQUIRE(hard >= 0.f && hard <= 1.f && (hard == 0.f || target), "lp_distill_fwd_bwd: a hard share of %g needs labels and lies in [0, 1]", (double)hard);
  DistillArgs a = {logits, ld, ids, ids_64, ld_ids, teacher, teacher_fp32, ld_teacher, K, weight, target, 1.f / temperature, temperature, hard, loss, reinterpret_cast<bf16*>(dlogits), ldd, V, Vp};
  note_launch();
  const size_t smem = (size_t)K * 8;
  if (logits_fp32) distill_kernel<float><<<rows, 256, smem, stream>>>(a);
  else distill_kernel<bf16><<<rows, 256, smem, stream>>>(a);
  LP_CHECK_CUDA(cudaGetLastError());
  return 0;
}
