// Distillation from a teacher's top logits (forward, and forward with the gradient).
//   q = softmax(x / T), p = softmax(teacher / T) over the k given entries
//   KL = sum_j p_j (ln p_j - ln q_{id_j}),   d(T^2 KL)/dx = T (q - p)
// and with hard labels CE = lse(x) - x_label, dCE/dx = softmax(x) - onehot.
// One CTA per row: a pass for the maximum, one for the sums, one that writes the gradient of the
// dense part; the k entries and the label are then corrected one by one from the same fp32 values.
#include "m3_internal.h"
#include "m3_vocab.cuh"

namespace m3 {
namespace {

using namespace vocab;

constexpr int kThreads = 256, kWarps = kThreads / 32;

struct Params {
  int64_t rows;
  int vocab, k;
  float temperature, inv_t, hard, scale;  // scale: grad_scale, over the row count for an unweighted mean
  Rows lrow, grow;
  const void* logits;
  void* grad;
  const int64_t *ids, *labels;
  const float *teacher, *weights, *upstream;
  int64_t upstream_stride;
  const float* weight_sum;  // a mean's divisor, NULL = none
  float* row_loss;
};

__device__ __forceinline__ float block_sum(float v, float* sm) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sm[0];
  for (int w = 1; w < kWarps; ++w) v += sm[w];
  return v;
}
__device__ __forceinline__ float block_max(float v, float* sm) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sm[0];
  for (int w = 1; w < kWarps; ++w) v = fmaxf(v, sm[w]);
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) distill_kernel(const Params p) {
  __shared__ float fs[kWarps], amount[M3_MAX_TOP];
  __shared__ int64_t sid[M3_MAX_TOP];
  const int64_t row = blockIdx.x;
  const int V = p.vocab, tid = threadIdx.x;
  const T* x = reinterpret_cast<const T*>(p.logits) + p.lrow.at(row);
  T* g = p.grad ? reinterpret_cast<T*>(p.grad) + p.grow.at(row) : nullptr;
  const float w = p.weights ? p.weights[row] : 1.f;
  const int64_t label = p.labels ? p.labels[row] : -1;

  // the teacher's entries, one per thread
  const int64_t id = tid < p.k ? p.ids[row * p.k + tid] : -1;
  const float t = id >= 0 ? p.teacher[row * p.k + tid] : -INFINITY;
  if (tid < p.k) sid[tid] = id;
  const bool bad = __syncthreads_or(id >= V) || label >= V;
  const bool soft = __syncthreads_or(id >= 0) && p.hard < 1.f, hard = label >= 0 && p.hard > 0.f;
  if (w == 0.f || (!soft && !hard)) {
    if (tid == 0) p.row_loss[row] = 0.f;
    if (g)
      for (int i = tid; i < V; i += kThreads) stg<T>(g + i, 0.f);
    return;
  }
  if (bad) {
    if (tid == 0) p.row_loss[row] = NAN;
    if (g)
      for (int i = tid; i < V; i += kThreads) stg<T>(g + i, NAN);
    return;
  }
  const float xid = id >= 0 ? ld(x + id) : 0.f, xl = hard ? ld(x + label) : 0.f;
  const float tm = block_max(t, fs);
  const float d = (t - tm) * p.inv_t;
  const float e = id >= 0 ? expf(d) : 0.f;
  const float es = block_sum(e, fs);
  const float pj = id >= 0 ? e / es : 0.f;

  float m = -INFINITY;
  for (int i = tid; i < V; i += kThreads) m = fmaxf(m, ld(x + i));
  m = block_max(m, fs);
  const float c = p.inv_t * kLog2e;
  float s = 0.f, s1 = 0.f;
  for (int i = tid; i < V; i += kThreads) {
    const float dx = ld(x + i) - m;
    s += ex2(dx * c);
    if (hard) s1 += ex2(dx * kLog2e);
  }
  s = block_sum(s, fs);
  if (hard) s1 = block_sum(s1, fs);
  // p_j (ln p_j - ln q_j); an entry of probability 0 has no term
  const float term = pj > 0.f ? pj * (d - logf(es) - (xid - m) * p.inv_t + logf(s)) : (pj == pj ? 0.f : NAN);
  const float kl = block_sum(term, fs);
  const float wk = 1.f - p.hard, T2 = p.temperature * p.temperature;
  if (tid == 0) {
    float loss = soft ? wk * T2 * kl : 0.f;
    if (hard) loss += p.hard * (logf(s1) - (xl - m));
    p.row_loss[row] = w * loss;
  }
  if (!g) return;
  float rs = p.scale * w;
  if (p.weight_sum) rs /= *p.weight_sum;
  if (p.upstream) rs *= p.upstream[row * p.upstream_stride];
  const float as = soft ? rs * wk * p.temperature : 0.f, ah = hard ? rs * p.hard : 0.f;
  const float ks = as / s, kh = hard ? ah / s1 : 0.f;
  auto dense = [&](float xv) {
    const float dx = xv - m;
    float v = soft ? ks * ex2(dx * c) : 0.f;
    if (hard) v = fmaf(kh, ex2(dx * kLog2e), v);
    return v;
  };
  for (int i = tid; i < V; i += kThreads) stg<T>(g + i, dense(ld(x + i)));
  if (tid < p.k) amount[tid] = as * pj;
  __syncthreads();
  // each id once, by its first entry; the label by itself where no entry has it
  if (tid < p.k && id >= 0) {
    float a = 0.f;
    bool first = true;
    for (int j = 0; j < p.k; ++j)
      if (sid[j] == id) {
        a += amount[j];
        if (j < tid) first = false;
      }
    if (id == label) a += ah;
    if (first) stg<T>(g + id, dense(xid) - a);
  }
  const bool hit = __syncthreads_or(tid < p.k && id >= 0 && id == label);
  if (hard && !hit && tid == 0) stg<T>(g + label, dense(xl) - ah);
}

// out = sum over v (n values), one CTA, a fixed order; over the sum of weights (or n) for a mean.
__global__ void __launch_bounds__(1024) sum_kernel(const float* __restrict__ v, int64_t n, const float* div_by,
                                                   float scale, float* out) {
  __shared__ float sm[32];
  float s = 0.f;
  for (int64_t i = threadIdx.x; i < n; i += 1024) s += v[i];
  s = warp_sum(s);
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x < 32) {
    s = warp_sum(sm[threadIdx.x]);
    if (threadIdx.x == 0) *out = s * scale / (div_by ? *div_by : 1.f);
  }
}

}  // namespace
}  // namespace m3

using namespace m3;

extern "C" int m3_distill(const M3DistillArgs* args, void* stream) {
  if (!args) return set_error(M3_ERR_ARG, "m3_distill: args is NULL");
  const M3DistillArgs& a = *args;
  if (a.rows_outer < 0 || a.rows_inner < 0 || a.vocab <= 0 || a.k <= 0 || a.k > M3_MAX_TOP)
    return set_error(M3_ERR_SHAPE, "m3_distill: need rows >= 0, vocab > 0 and 1 <= k <= 128");
  if (a.logits_dtype != M3_DTYPE_F32 && a.logits_dtype != M3_DTYPE_BF16)
    return set_error(M3_ERR_UNSUPPORTED, "m3_distill: logits must be f32 or bf16");
  if (a.reduction < M3_REDUCE_NONE || a.reduction > M3_REDUCE_MEAN)
    return set_error(M3_ERR_ARG, "m3_distill: reduction must be NONE, SUM or MEAN");
  if (!(a.temperature > 0.f) || !(a.hard_weight >= 0.f && a.hard_weight <= 1.f))
    return set_error(M3_ERR_ARG, "m3_distill: need temperature > 0 and 0 <= hard_weight <= 1");
  const int64_t rows = (int64_t)a.rows_outer * a.rows_inner;
  if (rows > 0x7FFFFFFF) return set_error(M3_ERR_SHAPE, "m3_distill: more than 2^31 - 1 rows");
  if ((rows > 0 && (!a.logits || !a.ids || !a.teacher || !a.row_loss)) ||
      (a.hard_weight > 0.f && rows > 0 && !a.labels) || (a.reduction != M3_REDUCE_NONE && !a.loss))
    return set_error(M3_ERR_ARG, "m3_distill: NULL pointer");
  const bool wmean = a.reduction == M3_REDUCE_MEAN && a.weights && rows > 0;
  if (wmean && !a.weight_sum) return set_error(M3_ERR_ARG, "m3_distill: a mean with weights needs weight_sum");
  if (a.upstream_stride < 0 || a.upstream_stride > 1)
    return set_error(M3_ERR_ARG, "m3_distill: upstream_stride must be 0 or 1");
  cudaStream_t s = (cudaStream_t)stream;
  Params p;
  p.rows = rows;
  p.vocab = a.vocab;
  p.k = a.k;
  p.temperature = a.temperature;
  p.inv_t = 1.f / a.temperature;
  p.hard = a.hard_weight;
  p.scale = a.grad_scale;
  if (a.reduction == M3_REDUCE_MEAN && !a.weights) p.scale /= (float)rows;
  p.lrow = Rows{a.rows_inner, a.ld_outer, a.ld_inner};
  p.grow = Rows{a.rows_inner, a.g_outer, a.g_inner};
  p.logits = a.logits;
  p.grad = a.grad;
  p.ids = a.ids;
  p.labels = a.hard_weight > 0.f ? a.labels : nullptr;
  p.teacher = a.teacher;
  p.weights = a.weights;
  p.upstream = a.upstream;
  p.upstream_stride = a.upstream_stride;
  p.weight_sum = wmean ? a.weight_sum : nullptr;
  p.row_loss = a.row_loss;
  if (wmean) sum_kernel<<<1, 1024, 0, s>>>(a.weights, rows, nullptr, 1.f, a.weight_sum);
  if (rows > 0) {
    if (a.logits_dtype == M3_DTYPE_BF16)
      distill_kernel<__nv_bfloat16><<<(unsigned)rows, kThreads, 0, s>>>(p);
    else
      distill_kernel<float><<<(unsigned)rows, kThreads, 0, s>>>(p);
  }
  if (a.reduction != M3_REDUCE_NONE)  // the mean of no rows is 0 / 0
    sum_kernel<<<1, 1024, 0, s>>>(a.row_loss, rows, p.weight_sum,
                                  a.reduction == M3_REDUCE_MEAN && !a.weights ? 1.f / (float)rows : 1.f, a.loss);
  return check_launch("m3_distill");
}
