// Log probabilities of given tokens, entropy and top alternatives of logits rows.
//   y = x / T, m = max y, Z = sum e^(y - m):  lse = m + ln Z,  entropy = ln Z - sum e d / Z, d = y - m
// One CTA per row: a pass for the maximum, one for the sums, then one pass per alternative (the
// largest entry below the previous one in the order (logit, lower index)).
#include "m3_internal.h"
#include "m3_vocab.cuh"

namespace m3 {
namespace {

using namespace vocab;

constexpr int kThreads = 256, kWarps = kThreads / 32;

struct Params {
  int64_t rows;
  int vocab, top;
  float inv_t;
  Rows lrow, trow;
  const void* logits;
  const int64_t* targets;
  float *logprob, *entropy, *lse, *top_logprob;
  int64_t* top_ids;
};

template <typename V, typename F>
__device__ __forceinline__ V block_reduce(V v, F f, V* sm) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sm[0];
  for (int w = 1; w < kWarps; ++w) v = f(v, sm[w]);
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) score_kernel(const Params p) {
  __shared__ float fs[kWarps];
  __shared__ uint64_t ws[kWarps];
  const int64_t row = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(p.logits) + p.lrow.at(row);
  const int V = p.vocab;
  auto sum = [](float a, float b) { return a + b; };
  float m = -INFINITY;
  for (int i = threadIdx.x; i < V; i += kThreads) m = fmaxf(m, ld(x + i));
  m = block_reduce(m, [](float a, float b) { return fmaxf(a, b); }, fs);
  // log2 units; a row without a finite maximum makes every term NaN
  const float c = p.inv_t * kLog2e;
  float s = 0.f, u = 0.f;
  for (int i = threadIdx.x; i < V; i += kThreads) {
    const float d = (ld(x + i) - m) * c;
    const float e = ex2(d);
    s += e;
    u = fmaf(e, fmaxf(d, -1e4f), u);  // e = 0 below -150: 0 * -inf is 0
  }
  s = block_reduce(s, sum, fs);
  u = block_reduce(u, sum, fs);
  const float l2 = log2f(s);
  const float lse = m * p.inv_t + l2 * kLn2;
  if (threadIdx.x == 0) {
    p.lse[row] = lse;
    p.entropy[row] = (l2 - u / s) * kLn2;
    if (p.targets) {
      const int64_t t = p.targets[p.trow.at(row)];
      p.logprob[row] = t < 0 ? 0.f : t >= V ? NAN : (ld(x + t) - m) * p.inv_t - l2 * kLn2;
    }
  }
  uint64_t prev = ~0ull;
  for (int j = 0; j < p.top; ++j) {
    uint64_t best = 0;
    for (int i = threadIdx.x; i < V; i += kThreads) {
      const uint64_t w = rank_word(ld(x + i), i);
      if ((w < prev || j == 0) && w > best) best = w;  // (NaN, 0) has the top word
    }
    best = block_reduce(best, [](uint64_t a, uint64_t b) { return a > b ? a : b; }, ws);
    if (threadIdx.x == 0) {
      p.top_ids[row * p.top + j] = rank_index(best);
      p.top_logprob[row * p.top + j] = (key_value((uint32_t)(best >> 32)) - m) * p.inv_t - l2 * kLn2;
    }
    prev = best;
  }
}

}  // namespace
}  // namespace m3

using namespace m3;

extern "C" int m3_token_logprobs(const M3ScoreArgs* args, void* stream) {
  if (!args) return set_error(M3_ERR_ARG, "m3_token_logprobs: args is NULL");
  const M3ScoreArgs& a = *args;
  if (a.rows_outer < 0 || a.rows_inner < 0 || a.vocab <= 0 || a.top < 0 || a.top > M3_MAX_TOP || a.top > a.vocab)
    return set_error(M3_ERR_SHAPE, "m3_token_logprobs: need rows >= 0, vocab > 0 and 0 <= top <= min(vocab, 128)");
  if (a.logits_dtype != M3_DTYPE_F32 && a.logits_dtype != M3_DTYPE_BF16)
    return set_error(M3_ERR_UNSUPPORTED, "m3_token_logprobs: logits must be f32 or bf16");
  if (!(a.temperature > 0.f)) return set_error(M3_ERR_ARG, "m3_token_logprobs: temperature must be > 0");
  const int64_t rows = (int64_t)a.rows_outer * a.rows_inner;
  if (rows == 0) return M3_OK;
  if (!a.logits || !a.entropy || !a.lse || (a.targets && !a.logprob) || (a.top > 0 && (!a.top_logprob || !a.top_ids)))
    return set_error(M3_ERR_ARG, "m3_token_logprobs: NULL pointer");
  if (rows > 0x7FFFFFFF) return set_error(M3_ERR_SHAPE, "m3_token_logprobs: more than 2^31 - 1 rows");
  Params p;
  p.rows = rows;
  p.vocab = a.vocab;
  p.top = a.top;
  p.inv_t = 1.f / a.temperature;
  p.lrow = Rows{a.rows_inner, a.ld_outer, a.ld_inner};
  p.trow = Rows{a.rows_inner, a.t_outer, a.t_inner};
  p.logits = a.logits;
  p.targets = a.targets;
  p.logprob = a.logprob;
  p.entropy = a.entropy;
  p.lse = a.lse;
  p.top_logprob = a.top_logprob;
  p.top_ids = a.top_ids;
  cudaStream_t s = (cudaStream_t)stream;
  if (a.logits_dtype == M3_DTYPE_BF16)
    score_kernel<__nv_bfloat16><<<(unsigned)rows, kThreads, 0, s>>>(p);
  else
    score_kernel<float><<<(unsigned)rows, kThreads, 0, s>>>(p);
  return check_launch("m3_token_logprobs");
}
