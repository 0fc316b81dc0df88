// Shared by the kernels over logits rows (m3_score.cu, m3_distill.cu): rows behind two
// strides, the order of logits, and the running (max, sum) of a softmax.
#pragma once

#include "m3_common.cuh"

namespace m3 {
namespace vocab {

constexpr float kLn2 = 0.69314718055994530942f;

// Element offset of row r = (r / inner) * outer_stride + (r % inner) * inner_stride.
struct Rows {
  int inner;
  int64_t outer_stride, inner_stride;
  __device__ __forceinline__ int64_t at(int64_t r) const {
    const int64_t o = r / inner;
    return o * outer_stride + (r - o * inner) * inner_stride;
  }
};

// Order-preserving map of a logit (larger logit, larger key; -0 == +0; every NaN is the top).
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  if (x != x) return 0xFFFFFFFFu;
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  if (k == 0xFFFFFFFFu) return __uint_as_float(0x7FC00000u);
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}
// Descending order of (logit, then lower index): the larger rank word comes first.
__device__ __forceinline__ uint64_t rank_word(float x, int idx) {
  return ((uint64_t)key_of(x) << 32) | (uint32_t)~idx;
}
__device__ __forceinline__ int rank_index(uint64_t w) { return (int)~(uint32_t)w; }

}  // namespace vocab
}  // namespace m3
