// Shared by the kernels over logits rows (m3_score.cu, m3_distill.cu): rows behind two
// strides, the order of logits, and the running (max, sum) of a softmax.
#pragma once

#include "m3_common.cuh"

namespace m3 {
namespace vocab {

constexpr float kLn2 = 0.69314718055994530942f;
constexpr int kMaxVocab = 1 << 30;  // element and vector indices are ints

// The most 16-byte vectors that a row of n elements can touch: its start's place in a vector is the
// same for every row if both strides are whole vectors, else anything.
inline int most_vectors(const void* x, int n, int size, int64_t outer, int64_t inner) {
  const int e = 16 / size;
  const int shift = outer % e == 0 && inner % e == 0 ? (int)((uintptr_t)x % 16) / size : e - 1;
  return (shift + n + e - 1) / e;
}

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

// ---- a row as 16-byte vectors ---------------------------------------------------------------
// Vector q of a row that starts `shift` elements past a 16-byte boundary holds the elements
// [q E - shift, q E - shift + E); those outside [0, n) read as -inf, which has probability 0.
template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

template <typename T>
__device__ __forceinline__ int row_shift(const T* x) {
  return (int)(((uintptr_t)x & 15u) / sizeof(T));
}

template <typename T>
__device__ __forceinline__ uint4 neg_inf_vec() {
  const uint32_t w = sizeof(T) == 2 ? 0xFF80FF80u : 0xFF800000u;
  return make_uint4(w, w, w, w);
}

template <typename T>
__device__ __forceinline__ uint4 load_vec(const T* row, int lo, int n) {
  constexpr int E = kVec<T>;
  uint4 u;
  if (lo >= 0 && lo + E <= n) {  // read once: no place in L1
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
                 : "l"(row + lo));
    return u;
  }
  // the ragged ends of a row, element by element
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (sizeof(T) == 2) {
      const int i = lo + 2 * j;
      const uint32_t a = i >= 0 && i < n ? *reinterpret_cast<const uint16_t*>(row + i) : 0xFF80u;
      const uint32_t b = i + 1 >= 0 && i + 1 < n ? *reinterpret_cast<const uint16_t*>(row + i + 1) : 0xFF80u;
      w[j] = a | (b << 16);
    } else {
      const int i = lo + j;
      w[j] = i >= 0 && i < n ? *reinterpret_cast<const uint32_t*>(row + i) : 0xFF800000u;
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The vector's elements as pairs of floats.
template <typename T>
__device__ __forceinline__ void unpack(const uint4& u, float2 (&f)[kVec<T> / 2]) {
  if constexpr (sizeof(T) == 2) {
    f[0] = bf2f(u.x);
    f[1] = bf2f(u.y);
    f[2] = bf2f(u.z);
    f[3] = bf2f(u.w);
  } else {
    f[0] = make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
    f[1] = make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
  }
}

// The largest element (NaN ignored).
template <typename T>
__device__ __forceinline__ float vec_max(const uint4& u) {
  if constexpr (sizeof(T) == 2) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
  } else {
    return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
  }
}

__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// ---- clusters -------------------------------------------------------------------------------
__device__ __forceinline__ int cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return (int)r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// The address of this CTA's shared `p` in CTA `rank` of the cluster.
template <typename P>
__device__ __forceinline__ P* peer(P* p, int rank) {
  uint64_t a;
  asm volatile("mapa.u64 %0, %1, %2;" : "=l"(a) : "l"((uint64_t)p), "r"(rank));
  return reinterpret_cast<P*>(a);
}

}  // namespace vocab
}  // namespace m3
