// Shared by the kernels over logits rows (m3_score.cu, m3_distill.cu): rows behind two
// strides, the order of logits, and the running (max, sum) of a softmax.
#pragma once

#include <string>

#include "m3_common.cuh"
#include "m3_internal.h"

namespace m3 {
namespace vocab {

constexpr float kLn2 = 0.69314718055994530942f;
constexpr int kMaxVocab = 1 << 30, kMaxRows = 1 << 30;  // element, vector and row indices are ints

// The most 16-byte vectors that a row of n elements can touch: its start's place in a vector is the
// same for every row if both strides are whole vectors, else anything.
inline int most_vectors(const void* x, int n, int size, int64_t outer, int64_t inner) {
  const int e = 16 / size;
  const int shift = outer % e == 0 && inner % e == 0 ? (int)((uintptr_t)x % 16) / size : e - 1;
  return (shift + n + e - 1) / e;
}

// Rows a warp takes: several waves of CTAs, so that the last one costs little (at 27 rows a warp,
// 131072 rows were 607 CTAs for 592 places, and took 142 us instead of 85).
inline int warp_batch(int rows, int sms) {
  const int batch = rows / (sms * 128);
  return batch < 1 ? 1 : batch > 32 ? 32 : batch;
}

// n / d for 0 <= n < 2^31, 1 <= d < 2^31, by one multiplication: with s = ceil(log2 d) and
// m = ceil(2^(31 + s) / d) < 2^32, m d exceeds 2^(31 + s) by less than d <= 2^s,
// so n m / 2^(31 + s) exceeds n / d by less than 1 / d.
struct Divider {
  uint32_t m;
  int shift, d;
  Divider() = default;
  explicit Divider(int div) : d(div) {
    int s = 0;
    while (((int64_t)1 << s) < div) ++s;
    shift = 31 + s;
    m = (uint32_t)((((uint64_t)1 << shift) + div - 1) / div);
  }
  __device__ __forceinline__ int div(int n) const { return (int)((uint64_t)(uint32_t)n * m >> shift); }
};

// Element offset of row r = (r / inner) * outer_stride + (r % inner) * inner_stride.  (A 64-bit
// division by every thread cost as much as 20 logits each.)  `flat`: one stride does for all rows.
struct Rows {
  Divider inner;
  bool flat;
  int64_t outer_stride, inner_stride;
  Rows() = default;
  Rows(int n_outer, int n, int64_t outer, int64_t in)
      : inner(n > 0 ? n : 1), flat(n_outer <= 1 || outer == n * in || n <= 1), outer_stride(outer),
        inner_stride(n <= 1 ? outer : in) {}
  __device__ __forceinline__ int64_t at(int r) const {
    if (flat) return r * inner_stride;
    const int o = inner.div(r);
    return o * outer_stride + (r - o * inner.d) * inner_stride;
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
template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

template <typename T>
__device__ __forceinline__ int row_shift(const T* x) {  // elements past a 16-byte boundary
  return (int)(((uintptr_t)x & 15u) / sizeof(T));
}

template <typename T>
__device__ __forceinline__ uint4 neg_inf_vec() {  // probability 0
  const uint32_t w = sizeof(T) == 2 ? 0xFF80FF80u : 0xFF800000u;
  return make_uint4(w, w, w, w);
}

// Logits pass through L1 without a place there.  In L2 they either stay for a second walk of the row
// or go first; a gradient goes first as well, so that it does not displace the rows in flight.
enum class Keep { kNo, kYes };

__device__ __forceinline__ uint64_t l2_policy(Keep keep) {
  uint64_t p;
  if (keep == Keep::kYes)
    asm volatile("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(p));
  else
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ uint4 load_stream(const uint4* p, uint64_t policy) {
  uint4 u;
  asm volatile("ld.global.L1::no_allocate.L2::cache_hint.v4.u32 {%0,%1,%2,%3}, [%4], %5;"
               : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
               : "l"(p), "l"(policy));
  return u;
}
__device__ __forceinline__ uint4 load_once(const uint4* p) {
  uint4 u;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
               : "l"(p));
  return u;
}
__device__ __forceinline__ void store_stream(void* p, const uint4& u, uint64_t policy) {
  asm volatile("st.global.L2::cache_hint.v4.u32 [%0], {%1,%2,%3,%4}, %5;" ::"l"(p), "r"(u.x), "r"(u.y), "r"(u.z),
               "r"(u.w), "l"(policy)
               : "memory");
}

// Vector of the elements [lo, lo + E) of a row, those outside [0, n) as -inf.
template <typename T>
__device__ __forceinline__ uint4 load_vec(const T* row, int lo, int n) {
  constexpr int E = kVec<T>;
  if (lo >= 0 && lo + E <= n) return load_once(reinterpret_cast<const uint4*>(row + lo));
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

// A row of n elements as `head` elements, `full` aligned vectors and `tail` elements.  The first CTA
// of a row's cluster takes the head and the last one the tail: lanes 0.. and 16.. of one warp.
struct Split {
  int head, full, tail, n;
};
template <typename T>
__device__ __forceinline__ Split split_row(const T* x, int n) {
  constexpr int E = kVec<T>;
  Split r;
  r.n = n;
  r.head = min(n, (E - row_shift(x)) & (E - 1));
  r.full = (n - r.head) / E;
  r.tail = n - r.head - r.full * E;
  return r;
}
__device__ __forceinline__ int edge_index(const Split& r, int lane, bool first, bool last) {  // -1: none
  if (first && lane < r.head) return lane;
  return last && lane >= 16 && lane - 16 < r.tail ? r.n - r.tail + lane - 16 : -1;
}

// Walks n vectors by TB threads, NV a thread and tile: f(d, base, full) with d[j] = v[base + j TB +
// thread], -inf past the end.  `full` tiles have no bounds to check, which halves the instructions of
// the loop; in the last one, f skips the j with base + j TB >= n.
template <bool B>
struct Flag {
  static constexpr bool value = B;
};
template <typename T, int NV, int TB, typename F>
__device__ __forceinline__ void walk(const uint4* v, int n, int thread, Keep keep, F f) {
  const uint64_t policy = l2_policy(keep);
  int base = 0;
  for (; base + NV * TB <= n; base += NV * TB) {
    const uint4* q = v + base + thread;
    uint4 d[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) d[j] = load_stream(q + j * TB, policy);
    f(d, base, Flag<true>());
  }
  if (base < n) {
    uint4 d[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int i = base + j * TB + thread;
      d[j] = neg_inf_vec<T>();
      if (i < n) d[j] = load_stream(v + i, policy);
    }
    f(d, base, Flag<false>());
  }
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

// The largest elements of a vector (NaN ignored), two side by side for bf16.
template <typename T>
struct VecMax;
template <>
struct VecMax<__nv_bfloat16> {
  __nv_bfloat162 m;
  __device__ __forceinline__ void of(const uint4& u) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
    m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  }
  __device__ __forceinline__ void none() { m = __float2bfloat162_rn(-INFINITY); }
  __device__ __forceinline__ void join(const VecMax& o) { m = __hmax2(m, o.m); }
  __device__ __forceinline__ float value() const { return fmaxf(__low2float(m), __high2float(m)); }
  // some element is at least b, a logit (so that bf16 holds it)
  __device__ __forceinline__ bool reaches(float b) const { return !__hblt2(m, __float2bfloat162_rn(b)); }
};
template <>
struct VecMax<float> {
  float m;
  __device__ __forceinline__ void of(const uint4& u) {
    m = fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
  }
  __device__ __forceinline__ void none() { m = -INFINITY; }
  __device__ __forceinline__ void join(const VecMax& o) { m = fmaxf(m, o.m); }
  __device__ __forceinline__ float value() const { return m; }
  __device__ __forceinline__ bool reaches(float b) const { return m >= b; }
};

// The largest element of the vectors with `use(j)`; vm: of each of them.
template <typename T, int NV, typename F>
__device__ __forceinline__ float vecs_max(const uint4 (&d)[NV], VecMax<T> (&vm)[NV], F use) {
  VecMax<T> m;
  m.none();
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (use(j)) {
      vm[j].of(d[j]);
      m.join(vm[j]);
    }
  return m.value();
}

// max(x, -1e30) per element, NaN kept: finite where -inf would make 0 * -inf.
template <typename T>
__device__ __forceinline__ uint4 clamp_low(const uint4& u) {
  uint4 r;
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  uint32_t o[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (sizeof(T) == 2)  // 0xF149 = bf16(-1e30)
      asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(o[j]) : "r"(w[j]), "r"(0xF149F149u));
    else
      asm("max.NaN.f32 %0, %1, %2;" : "=r"(o[j]) : "r"(w[j]), "r"(0xF149F2CAu));
  }
  r = make_uint4(o[0], o[1], o[2], o[3]);
  return r;
}

__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// ---- the sums of a softmax ------------------------------------------------------------------
// In log2 units: c = log2(e) / T, terms 2^(c x - R) by one fused multiply-add and one SFU exponential.
// R is the ceiling of c times the largest logit so far: a whole number, so that sums against different
// R are joined by exact powers of two and the result does not depend on how R was rounded.  Holds for
// |c x| up to 1e19 ("plain" rows).  A row whose largest logit is beyond that (a mask of the type's lowest
// value over every entry, infinities, NaN) is summed again as 2^(c (x - max)).
constexpr float kLowRef = -1e20f;

__device__ __forceinline__ float ref_of(float m, float c) { return fmaxf(ceilf(m * c), kLowRef); }
// 1 / T and log2(e) / T are ordinary numbers.
inline bool temperature_ok(float t) { return t >= 1e-30f && t <= 1e30f; }
// The most that |max| c may be for a plain row; none is with c so small or large that the clamp at
// -1e30 would not lie between kLowRef and fp32's range.
inline float plain_most(float c) { return c >= 1e-9f && c <= 1e8f ? 1e19f : -1.f; }

// The logarithm of the distribution at x, given either form's reference (R, or the maximum) and log2 of the sum.
struct Log2P {
  bool plain;
  float c, ref, l2;
  __device__ __forceinline__ float exponent(float x) const { return plain ? fmaf(x, c, -ref) : (x - ref) * c; }
  __device__ __forceinline__ float lse(float inv_t) const {  // natural, of x / T
    return plain ? (ref + l2) * kLn2 : fmaf(ref, inv_t, l2 * kLn2);
  }
  __device__ __forceinline__ float ln(float x, float inv_t) const {
    const float d = exponent(x);
    // log2(e) x may overflow where x does not
    const float r = fabsf(d) == INFINITY && fabsf(x) != INFINITY ? fmaf(x, inv_t, -lse(inv_t)) : (d - l2) * kLn2;
    return r > 0.f ? 0.f : r;  // above 0 by rounding; NaN stays
  }
};

// ---- clusters -------------------------------------------------------------------------------
__device__ __forceinline__ int cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return (int)r;
}
// Only that the peers have started: nothing written before it is waited for.
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// The address of this CTA's shared `p` in CTA `rank` of the cluster.
template <typename P>
__device__ __forceinline__ P* peer(P* p, int rank) {
  uint64_t a;
  asm volatile("mapa.u64 %0, %1, %2;" : "=l"(a) : "l"((uint64_t)p), "r"(rank));
  return reinterpret_cast<P*>(a);
}

// ---- launches that overlap -------------------------------------------------------------------
// A kernel launched `early` may start before the one in front of it in the stream has ended (from that
// one's next_may_start on, or as its CTAs end); what it needs of that one's results it reads behind
// after_previous().
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void next_may_start() { asm volatile("griddepcontrol.launch_dependents;"); }

template <typename... P, typename... A>
int launch_ex(const char* what, void (*kern)(P...), dim3 grid, int block, size_t smem, int cluster, bool early,
              cudaStream_t s, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(block, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  cfg.attrs = at;
  if (cluster > 1) {
    at[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    at[cfg.numAttrs].val.clusterDim.x = cluster;
    at[cfg.numAttrs].val.clusterDim.y = at[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  if (early) {
    at[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
  if (e == cudaSuccess) return M3_OK;
  cudaGetLastError();  // else the next call's check would report it again
  return set_error(M3_ERR_LAUNCH, std::string(what) + ": " + cudaGetErrorString(e));
}

}  // namespace vocab
}  // namespace m3
