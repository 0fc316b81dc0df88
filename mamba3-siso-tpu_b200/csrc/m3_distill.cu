// Distillation from a teacher's top logits (forward, and forward with the gradient).
//   q = softmax(x / T), p = softmax(teacher / T) over the k given entries
//   KL = sum_j p_j (ln p_j - ln q_{id_j}),   d(T^2 KL)/dx = T (q - p)
// and with hard labels CE = lse(x) - x_label, dCE/dx = softmax(x) - onehot.
// One read of the logits from memory and one write of their gradient.  Each warp walks its share of a
// row with a running maximum and sums against it; the parts of the row's warps meet at one barrier;
// then the row is walked again, from L2 (so that the rows in flight have to fit there), and its
// gradient written.  One warp holds the teacher's entries, four to a lane.  The dense gradient k_s q is stored
// first; then each entry's place is stored again as k_s q - p, from the same fp32 values, so that
// every element is rounded once.
#include "m3_internal.h"
#include "m3_vocab.cuh"

namespace m3 {
namespace {

using namespace vocab;

constexpr int kNV = 8;          // vectors a thread loads at a time
constexpr int kMaxCluster = 8;  // CTAs per row (portable size)
constexpr int kEnt = M3_MAX_TOP / 32;  // entries a lane holds

struct Params {
  int rows, vocab, k, cluster, log2_cluster;
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

// Sums against a maximum: s = sum e^((x - m) / T), s1 = sum e^(x - m) (only with hard labels).
struct Part {
  float m, s, s1;
};

__device__ __forceinline__ float finite_or_0(float m) { return m == -INFINITY ? 0.f : m; }

template <typename T, bool HARD>
__device__ __forceinline__ void add_vec(const uint4& v, float m, float c, float2& s, float2& s1) {
  float2 f[kVec<T> / 2];
  unpack<T>(v, f);
#pragma unroll
  for (int j = 0; j < kVec<T> / 2; ++j) {
    const float2 x = add2(f[j], f2s(-m));
    const float2 d = mul2(x, f2s(c));
    s = add2(s, f2(ex2(d.x), ex2(d.y)));
    if (HARD) {
      const float2 d1 = mul2(x, f2s(kLog2e));
      s1 = add2(s1, f2(ex2(d1.x), ex2(d1.y)));
    }
  }
}

template <bool HARD>
__device__ __forceinline__ Part join(Part p, float c) {
  Part r;
  r.m = warp_max(p.m);
  const bool none = p.m == -INFINITY;
  r.s = warp_sum(p.s * (none ? 0.f : ex2((p.m - r.m) * c)));
  r.s1 = HARD ? warp_sum(p.s1 * (none ? 0.f : ex2((p.m - r.m) * kLog2e))) : 1.f;
  return r;
}

// The teacher's entries of a row, held by one warp: entry lane + 32 e.
struct Entries {
  int id[kEnt];  // -1: absent
  float t[kEnt], x[kEnt];
};

enum { kSoft = 1, kHard = 2, kBad = 4 };  // a row's terms; kBad: an id or label past the vocabulary

// `ids` are loaded as they are, absent and bad ones become -1.
template <bool HARD>
__device__ __forceinline__ int load_entries(const Params& p, int row, float w, int64_t label, Entries& en) {
  const int lane = threadIdx.x & 31;
  bool any = false, bad = false;
#pragma unroll
  for (int e = 0; e < kEnt; ++e) {
    en.id[e] = -1;
    en.t[e] = -INFINITY;
    if (32 * e < p.k) {
      const int j = lane + 32 * e;
      if (j < p.k) {
        const int64_t id = p.ids[(int64_t)row * p.k + j];
        const float t = p.teacher[(int64_t)row * p.k + j];
        bad |= id >= p.vocab;
        if (id >= 0 && id < p.vocab) {
          en.id[e] = (int)id;
          en.t[e] = t;
          any = true;
        }
      }
    }
  }
  any = __any_sync(0xffffffffu, any || bad);
  bad = __any_sync(0xffffffffu, bad) || (HARD && label >= p.vocab);
  int f = (any && (!HARD || p.hard < 1.f) ? kSoft : 0) | (HARD && label >= 0 ? kHard : 0);
  if (w == 0.f) f = 0;
  return f && bad ? kBad : f;
}

// The teacher's probabilities and their logarithms; an absent entry has probability 0.
__device__ __forceinline__ void teacher_softmax(const Params& p, const Entries& en, float (&pr)[kEnt], float (&lp)[kEnt]) {
  float tm = -INFINITY, es = 0.f;
#pragma unroll
  for (int e = 0; e < kEnt; ++e)
    if (32 * e < p.k) tm = fmaxf(tm, en.t[e]);
  tm = warp_max(tm);
#pragma unroll
  for (int e = 0; e < kEnt; ++e)
    if (32 * e < p.k) {
      lp[e] = (en.t[e] - tm) * p.inv_t;
      pr[e] = en.id[e] >= 0 ? ex2(lp[e] * kLog2e) : 0.f;
      es += pr[e];
    }
  es = warp_sum(es);
  const float ls = log2f(es) * kLn2, inv = 1.f / es;
#pragma unroll
  for (int e = 0; e < kEnt; ++e)
    if (32 * e < p.k) {
      pr[e] *= inv;
      lp[e] -= ls;
    }
}

// The loss of a row, by the warp that holds its entries.
template <bool HARD>
__device__ __forceinline__ float row_loss(const Params& p, const Part& a, int flags, float w, const Entries& en,
                                          const float (&pr)[kEnt], const float (&lp)[kEnt], float xl) {
  if (flags == 0) return 0.f;
  if (flags & kBad) return NAN;
  const float ln_z = a.m == -INFINITY ? NAN : log2f(a.s) * kLn2;
  float kl = 0.f;
#pragma unroll
  for (int e = 0; e < kEnt; ++e)
    if (32 * e < p.k && en.id[e] >= 0 && pr[e] != 0.f) kl = fmaf(pr[e], lp[e] - (en.x[e] - a.m) * p.inv_t + ln_z, kl);
  kl = warp_sum(kl);
  float loss = flags & kSoft ? (1.f - p.hard) * p.temperature * p.temperature * kl : 0.f;
  if (HARD && (flags & kHard)) loss += p.hard * ((a.m == -INFINITY ? NAN : log2f(a.s1) * kLn2) - (xl - a.m));
  return w * loss;
}

// The gradient of a row at a logit x: ks e^((x - m) / T) + kh e^(x - m), less `as` p for an entry and
// `ah` for the label.
struct Coef {
  float m, c, ks, kh, as, ah;
  template <bool HARD>
  __device__ __forceinline__ float2 at(float2 x) const {
    const float2 y = add2(x, f2s(-m)), d = mul2(y, f2s(c));
    float2 g = mul2(f2(ex2(d.x), ex2(d.y)), f2s(ks));
    if (HARD) {
      const float2 d1 = mul2(y, f2s(kLog2e));
      g = fma2(f2(ex2(d1.x), ex2(d1.y)), f2s(kh), g);
    }
    return g;
  }
  // at an entry of probability `a` and / or the label, each share less its own target
  template <bool HARD>
  __device__ __forceinline__ float at_entry(float x, float a, bool label) const {
    float g = ks * ex2((x - m) * c) - as * a;
    if (HARD) g += kh * ex2((x - m) * kLog2e) - (label ? ah : 0.f);
    return g;
  }
};

template <bool HARD>
__device__ __forceinline__ Coef coefficients(const Params& p, const Part& a, int row, int flags, float w) {
  float r = p.scale * w;
  if (p.weight_sum) r /= *p.weight_sum;
  if (p.upstream) r *= p.upstream[row * p.upstream_stride];
  Coef g;
  g.m = a.m;
  g.c = p.inv_t * kLog2e;
  g.as = flags & kSoft ? r * (1.f - p.hard) * p.temperature : 0.f;
  g.ah = HARD && (flags & kHard) ? r * p.hard : 0.f;
  g.ks = flags & kSoft ? g.as / a.s : 0.f;
  g.kh = HARD && (flags & kHard) ? g.ah / a.s1 : 0.f;
  if (flags & kBad) g.ks = NAN;
  return g;
}

template <typename T, bool HARD>
__device__ __forceinline__ uint4 grad_vec(const uint4& v, const Coef& k) {
  float2 f[kVec<T> / 2];
  unpack<T>(v, f);
#pragma unroll
  for (int j = 0; j < kVec<T> / 2; ++j) f[j] = k.at<HARD>(f[j]);
  if constexpr (sizeof(T) == 2)
    return make_uint4(f2bf(f[0]), f2bf(f[1]), f2bf(f[2]), f2bf(f[3]));
  else
    return make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x), __float_as_uint(f[1].y));
}

// The E elements at g; `vec`: g is 16-byte aligned.
template <typename T>
__device__ __forceinline__ void store_vec(T* g, const uint4& u, bool vec, uint64_t policy) {
  if (vec) {
    store_stream(g, u, policy);
    return;
  }
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < kVec<T>; ++j) {
    if constexpr (sizeof(T) == 2)
      reinterpret_cast<uint16_t*>(g)[j] = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
    else
      reinterpret_cast<uint32_t*>(g)[j] = w[j];
  }
}

// Stores the gradient again at the entries (and the label) within [lo, hi), by the warp that holds
// them.  An id that occurs twice (its bit in `seen`, hi - lo clear bits, is set already; without
// `seen` it is always looked for) is stored once, with all its probabilities.  ids, amounts: k words of
// shared memory for that search.
template <typename T, bool HARD>
__device__ __forceinline__ void store_entries(const Params& p, T* g, int lo, int hi, const Coef& k, const Entries& en,
                                              const float (&pr)[kEnt], int64_t label, float xl, uint32_t* seen,
                                              int* ids, float* amounts) {
  const int lane = threadIdx.x & 31;
  const bool hard = HARD && k.ah != 0.f;
  bool twice = seen == nullptr, hit = false;
#pragma unroll
  for (int e = 0; e < kEnt; ++e)
    if (32 * e < p.k) {
      const int id = en.id[e];
      if (seen && id >= lo && id < hi) {
        const uint32_t bit = 1u << ((id - lo) & 31);
        twice |= (atomicOr(&seen[(id - lo) >> 5], bit) & bit) != 0u;
      }
      hit |= id >= 0 && id == label;
    }
  twice = __any_sync(0xffffffffu, twice);
  if (twice) {
#pragma unroll
    for (int e = 0; e < kEnt; ++e)
      if (lane + 32 * e < p.k) {
        ids[lane + 32 * e] = en.id[e];
        amounts[lane + 32 * e] = pr[e];
      }
    __syncwarp();
  }
#pragma unroll
  for (int e = 0; e < kEnt; ++e)
    if (32 * e < p.k) {
      const int id = en.id[e];
      bool first = id >= lo && id < hi;
      float a = pr[e];
      if (twice && first) {
        a = 0.f;
        for (int j = 0; j < p.k; ++j)
          if (ids[j] == id) {
            a += amounts[j];
            if (j < lane + 32 * e) first = false;
          }
      }
      if (first) stg<T>(g + id, k.at_entry<HARD>(en.x[e], a, id == label));
    }
  if (HARD) {
    hit = __any_sync(0xffffffffu, hit);
    if (hard && !hit && lane == 0 && label >= lo && label < hi) stg<T>(g + label, k.at_entry<HARD>(xl, 0.f, true));
  }
}

// ---- one CTA or one cluster per row -------------------------------------------------------
template <int TB, bool GRAD>
struct Smem {
  static constexpr int kSeen = GRAD ? 8 * TB : 4;  // a bit per element of a share of up to 256 TB
  Part part[TB / 32];
  Part parts[kMaxCluster];
  int flags;
  int ids[GRAD ? M3_MAX_TOP : 1];
  float amounts[GRAD ? M3_MAX_TOP : 1];
  alignas(16) uint32_t seen[kSeen];  // cleared as 16-byte vectors
};

template <typename T, int TB, bool HARD, bool GRAD>
__global__ void __launch_bounds__(TB, 1024 / TB) distill_kernel(const Params p) {
  constexpr int E = kVec<T>, NW = TB / 32;
  using S = Smem<TB, GRAD>;
  __shared__ S s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cl = p.cluster, rank = cl > 1 ? cluster_rank() : 0;
  const int row = (int)blockIdx.x >> p.log2_cluster;
  const int V = p.vocab;
  const T* x = reinterpret_cast<const T*>(p.logits) + p.lrow.at(row);
  const Split sp = split_row(x, V);
  const int per = (sp.full + cl - 1) >> p.log2_cluster, v0 = min(sp.full, rank * per), n = min(per, sp.full - v0);
  const uint4* v = reinterpret_cast<const uint4*>(x + sp.head) + v0;
  const float c = p.inv_t * kLog2e;
  if (cl > 1) cluster_arrive_relaxed();  // peers have started before anyone writes to their shared memory

  const float w = p.weights ? p.weights[row] : 1.f;
  const int64_t label = HARD ? p.labels[row] : -1;
  Entries en;
  float xl = 0.f, pr[kEnt], lp[kEnt];
  const bool holder = warp == 0 && (GRAD || rank == 0);  // this warp holds the entries
  if (warp == 0) {
    const int f = load_entries<HARD>(p, row, w, label, en);
    if (lane == 0) s.flags = f;
    if (holder) {  // read here: below, the gradient may overwrite the logits
#pragma unroll
      for (int e = 0; e < kEnt; ++e) en.x[e] = 32 * e < p.k && en.id[e] >= 0 ? ld(x + en.id[e]) : 0.f;
      if (HARD && label >= 0 && label < V) xl = ld(x + label);
    }
  }
  if constexpr (GRAD)
    for (int i = tid; i < S::kSeen / 4; i += TB) reinterpret_cast<uint4*>(s.seen)[i] = make_uint4(0u, 0u, 0u, 0u);

  float m = -INFINITY;  // the warp's maximum
  float2 s2 = f2s(0.f), t2 = f2s(0.f);
  auto raise = [&](float to) {  // the sums against a new maximum
    if (to > m) {
      if (m != -INFINITY) {
        s2 = mul2(s2, f2s(ex2((m - to) * c)));
        if (HARD) t2 = mul2(t2, f2s(ex2((m - to) * kLog2e)));
      }
      m = to;
    }
  };
  walk<T, kNV, TB>(v, n, tid, GRAD ? Keep::kYes : Keep::kNo, [&](const uint4(&d)[kNV], int base, auto full) {
    VecMax<T> vm[kNV];
    const float mt = vecs_max<T, kNV>(d, vm, [&](int j) { return full.value || base + j * TB < n; });
    raise(warp_max(mt));
    const float ref = finite_or_0(m);
#pragma unroll
    for (int j = 0; j < kNV; ++j)
      if (full.value || base + j * TB < n) add_vec<T, HARD>(d[j], ref, c, s2, t2);
  });
  int edge = -1;  // this lane's element of the row's edges
  float xe = -INFINITY;
  if (warp == NW - 1) {
    edge = edge_index(sp, lane, rank == 0, rank == cl - 1);
    if (edge >= 0) xe = ld(x + edge);
    raise(warp_max(xe));
    s2.x += ex2((xe - finite_or_0(m)) * c);
    if (HARD) t2.x += ex2((xe - finite_or_0(m)) * kLog2e);
  }
  Part a{m, warp_sum(s2.x + s2.y), HARD ? warp_sum(t2.x + t2.y) : 0.f};
  if (lane == 0) s.part[warp] = a;
  if (holder) teacher_softmax(p, en, pr, lp);
  __syncthreads();
  const Part none{-INFINITY, 0.f, 0.f};
  a = join<HARD>(lane < NW ? s.part[lane] : none, c);
  if (cl > 1) {
    __syncwarp();
    cluster_wait();
    if (tid < cl) *peer(&s.parts[rank], tid) = a;
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    a = join<HARD>(lane < cl ? s.parts[lane] : none, c);
  }
  const int flags = s.flags;
  if (warp == 0 && rank == 0) {
    const float loss = row_loss<HARD>(p, a, flags, w, en, pr, lp, xl);
    if (lane == 0) p.row_loss[row] = loss;
  }
  if constexpr (GRAD) {
    T* g = reinterpret_cast<T*>(p.grad) + p.grow.at(row);
    T* gv = g + sp.head + v0 * E;  // this share's vectors, aligned or not
    const bool vec = row_shift(gv) == 0;
    const Coef k = coefficients<HARD>(p, a, row, flags, w);
    const uint64_t first = l2_policy(Keep::kNo);
    if (flags) {
      walk<T, kNV, TB>(v, n, tid, Keep::kNo, [&](const uint4(&d)[kNV], int base, auto full) {
#pragma unroll
        for (int j = 0; j < kNV; ++j) {
          const int q = base + j * TB + tid;
          if (full.value || base + j * TB < n) {
            const uint4 u = grad_vec<T, HARD>(d[j], k);
            if (full.value || q < n) store_vec<T>(gv + (int64_t)q * E, u, vec, first);
          }
        }
      });
    } else {
      for (int q = tid; q < n; q += TB) store_vec<T>(gv + (int64_t)q * E, make_uint4(0u, 0u, 0u, 0u), vec, first);
    }
    if (edge >= 0) stg<T>(g + edge, flags ? k.at<HARD>(f2s(xe)).x : 0.f);
    __syncthreads();
    if (warp == 0 && flags && !(flags & kBad)) {
      const int lo = rank == 0 ? 0 : sp.head + v0 * E, hi = rank == cl - 1 ? V : sp.head + (v0 + n) * E;
      store_entries<T, HARD>(p, g, lo, hi, k, en, pr, label, xl, hi - lo <= 32 * S::kSeen ? s.seen : nullptr, s.ids,
                             s.amounts);
    }
  }
}

// ---- one warp per row ---------------------------------------------------------------------
constexpr int kWarpThreads = 256, kWarpRows = kWarpThreads / 32;

template <typename T, int NV, bool HARD, bool GRAD>
__global__ void __launch_bounds__(kWarpThreads) distill_warp_kernel(const Params p) {
  constexpr int E = kVec<T>, kSeen = NV * E;  // words of 32 bits: one bit per element
  __shared__ uint4 row_of[kWarpRows][NV * 32];
  __shared__ uint32_t seen_of[kWarpRows][GRAD ? kSeen : 1];
  __shared__ int ids_of[kWarpRows][GRAD ? M3_MAX_TOP : 1];
  __shared__ float amounts_of[kWarpRows][GRAD ? M3_MAX_TOP : 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, V = p.vocab;
  const int step = gridDim.x * kWarpRows;
  const float c = p.inv_t * kLog2e;
  int row = blockIdx.x * kWarpRows + warp;
  uint4 d[NV];
  int shift = 0;
  auto load = [&](int r) {
    const T* x = reinterpret_cast<const T*>(p.logits) + p.lrow.at(r);
    shift = row_shift(x);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int lo = (j * 32 + lane) * E - shift;
      d[j] = lo < V ? load_vec(x, lo, V) : neg_inf_vec<T>();
    }
  };
  if (row < p.rows) load(row);
  for (; row < p.rows; row += step) {
    const float w = p.weights ? p.weights[row] : 1.f;
    const int64_t label = HARD ? p.labels[row] : -1;
    Entries en;
    const int flags = load_entries<HARD>(p, row, w, label, en);
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      row_of[warp][j * 32 + lane] = d[j];
    }
    VecMax<T> vm[NV];
    m = vecs_max<T, NV>(d, vm, [](int) { return true; });
    if (GRAD)
      for (int i = lane; i < kSeen; i += 32) seen_of[warp][i] = 0u;
    m = warp_max(m);
    const float ref = finite_or_0(m);
    float2 s2 = f2s(0.f), t2 = f2s(0.f);
#pragma unroll
    for (int j = 0; j < NV; ++j) add_vec<T, HARD>(d[j], ref, c, s2, t2);
    __syncwarp();
    const T* xs = reinterpret_cast<const T*>(row_of[warp]) + shift;
#pragma unroll
    for (int e = 0; e < kEnt; ++e) en.x[e] = 32 * e < p.k && en.id[e] >= 0 ? ld(xs + en.id[e]) : 0.f;
    const float xl = HARD && label >= 0 && label < V ? ld(xs + label) : 0.f;
    float pr[kEnt], lp[kEnt];
    teacher_softmax(p, en, pr, lp);
    const Part a{m, warp_sum(s2.x + s2.y), HARD ? warp_sum(t2.x + t2.y) : 1.f};
    const float loss = row_loss<HARD>(p, a, flags, w, en, pr, lp, xl);
    if (lane == 0) p.row_loss[row] = loss;
    const int at = shift;
    uint4 u[GRAD ? NV : 1];
    Coef k;
    if constexpr (GRAD) {
      k = coefficients<HARD>(p, a, row, flags, w);
#pragma unroll
      for (int j = 0; j < NV; ++j) u[j] = flags ? grad_vec<T, HARD>(d[j], k) : make_uint4(0u, 0u, 0u, 0u);
    }
    if (row + step < p.rows) load(row + step);  // on its way while this row is finished
    if constexpr (GRAD) {
      T* g = reinterpret_cast<T*>(p.grad) + p.grow.at(row);
      const bool vec = row_shift(g) == at;
      const uint64_t first = l2_policy(Keep::kNo);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int lo = (j * 32 + lane) * E - at;
        if (lo >= 0 && lo + E <= V) {
          store_vec<T>(g + lo, u[j], vec, first);
        } else if (lo < V) {
          const T* e = reinterpret_cast<const T*>(&u[j]);
#pragma unroll
          for (int i = 0; i < E; ++i)
            if (lo + i >= 0 && lo + i < V) g[lo + i] = e[i];
        }
      }
      __syncwarp();
      if (flags && !(flags & kBad))
        store_entries<T, HARD>(p, g, 0, V, k, en, pr, label, xl, seen_of[warp], ids_of[warp], amounts_of[warp]);
    }
    __syncwarp();  // the row's shared memory is free again
  }
}

// out = scale * (sum of n values) / (*div_by, if given), by one cluster in a fixed order.
constexpr int kSumCtas = 8, kSumThreads = 1024;

__global__ void __cluster_dims__(kSumCtas, 1, 1) __launch_bounds__(kSumThreads)
    sum_kernel(const float* __restrict__ v, int64_t n, const float* div_by, float scale, float* out) {
  __shared__ float sm[32], total[kSumCtas];
  const int tid = threadIdx.x, rank = cluster_rank();
  cluster_arrive_relaxed();
  float s = 0.f;
#pragma unroll 4
  for (int64_t i = (int64_t)rank * kSumThreads + tid; i < n; i += kSumCtas * kSumThreads) s += v[i];
  s = warp_sum(s);
  if ((tid & 31) == 0) sm[tid >> 5] = s;
  __syncthreads();
  s = warp_sum(sm[tid & 31]);
  cluster_wait();
  if (tid == 0) *peer(&total[rank], 0) = s;
  __syncwarp();
  cluster_arrive();
  cluster_wait();
  if (rank == 0 && tid == 0) {
    s = 0.f;
    for (int r = 0; r < kSumCtas; ++r) s += total[r];
    *out = s * scale / (div_by ? *div_by : 1.f);
  }
}

int sm_count() {
  int dev = 0, c = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&c, cudaDevAttrMultiProcessorCount, dev);
  return c;
}

template <typename T, int TB, bool HARD, bool GRAD>
int launch_cta(const Params& p, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p.rows * p.cluster, 1, 1);
  cfg.blockDim = dim3(TB, 1, 1);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = p.cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = p.cluster > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, distill_kernel<T, TB, HARD, GRAD>, p);
  return e == cudaSuccess ? M3_OK : set_error(M3_ERR_LAUNCH, std::string("m3_distill: ") + cudaGetErrorString(e));
}

template <typename T, int NV, bool HARD, bool GRAD>
int launch_warp(const Params& p, cudaStream_t s) {
  const int want = (p.rows + kWarpRows - 1) / kWarpRows, most = sm_count() * 8;
  distill_warp_kernel<T, NV, HARD, GRAD><<<(unsigned)(want < most ? want : most), kWarpThreads, 0, s>>>(p);
  return check_launch("m3_distill");
}

// A row goes to a warp while its vectors fit the lanes' registers, else to a CTA, and with few rows to
// a cluster.
template <typename T, bool HARD, bool GRAD>
int launch(Params p, int nvec, cudaStream_t s) {
  if (nvec <= 32) return launch_warp<T, 1, HARD, GRAD>(p, s);
  if (nvec <= 64) return launch_warp<T, 2, HARD, GRAD>(p, s);
  if (nvec <= 128) return launch_warp<T, 4, HARD, GRAD>(p, s);
  if (nvec <= 256) return launch_warp<T, 8, HARD, GRAD>(p, s);
  // few rows: several CTAs per row until they cover the SMs
  const int sms = sm_count();
  int cl = 1;
  while (cl < kMaxCluster && (int64_t)p.rows * cl * 2 <= sms && nvec / (cl * 2) >= 128) cl *= 2;
  p.cluster = cl;
  while ((1 << p.log2_cluster) < cl) ++p.log2_cluster;
  if ((int64_t)p.rows * cl > 0x7FFFFFFF) return set_error(M3_ERR_SHAPE, "m3_distill: too many rows");
  // a second walk finds its row in L2 only while the rows in flight (1024 / threads per SM) fit there
  if (nvec <= kNV * 128 * cl) return launch_cta<T, 128, HARD, GRAD>(p, s);
  const bool fits = (int64_t)nvec * 16 * 4 * sms <= (int64_t)64 << 20;
  return (GRAD && !fits) || (int64_t)p.rows * cl <= 2 * sms ? launch_cta<T, 512, HARD, GRAD>(p, s)
                                                             : launch_cta<T, 256, HARD, GRAD>(p, s);
}

template <typename T>
int launch(const Params& p, int nvec, cudaStream_t s) {
  if (p.hard > 0.f) return p.grad ? launch<T, true, true>(p, nvec, s) : launch<T, true, false>(p, nvec, s);
  return p.grad ? launch<T, false, true>(p, nvec, s) : launch<T, false, false>(p, nvec, s);
}

}  // namespace
}  // namespace m3

using namespace m3;

extern "C" int m3_distill(const M3DistillArgs* args, void* stream) {
  if (!args) return set_error(M3_ERR_ARG, "m3_distill: args is NULL");
  const M3DistillArgs& a = *args;
  if (a.rows_outer < 0 || a.rows_inner < 0 || a.vocab <= 0 || a.vocab > kMaxVocab || a.k <= 0 || a.k > M3_MAX_TOP)
    return set_error(M3_ERR_SHAPE, "m3_distill: need rows >= 0, 0 < vocab <= 2^30 and 1 <= k <= 128");
  if (a.logits_dtype != M3_DTYPE_F32 && a.logits_dtype != M3_DTYPE_BF16)
    return set_error(M3_ERR_UNSUPPORTED, "m3_distill: logits must be f32 or bf16");
  if (a.reduction < M3_REDUCE_NONE || a.reduction > M3_REDUCE_MEAN)
    return set_error(M3_ERR_ARG, "m3_distill: reduction must be NONE, SUM or MEAN");
  if (!(a.temperature > 0.f) || !(a.hard_weight >= 0.f && a.hard_weight <= 1.f))
    return set_error(M3_ERR_ARG, "m3_distill: need temperature > 0 and 0 <= hard_weight <= 1");
  const int64_t rows = (int64_t)a.rows_outer * a.rows_inner;
  if (rows > kMaxRows) return set_error(M3_ERR_SHAPE, "m3_distill: more than 2^30 rows");
  if ((rows > 0 && (!a.logits || !a.ids || !a.teacher || !a.row_loss)) ||
      (a.hard_weight > 0.f && rows > 0 && !a.labels) || (a.reduction != M3_REDUCE_NONE && !a.loss))
    return set_error(M3_ERR_ARG, "m3_distill: NULL pointer");
  const bool wmean = a.reduction == M3_REDUCE_MEAN && a.weights && rows > 0;
  if (wmean && !a.weight_sum) return set_error(M3_ERR_ARG, "m3_distill: a mean with weights needs weight_sum");
  if (a.upstream_stride < 0 || a.upstream_stride > 1)
    return set_error(M3_ERR_ARG, "m3_distill: upstream_stride must be 0 or 1");
  const bool bf = a.logits_dtype == M3_DTYPE_BF16;
  const size_t size = bf ? 2 : 4;
  if (((uintptr_t)a.logits) % size || ((uintptr_t)a.grad) % size)
    return set_error(M3_ERR_ARG, "m3_distill: logits and grad must be aligned to their type");
  cudaStream_t s = (cudaStream_t)stream;
  Params p;
  p.rows = (int)rows;
  p.cluster = 1;
  p.log2_cluster = 0;
  p.vocab = a.vocab;
  p.k = a.k;
  p.temperature = a.temperature;
  p.inv_t = 1.f / a.temperature;
  p.hard = a.hard_weight;
  p.scale = a.grad_scale;
  if (a.reduction == M3_REDUCE_MEAN && !a.weights) p.scale /= (float)rows;
  p.lrow = Rows{a.rows_outer, a.rows_inner, a.ld_outer, a.ld_inner};
  p.grow = Rows{a.rows_outer, a.rows_inner, a.g_outer, a.g_inner};
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
  if (wmean) sum_kernel<<<kSumCtas, kSumThreads, 0, s>>>(a.weights, rows, nullptr, 1.f, a.weight_sum);
  if (rows > 0) {
    const int nvec = most_vectors(a.logits, a.vocab, bf ? 2 : 4, a.ld_outer, a.ld_inner);
    const int rc = bf ? launch<__nv_bfloat16>(p, nvec, s) : launch<float>(p, nvec, s);
    if (rc != M3_OK) return rc;
  }
  if (a.reduction != M3_REDUCE_NONE)  // the mean of no rows is 0 / 0
    sum_kernel<<<kSumCtas, kSumThreads, 0, s>>>(a.row_loss, rows, p.weight_sum,
                                                a.reduction == M3_REDUCE_MEAN && !a.weights ? 1.f / (float)rows : 1.f,
                                                a.loss);
  return check_launch("m3_distill");
}
