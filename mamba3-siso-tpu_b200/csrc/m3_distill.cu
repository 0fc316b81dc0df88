// Distillation from a teacher's top logits (forward, and forward with the gradient).
//   q = softmax(x / T), p = softmax(teacher / T) over the k given entries
//   KL = sum_j p_j (ln p_j - ln q_{id_j}),   d(T^2 KL)/dx = T (q - p)
// and with hard labels CE = lse(x) - x_label, dCE/dx = softmax(x) - onehot.
// One read of the logits from memory and one write of their gradient.  Each warp walks its share of a
// row with a running maximum and sums against it; the parts of the row's warps meet at one barrier;
// then the row is walked again, its first tile still in registers and its second in shared memory, the
// rest from L2 (so that the rows in flight have to fit there), and its gradient written.  One warp holds
// the teacher's entries.  The dense gradient k_s q is stored first; then each entry's place is stored
// again as k_s q - p, from the same fp32 values, so that every element is rounded once.
// Floor: one read and one write.  Measured with the gradient: 4096 x 128256 bf16 397 to 420 us (5.0 to 5.3 TB/s of
// the 6.4 that a copy reaches; the SFU is busy 62 % of the time with the exponentials and the issue slots 39 %, so
// that it is how the phases of two CTAs an SM overlap that decides), 32768 x 8192 f32 332 us (6.5 TB/s), 131072 x 256
// bf16 with weights 72 us (2.2 TB/s, bound by about 440 instructions a row).  Reading the whole row again from L2
// took 535 us at the first size with four rows an SM in flight (150 MB, more than L2), 430 with two.
// The loss alone: 168 us at the first size; with hard labels 427, as the 64 registers of a thread then hold a bf16
// tile only with 488 bytes of them spilled (f32, 4095 x 50257: 136 and 146).
#include "m3_internal.h"
#include "m3_vocab.cuh"

namespace m3 {
namespace {

using namespace vocab;

constexpr int kNV = 8;          // vectors a thread loads at a time
constexpr int kMaxCluster = 8;  // CTAs per row (portable size)
constexpr int kEnt = M3_MAX_TOP / 32;  // entries a lane holds at most
constexpr float kMostTemperature = 1e18f;  // T * T is a finite factor of the loss

struct Params {
  int rows, vocab, k, cluster, log2_cluster;
  float temperature, inv_t, c, plain_most, hard, scale;  // scale: grad_scale, over the row count for an unweighted mean
  Rows lrow, grow;
  const void* logits;
  void* grad;
  const int64_t *ids, *labels;
  const float *teacher, *weights, *upstream;
  int64_t upstream_stride;
  const float* weight_sum;  // a mean's divisor, NULL = none
  float* row_loss;
  bool ready;  // grad holds the gradient for an upstream of 1
  bool early;  // the sum of weights is the kernel in front of this one, which may start before that has ended
};

// The gradient is there already (the same for all threads).
__device__ __forceinline__ bool nothing_to_do(const Params& p) { return p.ready && *p.upstream == 1.f; }

// The maximum, and the sums s = sum 2^(c x - r) and, with hard labels, s1 = sum 2^(log2(e) x - r1).
struct Part {
  float m, r, s, r1, s1;
};
__device__ __forceinline__ Part no_part() { return Part{-INFINITY, kLowRef, 0.f, kLowRef, 0.f}; }

template <typename T, bool HARD>
__device__ __forceinline__ void add_vec(const uint4& v, float r, float r1, float c, float2& s, float2& s1) {
  float2 f[kVec<T> / 2];
  unpack<T>(v, f);
#pragma unroll
  for (int j = 0; j < kVec<T> / 2; ++j) {
    const float2 d = fma2(f[j], f2s(c), f2s(-r));
    s = add2(s, f2(ex2(d.x), ex2(d.y)));
    if (HARD) {
      const float2 d1 = fma2(f[j], f2s(kLog2e), f2s(-r1));
      s1 = add2(s1, f2(ex2(d1.x), ex2(d1.y)));
    }
  }
}

template <bool HARD>
__device__ __forceinline__ Part join(Part p) {
  Part q;
  q.m = warp_max(p.m);
  q.r = warp_max(p.r);
  q.s = warp_sum(p.s * ex2(p.r - q.r));
  q.r1 = HARD ? warp_max(p.r1) : 0.f;
  q.s1 = HARD ? warp_sum(p.s1 * ex2(p.r1 - q.r1)) : 1.f;
  return q;
}

// The terms [lo, hi) of a row that is not plain, every `step`-th from lo + first, against its maximum.
template <typename T>
__device__ __noinline__ Part slow_part(const T* x, int lo, int hi, int first, int step, float m, float c) {
  float s = 0.f, s1 = 0.f;
  for (int i = lo + first; i < hi; i += step) {
    const float d = ld(x + i) - m;
    s += ex2(d * c);
    s1 += ex2(d * kLog2e);
  }
  return Part{m, 0.f, s, 0.f, s1};
}

// A row's distributions (at T, and at 1 for the label) and the factors of its gradient
//   ks 2^(c x - ref) + kh 2^(log2(e) x - ref1),  less `as` p at an entry and `ah` at the label.
struct Row {
  Log2P q, q1;
  float s, s1, ks, kh, as, ah;
  template <bool HARD>
  __device__ __forceinline__ float2 plain(float2 x) const {
    const float2 d = fma2(x, f2s(q.c), f2s(-q.ref));
    float2 g = mul2(f2(ex2(d.x), ex2(d.y)), f2s(ks));
    if (HARD) {
      const float2 d1 = fma2(x, f2s(kLog2e), f2s(-q1.ref));
      g = fma2(f2(ex2(d1.x), ex2(d1.y)), f2s(kh), g);
    }
    return g;
  }
  template <bool HARD>
  __device__ __forceinline__ float dense(float x) const {
    const float g = ks * ex2(q.exponent(x));
    return HARD ? fmaf(kh, ex2(q1.exponent(x)), g) : g;
  }
  // At an entry given probability `a`, or the label: each share's probability less its target before the
  // factor, so that equal ones cancel exactly.
  template <bool HARD>
  __device__ __forceinline__ float at(float x, float a, bool label) const {
    const float g = as * (ex2(q.exponent(x)) / s - a);
    return HARD ? g + ah * (ex2(q1.exponent(x)) / s1 - (label ? 1.f : 0.f)) : g;
  }
};

template <typename T, bool HARD>
__device__ __forceinline__ uint4 grad_vec(const uint4& v, const Row& r) {
  float2 f[kVec<T> / 2];
  unpack<T>(v, f);
#pragma unroll
  for (int j = 0; j < kVec<T> / 2; ++j) f[j] = r.plain<HARD>(f[j]);
  if constexpr (sizeof(T) == 2)
    return make_uint4(f2bf(f[0]), f2bf(f[1]), f2bf(f[2]), f2bf(f[3]));
  else
    return make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x), __float_as_uint(f[1].y));
}

// The E elements at g, whatever its alignment.
template <typename T>
__device__ __forceinline__ void store_elements(T* g, const uint4& u) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < kVec<T>; ++j) {
    if constexpr (sizeof(T) == 2)
      reinterpret_cast<uint16_t*>(g)[j] = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
    else
      reinterpret_cast<uint32_t*>(g)[j] = w[j];
  }
}

// ---- the teacher's entries, by the warp that holds them: entry lane + 32 e in place e of a lane ----
template <int KE>
struct Entries {
  int id[KE];  // -1: absent
  float x[KE], p[KE], lp[KE];  // logit; probability and its logarithm
};

enum { kSoft = 1, kHard = 2, kBad = 4 };  // a row's terms; kBad: an id or label past the vocabulary

// Entry e, its id and teacher logit as they are given.  1: present, 2: bad.
template <int KE>
__device__ __forceinline__ int put_entry(Entries<KE>& en, int e, int64_t id, float t, int vocab) {
  const bool there = id >= 0 && id < vocab;
  en.id[e] = there ? (int)id : -1;
  en.lp[e] = there ? t : -INFINITY;
  return there ? 1 : id >= vocab ? 2 : 0;
}
// The row's terms from the `or` of put_entry over its entries.
template <bool HARD>
__device__ __forceinline__ int row_flags(const Params& p, int found, float w, int64_t label) {
  found = __reduce_or_sync(0xffffffffu, found);
  const bool bad = (found & 2) || (HARD && label >= p.vocab);
  int f = (found && (!HARD || p.hard < 1.f) ? kSoft : 0) | (HARD && label >= 0 ? kHard : 0);
  if (w == 0.f || !(f || bad)) return 0;
  return bad ? kBad : f;
}

template <int KE>
__device__ __forceinline__ void teacher_softmax(const Params& p, Entries<KE>& en) {
  float tm = -INFINITY, es = 0.f;
#pragma unroll
  for (int e = 0; e < KE; ++e) tm = fmaxf(tm, en.lp[e]);
  tm = warp_max(tm);
#pragma unroll
  for (int e = 0; e < KE; ++e) {
    en.lp[e] = (en.lp[e] - tm) * p.inv_t;
    en.p[e] = en.id[e] >= 0 ? ex2(en.lp[e] * kLog2e) : 0.f;
    es += en.p[e];
  }
  es = warp_sum(es);
  const float ls = log2f(es) * kLn2, inv = rcp_approx(es);
#pragma unroll
  for (int e = 0; e < KE; ++e) {
    en.p[e] = en.id[e] >= 0 ? en.p[e] * inv : 0.f;
    en.lp[e] -= ls;
  }
}

template <bool HARD, int KE>
__device__ __forceinline__ float row_loss(const Params& p, const Row& r, int flags, float w, const Entries<KE>& en,
                                          float xl) {
  if (flags == 0) return 0.f;
  if (flags & kBad) return NAN;
  float kl = 0.f;
#pragma unroll
  for (int e = 0; e < KE; ++e)  // an entry of probability 0 has no term
    if (en.p[e] != 0.f) kl = fmaf(en.p[e], en.lp[e] - r.q.ln(en.x[e], p.inv_t), kl);
  kl = warp_sum(kl);
  // KL grows as 1 / T where T is small: T * T would leave fp32's range before T * (T * KL) does
  float loss = flags & kSoft ? (1.f - p.hard) * (p.temperature * (p.temperature * kl)) : 0.f;
  if (HARD && (flags & kHard)) loss -= p.hard * r.q1.ln(xl, 1.f);
  return w * loss;
}

// `norm`: grad_scale over the mean's divisor.
template <bool HARD>
__device__ __forceinline__ Row make_row(const Params& p, const Part& a, bool plain, int row, int flags, float w, float norm) {
  Row r;
  r.s = a.s;
  r.s1 = a.s1;
  r.q = Log2P{plain, p.c, plain ? a.r : a.m, log2f(a.s)};
  r.q1 = Log2P{plain, kLog2e, plain ? a.r1 : a.m, HARD ? log2f(a.s1) : 0.f};
  float g = norm * w;
  if (p.upstream) g *= p.upstream[row * p.upstream_stride];
  r.as = flags & kSoft ? g * (1.f - p.hard) * p.temperature : 0.f;
  r.ah = HARD && (flags & kHard) ? g * p.hard : 0.f;
  r.ks = flags & kBad ? NAN : flags & kSoft ? r.as * rcp_approx(a.s) : 0.f;
  r.kh = HARD && (flags & kHard) ? r.ah * rcp_approx(a.s1) : 0.f;
  return r;
}

// Stores the gradient again at the entries (and the label) within [lo, hi).  An id that occurs twice (its
// bit in `seen`, hi - lo clear bits, is set already; without `seen` it is always looked for) is stored once,
// with all its probabilities.  ids, probs: k words each for that search.
template <typename T, bool HARD, int KE>
__device__ __forceinline__ void store_entries(const Params& p, T* g, int lo, int hi, const Row& r, int flags,
                                              const Entries<KE>& en, int64_t label, float xl, uint32_t* seen, int* ids,
                                              float* probs) {
  const int lane = threadIdx.x & 31;
  const bool hard = HARD && (flags & kHard);  // a share that is off has a factor of 0
  bool twice = seen == nullptr, hit = false;
#pragma unroll
  for (int e = 0; e < KE; ++e) {
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
    for (int e = 0; e < KE; ++e)
      if (lane + 32 * e < p.k) {
        ids[lane + 32 * e] = en.id[e];
        probs[lane + 32 * e] = en.p[e];
      }
    __syncwarp();
  }
#pragma unroll
  for (int e = 0; e < KE; ++e) {
    const int id = en.id[e];
    bool first = id >= lo && id < hi;
    float a = en.p[e];
    if (twice && first) {
      a = 0.f;
      for (int i = 0; i < p.k; ++i)
        if (ids[i] == id) {
          a += probs[i];
          if (i < lane + 32 * e) first = false;
        }
    }
    if (first) stg<T>(g + id, r.at<HARD>(en.x[e], a, id == label));
  }
  if (HARD) {
    hit = __any_sync(0xffffffffu, hit);
    if (hard && !hit && lane == 0 && label >= lo && label < hi) stg<T>(g + label, r.at<HARD>(xl, 0.f, true));
  }
}

// ---- one CTA or one cluster per row -------------------------------------------------------
template <int TB, bool GRAD>
struct alignas(16) Smem {
  static constexpr int kSeen = GRAD ? 8 * TB : 4;  // a bit per element of a share of up to 256 TB
  alignas(16) uint32_t seen[kSeen];                // cleared as 16-byte vectors
  int ids[M3_MAX_TOP];
  float probs[M3_MAX_TOP];
  Part part[TB / 32];
  Part parts[kMaxCluster], again[kMaxCluster];
  int flags;
};

template <typename T, int TB, bool HARD, bool GRAD>
__global__ void __launch_bounds__(TB, 1024 / TB) distill_kernel(const Params p) {
  constexpr int E = kVec<T>, NW = TB / 32, kTile = kNV * TB;
  using S = Smem<TB, GRAD>;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  S& s = *reinterpret_cast<S*>(smem_raw);
  uint4* cache = reinterpret_cast<uint4*>(smem_raw + sizeof(S));  // GRAD: the second tile
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cl = p.cluster, rank = cl > 1 ? cluster_rank() : 0;
  const int row = (int)blockIdx.x >> p.log2_cluster;
  const int V = p.vocab;
  if (GRAD && nothing_to_do(p)) return;
  const T* x = reinterpret_cast<const T*>(p.logits) + p.lrow.at(row);
  const Split sp = split_row(x, V);
  const int per = (sp.full + cl - 1) >> p.log2_cluster, v0 = min(sp.full, rank * per), n = min(per, sp.full - v0);
  const uint4* v = reinterpret_cast<const uint4*>(x + sp.head) + v0;
  // this share's entries, its vectors' first
  const int first = sp.head + v0 * E, lo = rank == 0 ? 0 : first, hi = rank == cl - 1 ? V : first + n * E;
  const float c = p.c;
  if (cl > 1) cluster_arrive_relaxed();  // peers have started before anyone writes to their shared memory

  const float w = p.weights ? p.weights[row] : 1.f;
  const int64_t label = HARD ? p.labels[row] : -1;
  float xl = 0.f;
  const bool holder = warp == 0 && (GRAD || rank == 0);
  Entries<kEnt> en;
  int64_t given[kEnt];
  float logit[kEnt];
  if (warp == 0) {
#pragma unroll
    for (int e = 0; e < kEnt; ++e) {
      const int j = lane + 32 * e;
      given[e] = j < p.k ? p.ids[(int64_t)row * p.k + j] : -1;
      logit[e] = j < p.k ? p.teacher[(int64_t)row * p.k + j] : 0.f;
    }
  }
  auto gather = [&]() {  // once the first tile is on its way; before the gradient may overwrite the logits
    int found = 0;
#pragma unroll
    for (int e = 0; e < kEnt; ++e) found |= put_entry(en, e, given[e], logit[e], V);
    const int f = row_flags<HARD>(p, found, w, label);
    if (lane == 0) s.flags = f;
#pragma unroll
    for (int e = 0; e < kEnt; ++e) en.x[e] = en.id[e] >= 0 ? ld(x + en.id[e]) : 0.f;
    if (HARD && label >= 0 && label < V) xl = ld(x + label);
  };
  if constexpr (GRAD)
    for (int i = tid; i < S::kSeen / 4; i += TB) reinterpret_cast<uint4*>(s.seen)[i] = make_uint4(0u, 0u, 0u, 0u);

  float m = -INFINITY, ref = kLowRef, ref1 = kLowRef;  // the warp's maximum and references
  float2 s2 = f2s(0.f), t2 = f2s(0.f);
  auto raise = [&](float to) {  // the sums against a new maximum
    if (to > m) {
      m = to;
      const float r = ref_of(m, c);
      s2 = mul2(s2, f2s(ex2(ref - r)));
      ref = r;
      if (HARD) {
        const float r1 = ref_of(m, kLog2e);
        t2 = mul2(t2, f2s(ex2(ref1 - r1)));
        ref1 = r1;
      }
    }
  };
  const uint64_t policy = l2_policy(GRAD ? Keep::kYes : Keep::kNo);
  uint4 d[kNV];
  auto load = [&](int base, uint64_t pol) {
#pragma unroll
    for (int j = 0; j < kNV; ++j) d[j] = load_stream(v + base + tid + j * TB, pol);
  };
  auto sum = [&](int base, auto full) {
    VecMax<T> vm[kNV];
    const float mt = vecs_max<T, kNV>(d, vm, [&](int j) { return full.value || base + j * TB < n; });
    raise(warp_max(mt));
#pragma unroll
    for (int j = 0; j < kNV; ++j)
      if (full.value || base + j * TB < n) add_vec<T, HARD>(d[j], ref, ref1, c, s2, t2);
  };
  auto load_rest = [&](int base, uint64_t pol) {
#pragma unroll
    for (int j = 0; j < kNV; ++j) {
      const int i = base + j * TB + tid;
      d[j] = neg_inf_vec<T>();
      if (i < n) d[j] = load_stream(v + i, pol);
    }
  };
  // the ragged tile first, then the full ones down to tile 0, which stays in d
  const int tiles = n / kTile, rest = tiles * kTile;
  if (rest < n)
    load_rest(rest, policy);
  else if (tiles > 0)
    load(rest - kTile, policy);
  if (warp == 0) gather();
  if (rest < n) {
    sum(rest, Flag<false>());
    if (tiles > 0) load(rest - kTile, policy);
  }
  for (int t = tiles - 1; t >= 0; --t) {
    sum(t * kTile, Flag<true>());
    if (GRAD && t == 1) {
#pragma unroll
      for (int j = 0; j < kNV; ++j) cache[j * TB + tid] = d[j];
    }
    if (t > 0) load((t - 1) * kTile, policy);
  }
  int edge = -1;  // this lane's element of the row's edges
  float xe = -INFINITY;
  if (warp == NW - 1) {
    edge = edge_index(sp, lane, rank == 0, rank == cl - 1);
    if (edge >= 0) xe = ld(x + edge);
    raise(warp_max(xe));
    s2.x += ex2(fmaf(xe, c, -ref));
    if (HARD) t2.x += ex2(fmaf(xe, kLog2e, -ref1));
  }
  Part a{m, ref, warp_sum(s2.x + s2.y), ref1, HARD ? warp_sum(t2.x + t2.y) : 0.f};
  if (lane == 0) s.part[warp] = a;
  if (holder) teacher_softmax(p, en);
  __syncthreads();
  a = join<HARD>(lane < NW ? s.part[lane] : no_part());
  auto exchange = [&](Part(&parts)[kMaxCluster], const Part& none) {
    __syncwarp();
    if (tid < cl) *peer(&parts[rank], tid) = a;
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    a = join<HARD>(lane < cl ? parts[lane] : none);
  };
  if (cl > 1) {
    __syncwarp();
    cluster_wait();
    exchange(s.parts, no_part());
  }
  const bool plain = fabsf(a.m) * fmaxf(c, kLog2e) <= p.plain_most;
  if (!plain) {  // the same for all threads of the row
    const Part none{a.m, 0.f, 0.f, 0.f, 0.f};
    a = slow_part(x, lo, hi, tid, TB, a.m, c);
    a.s = warp_sum(a.s);
    a.s1 = warp_sum(a.s1);
    __syncthreads();
    if (lane == 0) s.part[warp] = a;
    __syncthreads();
    a = join<HARD>(lane < NW ? s.part[lane] : none);
    if (cl > 1) exchange(s.again, none);
    a.m = none.m;
  }
  const int flags = s.flags;
  float norm = p.scale;
  after_previous();
  if (GRAD && p.weight_sum) norm /= *p.weight_sum;
  const Row r = make_row<HARD>(p, a, plain, row, flags, w, norm);
  if (warp == 0 && rank == 0 && p.row_loss) {
    const float loss = row_loss<HARD>(p, r, flags, w, en, xl);
    if (lane == 0) p.row_loss[row] = loss;
  }
  if constexpr (GRAD) {
    T* g = reinterpret_cast<T*>(p.grad) + p.grow.at(row);
    T* gv = g + first;  // this share's vectors
    const uint64_t go = l2_policy(Keep::kNo);
    if (flags == 0) {
      for (int i = lo + tid; i < hi; i += TB) stg<T>(g + i, 0.f);
    } else if (!plain) {
      for (int i = lo + tid; i < hi; i += TB) stg<T>(g + i, r.dense<HARD>(ld(x + i)));
    } else {
      auto write = [&](int b, auto full, auto aligned) {
#pragma unroll
        for (int j = 0; j < kNV; ++j)
          if (full.value || b + j * TB < n) {
            const uint4 u = grad_vec<T, HARD>(d[j], r);
            if (full.value || b + j * TB + tid < n) {
              if (aligned.value)
                store_stream(reinterpret_cast<uint4*>(gv) + b + tid + j * TB, u, go);
              else
                store_elements(gv + (int64_t)(b + tid + j * TB) * E, u);
            }
          }
      };
      auto walk_again = [&](auto aligned) {
        if (tiles > 0) write(0, Flag<true>(), aligned);
        if (tiles > 1) {
#pragma unroll
          for (int j = 0; j < kNV; ++j) d[j] = cache[j * TB + tid];
          write(kTile, Flag<true>(), aligned);
        }
        for (int t = 2; t < tiles; ++t) {
          load(t * kTile, go);
          write(t * kTile, Flag<true>(), aligned);
        }
        if (rest < n) {
          if (tiles > 0) load_rest(rest, go);
          write(rest, Flag<false>(), aligned);
        }
      };
      if (row_shift(gv) == 0)
        walk_again(Flag<true>());
      else
        walk_again(Flag<false>());
      if (edge >= 0) stg<T>(g + edge, r.plain<HARD>(f2s(xe)).x);
    }
    __syncthreads();
    if (warp == 0 && flags && !(flags & kBad))
      store_entries<T, HARD>(p, g, lo, hi, r, flags, en, label, xl, hi - lo <= 32 * S::kSeen ? s.seen : nullptr, s.ids,
                             s.probs);
  }
}

// ---- one warp per row ---------------------------------------------------------------------
// A warp takes `batch` (at most 32) rows one after the other, the next one's vectors and entries on
// their way; lane i keeps row i's weight, label and loss.
constexpr int kWarpThreads = 256, kWarps = kWarpThreads / 32;

// The entries' logits come from a copy of a short row in shared memory, of a longer one from L2.
template <int NV>
constexpr bool kCopy = NV <= 8;

template <typename T, int NV, bool GRAD>
struct alignas(16) WarpSmem {
  uint4 row[kCopy<NV> ? NV * 32 : 1];
  int ids[GRAD ? M3_MAX_TOP : 1];
  float probs[GRAD ? M3_MAX_TOP : 1];
  uint32_t seen[GRAD ? NV * kVec<T> : 1];  // a bit per element
};

// CTAs that have to fit an SM, which bounds the registers.  Measured, without a bound against this one: 65536 x 4096
// bf16 with gradient 355 -> 272 us, 131072 x 2048 bf16 260 -> 241, with 64 entries for 1024 181 -> 165, with
// hard labels for 1024 212 -> 181; one CTA more for each spills and is slower (1024, 64 entries: 185).
template <int NV, int KE, bool HARD>
constexpr int kWarpCtas = NV == 1   ? 0  // the compiler's own choice
                          : NV == 2 ? 4
                          : NV == 4 ? (KE > 1 ? 3 : HARD ? 4 : 0)
                          : NV == 8 ? (KE > 1 ? 2 : 3)
                                    : 2;

// KE: 1 for up to 32 entries, which are most lists, else kEnt.
template <typename T, int NV, int KE, bool HARD, bool GRAD>
__global__ void __launch_bounds__(kWarpThreads, kWarpCtas<NV, KE, HARD>) distill_warp_kernel(const Params p, int batch) {
  constexpr int E = kVec<T>;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  WarpSmem<T, NV, GRAD>& s = reinterpret_cast<WarpSmem<T, NV, GRAD>*>(smem_raw)[threadIdx.x >> 5];
  const int lane = threadIdx.x & 31, V = p.vocab;
  const float c = p.c;
  const int row0 = (blockIdx.x * kWarps + (threadIdx.x >> 5)) * batch, rows = min(batch, p.rows - row0);
  if (rows <= 0 || (GRAD && nothing_to_do(p))) return;
  const float w_all = lane < rows && p.weights ? p.weights[row0 + lane] : 1.f;
  const int64_t label_all = HARD && lane < rows ? p.labels[row0 + lane] : -1;
  uint4 d[NV];
  int shift = 0;
  int64_t id[KE];
  float t[KE];
  auto load = [&](int row) {
    const T* x = reinterpret_cast<const T*>(p.logits) + p.lrow.at(row);
    shift = row_shift(x);
    const bool whole = shift == 0 && V % E == 0;  // no ragged vector
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int lo = (j * 32 + lane) * E - shift;
      d[j] = neg_inf_vec<T>();
      if (whole) {
        if (lo < V) d[j] = load_once(reinterpret_cast<const uint4*>(x + lo));
      } else if (lo < V) {
        d[j] = load_vec(x, lo, V);
      }
    }
#pragma unroll
    for (int e = 0; e < KE; ++e) {
      const int j = lane + 32 * e;
      id[e] = j < p.k ? p.ids[(int64_t)row * p.k + j] : -1;
      t[e] = j < p.k ? p.teacher[(int64_t)row * p.k + j] : 0.f;
    }
  };
  load(row0);
  after_previous();
  const float norm = GRAD && p.weight_sum ? p.scale / *p.weight_sum : p.scale;
  float loss_all = 0.f;
  for (int i = 0; i < rows; ++i) {
    const int row = row0 + i, at = shift;
    const float w = __shfl_sync(0xffffffffu, w_all, i);
    const int64_t label = HARD ? __shfl_sync(0xffffffffu, label_all, i) : -1;
    const T* xs = reinterpret_cast<const T*>(p.logits) + p.lrow.at(row);
    if constexpr (kCopy<NV>) {
#pragma unroll
      for (int j = 0; j < NV; ++j) s.row[j * 32 + lane] = d[j];
      xs = reinterpret_cast<const T*>(s.row) + at;
    }
    if (GRAD)
      for (int j = lane; j < NV * E; j += 32) s.seen[j] = 0u;
    Entries<KE> en;
    int found = 0;
    float xl = 0.f;
    auto gather = [&]() {
#pragma unroll
      for (int e = 0; e < KE; ++e) {
        found |= put_entry(en, e, id[e], t[e], V);
        en.x[e] = en.id[e] >= 0 ? ld(xs + en.id[e]) : 0.f;
      }
      if (HARD && label >= 0 && label < V) xl = ld(xs + label);
    };
    if constexpr (!kCopy<NV>) gather();  // on their way during the sums
    Part a = no_part();
    VecMax<T> vm[NV];
    a.m = warp_max(vecs_max<T, NV>(d, vm, [](int) { return true; }));
    a.r = ref_of(a.m, c);
    a.r1 = ref_of(a.m, kLog2e);
    float2 s2 = f2s(0.f), t2 = f2s(0.f);
#pragma unroll
    for (int j = 0; j < NV; ++j) add_vec<T, HARD>(d[j], a.r, a.r1, c, s2, t2);
    __syncwarp();
    if constexpr (kCopy<NV>) gather();
    const int flags = row_flags<HARD>(p, found, w, label);
    teacher_softmax(p, en);
    a.s = warp_sum(s2.x + s2.y);
    a.s1 = HARD ? warp_sum(t2.x + t2.y) : 1.f;
    const bool plain = fabsf(a.m) * fmaxf(c, kLog2e) <= p.plain_most;
    if (!plain) {
      a = slow_part(xs, 0, V, lane, 32, a.m, c);
      a.s = warp_sum(a.s);
      a.s1 = warp_sum(a.s1);
    }
    const Row r = make_row<HARD>(p, a, plain, row, flags, w, norm);
    const float loss = row_loss<HARD>(p, r, flags, w, en, xl);
    if (lane == i) loss_all = loss;
    if constexpr (GRAD) {
      T* g = reinterpret_cast<T*>(p.grad) + p.grow.at(row);
      if (flags == 0) {
        for (int e = lane; e < V; e += 32) stg<T>(g + e, 0.f);
      } else if (!plain) {
        for (int e = lane; e < V; e += 32) stg<T>(g + e, r.dense<HARD>(ld(xs + e)));
      } else {
        const bool aligned = row_shift(g) == at;
        const uint64_t go = l2_policy(Keep::kNo);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const int lo = (j * 32 + lane) * E - at;
          const uint4 u = grad_vec<T, HARD>(d[j], r);
          if (lo >= 0 && lo + E <= V) {
            if (aligned)
              store_stream(g + lo, u, go);
            else
              store_elements(g + lo, u);
          } else if (lo < V) {
            const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
            for (int q = 0; q < E; ++q)
              if (lo + q >= 0 && lo + q < V) g[lo + q] = e[q];
          }
        }
      }
      if (i + 1 < rows) load(row + 1);
      __syncwarp();
      if (flags && !(flags & kBad)) store_entries<T, HARD>(p, g, 0, V, r, flags, en, label, xl, s.seen, s.ids, s.probs);
    } else {
      if (i + 1 < rows) load(row + 1);
    }
    __syncwarp();  // the row's shared memory is free again
  }
  if (lane < rows && p.row_loss) p.row_loss[row0 + lane] = loss_all;
}

// out = scale * (sum of n values) / (*div_by, if given), by one cluster in a fixed order.
// v is not __restrict__: the kernel in front may still be writing it when this one starts, and a load through
// the read-only path, which __restrict__ allows, need not stay behind after_previous().
constexpr int kSumCtas = 8, kSumThreads = 1024;

__global__ void __launch_bounds__(kSumThreads)
    sum_kernel(const float* v, int64_t n, const float* div_by, float scale, float* out) {
  __shared__ float sm[32], total[kSumCtas];
  const int tid = threadIdx.x, rank = cluster_rank();
  next_may_start();
  cluster_arrive_relaxed();
  after_previous();
  float s = 0.f;
#pragma unroll 16
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
    const float by = div_by ? *div_by : 1.f;
    *out = s == 0.f && by == 0.f ? 0.f : s * scale / by;  // no row has a weight: 0, as the gradient
  }
}

int sm_count() {
  int dev = 0, c = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&c, cudaDevAttrMultiProcessorCount, dev);
  return c;
}

// Allows a kernel its shared memory, once per device (`done`: the kernel's own).
template <typename K>
int allow_smem(K kern, size_t bytes, bool (&done)[64]) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (bytes <= 48 * 1024 || (dev < 64 && done[dev])) return M3_OK;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != cudaSuccess)
    return check_launch("m3_distill: cudaFuncSetAttribute");
  if (dev < 64) done[dev] = true;
  return M3_OK;
}

template <typename T, int TB, bool HARD, bool GRAD>
int launch_cta(const Params& p, cudaStream_t s) {
  static bool done[64] = {};
  constexpr size_t kSmem = sizeof(Smem<TB, GRAD>) + (GRAD ? sizeof(uint4) * kNV * TB : 0);
  auto* kern = distill_kernel<T, TB, HARD, GRAD>;
  if (const int rc = allow_smem(kern, kSmem, done)) return rc;
  return launch_ex("m3_distill", kern, (unsigned)p.rows * p.cluster, TB, kSmem, p.cluster, p.early, s, p);
}

template <typename T, int NV, int KE, bool HARD, bool GRAD>
int launch_warp_k(const Params& p, cudaStream_t s) {
  static bool done[64] = {};
  const int batch = warp_batch(p.rows, sm_count());
  const int warps = (p.rows + batch - 1) / batch;
  constexpr size_t kSmem = kWarps * sizeof(WarpSmem<T, NV, GRAD>);
  auto* kern = distill_warp_kernel<T, NV, KE, HARD, GRAD>;
  if (const int rc = allow_smem(kern, kSmem, done)) return rc;
  return launch_ex("m3_distill", kern, (unsigned)((warps + kWarps - 1) / kWarps), kWarpThreads, kSmem, 1, p.early, s, p, batch);
}

template <typename T, int NV, bool HARD, bool GRAD>
int launch_warp(const Params& p, cudaStream_t s) {
  return p.k <= 32 ? launch_warp_k<T, NV, 1, HARD, GRAD>(p, s) : launch_warp_k<T, NV, kEnt, HARD, GRAD>(p, s);
}

// A row goes to a warp while its vectors fit the lanes' registers, else to a CTA, and with few rows to
// a cluster.
template <typename T, bool HARD, bool GRAD>
int launch(Params p, int nvec, cudaStream_t s) {
  if (nvec <= 32) return launch_warp<T, 1, HARD, GRAD>(p, s);
  if (nvec <= 64) return launch_warp<T, 2, HARD, GRAD>(p, s);
  if (nvec <= 128) return launch_warp<T, 4, HARD, GRAD>(p, s);
  if (nvec <= 256) return launch_warp<T, 8, HARD, GRAD>(p, s);
  if (nvec <= 512 && p.rows >= 16 * sm_count()) return launch_warp<T, 16, HARD, GRAD>(p, s);
  // few rows: several CTAs per row until they cover the SMs
  const int sms = sm_count();
  int cl = 1;
  while (cl < kMaxCluster && (int64_t)p.rows * cl * 2 <= sms && nvec / (cl * 2) >= 128) cl *= 2;
  p.cluster = cl;
  while ((1 << p.log2_cluster) < cl) ++p.log2_cluster;
  if ((int64_t)p.rows * cl > 0x7FFFFFFF) return set_error(M3_ERR_SHAPE, "m3_distill: too many rows");
  // the fewest threads for which two tiles are the row; longer rows are read again from L2, which holds
  // the rows in flight of two CTAs per SM better than of four
  if (nvec <= 2 * kNV * 128 * cl) return launch_cta<T, 128, HARD, GRAD>(p, s);
  if (nvec <= 2 * kNV * 256 * cl && (int64_t)p.rows * cl > 2 * sms) return launch_cta<T, 256, HARD, GRAD>(p, s);
  // rows too long for L2 even so, where one exponential an element leaves one CTA an SM time to spare: 394 us
  // instead of 443 at 2048 x 128256 f32 (with 512 threads 371 instead of 400 at 4000 x 64000)
  if constexpr (GRAD && !HARD && sizeof(T) == 4)
    if (nvec > 5 * kNV * 512 * cl) return launch_cta<T, 1024, HARD, GRAD>(p, s);
  return launch_cta<T, 512, HARD, GRAD>(p, s);
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
  if (!temperature_ok(a.temperature) || a.temperature > kMostTemperature || !(a.hard_weight >= 0.f && a.hard_weight <= 1.f))
    return set_error(M3_ERR_ARG, "m3_distill: need a temperature in [1e-30, 1e18] and 0 <= hard_weight <= 1");
  const int64_t rows = (int64_t)a.rows_outer * a.rows_inner;
  if (rows > kMaxRows) return set_error(M3_ERR_SHAPE, "m3_distill: more than 2^30 rows");
  const bool only_grad = a.grad && !a.row_loss && !a.loss;
  if ((rows > 0 && (!a.logits || !a.ids || !a.teacher || (!a.row_loss && !only_grad))) ||
      (a.hard_weight > 0.f && rows > 0 && !a.labels) || (a.reduction != M3_REDUCE_NONE && !a.loss && !only_grad))
    return set_error(M3_ERR_ARG, "m3_distill: NULL pointer");
  if ((a.ready & M3_READY_GRAD) && (!only_grad || !a.upstream || a.upstream_stride != 0))
    return set_error(M3_ERR_ARG, "m3_distill: a ready gradient needs one upstream value and no losses");
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
  p.c = kLog2e / a.temperature;
  p.plain_most = plain_most(p.c);
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
  p.ready = (a.ready & M3_READY_GRAD) != 0;
  const bool sum_weights = wmean && !(a.ready & M3_READY_WEIGHTS);
  p.early = sum_weights && !p.ready;  // with nothing to do it would end without waiting for the sum
  p.row_loss = a.row_loss;
  auto sum = [&](const float* v, const float* div_by, float scale, float* out, bool early) {
    return launch_ex("m3_distill", sum_kernel, kSumCtas, kSumThreads, 0, kSumCtas, early, s, v, (int64_t)rows, div_by, scale, out);
  };
  int rc = M3_OK;
  if (sum_weights) rc = sum(a.weights, nullptr, 1.f, a.weight_sum, false);
  if (rc == M3_OK && rows > 0) {
    const int nvec = most_vectors(a.logits, a.vocab, bf ? 2 : 4, a.ld_outer, a.ld_inner);
    rc = bf ? launch<__nv_bfloat16>(p, nvec, s) : launch<float>(p, nvec, s);
  }
  if (rc == M3_OK && a.loss && a.reduction != M3_REDUCE_NONE)  // the mean of no rows is 0 / 0
    rc = sum(a.row_loss, p.weight_sum, a.reduction == M3_REDUCE_MEAN && !a.weights ? 1.f / (float)rows : 1.f, a.loss,
             rows > 0);
  return rc;
}
