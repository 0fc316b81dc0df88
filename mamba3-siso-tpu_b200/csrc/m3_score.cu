// Log probabilities of given tokens, entropy and top alternatives of logits rows.
//   y = x / T, m = max y, Z = sum e^(y - m):  lse = m + ln Z,  entropy = ln Z - sum e d / Z, d = y - m
// One read of the logits, which is the floor: about 6 instructions an element (load, unpack, maximum,
// multiply-add, exponential, two sums) against 0.3 ns an element that memory gives an SM in bf16, so the
// loops have to stay lean.  Measured at 4096 x 128256 bf16: 157 us without alternatives (6.7 TB/s), 223 to 242
// with 32 (1.7 times the instructions); 4092 x 50257 f32: 124 us (6.5 TB/s); 131072 x 256 bf16 with 8: 57 us
// (1.4 TB/s), bound by about 400 instructions a row.
//
// Rows go to threads by their length (see launch): a warp that holds a short row in registers, a warp that
// walks a row of some thousand entries, or a CTA that walks a long one.  Each warp walks its share with a
// running maximum and sums against it; the (max, sum, sum e d) triples of a row's warps meet at one barrier.
// Earlier a row was held by a cluster of CTAs: at 4092 x 50257 that took 247 us instead of 126, in barriers.
//
// Alternatives: every warp keeps the r-th largest of its lanes' maxima so far, r = ceil(top / warps);
// the smallest of these over the warps has at least `top` elements at or above it, so every
// alternative is at or above it as well, and it only rises.  Vectors that reach it when they pass are
// put aside (on rows without order about 2 top ln(tiles) of them), their elements that reach the
// final bound are ranked, and the CTAs' sorted lists are merged.  Rows that defeat the bound (a mask that leaves
// so few ids that some warp's r-th maximum is -inf, many equal logits, rising rows, NaN) take an exact selection by
// bits, some fifty walks of the row.  Measured with 20 alternatives, against rows without a mask: one row of 128256
// by a cluster of eight CTAs 92 us instead of 31, 64 rows by clusters of two 334 instead of 29, 4096 rows by a CTA
// each 17.2 ms instead of 0.22, 16384 x 4096 by a warp each (10 ids left) 1.49 ms instead of 0.07.
#include "m3_internal.h"
#include "m3_vocab.cuh"

namespace m3 {
namespace {

using namespace vocab;

constexpr int kNV = 8;          // vectors a thread loads at a time
constexpr int kMaxCluster = 8;  // CTAs per row (portable size)
constexpr int kCandCap = 1024;  // a power of two

struct Params {
  int rows, vocab, top, cluster, log2_cluster;
  float inv_t, c, plain_most;
  Rows lrow, trow;
  const void* logits;
  const int64_t* targets;
  float *logprob, *entropy, *lse, *top_logprob;
  int64_t* top_ids;
};

// The maximum, and against the reference r: s = sum 2^d, u = sum 2^d d.
struct Part {
  float m, r, s, u;
};
__device__ __forceinline__ Part no_part() { return Part{-INFINITY, kLowRef, 0.f, 0.f}; }

template <typename T>
__device__ __forceinline__ void add_vec(const uint4& v, float r, float c, float2& s, float2& u) {
  float2 f[kVec<T> / 2];
  unpack<T>(clamp_low<T>(v), f);
#pragma unroll
  for (int j = 0; j < kVec<T> / 2; ++j) {
    const float2 d = fma2(f[j], f2s(c), f2s(-r));
    const float2 e = f2(ex2(d.x), ex2(d.y));
    s = add2(s, e);
    u = fma2(e, d, u);
  }
}

// Joins the parts held by the lanes of a warp.
__device__ __forceinline__ Part join(Part p) {
  Part r;
  r.m = warp_max(p.m);
  r.r = warp_max(p.r);
  const float d = p.r - r.r, e = ex2(d);  // 0 for a lane without a part
  r.s = warp_sum(p.s * e);
  r.u = warp_sum((p.u + p.s * d) * e);
  return r;
}

// The terms [lo, hi) of a row that is not plain, every `step`-th from lo + first, against its maximum.
template <typename T>
__device__ __noinline__ Part slow_part(const T* x, int lo, int hi, int first, int step, float m, float c) {
  float s = 0.f, u = 0.f;
  for (int i = lo + first; i < hi; i += step) {
    const float d = (ld(x + i) - m) * c, e = ex2(d);
    s += e;
    u = fmaf(e, fmaxf(d, -1e4f), u);  // e is 0 there: 0 * -inf would not be
  }
  return Part{m, 0.f, s, u};
}

__device__ __forceinline__ Log2P distribution(const Part& a, bool plain, float c) {
  return Log2P{plain, c, plain ? a.r : a.m, log2f(a.s)};
}
__device__ __forceinline__ void write_row(const Params& p, const Part& a, const Log2P& q, int row) {
  p.lse[row] = q.lse(p.inv_t);
  const float h = (q.l2 - a.u / a.s) * kLn2;
  p.entropy[row] = h < 0.f ? 0.f : h;  // below 0 by rounding; NaN stays
}
__device__ __forceinline__ void write_target(const Params& p, const Log2P& q, int row, int64_t t, float xt) {
  p.logprob[row] = t < 0 ? 0.f : t >= p.vocab ? NAN : q.ln(xt, p.inv_t);
}

// Everything a row has but its alternatives, by one thread.
template <typename T>
__device__ __forceinline__ void finish_row(const Params& p, const Part& a, int row) {
  const Log2P q = distribution(a, fabsf(a.m) * p.c <= p.plain_most, p.c);
  write_row(p, a, q, row);
  if (p.targets) {
    const int64_t t = p.targets[p.trow.at(row)];
    const T* x = reinterpret_cast<const T*>(p.logits) + p.lrow.at(row);
    write_target(p, q, row, t, t >= 0 && t < p.vocab ? ld(x + t) : 0.f);
  }
}

// ---- one CTA or one cluster per row -------------------------------------------------------
template <int NW, bool TOP>
struct Smem {
  Part part[NW];
  Part parts[kMaxCluster], again[kMaxCluster];
};
template <int NW>
constexpr int kVecCap = NW <= 4 ? 512 : 1024;  // vectors put aside
template <int NW>
struct Smem<NW, true> {
  Part part[NW];
  Part parts[kMaxCluster], again[kMaxCluster];
  float bound[NW];
  int n_vec, n_cand;
  int vec_at[kVecCap<NW>];
  uint4 vec[kVecCap<NW>];
  uint64_t cand[kCandCap];
  uint64_t list[kMaxCluster][M3_MAX_TOP];  // every CTA's alternatives, descending, 0 past the end
  int before[M3_MAX_TOP];                  // entries of the row above this CTA's i-th
  int count[NW];
};

// The threads that work on a share together.
template <int TB, typename S>
struct CtaGroup {
  S& s;
  static constexpr int kSize = TB;
  __device__ __forceinline__ int id() const { return threadIdx.x; }
  __device__ __forceinline__ void sync() const { __syncthreads(); }
  __device__ __forceinline__ int sum(int n) const {
    n = __reduce_add_sync(0xffffffffu, n);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.count[threadIdx.x >> 5] = n;
    __syncthreads();
    n = 0;
    for (int w = 0; w < TB / 32; ++w) n += s.count[w];
    return n;
  }
};
struct WarpGroup {
  static constexpr int kSize = 32;
  __device__ __forceinline__ int id() const { return threadIdx.x & 31; }
  __device__ __forceinline__ void sync() const { __syncwarp(); }
  __device__ __forceinline__ int sum(int n) const { return __reduce_add_sync(0xffffffffu, n); }
};

// The `need` first of the entries [lo, hi) in the order of rank_word into cand[0, need), unsorted, by
// selection on the bits of the key and then of the index.  All threads of the group; n_cand: shared.
template <typename T, typename G>
__device__ __noinline__ void exact_top(const T* x, int lo, int hi, int need, uint64_t* cand, int* n_cand, G g) {
  auto count = [&](auto pred) {
    int n = 0;
    for (int i = lo + g.id(); i < hi; i += G::kSize) n += pred(key_of(ld(x + i)), i) ? 1 : 0;
    return g.sum(n);
  };
  uint32_t key = 0;  // the need-th largest key
  for (int b = 31; b >= 0; --b) {
    const uint32_t t = key | (1u << b);
    if (count([&](uint32_t k, int) { return k >= t; }) >= need) key = t;
  }
  const int ties = need - count([&](uint32_t k, int) { return k > key; });
  int last = 0;  // the index of the last tie taken
  for (int b = 31 - __clz(hi); b >= 0; --b) {
    const int t = last | (1 << b);
    if (count([&](uint32_t k, int i) { return k == key && i < t; }) < ties) last = t;
  }
  if (g.id() == 0) *n_cand = 0;
  g.sync();
  for (int i = lo + g.id(); i < hi; i += G::kSize) {
    const float v = ld(x + i);
    const uint32_t k = key_of(v);
    if (k > key || (k == key && i <= last)) cand[atomicAdd(n_cand, 1)] = rank_word(v, i);
  }
  g.sync();
}

// Counting ranks n candidates in n^2 / TB steps, a bitonic network in n log^2 n / 4 TB.
constexpr int kCountMost = 192;

// cand[0, n), n <= kCandCap, into descending order (Batcher's bitonic network), 0 behind them.
template <int TB>
__device__ __noinline__ void sort_candidates(uint64_t* cand, int n) {
  int size = 1;
  while (size < n) size *= 2;
  for (int i = n + threadIdx.x; i < size; i += TB) cand[i] = 0;
  __syncthreads();
  for (int len = 2; len <= size; len *= 2)
    for (int gap = len / 2; gap > 0; gap /= 2) {
      for (int t = threadIdx.x; t < size / 2; t += TB) {
        const int i = 2 * t - (t & (gap - 1)), j = i + gap;
        const uint64_t a = cand[i], b = cand[j];
        if ((a < b) == ((i & len) == 0)) {
          cand[i] = b;
          cand[j] = a;
        }
      }
      __syncthreads();
    }
}

template <typename T, int TB, bool TOP>
__global__ void __launch_bounds__(TB, 1024 / TB) score_kernel(const Params p) {
  constexpr int E = kVec<T>, NW = TB / 32;
  __shared__ Smem<NW, TOP> s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cl = p.cluster, rank = cl > 1 ? cluster_rank() : 0;
  const int row = (int)blockIdx.x >> p.log2_cluster;
  const int V = p.vocab;
  const T* x = reinterpret_cast<const T*>(p.logits) + p.lrow.at(row);
  const Split sp = split_row(x, V);
  const int per = (sp.full + cl - 1) >> p.log2_cluster, v0 = min(sp.full, rank * per), n = min(per, sp.full - v0);
  const uint4* v = reinterpret_cast<const uint4*>(x + sp.head) + v0;
  const float c = p.c;
  if (cl > 1) cluster_arrive_relaxed();  // peers have started before anyone writes to their shared memory

  int64_t t = -1;
  float xt = 0.f;
  if (p.targets && rank == 0 && tid == 0) {
    t = p.targets[p.trow.at(row)];
    if (t >= 0 && t < V) xt = ld(x + t);
  }
  float m = -INFINITY, ref = kLowRef, mine = -INFINITY;  // the warp's maximum and reference, this lane's maximum
  float2 s2 = f2s(0.f), u2 = f2s(0.f);
  auto raise = [&](float to) {  // the sums against a new maximum
    if (to > m) {
      m = to;
      const float r = ref_of(m, c);
      if (r > ref) {
        const float dr = ref - r, e = ex2(dr);
        u2 = mul2(fma2(s2, f2s(dr), u2), f2s(e));
        s2 = mul2(s2, f2s(e));
        ref = r;
      }
    }
  };
  // warps all of whose lanes see a vector, and how many lane maxima each of them gives
  const int wide = min(NW, n >> 5), r = wide ? (p.top + wide - 1) / wide : 33;
  float bound = -INFINITY, own = -INFINITY;  // of the row, of this warp
  if constexpr (TOP) {
    if (lane == 0) s.bound[warp] = r <= 32 && warp >= wide ? INFINITY : -INFINITY;
    if (tid == 0) s.n_vec = s.n_cand = 0;
    __syncthreads();
  }
  auto raise_bound = [&]() {  // after a change of a lane's maximum
    if constexpr (TOP) {
      if (r > 32 || warp >= wide) return;
      float left = mine;
      for (int i = 0; i < r; ++i) {
        own = warp_max(left);
        const unsigned at = __ballot_sync(0xffffffffu, left == own);
        if (lane == __ffs(at) - 1) left = -INFINITY;
      }
      if (lane == 0) *(volatile float*)&s.bound[warp] = own;
    }
  };
  walk<T, kNV, TB>(v, n, tid, Keep::kNo, [&](const uint4(&d)[kNV], int base, auto full) {
    VecMax<T> vm[kNV];
    const float mt = vecs_max<T, kNV>(d, vm, [&](int j) { return full.value || base + j * TB < n; });
    raise(warp_max(mt));
#pragma unroll
    for (int j = 0; j < kNV; ++j)
      if (full.value || base + j * TB < n) add_vec<T>(d[j], ref, c, s2, u2);
    if constexpr (TOP) {
      const bool higher = mt > mine && mt > own;  // below `own` nothing changes the r-th largest
      mine = fmaxf(mine, mt);
      if (__any_sync(0xffffffffu, higher)) raise_bound();
      if (base == 0) __syncthreads();  // a first bound from every warp; later ones may be read late
      __syncwarp();
      bound = -warp_max(lane < NW ? -*(volatile float*)&s.bound[lane] : -INFINITY);
      if (mt >= bound) {
#pragma unroll
        for (int j = 0; j < kNV; ++j) {
          const int q = base + j * TB + tid;
          if ((full.value || q < n) && vm[j].reaches(bound)) {
            const int at = atomicAdd(&s.n_vec, 1);
            if (at < kVecCap<NW>) {
              s.vec[at] = d[j];
              s.vec_at[at] = q;
            }
          }
        }
      }
      __syncwarp();
    }
  });
  if (warp == NW - 1) {  // the row's edges
    const int i = edge_index(sp, lane, rank == 0, rank == cl - 1);
    const float xe = i >= 0 ? ld(x + i) : -INFINITY;
    raise(warp_max(xe));
    const float d = fmaf(xe > -1e30f || xe != xe ? xe : -1e30f, c, -ref), e = ex2(d);
    s2.x += e;
    u2.x = fmaf(e, d, u2.x);
    if constexpr (TOP)
      if (i >= 0) s.cand[atomicAdd(&s.n_cand, 1)] = rank_word(xe, i);
  }
  Part a{m, ref, warp_sum(s2.x + s2.y), warp_sum(u2.x + u2.y)};
  if (lane == 0) s.part[warp] = a;
  __syncthreads();
  a = join(lane < NW ? s.part[lane] : no_part());
  // this share's entries, its vectors' first
  const int first = sp.head + v0 * E, lo = rank == 0 ? 0 : first, hi = rank == cl - 1 ? V : first + n * E;

  if constexpr (TOP) {
    const int k = p.top;
    bound = -warp_max(lane < NW ? -s.bound[lane] : -INFINITY);
    const int nv = s.n_vec;
    if (nv <= kVecCap<NW>)
      for (int i0 = warp * 32; i0 < nv * E; i0 += TB) {
        const int i = i0 + lane;
        const float xv = i < nv * E ? ld(reinterpret_cast<const T*>(s.vec) + i) : -INFINITY;
        const unsigned who = __ballot_sync(0xffffffffu, i < nv * E && xv >= bound);
        int at = 0;
        if (lane == 0 && who) at = atomicAdd(&s.n_cand, __popc(who));
        at = __shfl_sync(0xffffffffu, at, 0) + __popc(who & ((1u << lane) - 1u));
        if ((who >> lane & 1u) && at < kCandCap) s.cand[at] = rank_word(xv, first + s.vec_at[i / E] * E + i % E);
      }
    __syncthreads();
    // the sum is NaN iff the share holds NaN or +inf, which the comparisons above do not order
    if (nv > kVecCap<NW> || s.n_cand > kCandCap || a.s != a.s) {
      exact_top(x, lo, hi, min(k, hi - lo), s.cand, &s.n_cand, CtaGroup<TB, Smem<NW, TOP>>{s});
    }
    const int nc = s.n_cand;
    uint64_t* list = s.list[rank];
    if (nc <= kCountMost) {
      for (int i = tid; i < nc; i += TB) {
        const uint64_t w = s.cand[i];
        int above = 0;
        for (int j = 0; j < nc; ++j) above += s.cand[j] > w ? 1 : 0;
        if (above < k) list[above] = w;
      }
      for (int i = nc + tid; i < k; i += TB) list[i] = 0;
    } else {
      sort_candidates<TB>(s.cand, nc);
      for (int i = tid; i < k; i += TB) list[i] = s.cand[i];
    }
    for (int i = tid; i < k; i += TB) s.before[i] = i;
    __syncthreads();
  }

  if (cl > 1) {
    __syncwarp();
    cluster_wait();
    if (tid < cl) *peer(&s.parts[rank], tid) = a;
    if constexpr (TOP)
      for (int i = tid; i < p.top * cl; i += TB) {
        const int r = i / p.top, j = i - r * p.top;
        if (r != rank) *peer(&s.list[rank][j], r) = s.list[rank][j];
      }
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    a = join(lane < cl ? s.parts[lane] : no_part());
  }
  const bool plain = fabsf(a.m) * c <= p.plain_most;
  if (!plain) {  // the same for all threads of the row
    a = slow_part(x, lo, hi, tid, TB, a.m, c);
    a.s = warp_sum(a.s);
    a.u = warp_sum(a.u);
    __syncthreads();
    if (lane == 0) s.part[warp] = a;
    __syncthreads();
    const float m_all = a.m;
    a = join(lane < NW ? s.part[lane] : Part{m_all, 0.f, 0.f, 0.f});
    if (cl > 1) {
      if (tid < cl) *peer(&s.again[rank], tid) = a;
      __syncwarp();
      cluster_arrive();
      cluster_wait();
      a = join(lane < cl ? s.again[lane] : Part{m_all, 0.f, 0.f, 0.f});
    }
    a.m = m_all;
  }
  const Log2P w = distribution(a, plain, c);
  if (rank == 0 && tid == 0) {
    write_row(p, a, w, row);
    if (p.targets) write_target(p, w, row, t, xt);
  }

  if constexpr (TOP) {
    const int k = p.top;
    if (cl > 1) {  // entries of the other lists above each of this one's
      for (int i = tid; i < k * cl; i += TB) {
        const int r = i / k, j = i - r * k;
        const uint64_t e = s.list[rank][j];
        if (r == rank || e == 0) continue;
        int lo = 0, hi = k;
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          if (s.list[r][mid] > e)
            lo = mid + 1;
          else
            hi = mid;
        }
        atomicAdd(&s.before[j], lo);
      }
      __syncthreads();
    }
    for (int i = tid; i < k; i += TB) {
      const uint64_t e = s.list[rank][i];
      const int at = s.before[i];
      if (e != 0 && at < k) {
        p.top_ids[(int64_t)row * k + at] = rank_index(e);
        p.top_logprob[(int64_t)row * k + at] = w.ln(key_value((uint32_t)(e >> 32)), p.inv_t);
      }
    }
  }
}

// ---- one warp per row ---------------------------------------------------------------------
// The (logit, lower index) order as one word; 0 is below every entry.  bf16: the 16-bit key and the
// complement of the index, for rows of at most 512 entries.
template <typename T>
struct Word;
template <>
struct Word<__nv_bfloat16> {
  using type = uint32_t;
  static __device__ __forceinline__ void make(const uint4& v, int i0, type* w) {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t k;  // + 0: -0 becomes 0, every NaN 0x7FFF; then the order of the bits, both halves at once
      asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(k) : "r"(u[j]), "r"(0u));
      k ^= ((k >> 15) & 0x00010001u) * 0x7FFFu ^ 0x80008000u;
      w[2 * j] = k * 65536u + (uint32_t)(0xFFFF - i0 - 2 * j);
      w[2 * j + 1] = (k & 0xFFFF0000u) + (uint32_t)(0xFFFF - i0 - 2 * j - 1);
    }
  }
  static __device__ __forceinline__ float value(type w) {
    const uint32_t b = w & 0xFFFF0000u;
    return __uint_as_float(w & 0x80000000u ? b & 0x7FFF0000u : ~b & 0xFFFF0000u);
  }
  static __device__ __forceinline__ int index(type w) { return 0xFFFF - (int)(w & 0xFFFFu); }
  static __device__ __forceinline__ type max(type w) { return __reduce_max_sync(0xffffffffu, w); }
};
template <>
struct Word<float> {
  using type = uint64_t;
  static __device__ __forceinline__ void make(const uint4& v, int i0, type* w) {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = rank_word(__uint_as_float(u[j]), i0 + j);
  }
  static __device__ __forceinline__ float value(type w) { return key_value((uint32_t)(w >> 32)); }
  static __device__ __forceinline__ int index(type w) { return rank_index(w); }
  static __device__ __forceinline__ type max(type w) {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(w >> 32));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(w >> 32) == hi ? (uint32_t)w : 0u);
    return ((uint64_t)hi << 32) | lo;
  }
};

// Descending, by Batcher's odd-even merge exchange (Knuth, TAOCP vol. 3, 5.2.2, algorithm M).
template <int N, typename W>
__device__ __forceinline__ void sort_desc(W (&w)[N]) {
#pragma unroll
  for (int p = 1; p < N; p *= 2)
#pragma unroll
    for (int k = p; k >= 1; k /= 2)
#pragma unroll
      for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
        for (int i = 0; i < k; ++i)
          if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
            const W a = w[i + j], b = w[i + j + k];
            w[i + j] = a > b ? a : b;
            w[i + j + k] = a > b ? b : a;
          }
}

// A warp takes `batch` (at most 32) rows one after the other, the next one's vectors on their way, and
// keeps row i's sums in lane i, so that what is done once per row is done for all of them at once.
constexpr int kWarpThreads = 256, kWarps = kWarpThreads / 32;

template <typename T, int NV, bool TOP>
__global__ void __launch_bounds__(kWarpThreads) score_warp_kernel(const Params p, int batch) {
  constexpr int E = kVec<T>, N = NV * E;
  const int lane = threadIdx.x & 31, V = p.vocab;
  const float c = p.c;
  const int row0 = (blockIdx.x * kWarps + (threadIdx.x >> 5)) * batch, rows = min(batch, p.rows - row0);
  if (rows <= 0) return;
  uint4 d[NV];
  int shift = 0;
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
  };
  load(row0);
  Part keep = no_part();
  for (int i = 0; i < rows; ++i) {
    const int at = shift;
    Part a = no_part();
    VecMax<T> vm[NV];
    a.m = warp_max(vecs_max<T, NV>(d, vm, [](int) { return true; }));
    a.r = ref_of(a.m, c);
    float2 s2 = f2s(0.f), u2 = f2s(0.f);
#pragma unroll
    for (int j = 0; j < NV; ++j) add_vec<T>(d[j], a.r, c, s2, u2);
    typename Word<T>::type wd[TOP ? N : 1];
    if constexpr (TOP) {
#pragma unroll
      for (int j = 0; j < NV; ++j) Word<T>::make(d[j], (j * 32 + lane) * E - at, wd + j * E);
      // entries before the row's start rank nowhere; those past its end lose to all of its own
      if (at > 0) {
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (lane == 0 && j < at) wd[j] = 0;
      }
    }
    if (i + 1 < rows) load(row0 + i + 1);
    a.s = warp_sum(s2.x + s2.y);
    a.u = warp_sum(u2.x + u2.y);
    const bool plain = fabsf(a.m) * c <= p.plain_most;
    if (!plain) {
      a = slow_part(reinterpret_cast<const T*>(p.logits) + p.lrow.at(row0 + i), 0, V, lane, 32, a.m, c);
      a.s = warp_sum(a.s);
      a.u = warp_sum(a.u);
    }
    if (lane == i) keep = a;
    if constexpr (TOP) {
      const Log2P q = distribution(a, plain, c);
      const int64_t out = (int64_t)(row0 + i) * p.top;
      sort_desc(wd);
      typename Word<T>::type mine = 0;
      auto take = [&](int left) {  // the largest word leaves its lane's list, of which `left` words still matter
        const auto best = Word<T>::max(wd[0]);
        if (wd[0] == best) {
#pragma unroll
          for (int e = 0; e + 1 < N; ++e)
            if (e < left) wd[e] = wd[e + 1];
          wd[N - 1] = 0;
        }
        return best;
      };
      auto put = [&](int k0, int n) {
        if (lane < n) {
          p.top_ids[out + k0 + lane] = Word<T>::index(mine);
          p.top_logprob[out + k0 + lane] = q.ln(Word<T>::value(mine), p.inv_t);
        }
      };
      if (p.top <= 8) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j < p.top) {
            const auto best = take(7 - j);
            if (lane == j) mine = best;
          }
        put(0, p.top);
      } else {
        for (int k0 = 0; k0 < p.top; k0 += 32) {
          const int n = min(32, p.top - k0);
          for (int j = 0; j < n; ++j) {
            const auto best = take(N);
            if (lane == j) mine = best;
          }
          put(k0, n);
        }
      }
    }
  }
  if (lane < rows) finish_row<T>(p, keep, row0 + lane);
}

// ---- one warp per longer row --------------------------------------------------------------
// The CTA's walk by a single warp, without barriers: rows of up to some thousand entries are over too
// soon for a CTA's.  BEST: 0 without alternatives; else the bound is the top-th largest of every lane's BEST
// largest vector maxima (1 for up to 8 alternatives; 2 for up to 32, where the lanes' maxima alone would
// let a hundred candidates through and overflow the lists).
// NV: vectors a lane loads at a time, no more than the row has, and registers bounded so that 3 to 5 CTAs are
// resident; the selection hides its latency behind other warps, and a few spilled registers cost it less than
// a CTA.  Measured, with tiles of 8 without a bound against these: 262144 x 1024 bf16 without alternatives
// 141 -> 112 us, with 8 413 -> 258; 131072 x 2048 f32 with 8 302 -> 237; 38400 x 256 f32 with 1 46 -> 28.
// Tiles of 4 for the longer rows too: with 8 alternatives 237 -> 266 us, as their bound rises more often.
constexpr int kRowVecCap = 96, kRowCandCap = 128, kRowMostTop = 32;

struct RowSmem {
  uint4 vec[kRowVecCap];
  int vec_at[kRowVecCap];
  uint64_t cand[kRowCandCap];
  int n_cand;
};

template <typename T, int NV, int BEST>
__global__ void __launch_bounds__(kWarpThreads, NV == 2 ? 5 : NV == 4 || BEST ? 4 : 3) score_rows_kernel(
    const Params p, int batch) {
  constexpr int E = kVec<T>;
  constexpr bool TOP = BEST > 0;
  __shared__ RowSmem smem[TOP ? kWarps : 1];
  RowSmem& s = smem[TOP ? threadIdx.x >> 5 : 0];
  const int lane = threadIdx.x & 31, V = p.vocab, k = p.top;
  const unsigned lt = (1u << lane) - 1u;
  const float c = p.c;
  const int row0 = (blockIdx.x * kWarps + (threadIdx.x >> 5)) * batch, rows = min(batch, p.rows - row0);
  if (rows <= 0) return;
  Part keep = no_part();
  for (int i = 0; i < rows; ++i) {
    const T* x = reinterpret_cast<const T*>(p.logits) + p.lrow.at(row0 + i);
    const Split sp = split_row(x, V);
    const uint4* v = reinterpret_cast<const uint4*>(x + sp.head);
    const int n = sp.full;
    float m = -INFINITY, ref = kLowRef, best[2] = {-INFINITY, -INFINITY}, bound = -INFINITY;
    float2 s2 = f2s(0.f), u2 = f2s(0.f);
    int nv = 0, nc = 0;  // vectors and candidates put aside
    auto raise = [&](float to) {
      if (to > m) {
        m = to;
        const float r = ref_of(m, c), dr = ref - r, e = ex2(dr);
        u2 = mul2(fma2(s2, f2s(dr), u2), f2s(e));
        s2 = mul2(s2, f2s(e));
        ref = r;
      }
    };
    walk<T, NV, 32>(v, n, lane, Keep::kNo, [&](const uint4(&d)[NV], int base, auto full) {
      VecMax<T> vm[NV];
      const float mt = vecs_max<T, NV>(d, vm, [&](int j) { return full.value || base + j * 32 < n; });
      raise(warp_max(mt));
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (full.value || base + j * 32 < n) add_vec<T>(d[j], ref, c, s2, u2);
      if constexpr (TOP) {
        bool higher;  // a change of the top-th largest
        if (BEST == 1) {
          higher = mt > best[0] && mt > bound;
          best[0] = fmaxf(best[0], mt);
        } else {
          const float before = best[1];
#pragma unroll
          for (int j = 0; j < NV; ++j)
            if (full.value || base + j * 32 < n) {
              const float f = vm[j].value();
              best[1] = fmaxf(best[1], fminf(best[0], f));
              best[0] = fmaxf(best[0], f);
            }
          higher = mt > before && mt > bound;
        }
        if (__any_sync(0xffffffffu, higher)) {
          float left = best[0], next = BEST > 1 ? best[1] : -INFINITY;
          for (int q = 0; q < k; ++q) {
            bound = warp_max(left);
            const unsigned at = __ballot_sync(0xffffffffu, left == bound);
            if (lane == __ffs(at) - 1) {
              left = next;
              next = -INFINITY;
            }
          }
        }
        if (__any_sync(0xffffffffu, mt >= bound)) {
#pragma unroll
          for (int j = 0; j < NV; ++j) {
            if (!full.value && base + j * 32 >= n) break;
            const bool put = (full.value || base + j * 32 + lane < n) && vm[j].reaches(bound);
            const unsigned who = __ballot_sync(0xffffffffu, put);
            const int at = nv + __popc(who & lt);
            if (put && at < kRowVecCap) {
              s.vec[at] = d[j];
              s.vec_at[at] = base + j * 32 + lane;
            }
            nv += __popc(who);
          }
        }
      }
    });
    {
      const int q = edge_index(sp, lane, true, true);
      const float xe = q >= 0 ? ld(x + q) : -INFINITY;
      raise(warp_max(xe));
      const float d = fmaf(xe > -1e30f || xe != xe ? xe : -1e30f, c, -ref), e = ex2(d);
      s2.x += e;
      u2.x = fmaf(e, d, u2.x);
      if constexpr (TOP) {
        const unsigned who = __ballot_sync(0xffffffffu, q >= 0);
        if (q >= 0) s.cand[__popc(who & lt)] = rank_word(xe, q);
        nc = __popc(who);
      }
    }
    Part a{m, ref, warp_sum(s2.x + s2.y), warp_sum(u2.x + u2.y)};
    const bool odd = a.s != a.s, plain = fabsf(a.m) * c <= p.plain_most;
    if (!plain) {
      a = slow_part(x, 0, V, lane, 32, a.m, c);
      a.s = warp_sum(a.s);
      a.u = warp_sum(a.u);
    }
    if (lane == i) keep = a;
    if constexpr (TOP) {
      __syncwarp();
      if (nv <= kRowVecCap)
        for (int j0 = 0; j0 < nv * E; j0 += 32) {
          const int j = j0 + lane;
          const float xv = j < nv * E ? ld(reinterpret_cast<const T*>(s.vec) + j) : -INFINITY;
          const bool put = j < nv * E && xv >= bound;
          const unsigned who = __ballot_sync(0xffffffffu, put);
          const int at = nc + __popc(who & lt);
          if (put && at < kRowCandCap) s.cand[at] = rank_word(xv, sp.head + s.vec_at[j / E] * E + j % E);
          nc += __popc(who);
        }
      __syncwarp();
      if (nv > kRowVecCap || nc > kRowCandCap || odd) {
        exact_top(x, 0, V, k, s.cand, &s.n_cand, WarpGroup{});
        nc = k;
      }
      const Log2P q = distribution(a, plain, c);
      const int64_t out = (int64_t)(row0 + i) * k;
      for (int j = lane; j < nc; j += 32) {
        const uint64_t w = s.cand[j];
        int above = 0;
        for (int o = 0; o < nc; ++o) above += s.cand[o] > w ? 1 : 0;
        if (above < k) {
          p.top_ids[out + above] = rank_index(w);
          p.top_logprob[out + above] = q.ln(key_value((uint32_t)(w >> 32)), p.inv_t);
        }
      }
      __syncwarp();  // the lists are free again
    }
  }
  if (lane < rows) finish_row<T>(p, keep, row0 + lane);
}

int sm_count() {
  int dev = 0, c = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&c, cudaDevAttrMultiProcessorCount, dev);
  return c;
}

template <typename T, int TB, bool TOP>
int launch_cta(const Params& p, cudaStream_t s) {
  return launch_ex("m3_token_logprobs", score_kernel<T, TB, TOP>, (unsigned)p.rows * p.cluster, TB, 0, p.cluster, false, s,
                   p);
}

template <typename T, int NV, bool TOP>
int launch_warp(const Params& p, cudaStream_t s) {
  const int batch = warp_batch(p.rows, sm_count());
  const int warps = (p.rows + batch - 1) / batch;
  score_warp_kernel<T, NV, TOP><<<(unsigned)((warps + kWarps - 1) / kWarps), kWarpThreads, 0, s>>>(p, batch);
  return check_launch("m3_token_logprobs");
}

template <typename T, int NV, int BEST>
int launch_rows_n(const Params& p, cudaStream_t s) {
  const int batch = warp_batch(p.rows, sm_count());
  const int warps = (p.rows + batch - 1) / batch;
  score_rows_kernel<T, NV, BEST><<<(unsigned)((warps + kWarps - 1) / kWarps), kWarpThreads, 0, s>>>(p, batch);
  return check_launch("m3_token_logprobs");
}

// Tiles no larger than the row: fewer registers, more warps.
template <typename T, int BEST>
int launch_rows(const Params& p, int nvec, cudaStream_t s) {
  if (nvec <= 64) return launch_rows_n<T, 2, BEST>(p, s);
  if (nvec <= 128) return launch_rows_n<T, 4, BEST>(p, s);
  return launch_rows_n<T, 8, BEST>(p, s);
}

// A row goes to a warp while its vectors fit the lanes' registers (one each; with many alternatives two, which
// a lane can keep sorted), or while there are warps' worth of rows and it is a few tiles; else to a CTA, and
// with few rows to a cluster.
template <typename T, bool TOP>
int launch(Params p, int nvec, cudaStream_t s) {
  if (nvec <= 32) return launch_warp<T, 1, TOP>(p, s);
  const bool few = !TOP || p.top <= kRowMostTop;
  if (few && (nvec <= 32 * kNV || (nvec <= 4 * 32 * kNV && p.rows >= 16 * sm_count()))) {
    if constexpr (!TOP) return launch_rows<T, 0>(p, nvec, s);
    return p.top <= 8 ? launch_rows<T, 1>(p, nvec, s) : launch_rows<T, 2>(p, nvec, s);
  }
  if constexpr (TOP)
    if (nvec <= 64) return launch_warp<T, 2, TOP>(p, s);
  // few rows: several CTAs per row until they cover the SMs
  const int sms = sm_count();
  int cl = 1;
  while (cl < kMaxCluster && (int64_t)p.rows * cl * 2 <= sms && nvec / (cl * 2) >= 128) cl *= 2;
  p.cluster = cl;
  while ((1 << p.log2_cluster) < cl) ++p.log2_cluster;
  if ((int64_t)p.rows * cl > 0x7FFFFFFF) return set_error(M3_ERR_SHAPE, "m3_token_logprobs: too many rows");
  if (nvec <= kNV * 128 * cl) return launch_cta<T, 128, TOP>(p, s);
  return (int64_t)p.rows * cl <= 2 * sms ? launch_cta<T, 512, TOP>(p, s) : launch_cta<T, 256, TOP>(p, s);
}

}  // namespace
}  // namespace m3

using namespace m3;

extern "C" int m3_token_logprobs(const M3ScoreArgs* args, void* stream) {
  if (!args) return set_error(M3_ERR_ARG, "m3_token_logprobs: args is NULL");
  const M3ScoreArgs& a = *args;
  if (a.rows_outer < 0 || a.rows_inner < 0 || a.vocab <= 0 || a.vocab > kMaxVocab || a.top < 0 ||
      a.top > M3_MAX_TOP || a.top > a.vocab)
    return set_error(M3_ERR_SHAPE, "m3_token_logprobs: need rows >= 0, 0 < vocab <= 2^30 and 0 <= top <= min(vocab, 128)");
  if (a.logits_dtype != M3_DTYPE_F32 && a.logits_dtype != M3_DTYPE_BF16)
    return set_error(M3_ERR_UNSUPPORTED, "m3_token_logprobs: logits must be f32 or bf16");
  if (!temperature_ok(a.temperature))
    return set_error(M3_ERR_ARG, "m3_token_logprobs: temperature must be > 0, finite and not so small that 1 / T overflows");
  const int64_t rows = (int64_t)a.rows_outer * a.rows_inner;
  if (rows > kMaxRows) return set_error(M3_ERR_SHAPE, "m3_token_logprobs: more than 2^30 rows");
  if (rows == 0) return M3_OK;
  if (!a.logits || !a.entropy || !a.lse || (a.targets && !a.logprob) || (a.top > 0 && (!a.top_logprob || !a.top_ids)))
    return set_error(M3_ERR_ARG, "m3_token_logprobs: NULL pointer");
  const bool bf = a.logits_dtype == M3_DTYPE_BF16;
  if (((uintptr_t)a.logits) % (bf ? 2 : 4)) return set_error(M3_ERR_ARG, "m3_token_logprobs: logits are not aligned to their type");
  Params p;
  p.rows = (int)rows;
  p.vocab = a.vocab;
  p.top = a.top;
  p.cluster = 1;
  p.log2_cluster = 0;
  p.inv_t = 1.f / a.temperature;
  p.c = kLog2e / a.temperature;
  p.plain_most = plain_most(p.c);
  p.lrow = Rows{a.rows_outer, a.rows_inner, a.ld_outer, a.ld_inner};
  p.trow = Rows{a.rows_outer, a.rows_inner, a.t_outer, a.t_inner};
  p.logits = a.logits;
  p.targets = a.targets;
  p.logprob = a.logprob;
  p.entropy = a.entropy;
  p.lse = a.lse;
  p.top_logprob = a.top_logprob;
  p.top_ids = a.top_ids;
  cudaStream_t s = (cudaStream_t)stream;
  const int nvec = most_vectors(a.logits, a.vocab, bf ? 2 : 4, a.ld_outer, a.ld_inner);
  if (bf) return a.top ? launch<__nv_bfloat16, true>(p, nvec, s) : launch<__nv_bfloat16, false>(p, nvec, s);
  return a.top ? launch<float, true>(p, nvec, s) : launch<float, false>(p, nvec, s);
}
