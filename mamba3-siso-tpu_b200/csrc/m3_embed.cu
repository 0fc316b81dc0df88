// Embedding lookup with scaling, and the table's gradient by sorted tokens.
//   out[r] = scale * table[token r]              grad[v] = scale * sum of dy[r] over token r == v
// The gradient's rows are summed in the order of r (fp32), so that it is the same every call:
// (token, r) pairs are put in order by a stable radix sort (one cluster of up to 16 CTAs), the sorted list is cut
// into chunks of equal length, each summed by one group of threads, and the pieces of tokens longer
// than that are joined.  The cuts depend on the sizes alone, so the result is the same every call.
// Floor: the rows once in, the gradient once out.  Measured, lookup and gradient together: 16384 positions
// over 128256 x 2048 fp32 232 us (5.7 TB/s: the clear runs beside the sort at the rate of writes), 131072
// positions over 256 x 512 94 us (2.9 TB/s: lookup 29, sort 17, chunk sums 30, join 15 by themselves; the
// gradient's launches overlap, without that 98).
#include <cooperative_groups.h>

#include "m3_internal.h"
#include "m3_vocab.cuh"

namespace m3 {
namespace {

using namespace vocab;

constexpr int kThreads = 256;
constexpr int64_t kMaxLd = 1 << 30;  // elements between rows of a table

// The threads of a CTA as groups over a row's columns, N columns a thread: at most kThreads threads a
// group, wider rows take several CTAs (blockIdx.y).
struct Columns {
  int width, groups;  // threads per group, groups per CTA
  __device__ __forceinline__ int group() const { return (int)threadIdx.x / width; }
  __device__ __forceinline__ int first(int n) const {
    return ((int)threadIdx.x - group() * width + (int)blockIdx.y * width) * n;
  }
};

// ---- lookup -------------------------------------------------------------------------------
struct FwdParams {
  int rows, vocab, dim, table_ld, out_ld;  // 32-bit strides: one multiplication per address
  float scale;
  Rows trow;
  const int64_t* tokens;
  const void* table;
  void* out;
  Columns cols;
};

// N consecutive elements, as loaded (so that many loads can be under way before the first is looked
// at) and as floats; the address is aligned to all of them.  (Eight floats are one 256-bit access: two
// of 128 bits would each touch half of every 32-byte sector.)
template <int N, typename T>
struct Raw;
template <>
struct Raw<8, float> {
  float f8[8];
  __device__ __forceinline__ void load(const float* p) { ldg8(p, f8); }
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = f8[i];
  }
};
template <>
struct Raw<8, __nv_bfloat16> {
  uint4 u;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { u = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const float2 a = bf2f(u.x), b = bf2f(u.y), c = bf2f(u.z), d = bf2f(u.w);
    f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y, f[4] = c.x, f[5] = c.y, f[6] = d.x, f[7] = d.y;
  }
};
template <>
struct Raw<2, float> {
  float2 a;
  __device__ __forceinline__ void load(const float* p) { a = *reinterpret_cast<const float2*>(p); }
  __device__ __forceinline__ void get(float (&f)[2]) const { f[0] = a.x, f[1] = a.y; }
};
template <>
struct Raw<2, __nv_bfloat16> {
  uint32_t u;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { u = *reinterpret_cast<const uint32_t*>(p); }
  __device__ __forceinline__ void get(float (&f)[2]) const {
    const float2 a = bf2f(u);
    f[0] = a.x, f[1] = a.y;
  }
};
template <typename T>
struct Raw<1, T> {
  T u;
  __device__ __forceinline__ void load(const T* p) { u = *p; }
  __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = ld(&u); }
};
template <int N, typename T>
__device__ __forceinline__ void load_n(const T* p, float (&f)[N]) {
  Raw<N, T> r;
  r.load(p);
  r.get(f);
}
template <int N, typename T>
__device__ __forceinline__ void store_n(T* p, const float (&f)[N]) {
  if constexpr (N == 8 && sizeof(T) == 4) {
    asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]),
                 "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7])
                 : "memory");
  } else if constexpr (N == 8) {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(f2bf(f2(f[0], f[1])), f2bf(f2(f[2], f[3])), f2bf(f2(f[4], f[5])), f2bf(f2(f[6], f[7])));
  } else if constexpr (N == 2 && sizeof(T) == 4) {
    *reinterpret_cast<float2*>(p) = make_float2(f[0], f[1]);
  } else if constexpr (N == 2) {
    *reinterpret_cast<uint32_t*>(p) = f2bf(f2(f[0], f[1]));
  } else {
    stg<T>(p, f[0]);
  }
}

constexpr int kRows = 4;  // rows in flight

template <typename T, typename O, int N>
__global__ void __launch_bounds__(kThreads) embed_kernel(const FwdParams p) {
  const int g = p.cols.group(), c = p.cols.first(N);
  if (g >= p.cols.groups || c >= p.dim) return;
  const T* table = reinterpret_cast<const T*>(p.table) + c;
  O* out = reinterpret_cast<O*>(p.out) + c;
  const int step = gridDim.x * p.cols.groups, start = blockIdx.x * p.cols.groups + g;
  int next[kRows];  // table rows; -1: padding, -2: past the table
  auto fetch = [&](int r0) {
    int64_t t[kRows];
#pragma unroll
    for (int j = 0; j < kRows; ++j) t[j] = r0 + j * step < p.rows ? p.tokens[p.trow.at(r0 + j * step)] : -1;
#pragma unroll
    for (int j = 0; j < kRows; ++j) next[j] = t[j] < 0 ? -1 : t[j] < p.vocab ? (int)t[j] : -2;
  };
  fetch(start);
  for (int r0 = start; r0 < p.rows; r0 += step * kRows) {
    int t[kRows];
    Raw<N, T> v[kRows];
#pragma unroll
    for (int j = 0; j < kRows; ++j) t[j] = next[j];
#pragma unroll
    for (int j = 0; j < kRows; ++j) v[j].load(table + (int64_t)max(t[j], 0) * p.table_ld);
    fetch(r0 + step * kRows);
#pragma unroll
    for (int j = 0; j < kRows; ++j)
      if (r0 + j * step < p.rows) {
        float f[N];
        if (t[j] >= 0) {
          v[j].get(f);
#pragma unroll
          for (int i = 0; i < N; ++i) f[i] *= p.scale;
        } else {
#pragma unroll
          for (int i = 0; i < N; ++i) f[i] = t[j] == -1 ? 0.f : NAN;
        }
        store_n<N>(out + (int64_t)(r0 + j * step) * p.out_ld, f);
      }
  }
}

// ---- stable radix sort of (token, r) ------------------------------------------------------
constexpr int kSortMostCtas = 16, kSortThreads = 1024, kSortWarps = kSortThreads / 32;
constexpr int kMaxBits = 9, kMaxBins = 1 << kMaxBits;
constexpr int kSortAhead = 8;  // entries a lane has in flight

struct SortParams {
  int64_t rows;
  int vocab, passes, bits;  // `passes` digits of `bits` bits
  Rows trow;
  const int64_t* tokens;
  uint2* buf[2];  // (token, r); the result is in buf[(passes - 1) & 1]
  int* count;     // entries in the result: the tokens inside [0, vocab)
};

struct ClearParams {
  int rows, vocab;
  Rows trow;
  const int64_t* tokens;
  unsigned char* grad;
  int64_t row_bytes, ld_bytes;
};

struct SortSmem {
  int hist[kSortWarps][kMaxBins];  // per warp, then its next output position per digit
  int total[kMaxBins];             // this CTA's count per digit, read by the cluster
  int wsum[kSortWarps];
};

// Clears the gradient's rows of the tokens that do not occur while the cluster before it in the stream
// sorts: every CTA marks all tokens in a bitmap of its own, then clears its share.
constexpr int kClearThreads = 1024, kClearWarps = kClearThreads / 32, kClearAhead = 8;
constexpr int kClearMostVocab = 48 * 1024 * 8;  // bits of the bitmap

__global__ void __launch_bounds__(kClearThreads) clear_kernel(const ClearParams p) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  uint32_t* seen = reinterpret_cast<uint32_t*>(smem_raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = tid; i < (p.vocab + 31) / 32; i += kClearThreads) seen[i] = 0u;
  __syncthreads();
  for (int64_t i = tid; i < p.rows; i += kClearThreads * kClearAhead) {
    int64_t t[kClearAhead];
#pragma unroll
    for (int j = 0; j < kClearAhead; ++j) {
      const int64_t at = i + j * kClearThreads;
      t[j] = at < p.rows ? p.tokens[p.trow.at((int)at)] : -1;
    }
#pragma unroll
    for (int j = 0; j < kClearAhead; ++j)
      if (t[j] >= 0 && t[j] < p.vocab) atomicOr(&seen[t[j] >> 5], 1u << (t[j] & 31));
  }
  __syncthreads();
  const bool wide = ((uintptr_t)p.grad | (uint64_t)p.ld_bytes | (uint64_t)p.row_bytes) % 16 == 0;
  for (int64_t v = (int64_t)blockIdx.x * kClearWarps + warp; v < p.vocab; v += (int64_t)gridDim.x * kClearWarps) {
    if (seen[v >> 5] >> (v & 31) & 1u) continue;
    unsigned char* g = p.grad + v * p.ld_bytes;
    if (wide) {
      for (int64_t b = lane * 16; b < p.row_bytes; b += 512) *reinterpret_cast<uint4*>(g + b) = make_uint4(0u, 0u, 0u, 0u);
    } else {
      for (int64_t b = lane * 2; b < p.row_bytes; b += 64) *reinterpret_cast<uint16_t*>(g + b) = 0;
    }
  }
  after_previous();  // the kernel behind this one reads what the sort writes
}

// Each of the cluster's warps owns a contiguous piece of the input; positions are handed out
// digit by digit, then CTA by CTA, warp by warp and lane by lane, so equal digits keep their order.
__global__ void __launch_bounds__(kSortThreads) sort_kernel(const SortParams p) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  extern __shared__ __align__(16) unsigned char smem_raw[];
  SortSmem& s = *reinterpret_cast<SortSmem*>(smem_raw);
  next_may_start();  // the clear needs nothing of this kernel; the sums wait in place
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = (int)cluster.block_rank();
  const int ctas = (int)cluster.num_blocks();
  const int bins = 1 << p.bits;
  const unsigned lt = (1u << lane) - 1u;
  int64_t n = p.rows;
  for (int pass = 0; pass < p.passes; ++pass) {
    const int shift = pass * p.bits;
    const uint2* src = p.buf[(pass + 1) & 1];
    uint2* dst = p.buf[pass & 1];
    const int64_t piece = (n + ctas * kSortWarps * 32 - 1) / (ctas * kSortWarps * 32) * 32;
    int64_t i0 = (int64_t)(rank * kSortWarps + warp) * piece, i1 = i0 + piece;
    if (i0 > n) i0 = n;
    if (i1 > n) i1 = n;
    // the first pass reads the tokens and leaves out those outside the table (their token becomes -1)
    auto fetch = [&](int64_t i, uint2(&e)[kSortAhead]) {
      if (pass > 0) {
#pragma unroll
        for (int j = 0; j < kSortAhead; ++j) {
          const int64_t at = i + 32 * j + lane;
          e[j] = at < i1 ? __ldcg(src + at) : make_uint2(~0u, 0u);
        }
      } else {
        int64_t t[kSortAhead];
#pragma unroll
        for (int j = 0; j < kSortAhead; ++j) {
          const int64_t at = i + 32 * j + lane;
          t[j] = at < i1 ? p.tokens[p.trow.at((int)at)] : -1;
        }
#pragma unroll
        for (int j = 0; j < kSortAhead; ++j)
          e[j] = make_uint2(t[j] >= 0 && t[j] < p.vocab ? (uint32_t)t[j] : ~0u, (uint32_t)(i + 32 * j + lane));
      }
    };
    for (int b = lane; b < bins; b += 32) s.hist[warp][b] = 0;
    __syncwarp();
    for (int64_t i = i0; i < i1; i += 32 * kSortAhead) {
      uint2 e[kSortAhead];
      fetch(i, e);
#pragma unroll
      for (int j = 0; j < kSortAhead; ++j)
        if (e[j].x != ~0u) atomicAdd(&s.hist[warp][(e[j].x >> shift) & (bins - 1)], 1);
    }
    __syncthreads();
    if (tid < bins) {
      int run = 0;
      for (int w = 0; w < kSortWarps; ++w) {
        const int h = s.hist[w][tid];
        s.hist[w][tid] = run;
        run += h;
      }
      s.total[tid] = run;
    }
    cluster.sync();
    int all = 0, before = 0;
    if (tid < bins)
      for (int r = 0; r < ctas; ++r) {
        const int v = *cluster.map_shared_rank(&s.total[tid], r);
        before += r < rank ? v : 0;
        all += v;
      }
    // exclusive scan of `all` over the digits
    int incl = all;
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) s.wsum[warp] = incl;
    __syncthreads();
    int start = incl - all, sum = 0;
    for (int w = 0; w < kSortWarps; ++w) {
      if (w < warp) start += s.wsum[w];
      sum += s.wsum[w];
    }
    if (tid < bins)
      for (int w = 0; w < kSortWarps; ++w) s.hist[w][tid] += start + before;
    __syncthreads();
    for (int64_t i = i0; i < i1; i += 32 * kSortAhead) {
      uint2 e[kSortAhead];
      fetch(i, e);
#pragma unroll
      for (int j = 0; j < kSortAhead; ++j) {
        const bool in = e[j].x != ~0u;
        const int d = (int)((e[j].x >> shift) & (bins - 1));
        // the lanes with the same digit, by its bits (a match instruction took twice the kernel's time)
        unsigned same = __ballot_sync(0xffffffffu, in);
        for (int b = 0; b < p.bits; ++b) {
          const unsigned ones = __ballot_sync(0xffffffffu, (d >> b) & 1);
          same &= (d >> b) & 1 ? ones : ~ones;
        }
        int at = 0;
        if (in) at = s.hist[warp][d] + __popc(same & lt);
        __syncwarp();
        if (in && (same & lt) == 0u) s.hist[warp][d] += __popc(same);
        __syncwarp();
        if (in) dst[at] = e[j];
      }
    }
    n = sum;
    __threadfence();
    cluster.sync();  // the pass's output is complete; nobody still reads this CTA's totals
  }
  if (rank == 0 && tid == 0) *p.count = (int)n;
}

// ---- row sums -----------------------------------------------------------------------------
// Chunk k holds the sorted entries [k C, (k + 1) C).  A group walks its chunk and writes the rows of the
// tokens that begin in it, reading on where the last one ends within the next chunk (whose group then
// leaves those entries out).  Of a longer token every chunk writes a piece to `parts`: slot 2 k + 1 where it
// begins, 2 k in the others.
struct SumParams {
  int grad_ld, dim, chunk, vocab, accumulate, clear, sum_ctas;  // clear: rows of absent tokens are still to be cleared
  float scale;
  Rows drow;
  const uint2* sorted;
  const int* count;
  const void* dy;
  void* grad;
  float* parts;  // (2 chunks, dim)
  Columns cols;
};

template <int N, typename G>
__device__ __forceinline__ void write_row(const SumParams& p, uint32_t token, int c, float (&s)[N]) {
  G* g = reinterpret_cast<G*>(p.grad) + (int64_t)token * p.grad_ld + c;
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] *= p.scale;
  if (p.accumulate) {
    float old[N];
    load_n<N>(g, old);
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] += old[i];
  }
  store_n<N>(g, s);
}

__device__ __forceinline__ int lower_bound(const uint2* a, int n, uint32_t key) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a[mid].x < key)
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo;
}

// The token, which occurs before position b, does not occur from b on.
__device__ __forceinline__ bool ends_by(const uint2* a, int n, int64_t b, uint32_t token) {
  return b >= n || a[b].x != token;
}

constexpr int kAhead = 4;  // entries in flight (8, with half the warps an SM holds: 36 us instead of 30)

template <typename D, typename G, int N>
__global__ void __launch_bounds__(kThreads) sum_kernel(const SumParams p) {
  after_previous();
  const int n = *p.count;
  if ((int)blockIdx.x >= p.sum_ctas) {
    // the rows of tokens that do not occur: a warp looks 32 of them up and clears those
    const int lane = threadIdx.x & 31, warps = ((int)gridDim.x - p.sum_ctas) * (kThreads / 32);
    int64_t v0 = (int64_t)(((int)blockIdx.x - p.sum_ctas) * (kThreads / 32) + (int)(threadIdx.x >> 5)) * 32;
    const int span = p.cols.width * N, c0 = (int)blockIdx.y * span, c1 = min(p.dim, c0 + span);
    float zero[N];
#pragma unroll
    for (int i = 0; i < N; ++i) zero[i] = 0.f;
    for (; v0 < p.vocab; v0 += (int64_t)warps * 32) {
      const int64_t v = v0 + lane;
      bool absent = false;
      if (v < p.vocab) {
        const int i = lower_bound(p.sorted, n, (uint32_t)v);
        absent = i == n || p.sorted[i].x != (uint32_t)v;
      }
      for (unsigned m = __ballot_sync(0xffffffffu, absent); m; m &= m - 1) {
        G* g = reinterpret_cast<G*>(p.grad) + (v0 + __ffs(m) - 1) * p.grad_ld;
        for (int c = c0 + lane * N; c < c1; c += 32 * N) store_n<N>(g + c, zero);
      }
    }
    return;
  }
  const int g = p.cols.group(), c = p.cols.first(N);
  if (g >= p.cols.groups || c >= p.dim) return;
  const int64_t k = (int64_t)blockIdx.x * p.cols.groups + g, b0 = k * p.chunk;
  if (b0 >= n) return;
  const uint2* so = p.sorted;
  int i0 = (int)b0, i1 = (int)min((int64_t)n, b0 + p.chunk);
  const D* dy = reinterpret_cast<const D*>(p.dy) + c;
  const uint32_t last = so[i1 - 1].x;
  uint32_t token = so[i0].x;
  bool began = i0 > 0 && so[i0 - 1].x == token;  // the current token's entries began before the chunk
  bool goes_on = i1 < n && so[i1].x == last;
  if (goes_on && !(began && last == token) && ends_by(so, n, b0 + 2 * p.chunk, last)) {
    i1 += lower_bound(so + i1, min(p.chunk, n - i1), last + 1u);
    goes_on = false;
  }
  if (began && (i0 == p.chunk || so[i0 - p.chunk - 1].x != token) && ends_by(so, n, b0 + p.chunk, token)) {
    i0 += lower_bound(so + i0, min(p.chunk, n - i0), token + 1u);
    if (i0 >= i1) return;
    token = so[i0].x;
    began = false;
  }
  float acc[N];
#pragma unroll
  for (int j = 0; j < N; ++j) acc[j] = 0.f;
  uint2 e[kAhead];
#pragma unroll
  for (int j = 0; j < kAhead; ++j) e[j] = so[min(i0 + j, i1 - 1)];
  for (int i = i0; i < i1; i += kAhead) {
    Raw<N, D> v[kAhead];
    uint32_t t[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      v[j].load(dy + p.drow.at((int)e[j].y));
      t[j] = e[j].x;
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) e[j] = so[min(i + kAhead + j, i1 - 1)];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (i + j >= i1) break;
      if (t[j] != token) {
        if (began)
          store_n<N>(p.parts + 2 * k * p.dim + c, acc);
        else
          write_row<N, G>(p, token, c, acc);
        token = t[j];
        began = false;
#pragma unroll
        for (int q = 0; q < N; ++q) acc[q] = 0.f;
      }
      float f[N];
      v[j].get(f);
#pragma unroll
      for (int q = 0; q < N; ++q) acc[q] += f[q];
    }
  }
  if (began || goes_on)
    store_n<N>(p.parts + (2 * k + (began ? 0 : 1)) * p.dim + c, acc);
  else
    write_row<N, G>(p, token, c, acc);
}

// Joins the pieces of the long tokens.  A CTA looks at kJoinChunks chunks for tokens that begin in one and
// go on past the next, and takes kJoinWidth threads' columns of them: its groups sum the pieces in
// turn (a chunk whose first entry is still the token holds one), and their sums meet in a fixed order.
constexpr int kJoinWidth = 8, kJoinChunks = 16, kJoinAhead = 4;

template <typename G, int N>
__global__ void __launch_bounds__(kThreads) join_kernel(const SumParams p) {
  constexpr int kGroups = kThreads / kJoinWidth;
  after_previous();
  __shared__ float sums[kThreads / 32][kJoinWidth * N];
  const int n = *p.count, lane = threadIdx.x & 31;
  const int64_t k = (int64_t)blockIdx.x * kJoinChunks + lane, b1 = (k + 1) * p.chunk;
  bool goes_on = false;
  uint32_t token_at = 0;
  if (lane < kJoinChunks && b1 < n) {
    token_at = p.sorted[b1 - 1].x;
    goes_on = p.sorted[b1].x == token_at && !(k > 0 && p.sorted[b1 - p.chunk - 1].x == token_at) &&
              !ends_by(p.sorted, n, b1 + p.chunk, token_at);
  }
  const int g = threadIdx.x / kJoinWidth, w = threadIdx.x % kJoinWidth;
  const int c = (blockIdx.y * kJoinWidth + w) * N;
  for (unsigned m = __ballot_sync(0xffffffffu, goes_on); m; m &= m - 1) {  // the same in every warp
    const int64_t first = (int64_t)blockIdx.x * kJoinChunks + __ffs(m) - 1;
    const uint32_t token = __shfl_sync(0xffffffffu, token_at, __ffs(m) - 1);
    float acc[N];
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = 0.f;
    if (c < p.dim) {
      if (g == 0) load_n<N>(p.parts + (2 * first + 1) * p.dim + c, acc);
      bool more = true;
      for (int64_t q = first + 1 + g; more; q += kGroups * kJoinAhead) {
        Raw<N, float> v[kJoinAhead];
        uint32_t t[kJoinAhead];
#pragma unroll
        for (int j = 0; j < kJoinAhead; ++j) {
          const int64_t at = q + j * kGroups, b = at * p.chunk;
          t[j] = b < n ? p.sorted[b].x : ~0u;
          v[j].load(p.parts + 2 * (b < n ? at : first) * p.dim + c);
        }
#pragma unroll
        for (int j = 0; j < kJoinAhead; ++j) {
          more = more && t[j] == token;
          float f[N];
          v[j].get(f);
#pragma unroll
          for (int i = 0; i < N; ++i) acc[i] += more ? f[i] : 0.f;
        }
      }
    }
    // the groups of a warp, then the warps
#pragma unroll
    for (int o = kJoinWidth; o < 32; o *= 2)
#pragma unroll
      for (int j = 0; j < N; ++j) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], o);
    if (lane < kJoinWidth)
#pragma unroll
      for (int j = 0; j < N; ++j) sums[threadIdx.x >> 5][w * N + j] = acc[j];
    __syncthreads();
    if (threadIdx.x < kJoinWidth && c < p.dim) {
#pragma unroll
      for (int h = 1; h < kThreads / 32; ++h)
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] += sums[h][w * N + j];
      write_row<N, G>(p, token, c, acc);
    }
    __syncthreads();
  }
}

size_t align256(size_t b) { return (b + 255) & ~(size_t)255; }

int sm_count() {
  int dev = 0, c = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&c, cudaDevAttrMultiProcessorCount, dev);
  return c;
}

// Allows the sort its shared memory and its cluster of 16, once per device.
int sort_setup() {
  static bool done[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return check_launch("m3_embed_bwd: cudaGetDevice");
  if (dev < 64 && done[dev]) return M3_OK;
  if (cudaFuncSetAttribute(sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(SortSmem)) !=
          cudaSuccess ||
      cudaFuncSetAttribute(sort_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
    return check_launch("m3_embed_bwd: cudaFuncSetAttribute");
  if (dev < 64) done[dev] = true;
  return M3_OK;
}

bool dtype_ok(int d) { return d == M3_DTYPE_F32 || d == M3_DTYPE_BF16; }

Columns columns(int dim, int n) {
  const int all = (dim + n - 1) / n, width = all < kThreads ? all : kThreads;
  return Columns{width, kThreads / width};
}
int slabs(int dim, int n, const Columns& c) { return (dim + n * c.width - 1) / (n * c.width); }

// Whether rows of `size`-byte elements (base and strides) allow N elements at a time.
bool whole(const void* p, int size, int n, int dim, int64_t s0, int64_t s1) {
  return dim % n == 0 && ((uintptr_t)p) % (size * n) == 0 && s0 % n == 0 && s1 % n == 0;
}

template <typename T, typename O, int N>
void launch_embed(FwdParams p, cudaStream_t s) {
  p.cols = columns(p.dim, N);
  // a small table's columns are cut so that a CTA's share of it stays in L1
  const int keep = (128 << 10) / (int)(p.vocab < 4096 ? p.vocab * (int)sizeof(T) * N : 1 << 30);
  if (keep >= 8 && keep < p.cols.width && p.rows > 8 * (int64_t)p.vocab) p.cols = Columns{keep / 8 * 8, kThreads / (keep / 8 * 8)};
  const int y = slabs(p.dim, N, p.cols);
  const int want = (p.rows + p.cols.groups - 1) / p.cols.groups, most = (sm_count() * 8 + y - 1) / y;
  embed_kernel<T, O, N><<<dim3((unsigned)(want < most ? want : most), y), kThreads, 0, s>>>(p);
}

template <typename T, typename O>
void launch_embed(const FwdParams& p, cudaStream_t s) {
  auto fits = [&](int n) {
    return whole(p.table, sizeof(T), n, p.dim, p.table_ld, 0) && whole(p.out, sizeof(O), n, p.dim, p.out_ld, 0);
  };
  if (fits(8)) return launch_embed<T, O, 8>(p, s);
  if (fits(2)) return launch_embed<T, O, 2>(p, s);
  launch_embed<T, O, 1>(p, s);
}

// Entries per chunk: enough chunks for 1536 threads of 8 columns on each of 148 SMs.
constexpr int kMinChunk = 16, kMaxChunk = 256;

int chunk_of(int64_t rows, int dim) {
  int64_t c = rows * ((dim + 7) / 8) / (148 * 1536);  // not the device's: the sums' order depends on it
  c = (c + 7) / 8 * 8;
  return (int)(c < kMinChunk ? kMinChunk : c > kMaxChunk ? kMaxChunk : c);
}

template <typename D, typename G, int N>
int launch_sum(SumParams p, int64_t rows, cudaStream_t s) {
  p.cols = columns(p.dim, N);
  const int y = slabs(p.dim, N, p.cols);
  const int64_t chunks = (rows + p.chunk - 1) / p.chunk;
  p.sum_ctas = (int)((chunks + p.cols.groups - 1) / p.cols.groups);
  const int64_t want = (p.vocab + 32 * (kThreads / 32) - 1) / (32 * (kThreads / 32)), most = (int64_t)sm_count() * 8;
  const int64_t clear = !p.clear ? 0 : want < most ? want : most;
  int rc = M3_OK;
  if (p.sum_ctas + clear > 0)
    rc = launch_ex("m3_embed_bwd", sum_kernel<D, G, N>, dim3((unsigned)(p.sum_ctas + clear), y), kThreads, 0, 1, true, s, p);
  if (rc == M3_OK && chunks > 1)
    rc = launch_ex("m3_embed_bwd", join_kernel<G, N>,
                   dim3((unsigned)((chunks + kJoinChunks - 2) / kJoinChunks), (p.dim + N * kJoinWidth - 1) / (N * kJoinWidth)),
                   kThreads, 0, 1, true, s, p);
  return rc;
}

template <typename D, typename G>
int launch_sum(const SumParams& p, int n, int64_t rows, cudaStream_t s) {
  if (n == 8) return launch_sum<D, G, 8>(p, rows, s);
  if (n == 2) return launch_sum<D, G, 2>(p, rows, s);
  return launch_sum<D, G, 1>(p, rows, s);
}

// Columns a thread takes of the gradient's rows: what the alignment of both allows.
int sum_columns(const M3EmbedBwdArgs& a, int dy_size, int grad_size) {
  for (int n : {8, 2})
    if (whole(a.dy, dy_size, n, a.dim, a.dy_outer, a.dy_inner) && whole(a.grad, grad_size, n, a.dim, a.grad_ld, 0)) return n;
  return 1;
}
// Whether the grids of launch_sum's kernels reach all columns.
bool grids_reach(int dim, int n, bool join) {
  return slabs(dim, n, columns(dim, n)) <= 65535 && (!join || (dim + n * kJoinWidth - 1) / (n * kJoinWidth) <= 65535);
}

}  // namespace
}  // namespace m3

using namespace m3;

extern "C" int m3_embed(const M3EmbedArgs* args, void* stream) {
  if (!args) return set_error(M3_ERR_ARG, "m3_embed: args is NULL");
  const M3EmbedArgs& a = *args;
  if (a.rows_outer < 0 || a.rows_inner < 0 || a.vocab <= 0 || a.dim <= 0)
    return set_error(M3_ERR_SHAPE, "m3_embed: need rows >= 0, vocab > 0 and dim > 0");
  if (!dtype_ok(a.table_dtype) || !dtype_ok(a.out_dtype))
    return set_error(M3_ERR_UNSUPPORTED, "m3_embed: table and out must be f32 or bf16");
  const int64_t rows = (int64_t)a.rows_outer * a.rows_inner;
  if (rows > vocab::kMaxRows) return set_error(M3_ERR_SHAPE, "m3_embed: more than 2^30 rows");
  if (rows == 0) return M3_OK;
  if (!a.tokens || !a.table || !a.out) return set_error(M3_ERR_ARG, "m3_embed: NULL pointer");
  if (a.table_ld < a.dim || a.out_ld < a.dim || a.table_ld > kMaxLd || a.out_ld > kMaxLd) return set_error(M3_ERR_SHAPE, "m3_embed: bad leading dimension");
  const size_t ts = a.table_dtype == M3_DTYPE_BF16 ? 2 : 4, os = a.out_dtype == M3_DTYPE_BF16 ? 2 : 4;
  if (((uintptr_t)a.table) % ts || ((uintptr_t)a.out) % os)
    return set_error(M3_ERR_ARG, "m3_embed: table and out must be aligned to their types");
  const FwdParams p{(int)rows,
                    a.vocab,
                    a.dim,
                    (int)a.table_ld,
                    (int)a.out_ld,
                    a.scale,
                    Rows{a.rows_outer, a.rows_inner, a.t_outer, a.t_inner},
                    a.tokens,
                    a.table,
                    a.out,
                    Columns{}};
  cudaStream_t s = (cudaStream_t)stream;
  using bf16 = __nv_bfloat16;
  if (ts == 2)
    os == 2 ? launch_embed<bf16, bf16>(p, s) : launch_embed<bf16, float>(p, s);
  else
    os == 2 ? launch_embed<float, bf16>(p, s) : launch_embed<float, float>(p, s);
  return check_launch("m3_embed");
}

extern "C" size_t m3_embed_bwd_workspace_size(int64_t rows, int32_t dim) {
  if (rows < 0 || rows > vocab::kMaxRows || dim <= 0) return 0;
  const size_t chunks = ((size_t)rows + chunk_of(rows, dim) - 1) / chunk_of(rows, dim);
  return 256 + 2 * align256((size_t)rows * sizeof(uint2)) + 2 * chunks * dim * sizeof(float);
}

extern "C" int m3_embed_bwd(const M3EmbedBwdArgs* args, void* stream) {
  if (!args) return set_error(M3_ERR_ARG, "m3_embed_bwd: args is NULL");
  const M3EmbedBwdArgs& a = *args;
  if (a.rows_outer < 0 || a.rows_inner < 0 || a.vocab <= 0 || a.dim <= 0)
    return set_error(M3_ERR_SHAPE, "m3_embed_bwd: need rows >= 0, vocab > 0 and dim > 0");
  if (!dtype_ok(a.dy_dtype) || !dtype_ok(a.grad_dtype))
    return set_error(M3_ERR_UNSUPPORTED, "m3_embed_bwd: dy and grad must be f32 or bf16");
  const int64_t rows = (int64_t)a.rows_outer * a.rows_inner;
  if (rows > vocab::kMaxRows) return set_error(M3_ERR_SHAPE, "m3_embed_bwd: more than 2^30 rows");
  if (!a.grad || (rows > 0 && (!a.tokens || !a.dy))) return set_error(M3_ERR_ARG, "m3_embed_bwd: NULL pointer");
  if (a.grad_ld < a.dim || a.grad_ld > kMaxLd) return set_error(M3_ERR_SHAPE, "m3_embed_bwd: bad leading dimension");
  const size_t ds = a.dy_dtype == M3_DTYPE_BF16 ? 2 : 4, gs = a.grad_dtype == M3_DTYPE_BF16 ? 2 : 4;
  if (((uintptr_t)a.dy) % ds || ((uintptr_t)a.grad) % gs)
    return set_error(M3_ERR_ARG, "m3_embed_bwd: dy and grad must be aligned to their types");
  const int columns_at_once = sum_columns(a, (int)ds, (int)gs);
  if (!grids_reach(a.dim, columns_at_once, rows > chunk_of(rows, a.dim)))
    return set_error(M3_ERR_SHAPE, "m3_embed_bwd: dim is too large");
  const size_t need = m3_embed_bwd_workspace_size(rows, a.dim);
  if (!a.workspace || a.workspace_bytes < need || ((uintptr_t)a.workspace) % 256)
    return set_error(M3_ERR_WORKSPACE, "m3_embed_bwd: 256-byte aligned workspace of " + std::to_string(need) +
                                           " bytes required");
  cudaStream_t s = (cudaStream_t)stream;
  unsigned char* ws = (unsigned char*)a.workspace;
  int bits_all = 1;
  while (bits_all < 31 && ((int64_t)1 << bits_all) < a.vocab) ++bits_all;
  SortParams sp;
  sp.rows = rows;
  sp.vocab = a.vocab;
  sp.passes = (bits_all + kMaxBits - 1) / kMaxBits;
  sp.bits = (bits_all + sp.passes - 1) / sp.passes;
  sp.trow = Rows{a.rows_outer, a.rows_inner, a.t_outer, a.t_inner};
  sp.tokens = a.tokens;
  sp.count = (int*)ws;
  sp.buf[0] = (uint2*)(ws + 256);
  sp.buf[1] = (uint2*)(ws + 256 + align256((size_t)rows * sizeof(uint2)));
  if (const int rc = sort_setup()) return rc;
  // a CTA for every 2048 tokens: the cluster's barriers cost more than a few tokens a lane
  int sort_ctas = 1;
  while (sort_ctas < kSortMostCtas && rows > 2048 * sort_ctas) sort_ctas *= 2;
  if (const int rc = launch_ex("m3_embed_bwd", sort_kernel, (unsigned)sort_ctas, kSortThreads, sizeof(SortSmem), sort_ctas,
                               false, s, sp))
    return rc;
  // Rows of absent tokens are cleared beside the sort by CTAs that each read all tokens; where that is
  // more to read than there is to clear, or the bitmap does not fit, the sums' launch looks them up.
  const int64_t row_bytes = (int64_t)a.dim * (int64_t)gs, all_bytes = row_bytes * a.vocab;
  int64_t ctas = sm_count() - sort_ctas;
  if (ctas > all_bytes >> 17) ctas = all_bytes >> 17;  // at least 128 KB each
  const bool beside = !a.accumulate && ctas > 0 && ctas * rows * 8 <= all_bytes / 2 && a.vocab <= kClearMostVocab;
  if (beside) {
    const ClearParams cp{(int)rows, a.vocab, sp.trow, a.tokens, (unsigned char*)a.grad, row_bytes,
                         a.grad_ld * (int64_t)gs};
    if (const int rc = launch_ex("m3_embed_bwd", clear_kernel, (unsigned)ctas, kClearThreads, ((size_t)a.vocab + 31) / 32 * 4,
                                 1, true, s, cp))
      return rc;
  }
  const SumParams p{(int)a.grad_ld,
                    a.dim,
                    chunk_of(rows, a.dim),
                    a.vocab,
                    a.accumulate,
                    !a.accumulate && !beside,
                    0,
                    a.scale,
                    Rows{a.rows_outer, a.rows_inner, a.dy_outer, a.dy_inner},
                    sp.buf[(sp.passes - 1) & 1],
                    sp.count,
                    a.dy,
                    a.grad,
                    (float*)(ws + 256 + 2 * align256((size_t)rows * sizeof(uint2))),
                    Columns{}};
  using bf16 = __nv_bfloat16;
  const bool gb = a.grad_dtype == M3_DTYPE_BF16;
  if (a.dy_dtype == M3_DTYPE_BF16)
    return gb ? launch_sum<bf16, bf16>(p, columns_at_once, rows, s) : launch_sum<bf16, float>(p, columns_at_once, rows, s);
  return gb ? launch_sum<float, bf16>(p, columns_at_once, rows, s) : launch_sum<float, float>(p, columns_at_once, rows, s);
}
