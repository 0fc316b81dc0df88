// Embedding lookup with scaling, and the table's gradient by sorted tokens.
//   out[r] = scale * table[token r]              grad[v] = scale * sum of dy[r] over token r == v
// The gradient's rows are summed in the order of r (fp32), so that it is the same every call:
// (token, r) pairs are put in order by a stable radix sort (one 8-CTA cluster), then every
// vocabulary row sums its own range of the sorted list.
#include <cooperative_groups.h>

#include "m3_internal.h"
#include "m3_vocab.cuh"

namespace m3 {
namespace {

using vocab::Rows;

constexpr int kThreads = 256;

// ---- lookup -------------------------------------------------------------------------------
struct FwdParams {
  int64_t rows, table_ld, out_ld;
  int vocab, dim;
  float scale;
  Rows trow;
  const int64_t* tokens;
  const void* table;
  void* out;
};

template <typename T, typename O>
__global__ void __launch_bounds__(kThreads) embed_kernel(const FwdParams p) {
  const int64_t total = p.rows * p.dim;
  for (int64_t i = blockIdx.x * (int64_t)kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
    const int64_t r = i / p.dim;
    const int c = (int)(i - r * p.dim);
    const int64_t t = p.tokens[p.trow.at((int)r)];
    float v = t < 0 ? 0.f : NAN;
    if (t >= 0 && t < p.vocab) v = ld(reinterpret_cast<const T*>(p.table) + t * p.table_ld + c) * p.scale;
    stg<O>(reinterpret_cast<O*>(p.out) + r * p.out_ld + c, v);
  }
}

// ---- stable radix sort of (token, r) ------------------------------------------------------
constexpr int kSortCtas = 8, kSortThreads = 1024, kSortWarps = kSortThreads / 32;
constexpr int kMaxBits = 9, kMaxBins = 1 << kMaxBits;

struct SortParams {
  int64_t rows;
  int vocab, passes, bits;  // `passes` digits of `bits` bits
  Rows trow;
  const int64_t* tokens;
  uint2* buf[2];  // (token, r); the result is in buf[(passes - 1) & 1]
  int* count;     // entries in the result: the tokens inside [0, vocab)
};

struct SortSmem {
  int hist[kSortWarps][kMaxBins];  // per warp, then its next output position per digit
  int total[kMaxBins];             // this CTA's count per digit, read by the cluster
  int wsum[kSortWarps];
};

// Each of the cluster's 256 warps owns a contiguous piece of the input; positions are handed out
// digit by digit, then CTA by CTA, warp by warp and lane by lane, so equal digits keep their order.
__global__ void __cluster_dims__(kSortCtas, 1, 1) __launch_bounds__(kSortThreads) sort_kernel(const SortParams p) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  extern __shared__ __align__(16) unsigned char smem_raw[];
  SortSmem& s = *reinterpret_cast<SortSmem*>(smem_raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = (int)cluster.block_rank();
  const int bins = 1 << p.bits;
  const unsigned lt = (1u << lane) - 1u;
  int64_t n = p.rows;
  for (int pass = 0; pass < p.passes; ++pass) {
    const int shift = pass * p.bits;
    const uint2* src = p.buf[(pass + 1) & 1];
    uint2* dst = p.buf[pass & 1];
    const int64_t piece = (n + kSortCtas * kSortWarps * 32 - 1) / (kSortCtas * kSortWarps * 32) * 32;
    int64_t i0 = (int64_t)(rank * kSortWarps + warp) * piece, i1 = i0 + piece;
    if (i0 > n) i0 = n;
    if (i1 > n) i1 = n;
    // the first pass reads the tokens and leaves out those outside the table
    auto fetch = [&](int64_t i, uint2& e) -> bool {
      if (i >= i1) return false;
      if (pass > 0) {
        e = __ldcg(src + i);
        return true;
      }
      const int64_t t = p.tokens[p.trow.at((int)i)];
      e = make_uint2((uint32_t)t, (uint32_t)i);
      return t >= 0 && t < p.vocab;
    };
    for (int b = lane; b < bins; b += 32) s.hist[warp][b] = 0;
    __syncwarp();
    for (int64_t i = i0; i < i1; i += 32) {
      uint2 e;
      if (fetch(i + lane, e)) atomicAdd(&s.hist[warp][(e.x >> shift) & (bins - 1)], 1);
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
      for (int r = 0; r < kSortCtas; ++r) {
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
    for (int64_t i = i0; i < i1; i += 32) {
      uint2 e = make_uint2(0u, 0u);
      const bool in = fetch(i + lane, e);
      const int d = in ? (int)((e.x >> shift) & (bins - 1)) : bins;
      const unsigned same = __match_any_sync(0xffffffffu, d);
      int at = 0;
      if (in) at = s.hist[warp][d] + __popc(same & lt);
      __syncwarp();
      if (in && (same & lt) == 0u) s.hist[warp][d] += __popc(same);
      __syncwarp();
      if (in) dst[at] = e;
    }
    n = sum;
    __threadfence();
    cluster.sync();  // the pass's output is complete; nobody still reads this CTA's totals
  }
  if (rank == 0 && tid == 0) *p.count = (int)n;
}

// ---- row sums -----------------------------------------------------------------------------
struct SumParams {
  int64_t grad_ld;
  int dim, accumulate;
  float scale;
  Rows drow;
  const uint2* sorted;
  const int* count;
  const void* dy;
  void* grad;
};

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

template <typename D, typename G>
__global__ void __launch_bounds__(kThreads) sum_kernel(const SumParams p) {
  const int v = blockIdx.x, n = *p.count;
  const int i0 = lower_bound(p.sorted, n, (uint32_t)v), i1 = lower_bound(p.sorted, n, (uint32_t)v + 1u);
  if (p.accumulate && i0 == i1) return;
  G* g = reinterpret_cast<G*>(p.grad) + v * p.grad_ld;
  for (int c = threadIdx.x; c < p.dim; c += kThreads) {
    float s = 0.f;
    for (int i = i0; i < i1; ++i) s += ld(reinterpret_cast<const D*>(p.dy) + p.drow.at((int)p.sorted[i].y) + c);
    s *= p.scale;
    stg<G>(g + c, p.accumulate ? ld(g + c) + s : s);
  }
}

size_t align256(size_t b) { return (b + 255) & ~(size_t)255; }

int sm_count() {
  int dev = 0, c = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&c, cudaDevAttrMultiProcessorCount, dev);
  return c;
}

bool dtype_ok(int d) { return d == M3_DTYPE_F32 || d == M3_DTYPE_BF16; }

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
  if (a.table_ld < a.dim || a.out_ld < a.dim) return set_error(M3_ERR_SHAPE, "m3_embed: bad leading dimension");
  const FwdParams p{rows,     a.table_ld, a.out_ld, a.vocab, a.dim, a.scale, Rows{a.rows_inner, a.t_outer, a.t_inner},
                    a.tokens, a.table,    a.out};
  cudaStream_t s = (cudaStream_t)stream;
  const int64_t want = (rows * a.dim + kThreads - 1) / kThreads, most = (int64_t)sm_count() * 8;
  const unsigned grid = (unsigned)(want < most ? want : most);
  const bool tb = a.table_dtype == M3_DTYPE_BF16, ob = a.out_dtype == M3_DTYPE_BF16;
  auto* kern = tb ? (ob ? embed_kernel<__nv_bfloat16, __nv_bfloat16> : embed_kernel<__nv_bfloat16, float>)
                  : (ob ? embed_kernel<float, __nv_bfloat16> : embed_kernel<float, float>);
  kern<<<grid, kThreads, 0, s>>>(p);
  return check_launch("m3_embed");
}

extern "C" size_t m3_embed_bwd_workspace_size(int64_t rows, int32_t dim) {
  if (rows < 0 || rows > vocab::kMaxRows || dim <= 0) return 0;
  return 2 * align256((size_t)rows * sizeof(uint2)) + 256;
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
  if (a.grad_ld < a.dim) return set_error(M3_ERR_SHAPE, "m3_embed_bwd: bad leading dimension");
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
  sp.trow = Rows{a.rows_inner, a.t_outer, a.t_inner};
  sp.tokens = a.tokens;
  sp.count = (int*)ws;
  sp.buf[0] = (uint2*)(ws + 256);
  sp.buf[1] = (uint2*)(ws + 256 + align256((size_t)rows * sizeof(uint2)));
  static bool attr[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !attr[dev]) {
    if (cudaFuncSetAttribute(sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(SortSmem)) !=
        cudaSuccess)
      return check_launch("m3_embed_bwd: cudaFuncSetAttribute");
    if (dev < 64) attr[dev] = true;
  }
  sort_kernel<<<kSortCtas, kSortThreads, sizeof(SortSmem), s>>>(sp);
  const SumParams p{a.grad_ld, a.dim,    a.accumulate,
                    a.scale,   Rows{a.rows_inner, a.dy_outer, a.dy_inner},
                    sp.buf[(sp.passes - 1) & 1], sp.count, a.dy, a.grad};
  const bool db = a.dy_dtype == M3_DTYPE_BF16, gb = a.grad_dtype == M3_DTYPE_BF16;
  auto* kern = db ? (gb ? sum_kernel<__nv_bfloat16, __nv_bfloat16> : sum_kernel<__nv_bfloat16, float>)
                  : (gb ? sum_kernel<float, __nv_bfloat16> : sum_kernel<float, float>);
  kern<<<(unsigned)a.vocab, kThreads, 0, s>>>(p);
  return check_launch("m3_embed_bwd");
}
