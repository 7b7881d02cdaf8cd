// state_pages.cu — pages of a cache of recurrent states: copy, fork, free and
// compact, decided on the device so that the calls can be captured.
//
// Each call is a plan and a copy.  The plan (one CTA) turns the caller's
// indices and the `used` flags into a list of (source page, destination page)
// with distinct destinations, none of which is a source, so the copy may run
// in any order.  The copy is a grid over (pair, pool, piece of a page) and is
// bound by HBM: every moved byte is read once and written once.
#include <cuda_runtime.h>

#include <atomic>

#include "common.cuh"
#include "ptx.cuh"

namespace gdn {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kCopyThreads = 256;
constexpr int64_t kPiece = 32 * 1024;  // bytes of a page that one CTA moves at a time

struct CopyParams {
  pages_pool_t pool[PAGES_MAX_POOLS];
  int32_t first[PAGES_MAX_POOLS + 1];  // pieces of the pools before this one, per pair
  const int32_t* src;                  // pairs; negative = skip
  const int32_t* dst;
  const int32_t* pairs;                // their number, or NULL: n
  int32_t n_pools, n;
};

// Exclusive prefix sum of `x` over the CTA; *total = its sum.  Every thread calls it.
__device__ int block_scan(int x, int* total) {
  __shared__ int s_warp[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = x;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, inc, off);
    if (lane >= off) inc += y;
  }
  if (lane == 31) s_warp[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    int w = s_warp[lane];
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, w, off);
      if (lane >= off) w += y;
    }
    s_warp[lane] = w;
  }
  __syncthreads();
  const int before = warp ? s_warp[warp - 1] : 0;
  *total = s_warp[31];
  __syncthreads();
  return before + inc - x;
}

// ws: [n] destination of each pair, -1 = skip
__global__ void __launch_bounds__(kPlanThreads) copy_plan_kernel(const pages_args_t a) {
  extern __shared__ uint32_t s_bits[];  // sources | destinations | destinations seen twice
  const int words = (a.pages + 31) / 32;
  uint32_t *is_src = s_bits, *is_dst = s_bits + words, *twice = s_bits + 2 * words;
  pdl_launch_dependents();
  for (int i = threadIdx.x; i < 3 * words; i += kPlanThreads) s_bits[i] = 0;
  __syncthreads();
  pdl_wait();
  const auto in = [&](int p) { return p >= 0 && p < a.pages; };
  for (int i = threadIdx.x; i < a.n; i += kPlanThreads) {
    const int s = a.src[i], d = a.dst[i];
    if (!in(s) || !in(d) || s == d) continue;
    atomicOr(&is_src[s >> 5], 1u << (s & 31));
    if (atomicOr(&is_dst[d >> 5], 1u << (d & 31)) >> (d & 31) & 1u) atomicOr(&twice[d >> 5], 1u << (d & 31));
  }
  __syncthreads();
  bool bad = false;
  for (int i = threadIdx.x; i < a.n; i += kPlanThreads) {
    const int s = a.src[i], d = a.dst[i];
    bool take = false;
    if (s >= 0 && d >= 0) {
      if (!in(s) || !in(d)) {
        bad = true;
      } else if (s != d) {
        take = !((is_src[d >> 5] | twice[d >> 5]) >> (d & 31) & 1u);
        bad |= !take;
      }
    }
    a.workspace[i] = take ? d : -1;
  }
  if (__syncthreads_or(bad) && threadIdx.x == 0) report(a.status, GDN_DEVERR_BAD_INDEX);
}

// dst[i] = the page given to entry i; ws: [n] the free pages in order
__global__ void __launch_bounds__(kPlanThreads) fork_plan_kernel(const pages_args_t a) {
  pdl_launch_dependents();
  pdl_wait();
  bool bad = false, full = false;
  int wanted = 0;
  for (int i0 = 0; i0 < a.n; i0 += kPlanThreads) {
    const int i = i0 + threadIdx.x;
    bool take = i < a.n;
    if (take && a.src) {
      const int s = a.src[i];
      take = s >= 0 && s < a.pages && a.used[s] != 0;
      bad |= s >= 0 && !take;
    }
    int total;
    const int rank = wanted + block_scan(take, &total);
    if (i < a.n) a.dst[i] = take ? rank : -1;
    wanted += total;
  }
  int given = 0;
  for (int p0 = 0; p0 < a.pages; p0 += kPlanThreads) {
    const int p = p0 + threadIdx.x;
    const int flag = p < a.pages ? a.used[p] : 1;
    int total;
    const int rank = given + block_scan(flag == 0, &total);
    const bool give = flag == 0 && rank < wanted;
    if (give) a.workspace[rank] = p;
    if (p < a.pages) a.used_out[p] = give ? 1 : flag;
    given += total;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.n; i += kPlanThreads) {
    const int rank = a.dst[i];
    if (rank < 0) continue;
    full |= rank >= given;
    a.dst[i] = rank < given ? a.workspace[rank] : -1;
  }
  if (__syncthreads_or(bad) && threadIdx.x == 0) report(a.status, GDN_DEVERR_BAD_INDEX);
  if (__syncthreads_or(full) && threadIdx.x == 0) report(a.status, GDN_DEVERR_POOL_FULL);
}

__global__ void __launch_bounds__(kPlanThreads) free_kernel(const pages_args_t a) {
  pdl_launch_dependents();
  pdl_wait();
  if (a.used_out != a.used)
    for (int p = threadIdx.x; p < a.pages; p += kPlanThreads) a.used_out[p] = a.used[p];
  __syncthreads();
  bool bad = false;
  for (int i = threadIdx.x; i < a.n; i += kPlanThreads) {
    const int p = a.src[i];
    if (p < 0) continue;
    if (p >= a.pages) bad = true;
    else bad |= atomicExch(a.used_out + p, 0) == 0;
  }
  if (__syncthreads_or(bad) && threadIdx.x == 0) report(a.status, GDN_DEVERR_BAD_INDEX);
}

// ws: [pages/2] holes = destinations, [pages/2] movers = sources, [1] their number
__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(const pages_args_t a) {
  pdl_launch_dependents();
  pdl_wait();
  int32_t* hole = a.workspace;
  int32_t* mover = a.workspace + a.pages / 2;
  int mine = 0, count;
  for (int p = threadIdx.x; p < a.pages; p += kPlanThreads) mine += a.used[p] != 0;
  block_scan(mine, &count);
  int holes = 0, movers = 0;
  for (int p0 = 0; p0 < a.pages; p0 += kPlanThreads) {
    const int p = p0 + threadIdx.x;
    const bool used = p < a.pages && a.used[p] != 0;
    const bool is_hole = p < count && !used, is_mover = p >= count && used;
    int total;  // at most 1024 of each: both counts fit one word
    const int rank = block_scan(is_hole | is_mover << 16, &total);
    if (is_hole) hole[holes + (rank & 0xffff)] = p;
    if (is_mover) mover[movers + (rank >> 16)] = p;
    holes += total & 0xffff;
    movers += total >> 16;
    if (p < a.pages) a.remap[p] = used && !is_mover ? p : -1;
  }
  __syncthreads();
  for (int r = threadIdx.x; r < movers; r += kPlanThreads) a.remap[mover[r]] = hole[r];
  if (threadIdx.x == 0) {
    *a.count = count;
    a.workspace[a.pages / 2 * 2] = movers;
  }
  for (int p = threadIdx.x; p < a.pages; p += kPlanThreads) a.used_out[p] = p < count;
  __syncthreads();
  bool bad = false;
  for (int i = threadIdx.x; i < a.n; i += kPlanThreads) {
    const int p = a.src[i];
    const int to = p >= 0 && p < a.pages ? a.remap[p] : -1;
    bad |= p >= 0 && to < 0;
    a.dst[i] = to;
  }
  if (__syncthreads_or(bad) && threadIdx.x == 0) report(a.status, GDN_DEVERR_BAD_INDEX);
}

__global__ void __launch_bounds__(kCopyThreads) copy_kernel(const __grid_constant__ CopyParams c) {
  pdl_launch_dependents();
  pdl_wait();
  const int64_t pairs = c.pairs ? *c.pairs : c.n;
  const int64_t per = c.first[c.n_pools];
  for (int64_t u = blockIdx.x; u < pairs * per; u += gridDim.x) {
    const int64_t i = u / per;
    const int piece = static_cast<int>(u - i * per);
    const int s = c.src[i], d = c.dst[i];
    if (s < 0 || d < 0) continue;
    int l = 0;
    while (piece >= c.first[l + 1]) ++l;
    const pages_pool_t& pool = c.pool[l];
    const int64_t at = (piece - c.first[l]) * kPiece;
    const int64_t left = pool.page_bytes - at;
    const int n = static_cast<int>((left < kPiece ? left : kPiece) / 16);
    const uint4* from = reinterpret_cast<const uint4*>(static_cast<const char*>(pool.base) + s * pool.page_stride + at);
    uint4* to = reinterpret_cast<uint4*>(static_cast<char*>(pool.base) + d * pool.page_stride + at);
    uint4 x[kPiece / 16 / kCopyThreads];
#pragma unroll
    for (int e = 0; e < static_cast<int>(kPiece / 16 / kCopyThreads); ++e)
      if (e * kCopyThreads + static_cast<int>(threadIdx.x) < n) x[e] = __ldcs(from + e * kCopyThreads + threadIdx.x);
#pragma unroll
    for (int e = 0; e < static_cast<int>(kPiece / 16 / kCopyThreads); ++e)
      if (e * kCopyThreads + static_cast<int>(threadIdx.x) < n) to[e * kCopyThreads + threadIdx.x] = x[e];
  }
}

template <typename Kernel, typename Arg>
int launch_pdl(Kernel kern, unsigned grid, unsigned threads, size_t smem, cudaStream_t stream, const Arg& arg) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kern, arg) != cudaSuccess) {
    (void)cudaGetLastError();
    return GDN_ERR_LAUNCH;
  }
  return GDN_OK;
}

int launch_copy(const pages_args_t& a, const int32_t* src, const int32_t* dst, const int32_t* pairs, int64_t most,
                const DeviceInfo& di, cudaStream_t stream) {
  if (!a.n_pools || most < 1) return GDN_OK;
  CopyParams c;
  c.src = src;
  c.dst = dst;
  c.pairs = pairs;
  c.n_pools = a.n_pools;
  c.n = a.n;
  c.first[0] = 0;
  for (int l = 0; l < a.n_pools; ++l) {
    c.pool[l] = a.pools[l];
    const int64_t pieces = (a.pools[l].page_bytes + kPiece - 1) / kPiece;
    if (pieces > INT32_MAX - c.first[l]) return GDN_ERR_SHAPE;
    c.first[l + 1] = c.first[l] + static_cast<int32_t>(pieces);
  }
  const int64_t units = most * c.first[a.n_pools], ctas = di.sm_count * 4;
  return launch_pdl(copy_kernel, static_cast<unsigned>(units < ctas ? units : ctas), kCopyThreads, 0, stream, c);
}

// What every call checks; `moves`: the pools are read and written.
int validate(const pages_args_t* a, bool flags, bool moves) {
  if (!a) return GDN_ERR_NULL;
  if (a->pages < 1 || a->pages > PAGES_MAX_PAGES || a->n < 0) return GDN_ERR_SHAPE;
  if (flags && (!a->used || !a->used_out)) return GDN_ERR_NULL;
  if (!moves) return GDN_OK;
  if (a->n_pools < 0 || a->n_pools > PAGES_MAX_POOLS) return GDN_ERR_SHAPE;
  if (a->n_pools && !a->pools) return GDN_ERR_NULL;
  for (int l = 0; l < a->n_pools; ++l) {
    const pages_pool_t& p = a->pools[l];
    if (!p.base) return GDN_ERR_NULL;
    if (p.page_bytes < 16 || p.page_stride < p.page_bytes) return GDN_ERR_SHAPE;
    if (!aligned16(p.base) || (p.page_bytes & 15) || (p.page_stride & 15)) return GDN_ERR_ALIGN;
  }
  return GDN_OK;
}

int workspace_ok(const pages_args_t* a, size_t need) {
  if (!a->workspace || a->workspace_bytes < need) return GDN_ERR_WORKSPACE;
  return (reinterpret_cast<uintptr_t>(a->workspace) & 3) ? GDN_ERR_ALIGN : GDN_OK;
}

size_t list_bytes(const pages_args_t* a) { return static_cast<size_t>(a->n) * 4; }
size_t compact_bytes(const pages_args_t* a) { return (static_cast<size_t>(a->pages) / 2 * 2 + 1) * 4; }

}  // namespace
}  // namespace gdn

using namespace gdn;

extern "C" size_t pages_workspace_size(const pages_args_t* a) {
  if (!a || a->n < 0 || a->pages < 1 || a->pages > PAGES_MAX_PAGES) return 0;
  return a->remap ? compact_bytes(a) : list_bytes(a);
}

extern "C" int pages_copy_launch(const pages_args_t* a, gdn_stream_t stream) {
  int rc = validate(a, false, true);
  if (rc) return rc;
  if (a->n == 0) return GDN_OK;
  if (!a->src || !a->dst) return GDN_ERR_NULL;
  if ((rc = workspace_ok(a, list_bytes(a)))) return rc;
  DeviceInfo di;
  if ((rc = device_info(&di))) return rc;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const size_t smem = (static_cast<size_t>(a->pages) + 31) / 32 * 12;
  static std::atomic<uint64_t> attr_done{0};
  if ((rc = ensure_smem_attr(copy_plan_kernel, (PAGES_MAX_PAGES / 32) * 12, attr_done))) return rc;
  if ((rc = launch_pdl(copy_plan_kernel, 1, kPlanThreads, smem, st, *a))) return rc;
  return launch_copy(*a, a->src, a->workspace, nullptr, a->n, di, st);
}

extern "C" int pages_fork_launch(const pages_args_t* a, gdn_stream_t stream) {
  int rc = validate(a, true, a && a->src);
  if (rc) return rc;
  if (a->n && !a->dst) return GDN_ERR_NULL;
  if ((rc = workspace_ok(a, list_bytes(a))) && a->n) return rc;
  DeviceInfo di;
  if ((rc = device_info(&di))) return rc;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if ((rc = launch_pdl(fork_plan_kernel, 1, kPlanThreads, 0, st, *a))) return rc;
  return a->src ? launch_copy(*a, a->src, a->dst, nullptr, a->n, di, st) : GDN_OK;
}

extern "C" int pages_free_launch(const pages_args_t* a, gdn_stream_t stream) {
  int rc = validate(a, true, false);
  if (rc) return rc;
  if (a->n && !a->src) return GDN_ERR_NULL;
  DeviceInfo di;
  if ((rc = device_info(&di))) return rc;
  return launch_pdl(free_kernel, 1, kPlanThreads, 0, reinterpret_cast<cudaStream_t>(stream), *a);
}

extern "C" int pages_compact_launch(const pages_args_t* a, gdn_stream_t stream) {
  int rc = validate(a, true, true);
  if (rc) return rc;
  if (!a->remap || !a->count || (a->n && (!a->src || !a->dst))) return GDN_ERR_NULL;
  if ((rc = workspace_ok(a, compact_bytes(a)))) return rc;
  DeviceInfo di;
  if ((rc = device_info(&di))) return rc;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if ((rc = launch_pdl(compact_plan_kernel, 1, kPlanThreads, 0, st, *a))) return rc;
  return launch_copy(*a, a->workspace + a->pages / 2, a->workspace, a->workspace + a->pages / 2 * 2, a->pages / 2, di,
                     st);
}
