// state_pages.cu — pages of a cache of recurrent states: copy, fork, free and
// compact, decided on the device so that the calls can be captured.
//
// Each call is a plan and a copy.  The plan turns the caller's indices and the
// `used` flags into a list of (source page, destination page) with distinct
// destinations, none of which is a source, so the copy may run in any order.  The
// copy is a grid over (pair, pool, piece of a page) and is bound by HBM: every
// moved byte is read once and written once.
//
// Small plans (kSmall pages and entries) are made by every CTA of the copy for
// itself in shared memory, one launch in all; only the first CTA writes the
// caller's arrays.  Larger ones are made once, by a CTA of their own, into the
// workspace.
#include <cuda_runtime.h>

#include <atomic>

#include "common.cuh"
#include "page_runs.cuh"
#include "ptx.cuh"

namespace gdn {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kCopyThreads = 256;
constexpr int kSmall = 2048;           // pages and entries up to which the copy plans for itself
constexpr int64_t kPiece = 32 * 1024;  // bytes of a page that one CTA moves at a time
// CTAs of a copy: 16 for each SM, of which 4 or so run at a time (16 sources of 2 MB
// forked into 64 in 2 pools: 65 us with 4, 62 with 8, 58 with 16 and with 64, which
// each plan for themselves; one read for a run of copies of one source: 84 -> 65 us)
constexpr int kCtasPerSm = 16;

enum Op { kCopy, kFork, kCompact };

struct CopyParams {
  pages_args_t a;
  pages_pool_t pool[PAGES_MAX_POOLS];
  int32_t first[PAGES_MAX_POOLS + 1];  // pieces of the pools before this one, per pair
  int32_t n_pools;
  int32_t write_used;  // the kernel may write used_out: it is not read by another CTA
  // a plan made before: its pairs, and their number (or NULL: a.n)
  const int32_t* src;
  const int32_t* dst;
  const int32_t* pairs;
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
    int w = lane < static_cast<int>(blockDim.x >> 5) ? s_warp[lane] : 0;
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

// The plans below are called by every thread of a CTA; `out`: this CTA writes the
// caller's arrays and the status.

// to[i] = destination of entry i, -1 = skip; bits: 3 x ceil(pages / 32) words.
__device__ void plan_copy(const pages_args_t& a, bool out, uint32_t* bits, int32_t* to) {
  const int words = (a.pages + 31) / 32;
  uint32_t *is_src = bits, *is_dst = bits + words, *twice = bits + 2 * words;
  for (int i = threadIdx.x; i < 3 * words; i += blockDim.x) bits[i] = 0;
  __syncthreads();
  const auto in = [&](int p) { return p >= 0 && p < a.pages; };
  for (int i = threadIdx.x; i < a.n; i += blockDim.x) {
    const int s = a.src[i], d = a.dst[i];
    if (!in(s) || !in(d) || s == d) continue;
    atomicOr(&is_src[s >> 5], 1u << (s & 31));
    if (atomicOr(&is_dst[d >> 5], 1u << (d & 31)) >> (d & 31) & 1u) atomicOr(&twice[d >> 5], 1u << (d & 31));
  }
  __syncthreads();
  bool bad = false;
  for (int i = threadIdx.x; i < a.n; i += blockDim.x) {
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
    to[i] = take ? d : -1;
  }
  if (__syncthreads_or(bad) && out && threadIdx.x == 0) report(a.status, GDN_DEVERR_BAD_INDEX);
}

// to[i] = the page given to entry i; list: n words, the free pages in order.
__device__ void plan_fork(const pages_args_t& a, bool out, bool write_used, int32_t* list, int32_t* to) {
  bool bad = false, full = false;
  int wanted = 0;
  for (int i0 = 0; i0 < a.n; i0 += blockDim.x) {
    const int i = i0 + threadIdx.x;
    bool take = i < a.n;
    if (take && a.src) {
      const int s = a.src[i];
      take = s >= 0 && s < a.pages && a.used[s] != 0;
      bad |= s >= 0 && !take;
    }
    int total;
    const int rank = wanted + block_scan(take, &total);
    if (i < a.n) to[i] = take ? rank : -1;
    wanted += total;
  }
  int given = 0;
  for (int p0 = 0; p0 < a.pages; p0 += blockDim.x) {
    const int p = p0 + threadIdx.x;
    const int flag = p < a.pages ? a.used[p] : 1;
    int total;
    const int rank = given + block_scan(flag == 0, &total);
    const bool give = flag == 0 && rank < wanted;
    if (give) list[rank] = p;
    if (out && write_used && p < a.pages) a.used_out[p] = give ? 1 : flag;
    given += total;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.n; i += blockDim.x) {
    const int rank = to[i];
    if (rank < 0) continue;
    full |= rank >= given;
    to[i] = rank < given ? list[rank] : -1;
  }
  if (__syncthreads_or(bad) && out && threadIdx.x == 0) report(a.status, GDN_DEVERR_BAD_INDEX);
  if (__syncthreads_or(full) && out && threadIdx.x == 0) report(a.status, GDN_DEVERR_POOL_FULL);
}

// mover[r] -> hole[r], r < the result; each pages / 2 words.
__device__ int plan_compact(const pages_args_t& a, bool out, bool write_used, int32_t* mover, int32_t* hole) {
  int mine = 0, count;
  for (int p = threadIdx.x; p < a.pages; p += blockDim.x) mine += a.used[p] != 0;
  block_scan(mine, &count);
  int holes = 0, movers = 0;
  for (int p0 = 0; p0 < a.pages; p0 += blockDim.x) {
    const int p = p0 + threadIdx.x;
    const bool used = p < a.pages && a.used[p] != 0;
    const bool is_hole = p < count && !used, is_mover = p >= count && used;
    int total;  // at most 1024 of each: both counts fit one word
    const int rank = block_scan(is_hole | is_mover << 16, &total);
    if (is_hole) hole[holes + (rank & 0xffff)] = p;
    if (is_mover) mover[movers + (rank >> 16)] = p;
    holes += total & 0xffff;
    movers += total >> 16;
    if (out && p < a.pages) a.remap[p] = used && !is_mover ? p : -1;
  }
  __syncthreads();
  if (!out) return movers;
  for (int r = threadIdx.x; r < movers; r += blockDim.x) a.remap[mover[r]] = hole[r];
  if (threadIdx.x == 0) *a.count = count;
  if (write_used)
    for (int p = threadIdx.x; p < a.pages; p += blockDim.x) a.used_out[p] = p < count;
  __syncthreads();
  bool bad = false;
  for (int i = threadIdx.x; i < a.n; i += blockDim.x) {
    const int p = a.src[i];
    const int to = p >= 0 && p < a.pages ? a.remap[p] : -1;
    bad |= p >= 0 && to < 0;
    a.dst[i] = to;
  }
  if (__syncthreads_or(bad) && threadIdx.x == 0) report(a.status, GDN_DEVERR_BAD_INDEX);
  return movers;
}

// A plan by itself, into the workspace: kCopy [n] destinations; kFork [n] free pages
// (the destinations are the caller's dst); kCompact [pages / 2] holes, [pages / 2]
// movers, their number.
template <Op OP>
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const pages_args_t a) {
  extern __shared__ uint32_t s_bits[];
  pdl_launch_dependents();
  pdl_wait();
  if constexpr (OP == kCopy) plan_copy(a, true, s_bits, a.workspace);
  if constexpr (OP == kFork) plan_fork(a, true, true, a.workspace, a.dst);
  if constexpr (OP == kCompact) {
    const int half = a.pages / 2;
    const int movers = plan_compact(a, true, true, a.workspace + half, a.workspace);
    if (threadIdx.x == 0) a.workspace[2 * half] = movers;
  }
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

// `used` in place, after a copy whose CTAs have all read it.
template <Op OP>
__global__ void __launch_bounds__(kCopyThreads) mark_kernel(const pages_args_t a) {
  pdl_launch_dependents();
  pdl_wait();
  if constexpr (OP == kFork) {
    for (int i = threadIdx.x; i < a.n; i += kCopyThreads)
      if (a.dst[i] >= 0) a.used_out[a.dst[i]] = 1;
  } else {
    const int count = *a.count;
    for (int p = threadIdx.x; p < a.pages; p += kCopyThreads) a.used_out[p] = p < count;
  }
}

// SELF: the CTA makes the plan itself.
template <Op OP, bool SELF>
__global__ void __launch_bounds__(kCopyThreads) copy_kernel(const __grid_constant__ CopyParams c) {
  __shared__ int32_t s_from[SELF ? kSmall : 1], s_to[SELF ? kSmall : 1];
  pdl_launch_dependents();
  pdl_wait();
  const int32_t *src = c.src, *dst = c.dst;
  int64_t pairs = c.a.n;
  if constexpr (SELF) {
    const bool out = blockIdx.x == 0;
    src = c.a.src;
    dst = s_to;
    if constexpr (OP == kCopy) plan_copy(c.a, out, reinterpret_cast<uint32_t*>(s_from), s_to);
    if constexpr (OP == kFork) {
      plan_fork(c.a, out, c.write_used, s_from, s_to);
      if (out)
        for (int i = threadIdx.x; i < c.a.n; i += kCopyThreads) c.a.dst[i] = s_to[i];
    }
    if constexpr (OP == kCompact) {
      pairs = plan_compact(c.a, out, c.write_used, s_from, s_to);
      src = s_from;
    }
  } else {
    if (c.pairs) pairs = *c.pairs;
  }
  const int64_t per = c.first[c.n_pools];
  for (int64_t u = blockIdx.x; u < pairs * per; u += gridDim.x) {
    const int64_t i = u / per;
    const int piece = static_cast<int>(u - i * per);
    int64_t j = run_first(src, dst, pairs, i);
    if (j < 0) continue;
    const int s = src[i];
    int l = 0;
    while (piece >= c.first[l + 1]) ++l;
    const pages_pool_t& pool = c.pool[l];
    const int64_t at = (piece - c.first[l]) * kPiece;
    const int64_t left = pool.page_bytes - at;
    const int n = static_cast<int>((left < kPiece ? left : kPiece) / 16);
    char* const base = static_cast<char*>(pool.base) + at;
    const uint4* from = reinterpret_cast<const uint4*>(base + s * pool.page_stride);
    uint4 x[kPiece / 16 / kCopyThreads];
#pragma unroll
    for (int e = 0; e < static_cast<int>(kPiece / 16 / kCopyThreads); ++e)
      if (e * kCopyThreads + static_cast<int>(threadIdx.x) < n) x[e] = __ldcs(from + e * kCopyThreads + threadIdx.x);
    for (; j >= 0; j = run_next(src, pairs, j)) {
      if (dst[j] < 0) continue;
      uint4* to = reinterpret_cast<uint4*>(base + dst[j] * pool.page_stride);
#pragma unroll
      for (int e = 0; e < static_cast<int>(kPiece / 16 / kCopyThreads); ++e)
        if (e * kCopyThreads + static_cast<int>(threadIdx.x) < n) to[e * kCopyThreads + threadIdx.x] = x[e];
    }
  }
}

bool small(const pages_args_t& a) { return a.pages <= kSmall && a.n <= kSmall; }

// The pools, and the pieces of `most` pairs as a number of CTAs.
int fill(CopyParams* c, const pages_args_t& a, int64_t most, const DeviceInfo& di, unsigned* ctas) {
  c->a = a;
  c->a.pools = nullptr;  // (host memory)
  c->n_pools = a.n_pools;
  c->write_used = a.used_out != a.used;
  c->src = c->dst = c->pairs = nullptr;
  c->first[0] = 0;
  for (int l = 0; l < a.n_pools; ++l) {
    c->pool[l] = a.pools[l];
    const int64_t pieces = (a.pools[l].page_bytes + kPiece - 1) / kPiece;
    if (pieces > INT32_MAX - c->first[l]) return GDN_ERR_SHAPE;
    c->first[l + 1] = c->first[l] + static_cast<int32_t>(pieces);
  }
  const int64_t units = most * c->first[a.n_pools], limit = static_cast<int64_t>(di.sm_count) * kCtasPerSm;
  *ctas = static_cast<unsigned>(units < limit ? units : limit);
  return GDN_OK;
}

// The plan and the copy in one launch (two where `used` is updated in place).
template <Op OP>
int launch_self(const pages_args_t& a, int64_t most, const DeviceInfo& di, cudaStream_t st) {
  CopyParams c;
  unsigned ctas;
  int rc = fill(&c, a, most, di, &ctas);
  if (rc || (rc = launch_pdl(copy_kernel<OP, true>, ctas ? ctas : 1, kCopyThreads, 0, st, c))) return rc;
  if constexpr (OP != kCopy)
    if (!c.write_used) return launch_pdl(mark_kernel<OP>, 1, kCopyThreads, 0, st, a);
  return GDN_OK;
}

// The copy of a plan that the stream has made.
template <Op OP>
int launch_planned(const pages_args_t& a, const int32_t* src, const int32_t* dst, const int32_t* pairs, int64_t most,
                   const DeviceInfo& di, cudaStream_t st) {
  CopyParams c;
  unsigned ctas;
  const int rc = fill(&c, a, most, di, &ctas);
  if (rc || !ctas) return rc;
  c.src = src;
  c.dst = dst;
  c.pairs = pairs;
  return launch_pdl(copy_kernel<OP, false>, ctas, kCopyThreads, 0, st, c);
}

// What every call checks; `moves`: the pools are read and written.
int validate(const pages_args_t* a, bool flags, bool moves) {
  if (!a) return GDN_ERR_NULL;
  if (a->pages < 1 || a->pages > PAGES_MAX_PAGES || a->n < 0) return GDN_ERR_SHAPE;
  if (flags) {
    if (!a->used || !a->used_out) return GDN_ERR_NULL;
    if (a->used != a->used_out && a->used < a->used_out + a->pages && a->used_out < a->used + a->pages) return GDN_ERR_SHAPE;
  }
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
  if (!need) return GDN_OK;
  if (!a->workspace || a->workspace_bytes < need) return GDN_ERR_WORKSPACE;
  return (reinterpret_cast<uintptr_t>(a->workspace) & 3) ? GDN_ERR_ALIGN : GDN_OK;
}

size_t list_bytes(const pages_args_t* a) { return small(*a) ? 0 : static_cast<size_t>(a->n) * 4; }
size_t compact_bytes(const pages_args_t* a) {
  return small(*a) ? 0 : (static_cast<size_t>(a->pages) / 2 * 2 + 1) * 4;
}

// Whether two arrays of int32 share memory (`same` allowed: they may be the same one).
bool overlap(const int32_t* p, int64_t n, const int32_t* q, int64_t m, bool same) {
  return p && q && n && m && p < q + m && q < p + n && !(same && p == q);
}

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
  if (small(*a)) return launch_self<kCopy>(*a, a->n, di, st);
  static std::atomic<uint64_t> attr_done{0};
  if ((rc = ensure_smem_attr(plan_kernel<kCopy>, (PAGES_MAX_PAGES / 32) * 12, attr_done))) return rc;
  const size_t smem = (static_cast<size_t>(a->pages) + 31) / 32 * 12;
  if ((rc = launch_pdl(plan_kernel<kCopy>, 1, kPlanThreads, smem, st, *a))) return rc;
  return launch_planned<kCopy>(*a, a->src, a->workspace, nullptr, a->n, di, st);
}

extern "C" int pages_fork_launch(const pages_args_t* a, gdn_stream_t stream) {
  int rc = validate(a, true, a && a->src);
  if (rc) return rc;
  if (a->n && !a->dst) return GDN_ERR_NULL;
  if (overlap(a->dst, a->n, a->src, a->n, false) || overlap(a->dst, a->n, a->used, a->pages, false) ||
      overlap(a->dst, a->n, a->used_out, a->pages, false) || overlap(a->src, a->n, a->used_out, a->pages, false))
    return GDN_ERR_SHAPE;
  if ((rc = workspace_ok(a, list_bytes(a)))) return rc;
  DeviceInfo di;
  if ((rc = device_info(&di))) return rc;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  pages_args_t b = *a;
  if (!b.src) b.n_pools = 0;
  if (small(b)) return launch_self<kFork>(b, b.n, di, st);
  if ((rc = launch_pdl(plan_kernel<kFork>, 1, kPlanThreads, 0, st, b))) return rc;
  return launch_planned<kFork>(b, b.src, b.dst, nullptr, b.n, di, st);
}

extern "C" int pages_free_launch(const pages_args_t* a, gdn_stream_t stream) {
  int rc = validate(a, true, false);
  if (rc) return rc;
  if (a->n && !a->src) return GDN_ERR_NULL;
  if (overlap(a->src, a->n, a->used_out, a->pages, false)) return GDN_ERR_SHAPE;
  DeviceInfo di;
  if ((rc = device_info(&di))) return rc;
  return launch_pdl(free_kernel, 1, kPlanThreads, 0, reinterpret_cast<cudaStream_t>(stream), *a);
}

extern "C" int pages_compact_launch(const pages_args_t* a, gdn_stream_t stream) {
  int rc = validate(a, true, true);
  if (rc) return rc;
  if (!a->remap || !a->count || (a->n && (!a->src || !a->dst))) return GDN_ERR_NULL;
  const int32_t* const out[] = {a->remap, a->count, a->n ? a->dst : nullptr};
  const int64_t len[] = {a->pages, 1, a->n};
  for (int i = 0; i < 3; ++i) {
    if (overlap(out[i], len[i], a->used, a->pages, false) || overlap(out[i], len[i], a->used_out, a->pages, false) ||
        overlap(out[i], len[i], a->src, a->n, i == 2))
      return GDN_ERR_SHAPE;
    for (int j = 0; j < i; ++j)
      if (overlap(out[i], len[i], out[j], len[j], false)) return GDN_ERR_SHAPE;
  }
  if (overlap(a->src, a->n, a->used_out, a->pages, false)) return GDN_ERR_SHAPE;
  if ((rc = workspace_ok(a, compact_bytes(a)))) return rc;
  DeviceInfo di;
  if ((rc = device_info(&di))) return rc;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int half = a->pages / 2;
  if (small(*a)) return launch_self<kCompact>(*a, half, di, st);
  if ((rc = launch_pdl(plan_kernel<kCompact>, 1, kPlanThreads, 0, st, *a))) return rc;
  return launch_planned<kCompact>(*a, a->workspace + half, a->workspace, a->workspace + 2 * half, half, di, st);
}
