// lin_prefill.cu — linear attention with a decay per head over T tokens.
#include <cuda_runtime.h>

#include "common.cuh"
#include "ptx.cuh"

namespace gdn {
namespace {

constexpr int kThreads = 256;
constexpr int kCols = 64;

// Where sequence n lies: first row, tokens, page (-1: none).  ok: offsets are sound.
struct Seq {
  int64_t start;
  int len, page;
  bool ok, bad_page;
};

__device__ Seq find_seq(const lin_prefill_args_t& a, int n) {
  Seq s;
  s.ok = true;
  s.start = 0;
  s.len = a.T;
  if (a.cu_seqlens) {
    const int lo = a.cu_seqlens[n], hi = a.cu_seqlens[n + 1];
    s.ok = lo >= 0 && lo <= hi && hi <= a.T;
    s.start = lo;
    s.len = s.ok ? hi - lo : 0;
  }
  s.page = a.index ? a.index[n] : n;
  s.bad_page = s.page >= a.pages;
  return s;
}

template <int DK, typename IO>
__global__ void __launch_bounds__(kThreads) recurrent_kernel(const lin_prefill_args_t a) {
  constexpr int kParts = kThreads / kCols, kRows = DK / kParts;
  __shared__ float s_k[DK], s_q[DK], s_o[kParts][kCols];
  const int nvb = a.dv / kCols;
  const int h = blockIdx.x / nvb, vb = blockIdx.x - h * nvb, hq = h / (a.Hv / a.Hqk);
  const int n = blockIdx.y, tid = threadIdx.x, col = tid % kCols, part = tid / kCols;
  Seq s = find_seq(a, n);
  bool taken = false;
  if (a.index && s.page >= 0)
    for (int j = tid; j < n; j += kThreads) taken |= a.index[j] == s.page;
  if (__syncthreads_or(taken)) s.bad_page = true;
  if ((s.bad_page || !s.ok) && blockIdx.x == 0 && tid == 0) report(a.status, GDN_DEVERR_BAD_INDEX);
  if (!s.ok) return;
  if (s.bad_page) s.page = -1;
  const int64_t at = static_cast<int64_t>(h) * DK * a.dv + vb * kCols + col;
  float S[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i)
    S[i] = a.initial_state && s.page >= 0
               ? a.initial_state[s.page * a.initial_sp + at + static_cast<int64_t>(part * kRows + i) * a.dv]
               : 0.f;
  const int64_t b = a.cu_seqlens ? 0 : n;
  for (int t = 0; t < s.len; ++t) {
    const int64_t r = s.start + t;
    if (tid < DK) {
      s_k[tid] = to_f32(static_cast<const IO*>(a.k)[b * a.k_sb + r * a.k_st + hq * a.k_sh + tid]);
      s_q[tid] = to_f32(static_cast<const IO*>(a.q)[b * a.q_sb + r * a.q_st + hq * a.q_sh + tid]);
    }
    const float v = to_f32(static_cast<const IO*>(a.v)[b * a.v_sb + r * a.v_st + h * a.v_sh + vb * kCols + col]);
    const float alpha = expf(load_any(a.g, b * a.g_sb + r * a.g_st + h * a.g_sh, a.g_dtype));
    __syncthreads();
    float o = 0.f;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      S[i] = fmaf(alpha, S[i], s_k[part * kRows + i] * v);
      o = fmaf(s_q[part * kRows + i], S[i], o);
    }
    s_o[part][col] = o;
    __syncthreads();
    if (part == 0) {
      float x = 0.f;
#pragma unroll
      for (int p = 0; p < kParts; ++p) x += s_o[p][col];
      static_cast<IO*>(a.o)[b * a.o_sb + r * a.o_st + h * a.o_sh + vb * kCols + col] = from_f32<IO>(a.scale * x);
    }
  }
  if (s.page >= 0)
#pragma unroll
    for (int i = 0; i < kRows; ++i)
      a.final_state[s.page * a.final_sp + at + static_cast<int64_t>(part * kRows + i) * a.dv] = S[i];
}

int validate(const lin_prefill_args_t* a) {
  if (!a) return GDN_ERR_NULL;
  if (!a->q || !a->k || !a->v || !a->g || !a->final_state || !a->o) return GDN_ERR_NULL;
  if (a->B < 1 || a->B > 65535 || a->T < 1 || a->Hqk < 1 || a->Hv < 1 || a->Hv % a->Hqk) return GDN_ERR_SHAPE;
  if (a->pages < 1 || (!a->index && a->pages < a->B)) return GDN_ERR_SHAPE;
  if (a->dk != 64 && a->dk != 128) return GDN_ERR_SHAPE;
  if (a->dv < 64 || a->dv % 64) return GDN_ERR_SHAPE;
  const int64_t page = static_cast<int64_t>(a->Hv) * a->dk * a->dv;
  if (page > INT32_MAX || a->final_sp < page || (a->initial_state && a->initial_sp < page)) return GDN_ERR_SHAPE;
  if (a->io_dtype != GDN_DT_BF16 && a->io_dtype != GDN_DT_F16) return GDN_ERR_DTYPE;
  if (!dtype_valid(a->g_dtype)) return GDN_ERR_DTYPE;
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->o) || !aligned16(a->final_state) ||
      !aligned16(a->initial_state))
    return GDN_ERR_ALIGN;
  for (int64_t st : {a->q_sb, a->q_st, a->q_sh, a->k_sb, a->k_st, a->k_sh, a->v_sb, a->v_st, a->v_sh, a->o_sb, a->o_st,
                     a->o_sh}) {
    if (st < 0) return GDN_ERR_SHAPE;
    if (!stride_ok(st, 2)) return GDN_ERR_ALIGN;
  }
  if (!stride_ok(a->final_sp, 4) || (a->initial_state && !stride_ok(a->initial_sp, 4))) return GDN_ERR_ALIGN;
  if (a->initial_state && a->initial_state != a->final_state) {
    const float* i1 = a->initial_state + (a->pages - 1) * a->initial_sp + page;
    const float* f1 = a->final_state + (a->pages - 1) * a->final_sp + page;
    if (a->initial_state < f1 && a->final_state < i1) return GDN_ERR_SHAPE;
  } else if (a->initial_state && a->initial_sp != a->final_sp) {
    return GDN_ERR_SHAPE;
  }
  return GDN_OK;
}

}  // namespace
}  // namespace gdn

extern "C" size_t lin_prefill_workspace_size(const lin_prefill_args_t*) { return 0; }

extern "C" int lin_prefill_launch(const lin_prefill_args_t* a, gdn_stream_t stream) {
  int rc = gdn::validate(a);
  if (rc) return rc;
  gdn::DeviceInfo di;
  if ((rc = gdn::device_info(&di))) return rc;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid(a->Hv * (a->dv / gdn::kCols), a->B);
  const bool bf = a->io_dtype == GDN_DT_BF16;
  if (a->dk == 64 && bf) gdn::recurrent_kernel<64, __nv_bfloat16><<<grid, gdn::kThreads, 0, st>>>(*a);
  else if (a->dk == 64) gdn::recurrent_kernel<64, __half><<<grid, gdn::kThreads, 0, st>>>(*a);
  else if (bf) gdn::recurrent_kernel<128, __nv_bfloat16><<<grid, gdn::kThreads, 0, st>>>(*a);
  else gdn::recurrent_kernel<128, __half><<<grid, gdn::kThreads, 0, st>>>(*a);
  return cudaGetLastError() == cudaSuccess ? GDN_OK : GDN_ERR_LAUNCH;
}
