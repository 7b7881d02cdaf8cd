// lin_decode.cu — one token of linear attention with a decay per head:
//
//     S' = a S + k v^T            o = scale * S'^T q
//
// per (row, value head), the state fp32 and in place or in a pool of pages.
// Work: the state crosses HBM once in each direction (8 bytes per element, 5
// flops), so the kernel is bound by HBM; q, k, v and o are 1/100 of that.
//
// Unlike the delta rule nothing has to be reduced before the state can be
// written back: S' = a S + k v^T is elementwise, and o = q^T S' is summed on the
// side.  So there is no ring and no producer warp: a CTA takes one DK x BV slab of
// a head's state (columns are independent), every thread issues the loads of all
// its rows at once, and the CTAs resident on an SM hide each other's latency.
// B = 1024, H = 32, d = 128: 647 to 662 us, 6.5 to 6.7 TB/s of state, the measured copy's
// rate and what the GDN decode's ring reaches; with pages in random order 5% less.  d =
// 256 x 128, B = 512: 723 to 730 us, 0.91 of that rate.
#include <cuda_runtime.h>

#include "common.cuh"
#include "ptx.cuh"

namespace gdn {
namespace {

// 128 threads: at B = 1024, H = 32, d = 128, in bursts, a 128-column slab takes 641 us
// (6.70 TB/s of state) with 128 threads, 972 with 256 and 996 with 512.  More threads per slab
// mean fewer slabs on an SM, whose loads, arithmetic and stores then overlap less.
constexpr int kThreads = 128;

template <int DK, int BV, typename IO>
__global__ void __launch_bounds__(kThreads) lin_decode_kernel(const lin_decode_args_t a) {
  constexpr int kColGroups = BV / 4;                   // threads across a row, 4 columns each
  constexpr int kRowGroups = kThreads / kColGroups;
  constexpr int kRows = DK / kRowGroups;               // rows per thread
  constexpr int kWarps = kThreads / 32;
  static_assert(DK % kRowGroups == 0 && kColGroups <= 32, "slab shape");
  __shared__ float s_k[DK], s_q[DK];
  __shared__ float s_red[kWarps][BV];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cg = tid % kColGroups, rg = tid / kColGroups;
  const int nvb = a.dv / BV;
  const int h = blockIdx.x / nvb, vb = blockIdx.x - h * nvb;
  const int hq = h / (a.Hv / a.Hqk);

  pdl_launch_dependents();
  pdl_wait();
  for (int b = blockIdx.y; b < a.B; b += gridDim.y) {
    int page = a.index ? __ldg(a.index + b) : b;
    const bool outside = page >= a.pages;
    if (outside) page = -1;

    float4 s[kRows];
    const int64_t in = static_cast<int64_t>(h) * DK * a.dv + vb * BV + cg * 4;
    const float* src = a.state_in + page * a.state_in_sp + in;
    if (page >= 0) {
#pragma unroll
      for (int i = 0; i < kRows; ++i)
        s[i] = __ldcs(reinterpret_cast<const float4*>(src + static_cast<int64_t>(rg + i * kRowGroups) * a.dv));
    }
    const IO* q = static_cast<const IO*>(a.q) + b * a.q_sb + hq * a.q_sh;
    const IO* k = static_cast<const IO*>(a.k) + b * a.k_sb + hq * a.k_sh;
    for (int i = tid; i < DK; i += kThreads) {
      s_k[i] = to_f32(k[i]);
      s_q[i] = to_f32(q[i]);
    }
    // a page that an earlier row holds belongs to that row
    bool taken = false;
    if (a.index && page >= 0)
      for (int j = tid; j < b; j += kThreads) taken |= __ldg(a.index + j) == page;
    taken = __syncthreads_or(taken);

    const int64_t oo = b * a.o_sb + h * a.o_sh + vb * BV + cg * 4;
    if (page < 0 || taken) {
      if ((outside || taken) && blockIdx.x == 0 && tid == 0) report(a.status, GDN_DEVERR_BAD_INDEX);
      if (rg == 0) *reinterpret_cast<uint2*>(static_cast<IO*>(a.o) + oo) = make_uint2(0, 0);
      __syncthreads();
      continue;
    }
    const float g = load_any(a.g, b * a.g_sb + h * a.g_sh, a.g_dtype);
    const float alpha = a.gate_kind == GDN_GATE_LOG ? __expf(g) : g;
    const uint2 vw = __ldg(reinterpret_cast<const uint2*>(static_cast<const IO*>(a.v) + b * a.v_sb + h * a.v_sh +
                                                          vb * BV + cg * 4));
    const IO* vi = reinterpret_cast<const IO*>(&vw);
    const float4 v = make_float4(to_f32(vi[0]), to_f32(vi[1]), to_f32(vi[2]), to_f32(vi[3]));

    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float* dst = a.state_out + page * a.state_out_sp + in;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int row = rg + i * kRowGroups;
      const float kr = s_k[row], qr = s_q[row];
      float4 x = s[i];
      x.x = fmaf(alpha, x.x, kr * v.x);
      x.y = fmaf(alpha, x.y, kr * v.y);
      x.z = fmaf(alpha, x.z, kr * v.z);
      x.w = fmaf(alpha, x.w, kr * v.w);
      o.x = fmaf(qr, x.x, o.x);
      o.y = fmaf(qr, x.y, o.y);
      o.z = fmaf(qr, x.z, o.z);
      o.w = fmaf(qr, x.w, o.w);
      stg128(dst + static_cast<int64_t>(row) * a.dv, x);
    }
#pragma unroll
    for (int off = kColGroups; off < 32; off <<= 1) {
      o.x += __shfl_xor_sync(0xffffffffu, o.x, off);
      o.y += __shfl_xor_sync(0xffffffffu, o.y, off);
      o.z += __shfl_xor_sync(0xffffffffu, o.z, off);
      o.w += __shfl_xor_sync(0xffffffffu, o.w, off);
    }
    if (lane < kColGroups) *reinterpret_cast<float4*>(&s_red[warp][cg * 4]) = o;
    __syncthreads();
    if (tid < kColGroups) {
      o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float4 x = *reinterpret_cast<const float4*>(&s_red[w][tid * 4]);
        o.x += x.x; o.y += x.y; o.z += x.z; o.w += x.w;
      }
      IO ov[4] = {from_f32<IO>(a.scale * o.x), from_f32<IO>(a.scale * o.y), from_f32<IO>(a.scale * o.z),
                  from_f32<IO>(a.scale * o.w)};
      *reinterpret_cast<uint2*>(static_cast<IO*>(a.o) + oo) = *reinterpret_cast<const uint2*>(ov);
    }
  }
}

template <int DK, int BV, typename IO>
int launch(const lin_decode_args_t& a, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>(a.Hv * (a.dv / BV)), static_cast<unsigned>(a.B < 65535 ? a.B : 65535));
  return launch_pdl(lin_decode_kernel<DK, BV, IO>, grid, kThreads, 0, stream, a);
}

// The widest slab (at most 128 columns, and 128 registers of state a thread)
// that leaves four CTAs for each SM; at B = 8, H = 32, d = 128 (256 slabs of 128
// columns) 32 columns take 5.4 us, 64 5.7 and 128 5.8, at B = 64 47.4, 45.4 and 44.4.
int pick_cols(const lin_decode_args_t& a, int sms) {
  int cols = a.dk < 256 && a.dv % 128 == 0 ? 128 : 64;
  while (cols > 32 && static_cast<int64_t>(a.B) * a.Hv * (a.dv / cols) < 4 * static_cast<int64_t>(sms)) cols /= 2;
  return cols;
}

template <int DK, typename IO>
int dispatch_cols(const lin_decode_args_t& a, int cols, cudaStream_t stream) {
  if constexpr (DK < 256)
    if (cols == 128) return launch<DK, 128, IO>(a, stream);
  return cols == 64 ? launch<DK, 64, IO>(a, stream) : launch<DK, 32, IO>(a, stream);
}

template <typename IO>
int dispatch(const lin_decode_args_t& a, int sms, cudaStream_t stream) {
  const int cols = pick_cols(a, sms);
  if (a.dk == 64) return dispatch_cols<64, IO>(a, cols, stream);
  if (a.dk == 128) return dispatch_cols<128, IO>(a, cols, stream);
  return dispatch_cols<256, IO>(a, cols, stream);
}

int validate(const lin_decode_args_t* a) {
  if (!a) return GDN_ERR_NULL;
  if (!a->q || !a->k || !a->v || !a->g || !a->state_in || !a->state_out || !a->o) return GDN_ERR_NULL;
  if (a->B < 1 || a->Hqk < 1 || a->Hv < 1 || a->Hv % a->Hqk) return GDN_ERR_SHAPE;
  if (a->pages < 1 || (!a->index && a->pages < a->B)) return GDN_ERR_SHAPE;
  if (a->dk != 64 && a->dk != 128 && a->dk != 256) return GDN_ERR_SHAPE;
  if (a->dv < 64 || a->dv % 64) return GDN_ERR_SHAPE;
  const int64_t page = static_cast<int64_t>(a->Hv) * a->dk * a->dv;
  // the stride of an axis of one is free
  const bool rows = a->B > 1, many = a->pages > 1;
  if (page > INT32_MAX || (many && (a->state_in_sp < page || a->state_out_sp < page))) return GDN_ERR_SHAPE;
  if (a->io_dtype != GDN_DT_BF16 && a->io_dtype != GDN_DT_F16) return GDN_ERR_DTYPE;
  if (!dtype_valid(a->g_dtype)) return GDN_ERR_DTYPE;
  if (a->gate_kind != GDN_GATE_LOG && a->gate_kind != GDN_GATE_LINEAR) return GDN_ERR_DTYPE;
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->o) || !aligned16(a->state_in) ||
      !aligned16(a->state_out))
    return GDN_ERR_ALIGN;
  if (rows && (!stride_ok(a->q_sb, 2) || !stride_ok(a->k_sb, 2) || !stride_ok(a->v_sb, 2) || !stride_ok(a->o_sb, 2)))
    return GDN_ERR_ALIGN;
  if (a->Hqk > 1 && (!stride_ok(a->q_sh, 2) || !stride_ok(a->k_sh, 2))) return GDN_ERR_ALIGN;
  if (a->Hv > 1 && (!stride_ok(a->v_sh, 2) || !stride_ok(a->o_sh, 2))) return GDN_ERR_ALIGN;
  if (many && (!stride_ok(a->state_in_sp, 4) || !stride_ok(a->state_out_sp, 4))) return GDN_ERR_ALIGN;
  if ((rows && a->o_sb == 0) || (a->Hv > 1 && a->o_sh == 0)) return GDN_ERR_SHAPE;  // rows of o on one another
  if (a->state_in != a->state_out) {
    if (!pools_disjoint(a->state_in, a->state_in_sp, a->state_out, a->state_out_sp, page, a->pages)) return GDN_ERR_SHAPE;
  } else if (many && a->state_in_sp != a->state_out_sp) {
    return GDN_ERR_SHAPE;
  }
  return GDN_OK;
}

}  // namespace
}  // namespace gdn

extern "C" int lin_decode_launch(const lin_decode_args_t* args, gdn_stream_t stream) {
  int rc = gdn::validate(args);
  if (rc) return rc;
  gdn::DeviceInfo di;
  rc = gdn::device_info(&di);
  if (rc) return rc;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return args->io_dtype == GDN_DT_BF16 ? gdn::dispatch<__nv_bfloat16>(*args, di.sm_count, st)
                                            : gdn::dispatch<__half>(*args, di.sm_count, st);
}
