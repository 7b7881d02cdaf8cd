// lin_prefill.cu — linear attention with a decay per head over T tokens, in
// chunks of C = 128 on the tcgen05 tensor cores.
//
// With G the cumulative log gate inside a chunk and S the state before it:
//
//   P_ij = scale (q_i . k_j) e^(G_i - G_j)   (j <= i)
//   O    = (scale diag(e^G) Q) S + P V
//   S'   = e^(G_C) S + K^T diag(e^(G_C - G_j)) V
//
// Unlike the delta rule the state's increment does not depend on the state, so
// the only serial step from chunk to chunk is S' = gamma S + dS in registers;
// everything else pipelines.  One CTA takes one sequence, value head and block
// of BV value columns (columns are independent) through all its chunks, so q,
// k, v and o cross HBM once and the state stays on chip.  Per chunk of d = 128
// that is 128 KB against five 128^3 products.
//
// Warps (19): R 0-3 (a row of the chunk per thread), V 4-7, S 8-15, TMA 16,
// gates 17, MMA 18.  Per chunk, in the MMA warp's order:
//   SC  scores = Q K^T             both from shared memory; R turns them into
//                                  P, packed over the scores' own columns
//   LO  dS^T  = V''lo^T K          A from TMEM
//   QS  O     = Q' S               Q' = scale e^G Q in TMEM (R), S^T in shared memory
//   HI  dS^T += V''hi^T K          then S reads dS and rewrites S^T
//   PV  O    += P V                then V packs O into the Q tile and stores it
// V'' = e^(G_C - G_j) v is split into two parts of the I/O type, v'' = hi + lo,
// because the state is kept to fp32 accuracy: one 8-bit part would leave 2^-9
// of every term.  V writes both parts in turn to the same 64 columns, while the
// tensor cores are at SC and QS.
#include <cuda_runtime.h>

#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "tc.cuh"

namespace gdn {
namespace {

constexpr int kC = 128;             // tokens of a chunk
constexpr int kTile = kC * 128;     // bytes of a [128][64] 16-bit tile
constexpr int kThreads = 19 * 32;
constexpr int kWarpV = 4, kWarpS = 8, kWarpTma = 16, kWarpGate = 17, kWarpMma = 18;
constexpr float kLog2e = 1.4426950408889634f;
// log2 gates are cut off here: 2^-160 is zero in fp32, and cumulative sums stay finite
constexpr float kLowest = -160.f;

// TMEM columns
constexpr uint32_t kTmSC = 0;     // scores fp32 [128]; P over its first 64 columns
constexpr uint32_t kTmQ = 128;    // Q' bf16 [DK / 2]
constexpr uint32_t kTmV = 192;    // V'' [64]
constexpr uint32_t kTmO = 256;    // O fp32 [BV]
constexpr uint32_t kTmDS = 384;   // dS^T fp32 [DK]

template <int DK, int BV>
struct Layout {
  static constexpr int kQ = 0;
  static constexpr int kK = kQ + DK / 64 * kTile;
  static constexpr int kV = kK + DK / 64 * kTile;
  static constexpr int kStage = kV + BV / 64 * kTile;
  static constexpr int kStages = 2;
  static constexpr int kS = kStages * kStage;              // S^T bf16 [BV][DK], 64-wide blocks
  static constexpr int kSBlock = BV * 128;
  // O is staged in the chunk's Q tile where it fits
  static constexpr bool kOInQ = BV <= DK;
  static constexpr int kO = kS + DK / 64 * kSBlock;
  static constexpr int kGate = kO + (kOInQ ? 0 : BV / 64 * kTile);
  static constexpr int kGateStage = 2 * kC * 4;            // G, w
  static constexpr int kBars = kGate + 2 * kGateStage;
  static constexpr int kBytes = kBars + 256;
  static_assert(kBytes <= 232448, "shared memory");
};

struct Bars {
  uint64_t full[2], empty_kv[2], empty_q[2];
  uint64_t gfull[2], gempty[2];
  uint64_t sc_done, q_ready, p_ready, pv_done;
  uint64_t v_ready, v_free, o_free, ds_done, s_ready, drain;
  float gamma[2];
  uint32_t tmem;
  uint32_t pad;
};
static_assert(sizeof(Bars) <= 256, "barriers");

struct PrefillParams {
  lin_prefill_args_t a;
  int nvb;
};

// Where sequence n lies: first row, tokens, page (-1: none).
struct Seq {
  int start, len, page;
};

// Every thread of the CTA calls it.  Offsets out of range or descending give a
// sequence of -1 tokens; a page out of range or held by an earlier sequence none.
__device__ Seq find_seq(const lin_prefill_args_t& a, int n, bool reporter) {
  Seq s;
  s.start = 0;
  s.len = a.T;
  bool bad = false;
  if (a.cu_seqlens) {
    const int lo = a.cu_seqlens[n], hi = a.cu_seqlens[n + 1];
    bad = !(lo >= 0 && lo <= hi && hi <= a.T);
    s.start = lo;
    s.len = bad ? -1 : hi - lo;
  }
  s.page = a.index ? a.index[n] : n;
  bool taken = s.page >= a.pages;
  if (a.index && s.page >= 0)
    for (int j = threadIdx.x; j < n; j += blockDim.x) taken |= a.index[j] == s.page;
  if (__syncthreads_or(taken)) {
    bad = true;
    s.page = -1;
  }
  if (bad && reporter) report(a.status, GDN_DEVERR_BAD_INDEX);
  return s;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The log gate in powers of two, cut off below (a NaN stays one).
__device__ __forceinline__ float log2_gate(float g) {
  const float x = g * kLog2e;
  return x < kLowest ? kLowest : x;
}

// Waits for a phase; on a timeout reports `bits` and returns false.  For one
// thread; wait() is for a whole warp, whose lanes all get the same answer.
__device__ __forceinline__ bool wait1(uint64_t* bar, uint32_t parity, uint32_t* status, uint32_t bits) {
  if (mbar_wait_bounded(bar, parity)) return true;
  report(status, bits);
  return false;
}
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, uint32_t* status, uint32_t bits) {
  const bool ok = mbar_wait_bounded(bar, parity);
  if (__all_sync(0xffffffffu, ok)) return true;
  report(status, bits);
  return false;
}

template <int DK, int BV, typename IO>
__global__ void __launch_bounds__(kThreads, 1)
    lin_prefill_kernel(const __grid_constant__ PrefillParams p, const __grid_constant__ CUtensorMap map_q,
                       const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                       const __grid_constant__ CUtensorMap map_o) {
  using L = Layout<DK, BV>;
  constexpr bool BF16 = sizeof(IO) == 2 && std::is_same<IO, __nv_bfloat16>::value;
  extern __shared__ __align__(1024) unsigned char smem[];
  Bars& bar = *reinterpret_cast<Bars*>(smem + L::kBars);
  const lin_prefill_args_t& a = p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int h = blockIdx.x / p.nvb, vb = blockIdx.x - h * p.nvb, hq = h / (a.Hv / a.Hqk);
  const int n = blockIdx.y;
  const int batch = a.cu_seqlens ? 0 : n;

  if (warp == kWarpMma) tc::tmem_alloc(&bar.tmem, 512);
  if (tid == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bar.full[s], 1);
      mbar_init(&bar.empty_kv[s], 1);
      mbar_init(&bar.empty_q[s], 1);
      mbar_init(&bar.gfull[s], 1);
      mbar_init(&bar.gempty[s], 16);
    }
    mbar_init(&bar.sc_done, 1);
    mbar_init(&bar.q_ready, 4);
    mbar_init(&bar.p_ready, 4);
    mbar_init(&bar.pv_done, 1);
    mbar_init(&bar.v_ready, 4);
    mbar_init(&bar.v_free, 1);
    mbar_init(&bar.o_free, 4);
    mbar_init(&bar.ds_done, 1);
    mbar_init(&bar.s_ready, 8);
    mbar_init(&bar.drain, 1);
    fence_mbar_init();
  }
  pdl_launch_dependents();
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  pdl_wait();
  const Seq seq = find_seq(a, n, blockIdx.x == 0 && tid == 0);
  const int chunks = seq.len > 0 ? (seq.len + kC - 1) / kC : 0;
  const uint32_t tmem = bar.tmem;
  const uint32_t sb = smem_u32(smem);
  uint32_t* const status = a.status;

  if (warp < kWarpV) {
    // ------------------------------------------------ R: a row per thread
    const int row = tid;
    const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
    for (int c = 0; c < chunks; ++c) {
      const int st = c & 1;
      const uint32_t ph = (c >> 1) & 1;
      const unsigned char* stage = smem + st * L::kStage;
      const float* G = reinterpret_cast<const float*>(smem + L::kGate + st * L::kGateStage);
      if (!wait(&bar.gfull[st], ph, status, GDN_DEVERR_FULL_TIMEOUT)) break;
      if (!wait(&bar.full[st], ph, status, GDN_DEVERR_FULL_TIMEOUT)) break;
      // Q' = scale e^G Q over the columns that the last chunk's QS has read
      if (c && !wait(&bar.pv_done, (c - 1) & 1, status, GDN_DEVERR_MMA_TIMEOUT)) break;
      tc::fence_after_sync();
      const float Gi = G[row];
      const float f = a.scale * ex2(Gi);
#pragma unroll
      for (int b = 0; b < DK / 32; ++b) {
        uint32_t u[16];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int chunk = (b & 1) * 4 + e;
          const uint4 x = *reinterpret_cast<const uint4*>(stage + L::kQ + (b >> 1) * kTile + tc::sw128_offset(row, chunk));
          const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int i = 0; i < 4; ++i)
            u[e * 4 + i] = tc::pack2<true>(f * tc::unpack_lo<BF16>(w[i]), f * tc::unpack_hi<BF16>(w[i]));
        }
        tc::tmem_st16(tmem + lanes + kTmQ + b * 16, u);
      }
      tc::tmem_wait_st();
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.q_ready);

      if (!wait(&bar.sc_done, c & 1, status, GDN_DEVERR_MMA_TIMEOUT)) break;
      tc::fence_after_sync();
      // P in the I/O type over the scores: columns [16 b, 16 b + 16) go to [8 b, 8 b + 8)
#pragma unroll
      for (int b = 0; b < 8; ++b) {
        uint32_t u[8];
        if (b * 16 < warp * 32 + 32) {
          float s[16];
          tc::tmem_ld16(tmem + lanes + kTmSC + b * 16, s);
          float d[16];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float4 g = *reinterpret_cast<const float4*>(G + b * 16 + e * 4);
            d[e * 4 + 0] = a.scale * ex2(Gi - g.x);
            d[e * 4 + 1] = a.scale * ex2(Gi - g.y);
            d[e * 4 + 2] = a.scale * ex2(Gi - g.z);
            d[e * 4 + 3] = a.scale * ex2(Gi - g.w);
          }
          tc::tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e) s[e] = b * 16 + e <= row ? s[e] * d[e] : 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) u[e] = tc::pack2<BF16>(s[2 * e], s[2 * e + 1]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) u[e] = 0;
        }
        tc::tmem_st8(tmem + lanes + kTmSC + b * 8, u);
      }
      tc::tmem_wait_st();
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&bar.p_ready);
        mbar_arrive(&bar.gempty[st]);
      }
    }
  } else if (warp < kWarpS) {
    // ------------------------------------------------ V: V'' parts, and the output rows
    const int vt = tid - kWarpV * 32, quarter = warp - kWarpV;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const bool has_rows = quarter * 32 < BV;
    // A warp whose wait ran out keeps to the group's barriers until output(),
    // where the group agrees to stop.
    bool ok = true, stop = false;
    // part 0: lo, part 1: hi
    const auto parts = [&](int c, int part) {
      const int st = c & 1;
      const uint32_t tile = sb + st * L::kStage + L::kV;
      const float* w = reinterpret_cast<const float*>(smem + L::kGate + st * L::kGateStage) + kC;
      if (has_rows) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int dv = quarter * 32 + half * 16;  // of this warp's 16 rows
          const uint32_t block = tile + (dv >> 6) * kTile;
          const int chunk = ((dv & 63) >> 3) + ((lane >> 3) & 1);
#pragma unroll
          for (int t0 = 0; t0 < kC; t0 += 64) {
            uint32_t u[16];
#pragma unroll
            for (int tb = 0; tb < 4; ++tb) {
              const int t = t0 + tb * 16;
              uint32_t r[4];
              tc::ldsm_x4_trans(block + tc::sw128_offset(t + (lane >> 4) * 8 + (lane & 7), chunk), r);
              const float2 w0 = *reinterpret_cast<const float2*>(w + t + 2 * (lane & 3));
              const float2 w1 = *reinterpret_cast<const float2*>(w + t + 8 + 2 * (lane & 3));
#pragma unroll
              for (int m = 0; m < 4; ++m) {
                const float2 ww = m < 2 ? w0 : w1;
                const float x = ww.x * tc::unpack_lo<BF16>(r[m]), y = ww.y * tc::unpack_hi<BF16>(r[m]);
                uint32_t z = tc::pack2<BF16>(x, y);
                if (part == 0)  // what the leading part leaves, exact in fp32
                  z = tc::pack2<BF16>(x - tc::unpack_lo<BF16>(z), y - tc::unpack_hi<BF16>(z));
                u[tb * 4 + m] = z;
              }
            }
            tc::tmem_st_16x128b_x8(tmem + lanes + (static_cast<uint32_t>(half * 16) << 16) + kTmV + t0 / 2, u);
          }
        }
        tc::tmem_wait_st();
      }
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.v_ready);
    };
    // O of chunk c: packed into shared memory, then out
    const auto output = [&](int c) {
      const int st = c & 1;
      unsigned char* o = smem + (L::kOInQ ? st * L::kStage + L::kQ : L::kO);
      ok = ok && wait(&bar.pv_done, c & 1, status, GDN_DEVERR_MMA_TIMEOUT);
      stop = named_barrier_or(1, 128, !ok);
      if (stop) return;
      tc::fence_after_sync();
      if (!L::kOInQ && c) {  // the last store has read the tile
        if (vt == 0) bulk_wait_read();
        tc::group_sync(1, 128);
      }
#pragma unroll
      for (int b = 0; b < BV / 16; ++b) {
        float x[16];
        tc::tmem_ld16(tmem + lanes + kTmO + b * 16, x);
        tc::tmem_wait_ld();
        const uint32_t at = smem_u32(o) + (b >> 2) * kTile;
#pragma unroll
        for (int e = 0; e < 2; ++e)
          tc::sts128(at + tc::sw128_offset(vt, (b & 3) * 2 + e), tc::pack2<BF16>(x[8 * e], x[8 * e + 1]),
                     tc::pack2<BF16>(x[8 * e + 2], x[8 * e + 3]), tc::pack2<BF16>(x[8 * e + 4], x[8 * e + 5]),
                     tc::pack2<BF16>(x[8 * e + 6], x[8 * e + 7]));
      }
      tc::fence_before_sync();
      tc::fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.o_free);
      tc::group_sync(1, 128);
      const int rows = min(kC, seq.len - c * kC);
      if (rows == kC) {
        if (vt == 0) {
          for (int b = 0; b < BV / 64; ++b)
            tc::tma_store_4d(&map_o, o + b * kTile, vb * BV + b * 64, h, seq.start + c * kC, batch);
          bulk_commit();
          if (L::kOInQ) {
            bulk_wait_read();
            mbar_arrive(&bar.empty_q[st]);
          }
        }
      } else {  // the rows behind belong to another sequence, or to nobody
        IO* dst = static_cast<IO*>(a.o) + batch * a.o_sb + static_cast<int64_t>(seq.start + c * kC) * a.o_st + h * a.o_sh +
                  vb * BV;
        constexpr int kPer = BV / 8;  // 16-byte pieces of a row
        for (int i = vt; i < rows * kPer; i += 128) {
          const int r = i / kPer, piece = i - r * kPer;
          const uint4 x = *reinterpret_cast<const uint4*>(o + (piece >> 3) * kTile + tc::sw128_offset(r, piece & 7));
          *reinterpret_cast<uint4*>(dst + r * a.o_st + piece * 8) = x;
        }
      }
      if (!L::kOInQ && vt == 0) mbar_arrive(&bar.empty_q[st]);
    };
    for (int c = 0; c < chunks && !stop; ++c) {
      const int st = c & 1;
      const uint32_t ph = (c >> 1) & 1;
      ok = ok && wait(&bar.gfull[st], ph, status, GDN_DEVERR_FULL_TIMEOUT) &&
           wait(&bar.full[st], ph, status, GDN_DEVERR_FULL_TIMEOUT);
      const int rows = min(kC, seq.len - c * kC);
      if (rows < kC) {
        // rows of the next sequence, or outside: zero, whatever they hold, since
        // 0 x NaN would reach the sums over the chunk's tokens
        unsigned char* stage = smem + st * L::kStage;
        if (ok)
          for (int r = rows + quarter; r < kC; r += 4)
            for (int i = lane; i < (DK + BV) / 8; i += 32)
              *reinterpret_cast<uint4*>(stage + L::kK + (i >> 3) * kTile + tc::sw128_offset(r, i & 7)) = make_uint4(0, 0, 0, 0);
        tc::fence_proxy_async();
        tc::group_sync(1, 128);
      }
      ok = ok && (c == 0 || wait(&bar.v_free, 1, status, GDN_DEVERR_MMA_TIMEOUT));
      tc::fence_after_sync();
      if (ok) parts(c, 0);
      if (c) output(c - 1);
      ok = ok && wait(&bar.v_free, 0, status, GDN_DEVERR_MMA_TIMEOUT);
      tc::fence_after_sync();
      if (ok) parts(c, 1);
      if (lane == 0) mbar_arrive(&bar.gempty[st]);
    }
    if (chunks && !stop) output(chunks - 1);
    if (vt == 0) bulk_wait_all();
  } else if (warp < kWarpTma) {
    // ------------------------------------------------ S: the state, a value column per thread
    const int quarter = warp & 3, half = (warp - kWarpS) >> 2;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const int row = quarter * 32 + lane;  // value column of this CTA's block
    const bool has_rows = quarter * 32 < BV;
    constexpr int kN = DK / 2;            // d_k entries of this thread
    const int64_t at = (static_cast<int64_t>(h) * DK + half * kN) * a.dv + vb * BV + row;
    float S[kN];
    const bool load = has_rows && seq.page >= 0 && a.initial_state && seq.len >= 0;
    const float* from = a.initial_state + (load ? seq.page * a.initial_sp + at : 0);
#pragma unroll
    for (int i = 0; i < kN; ++i) S[i] = load ? from[static_cast<int64_t>(i) * a.dv] : 0.f;
    const auto publish = [&]() {  // S^T rounded to bf16, the QS product's operand
      if (has_rows) {
#pragma unroll
        for (int i = 0; i < kN / 8; ++i) {
          const int piece = half * (kN / 8) + i;
          tc::sts128(sb + L::kS + (piece >> 3) * L::kSBlock + tc::sw128_offset(row, piece & 7),
                     tc::pack2<true>(S[8 * i], S[8 * i + 1]), tc::pack2<true>(S[8 * i + 2], S[8 * i + 3]),
                     tc::pack2<true>(S[8 * i + 4], S[8 * i + 5]), tc::pack2<true>(S[8 * i + 6], S[8 * i + 7]));
        }
      }
      tc::fence_before_sync();
      tc::fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.s_ready);
    };
    publish();
    bool ok = true;
    for (int c = 0; c < chunks; ++c) {
      const int st = c & 1;
      ok = wait(&bar.gfull[st], (c >> 1) & 1, status, GDN_DEVERR_FULL_TIMEOUT) &&
           wait(&bar.ds_done, c & 1, status, GDN_DEVERR_MMA_TIMEOUT);
      if (!ok) break;
      tc::fence_after_sync();
      const float gamma = bar.gamma[st];
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.gempty[st]);
      if (has_rows) {
#pragma unroll
        for (int b = 0; b < kN / 16; ++b) {
          float d[16];
          tc::tmem_ld16(tmem + lanes + kTmDS + half * kN + b * 16, d);
          tc::tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e) S[b * 16 + e] = fmaf(gamma, S[b * 16 + e], d[e]);
        }
      }
      publish();
    }
    if (ok && has_rows && seq.page >= 0 && seq.len >= 0) {
      float* to = a.final_state + seq.page * a.final_sp + at;
#pragma unroll
      for (int i = 0; i < kN; ++i) to[static_cast<int64_t>(i) * a.dv] = S[i];
    }
  } else if (warp == kWarpTma) {
    if (lane == 0) {
      int c = 0;
      for (; c < chunks; ++c) {
        const int st = c & 1;
        unsigned char* stage = smem + st * L::kStage;
        const int t = seq.start + c * kC;
        if (c >= 2 && !wait1(&bar.empty_kv[st], ((c >> 1) & 1) ^ 1, status, GDN_DEVERR_EMPTY_TIMEOUT)) break;
        mbar_arrive_expect_tx(&bar.full[st], L::kStage);
        for (int b = 0; b < DK / 64; ++b) tc::tma_load_4d(stage + L::kK + b * kTile, &map_k, b * 64, hq, t, batch, &bar.full[st]);
        for (int b = 0; b < BV / 64; ++b)
          tc::tma_load_4d(stage + L::kV + b * kTile, &map_v, vb * BV + b * 64, h, t, batch, &bar.full[st]);
        if (c >= 2 && !wait1(&bar.empty_q[st], ((c >> 1) & 1) ^ 1, status, GDN_DEVERR_EMPTY_TIMEOUT)) {
          // give the rest of the stage up, so that the drain below ends on what was issued
          asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(&bar.full[st])),
                       "r"(static_cast<uint32_t>(L::kK))
                       : "memory");
          ++c;
          break;
        }
        for (int b = 0; b < DK / 64; ++b) tc::tma_load_4d(stage + L::kQ + b * kTile, &map_q, b * 64, hq, t, batch, &bar.full[st]);
      }
      // no copy may be in flight when the shared memory is released
      for (int j = max(0, c - 2); j < c; ++j)
        if (!wait1(&bar.full[j & 1], (j >> 1) & 1, status, GDN_DEVERR_DRAIN_TIMEOUT)) break;
    }
  } else if (warp == kWarpGate) {
    // ------------------------------------------------ gates: 4 tokens per lane
    const int64_t g0 = batch * a.g_sb + h * a.g_sh;
    const auto fetch = [&](int c, float (&x)[4]) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int t = c * kC + lane * 4 + e;
        x[e] = t < seq.len ? load_any(a.g, g0 + static_cast<int64_t>(seq.start + t) * a.g_st, a.g_dtype) : 0.f;
      }
    };
    float x[4];
    if (chunks) fetch(0, x);
    for (int c = 0; c < chunks; ++c) {
      const int st = c & 1;
      float* G = reinterpret_cast<float*>(smem + L::kGate + st * L::kGateStage);
      // cumulative in fp64: differences of far sums keep their small part
      double s[4];
      s[0] = log2_gate(x[0]);
#pragma unroll
      for (int e = 1; e < 4; ++e) s[e] = s[e - 1] + static_cast<double>(log2_gate(x[e]));
      double inc = s[3];
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, inc, off);
        if (lane >= off) inc += y;
      }
      const double before = inc - s[3], end = __shfl_sync(0xffffffffu, inc, 31);
      if (c + 1 < chunks) fetch(c + 1, x);
      if (c >= 2 && !wait(&bar.gempty[st], ((c >> 1) & 1) ^ 1, status, GDN_DEVERR_EMPTY_TIMEOUT)) break;
      float4 gv, wv;
      float* gp = &gv.x;
      float* wp = &wv.x;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const double Gt = before + s[e];
        gp[e] = static_cast<float>(Gt);
        wp[e] = c * kC + lane * 4 + e < seq.len ? exp2f(static_cast<float>(end - Gt)) : 0.f;
      }
      *reinterpret_cast<float4*>(G + lane * 4) = gv;
      *reinterpret_cast<float4*>(G + kC + lane * 4) = wv;
      if (lane == 0) bar.gamma[st] = exp2f(static_cast<float>(end));
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.gfull[st]);
    }
  } else if (lane == 0) {
    // ------------------------------------------------ MMA
    constexpr uint32_t kIdSC = tc::idesc_f16(128, kC, false, false, BF16);
    constexpr uint32_t kIdDS = tc::idesc_f16(128, DK, false, true, BF16);
    constexpr uint32_t kIdQS = tc::idesc_f16(128, BV, false, false, true);
    constexpr uint32_t kIdPV = tc::idesc_f16(128, BV, false, true, BF16);
    bool ok = true;
    for (int c = 0; c < chunks; ++c) {
      const int st = c & 1;
      const uint32_t q = sb + st * L::kStage + L::kQ, k = sb + st * L::kStage + L::kK, v = sb + st * L::kStage + L::kV;
      const auto add_ds = [&](bool first) {
#pragma unroll
        for (int s = 0; s < kC / 16; ++s)
          tc::mma_tmem_a(tmem + kTmDS, tmem + kTmV + s * 8, tc::mnmajor_desc(k, kTile, s), kIdDS, !first || s > 0);
      };
      ok = wait1(&bar.full[st], (c >> 1) & 1, status, GDN_DEVERR_FULL_TIMEOUT) &&
           (c == 0 || wait1(&bar.pv_done, (c - 1) & 1, status, GDN_DEVERR_MMA_TIMEOUT));
      if (!ok) break;
      tc::fence_after_sync();
#pragma unroll
      for (int s = 0; s < DK / 16; ++s)
        tc::mma(tmem + kTmSC, tc::kmajor_desc(q, kTile, s), tc::kmajor_desc(k, kTile, s), kIdSC, s > 0);
      tc::commit(&bar.sc_done);

      ok = wait1(&bar.s_ready, c & 1, status, GDN_DEVERR_MMA_TIMEOUT) &&
           wait1(&bar.v_ready, 0, status, GDN_DEVERR_MMA_TIMEOUT);
      if (!ok) break;
      tc::fence_after_sync();
      add_ds(true);
      tc::commit(&bar.v_free);

      ok = wait1(&bar.q_ready, c & 1, status, GDN_DEVERR_MMA_TIMEOUT) &&
           (c == 0 || wait1(&bar.o_free, (c - 1) & 1, status, GDN_DEVERR_MMA_TIMEOUT));
      if (!ok) break;
      tc::fence_after_sync();
#pragma unroll
      for (int s = 0; s < DK / 16; ++s)
        tc::mma_tmem_a(tmem + kTmO, tmem + kTmQ + s * 8, tc::kmajor_desc(sb + L::kS, L::kSBlock, s), kIdQS, s > 0);

      ok = wait1(&bar.v_ready, 1, status, GDN_DEVERR_MMA_TIMEOUT);
      if (!ok) break;
      tc::fence_after_sync();
      add_ds(false);
      tc::commit(&bar.v_free);
      tc::commit(&bar.ds_done);

      ok = wait1(&bar.p_ready, c & 1, status, GDN_DEVERR_MMA_TIMEOUT);
      if (!ok) break;
      tc::fence_after_sync();
#pragma unroll
      for (int s = 0; s < kC / 16; ++s)
        tc::mma_tmem_a(tmem + kTmO, tmem + kTmSC + s * 8, tc::mnmajor_desc(v, kTile, s), kIdPV, true);
      tc::commit(&bar.pv_done);
      tc::commit(&bar.empty_kv[st]);
    }
    if (!ok) {  // products in flight end before the tensor memory is released
      tc::commit(&bar.drain);
      wait1(&bar.drain, 0, status, GDN_DEVERR_DRAIN_TIMEOUT);
    }
  }
  __syncwarp();
  tc::fence_before_sync();
  __syncthreads();
  if (warp == kWarpMma) tc::tmem_dealloc(tmem, 512);
}

int io_map(CUtensorMap* m, bool bf16, const void* base, int d, int heads, int T, int B, int64_t sh, int64_t st, int64_t sb) {
  const uint64_t dims[4] = {static_cast<uint64_t>(d), static_cast<uint64_t>(heads), static_cast<uint64_t>(T),
                            static_cast<uint64_t>(B)};
  // the stride of an axis of one is free
  const uint64_t strides[3] = {static_cast<uint64_t>(heads > 1 ? sh : d) * 2, static_cast<uint64_t>(T > 1 ? st : d) * 2,
                               static_cast<uint64_t>(B > 1 ? sb : d) * 2};
  const uint32_t box[4] = {64, 1, kC, 1};
  return tensor_map(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, base, dims, strides,
                    box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int DK, int BV, typename IO>
int launch(const lin_prefill_args_t& a, cudaStream_t stream) {
  constexpr bool bf = std::is_same<IO, __nv_bfloat16>::value;
  using L = Layout<DK, BV>;
  static std::atomic<uint64_t> attr_done{0};
  PrefillParams p;
  p.a = a;
  p.nvb = a.dv / BV;
  const int B = a.cu_seqlens ? 1 : a.B;
  CUtensorMap mq, mk, mv, mo;
  int rc;
  if ((rc = io_map(&mq, bf, a.q, DK, a.Hqk, a.T, B, a.q_sh, a.q_st, a.q_sb)) ||
      (rc = io_map(&mk, bf, a.k, DK, a.Hqk, a.T, B, a.k_sh, a.k_st, a.k_sb)) ||
      (rc = io_map(&mv, bf, a.v, a.dv, a.Hv, a.T, B, a.v_sh, a.v_st, a.v_sb)) ||
      (rc = io_map(&mo, bf, a.o, a.dv, a.Hv, a.T, B, a.o_sh, a.o_st, a.o_sb)))
    return rc;
  auto kern = lin_prefill_kernel<DK, BV, IO>;
  if ((rc = ensure_smem_attr(kern, L::kBytes, attr_done))) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.Hv * p.nvb), static_cast<unsigned>(a.B));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = L::kBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kern, p, mq, mk, mv, mo) != cudaSuccess) {
    (void)cudaGetLastError();
    return GDN_ERR_LAUNCH;
  }
  return GDN_OK;
}

template <typename IO>
int dispatch(const lin_prefill_args_t& a, cudaStream_t stream) {
  const bool wide = a.dv % 128 == 0;
  if (a.dk == 64) return wide ? launch<64, 128, IO>(a, stream) : launch<64, 64, IO>(a, stream);
  return wide ? launch<128, 128, IO>(a, stream) : launch<128, 64, IO>(a, stream);
}

int validate(const lin_prefill_args_t* a) {
  if (!a) return GDN_ERR_NULL;
  if (!a->q || !a->k || !a->v || !a->g || !a->final_state || !a->o) return GDN_ERR_NULL;
  if (a->B < 1 || a->B > 65535 || a->T < 1 || a->Hqk < 1 || a->Hv < 1 || a->Hv % a->Hqk) return GDN_ERR_SHAPE;
  if (a->pages < 1 || (!a->index && a->pages < a->B)) return GDN_ERR_SHAPE;
  if (a->dk != 64 && a->dk != 128) return GDN_ERR_SHAPE;
  if (a->dv < 64 || a->dv % 64) return GDN_ERR_SHAPE;
  if (a->T > INT32_MAX - 2 * kC) return GDN_ERR_SHAPE;
  const int64_t page = static_cast<int64_t>(a->Hv) * a->dk * a->dv;
  if (page > INT32_MAX || a->final_sp < page || (a->initial_state && a->initial_sp < page)) return GDN_ERR_SHAPE;
  if (a->io_dtype != GDN_DT_BF16 && a->io_dtype != GDN_DT_F16) return GDN_ERR_DTYPE;
  if (!dtype_valid(a->g_dtype)) return GDN_ERR_DTYPE;
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->o) || !aligned16(a->final_state) ||
      !aligned16(a->initial_state))
    return GDN_ERR_ALIGN;
  const int64_t st[4][3] = {{a->q_sb, a->q_st, a->q_sh}, {a->k_sb, a->k_st, a->k_sh}, {a->v_sb, a->v_st, a->v_sh},
                            {a->o_sb, a->o_st, a->o_sh}};
  for (int i = 0; i < 4; ++i) {
    const int heads = i < 2 ? a->Hqk : a->Hv, B = a->cu_seqlens ? 1 : a->B;
    const int size[3] = {B, a->T, heads};
    for (int j = 0; j < 3; ++j) {
      if (size[j] > 1 && (st[i][j] < 1 || st[i][j] >= (1ll << 38))) return GDN_ERR_SHAPE;
      if (!stride_ok(st[i][j], 2)) return GDN_ERR_ALIGN;
    }
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
  return a->io_dtype == GDN_DT_BF16 ? gdn::dispatch<__nv_bfloat16>(*a, st) : gdn::dispatch<__half>(*a, st);
}
