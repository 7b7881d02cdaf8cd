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
// that is 128 KB against five 128^3 products (one more than the formulas have:
// the state's increment is two, see V'').  C = 128 and not 64: the state's update
// and its rounding to an operand cost the same per chunk, whatever its length.
//
// Warps (20): R 0-3 (a row of the chunk per thread), V 4-7, S 8-15, TMA loads 16,
// gates 17, MMA 18, TMA stores 19.  Per chunk, in the MMA warp's order:
//   SC  scores = Q K^T             Q copied into TMEM by R, which then turns the
//                                  scores into P, packed over their own columns
//   D0  dS^T  = V''^T K            of the chunk's first 64 tokens, V'' in TMEM (V)
//   QS  O     = Q S                S^T in shared memory
//   D1  dS^T += V''^T K            of the others; then S reads dS and rewrites S^T
//   PV  O    += P V                then V applies the rows' factors and stages O
// D0 and D1 lie between the others so that the tensor cores have work while R and
// V prepare the next operand.  All five take A from TMEM: a product with both
// operands in shared memory reads it at its full rate, and other warps' reads then
// take five times as long (4 ldmatrix.x4: 726 cycles against 141).
//
// V'' = w v, w = e^(G_C - G_j), is split into two parts of the I/O type, hi +
// lo: one part would leave half a step of the I/O type of every term (2^-8 in bf16) in a
// state that is fp32.  In bf16 so is w, which makes both parts a few packed fused
// multiply-adds: hi = v w_hi + v w_lo rounded once, lo = (v w_hi - hi) + v w_lo, the
// difference being exact.  Two parts of bf16 have 16 bits, and the state is off by up to
// 3.4e-6 of its norm; a third part, which would make that 2e-8, takes 14 instructions a
// pair of values in place of 5 and columns of TMEM that are all taken at d = 128.
//
// bf16 outputs are off by 2.4e-3: 1.7e-3 is their own rounding, P and the state that QS
// takes, each rounded to bf16 once as the operands that they are, give the rest.
//
// f16 I/O: w v, P and the state have no place in f16's range, and less than its precision
// in one part of bf16.  So w v is formed in fp32 and split times 2^-x, x by the largest of
// its value column (a part is lost only 2^-39 below that; the state is off by 2e-7); P is
// taken times 2^-y, y by its row; and QS, which R makes ready last and which then comes
// after PV, is a tf32 product, with 11 bits as f16 but fp32's range.  Outputs are off by
// 2.9e-4, 2.1e-4 of it their own rounding.  That costs V and R: at the shape below 185 to
// 200 us in bursts against bf16's 99 to 103.
//
// A value of V that is not finite belongs to the rows from its own on, but P V would
// bring it to the earlier ones of its chunk, as 0 x NaN.  It makes its column's dS NaN
// (its lower part is), which S sees; PV waits for that, the MMA warp puts zero in its
// place in the tile, and the epilogue writes NaN into its column from its row on.  (4% of
// the time, at d = 64 9%; a test of each value by V took 6% and 14%.)
//
// What bounds it (B = 4, T = 4096, Hqk = 16, H = 32, d = 128, bf16: 118 to 126 us, 403 MB,
// so 3.3 TB/s or 0.5 of the measured copy; 99 to 103 us in a burst, before the power limit
// takes the clock to 1.6 GHz): a CTA takes 4550 cycles a chunk.  The products take 0.49
// of them, and shared memory is at work in 0.92: operands 1280 cycles of 128 bytes, TMA
// 1000, the warps' reads, writes and barriers 1900.  Each answer from it takes some 250
// cycles then, in the chain Q, SC, P, PV of a chunk.  And instruction fetch: five
// roles of straight-line code pass through the SM's instruction cache once a chunk, at
// 0.89 hits.  So loops are kept rolled and call sites single where that is possible;
// unrolled throughout, the same kernel took 226 us.
#include <cuda_runtime.h>

#include <atomic>
#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "tc.cuh"

namespace gdn {
namespace {

constexpr int kC = 128;             // tokens of a chunk
constexpr int kTile = kC * 128;     // bytes of a [128][64] 16-bit tile
constexpr int kThreads = 20 * 32;
constexpr int kWarpV = 4, kWarpS = 8, kWarpTma = 16, kWarpGate = 17, kWarpMma = 18, kWarpStore = 19;
constexpr float kLog2e = 1.4426950408889634f;
// Up to so many sequences of a packed batch are put in order of length: 24 ragged ones
// (f16, d = 128 x 64, before its parts cost what they do now) took 89.6 us and not 98, 32
// of 20000 tokens 192 and not 203; 200, whose order takes each of 3200 CTAs 2 us to find,
// 409 and not 365.
constexpr int kRanked = 64;
// log2 gates are cut off here: 2^-160 is zero in fp32, and cumulative sums stay finite
constexpr float kLowest = -160.f;
// How a chunk's decays are factored, by the range of G (in powers of two):
//   kNear       G stays between -kLeast and kMost: e^(G_i) e^(-G_j)
//   kNearBlock  no gate grows or resets, and each block of 32 tokens spans at most kSpan:
//               e^(G_i - R_b) e^(R_b - G_j), R_b G at the end of j's block (where the
//               first of the two is zero so is P)
//   kFar        else, as across a reset: e^(G_i - G_j) by itself
// In bf16 O is summed without its rows' factors, which are 2^-kLeast at least, but with the
// scale's power of two (2^pow, |pow| <= 32): fp32 holds outputs of up to 2^47 then, and a
// row that decay leaves less of the state before the chunk takes 2^-80 of it.  The state
// itself is taken as it is: times a factor in the middle of the range, which may be 2^-80,
// it would leave bf16 from 2^-46 on.
constexpr float kSpan = 100.f;
constexpr float kLeast = 80.f, kMost = 40.f;
enum { kNear = 0, kNearBlock = 1, kFar = 2 };

// TMEM columns; all 512 are allocated, so they start at 0
constexpr uint32_t kTmSC = 0;     // scores fp32 [128]; P over its first 64 columns
constexpr uint32_t kTmQ = 128;    // Q, or Q' in bf16 [DK / 2]; f16: Q' in tf32 [DK] up to kTmV
constexpr uint32_t kTmV = 192;    // V'': lo [32], hi [32] of 64 tokens
constexpr uint32_t kTmO = 256;    // O fp32 [BV]
constexpr uint32_t kTmDS = 384;   // dS^T fp32 [DK]

template <int DK, int BV, bool BF16, bool FULL>
struct Layout {
  // K and V in two stages; Q, which R takes into TMEM, in one, and K too where a 32-bit
  // S^T needs its place
  static constexpr int kKStages = !BF16 && FULL && DK == 128 && BV == 128 ? 1 : 2;
  static constexpr int kKTile = DK / 64 * kTile, kVTile = BV / 64 * kTile;
  static constexpr int kK = 0;
  static constexpr int kV = kKStages * kKTile;
  static constexpr int kQ = kV + 2 * kVTile;
  static constexpr int kS = kQ + DK / 64 * kTile;          // S^T bf16 [BV][DK], 64-wide blocks; f16: tf32, 32-wide ones
  static constexpr int kSBlock = BV * 128;
  static constexpr int kO = kS + (BF16 || !FULL ? DK / 64 : DK / 32) * kSBlock;
  static constexpr int kGate = kO + BV / 64 * kTile;
  static constexpr int kGateStage = 2 * kC * 4;            // G or its factors, w
  static constexpr int kFirst = kGate + 2 * kGateStage;    // per value column, a byte: see Bars::bad
  static constexpr int kShift = kFirst + 128;              // f16: x of V'' per value column, by chunk, a byte
  static constexpr int kRow = kShift + 2 * 128;            // f16: y of P per row, by chunk, a byte
  static constexpr int kBars = kRow + 2 * 128;
  static constexpr int kBytes = kBars + 368;
  static_assert(kBytes <= 232448, "shared memory");
};

enum { kTileQ = 0, kTileK = 1, kTileV = 2 };

struct Bars {
  uint64_t full[3][2], empty[3][2];  // of the Q (one stage), K, V tiles
  uint64_t gfull[2], gempty[2];
  uint64_t sc_done, q_ready, q2_ready, qs_done, p_ready, pv_done;
  uint64_t v_ready[2], v_free[2], ds_done, seen, ds_free, s_ready;
  uint64_t o_free, o_staged, o_stored, zeroed, drain;
  float gamma[2];
  float ref[2][4];  // R_b
  int grow[2];      // f16: no G_i - G_j, i >= j, of the chunk is larger
  int form[2];      // kNear, kNearBlock, kFar
  // 1 + the last chunk in which dS is NaN; kFirst then holds, per value column, the first
  // token whose value is not finite (kC: none)
  int bad;
  int call;         // the MMA thread to the rest of its warp
  uint32_t tmem;
};
static_assert(sizeof(Bars) <= 368, "barriers");

struct PrefillParams {
  lin_prefill_args_t a;
  int nvb;
  // Few rows and a long time axis: sequences of more than `piece` tokens are cut
  // into pieces (0: none is).  A slot of the workspace per piece of a cut sequence
  // holds the state that the piece starts from, and first the piece before's own
  // contribution; `decay` the pieces' products of gates, [slot][head].
  int piece, pieces, slots;  // pieces: of every sequence, in the dense form
  int ranked;                // packed sequences are taken longest first
  // scale = rest * 2^pow; bf16 and not kFar: P and the state carry 2^pow, the epilogue
  // applies the rest
  float pow, pow2, rest;
  float* slot_state;
  float* decay;
};

// What a CTA works on: `len` tokens from row `start` (-1: nothing), beginning with
// the state `from` (NULL: zero) and leaving it in `to` (NULL: nowhere).
struct Item {
  int start, len;
  const float* from;
  float* to;
};

struct Seq {
  int start, len, page;
};

// Sequence n's rows; offsets out of range or descending give -1 tokens.
__device__ __forceinline__ void find_rows(const lin_prefill_args_t& a, int n, Seq& s) {
  s.start = 0;
  s.len = a.T;
  if (a.cu_seqlens) {
    const int lo = a.cu_seqlens[n], hi = a.cu_seqlens[n + 1];
    s.start = lo;
    s.len = lo >= 0 && lo <= hi && hi <= a.T ? hi - lo : -1;
  }
}

// Every thread of the CTA calls it.  A page out of range or held by an earlier
// sequence is none (-1).
__device__ Seq find_seq(const lin_prefill_args_t& a, int n, bool reporter) {
  Seq s;
  s.page = a.index ? a.index[n] : n;
  // the first of the earlier pages, asked for together with this one's
  const int j0 = threadIdx.x;
  const int other = a.index && j0 < n ? a.index[j0] : -1;
  find_rows(a, n, s);
  bool bad = s.len < 0;
  bool taken = s.page >= a.pages || (other >= 0 && other == s.page);
  if (a.index && s.page >= 0)
    for (int j = j0 + blockDim.x; j < n; j += blockDim.x) taken |= a.index[j] == s.page;
  if (__syncthreads_or(taken)) {
    bad = true;
    s.page = -1;
  }
  if (bad && reporter) report(a.status, GDN_DEVERR_BAD_INDEX);
  return s;
}

// Slots of sequence n: one per piece if it is cut.
__device__ __forceinline__ int slots_of(const PrefillParams& p, int n) {
  if (n >= p.a.B) return 0;
  Seq s;
  find_rows(p.a, n, s);
  return s.len > p.piece ? (s.len + p.piece - 1) / p.piece : 0;
}

// Whole warps: the sequence that slot y belongs to (-1: none) and the piece, or,
// with y < 0, the first slot of sequence *n.
__device__ int find_slot(const PrefillParams& p, int y, int* n) {
  if (!p.a.cu_seqlens) {
    if (y < 0) return *n * p.pieces;
    *n = y / p.pieces;
    return y - *n * p.pieces;
  }
  const int lane = threadIdx.x & 31;
  const int until = y < 0 ? *n : p.a.B;
  int run = 0;
  for (int n0 = 0; n0 < until; n0 += 32) {
    const int v = n0 + lane < until ? slots_of(p, n0 + lane) : 0;
    int inc = v;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, inc, off);
      if (lane >= off) inc += x;
    }
    const unsigned past = __ballot_sync(0xffffffffu, y >= 0 && y < run + inc);
    if (past) {
      const int hit = __ffs(past) - 1;
      *n = n0 + hit;
      return y - run - __shfl_sync(0xffffffffu, inc - v, hit);
    }
    run += __shfl_sync(0xffffffffu, inc, 31);
  }
  if (y < 0) return run;
  *n = -1;
  return 0;
}

// Every thread of the CTA calls it: the sequence that comes y-th by falling number of
// chunks (equal ones in order).  With more CTAs than SMs the longest start first, so
// that no long one is left alone at the end.
__device__ int nth_longest(const lin_prefill_args_t& a, int y, uint32_t* key) {
  const int j = threadIdx.x, padded = (a.B + 3) & ~3;
  if (j < padded) {
    uint32_t x = 0;
    if (j < a.B) {
      Seq s;
      find_rows(a, j, s);
      x = static_cast<uint32_t>((s.len + kC - 1) / kC) << 8 | (kRanked - 1 - j);
    }
    key[j] = x;
  }
  __syncthreads();
  if (j < a.B) {
    const uint32_t mine = key[j];
    int longer = 0;
    for (int i = 0; i < padded; i += 4) {
      const uint4 x = *reinterpret_cast<const uint4*>(key + i);
      longer += (x.x > mine) + (x.y > mine) + (x.z > mine) + (x.w > mine);
    }
    if (longer == y) key[kRanked] = j;
  }
  __syncthreads();
  return key[kRanked];
}

template <bool FULL>
__device__ Item find_item(const PrefillParams& p, int y, bool reporter, uint32_t* scratch) {
  const lin_prefill_args_t& a = p.a;
  const int64_t page = static_cast<int64_t>(a.Hv) * a.dk * a.dv;
  Item it{0, -1, nullptr, nullptr};
  int n = y, at = 0;
  const bool slot = p.piece && y < p.slots;
  if (slot) {
    at = find_slot(p, y, &n);
    if (n < 0) return it;
  } else if (p.piece) {
    n = y - p.slots;
  }
  if (FULL && !slot && p.ranked) n = nth_longest(a, n, scratch);
  const Seq s = find_seq(a, n, reporter);
  if (s.len < 0) return it;
  const bool cut = p.piece && s.len > p.piece;
  if (!slot) {
    if (cut) return it;
    it.start = s.start;
    it.len = s.len;
    if (s.page >= 0 && a.initial_state) it.from = a.initial_state + s.page * a.initial_sp;
    if (s.page >= 0) it.to = a.final_state + s.page * a.final_sp;
    return it;
  }
  const bool last = (at + 1) * p.piece >= s.len;
  // (overlapping sequences, which unsound offsets allow, could ask for more slots)
  if (!FULL && (last || y + 1 >= p.slots)) return it;
  it.start = s.start + at * p.piece;
  it.len = last ? s.len - at * p.piece : p.piece;
  if (FULL) {
    it.from = p.slot_state + y * page;
    if (last && s.page >= 0) it.to = a.final_state + s.page * a.final_sp;
  } else {
    it.to = p.slot_state + (y + 1) * page;
  }
  return it;
}

// Shared-memory loads that stay where they are written: ahead of the arithmetic.
template <typename T>
__device__ __forceinline__ void lds128(const void* p, T* x) {
  uint32_t* u = reinterpret_cast<uint32_t*>(x);
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3])
               : "r"(smem_u32(p)));
}
__device__ __forceinline__ void lds64(const void* p, uint32_t* u) {
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(u[0]), "=r"(u[1]) : "r"(smem_u32(p)));
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

// The lower half of the clock, in ns: two dozen copies of the waits below share the
// instruction cache with the roles' loops.  (Read after the first failed try only: 104.7
// us in bursts of the batch case; the whole of it 103.5; this 101.9.)
__device__ __forceinline__ uint32_t now_ns() {
  uint32_t t;
  asm volatile("mov.u32 %0, %%globaltimer_lo;" : "=r"(t));
  return t;
}
static_assert(kWaitLimitNs < 1ull << 31, "half a clock");

// Waits for a phase; false after kWaitLimitNs.  wait1() is for one thread; wait() for a
// whole warp, whose lanes all get the same answer.
__device__ __forceinline__ bool wait1(uint64_t* bar, uint32_t parity) {
  const uint32_t at = smem_u32(bar);
  const uint32_t t0 = now_ns();
  uint32_t ok;
  do {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(at), "r"(parity)
        : "memory");
  } while (!ok && now_ns() - t0 < static_cast<uint32_t>(kWaitLimitNs));
  return ok != 0;
}
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, wait1(bar, parity));
}
// Two or three at once: while products read shared memory an answer takes some 250
// cycles, and these overlap (batch case 103.2 against 99.7 us in bursts).  On a fresh
// barrier parity 1 counts as complete: that of the chunk before the first.
__device__ __forceinline__ bool wait1(uint64_t* b0, uint32_t p0, uint64_t* b1, uint32_t p1, uint64_t* b2, uint32_t p2) {
  const uint32_t at0 = smem_u32(b0), at1 = smem_u32(b1), at2 = smem_u32(b2);
  const uint32_t t0 = now_ns();
  uint32_t ok;
  do {
    asm volatile(
        "{\n\t.reg .pred p, q, r;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 q, [%3], %4;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 r, [%5], %6;\n\t"
        "and.pred p, p, q;\n\t"
        "and.pred p, p, r;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(at0), "r"(p0), "r"(at1), "r"(p1), "r"(at2), "r"(p2)
        : "memory");
  } while (!ok && now_ns() - t0 < static_cast<uint32_t>(kWaitLimitNs));
  return ok != 0;
}
__device__ __forceinline__ bool wait(uint64_t* b0, uint32_t p0, uint64_t* b1, uint32_t p1, uint64_t* b2, uint32_t p2) {
  return __all_sync(0xffffffffu, wait1(b0, p0, b1, p1, b2, p2));
}
__device__ __forceinline__ bool wait(uint64_t* b0, uint32_t p0, uint64_t* b1, uint32_t p1) {
  return __all_sync(0xffffffffu, wait1(b0, p0, b1, p1, b1, p1));
}

// A warp: puts zero in the place of what is not finite in a tile of V and leaves the first
// token of which that is so in first[column] (kC: none; dS is NaN for a key's sake too).
__device__ __noinline__ void clear_values(unsigned char* tile, int columns, uint32_t exponent, unsigned char* first) {
  for (int x = (threadIdx.x & 31) * 2; x < columns; x += 64) {
    unsigned char* at = tile + (x >> 6) * kTile + (x & 7) * 2;
    int first0 = kC, first1 = kC;
#pragma unroll 1
    for (int t0 = kC - 8; t0 >= 0; t0 -= 8) {  // rows of one swizzle atom, loads first
      uint32_t u[8];
#pragma unroll
      for (int t = 0; t < 8; ++t) u[t] = *reinterpret_cast<uint32_t*>(at + tc::sw128_offset(t0 + t, (x & 63) >> 3));
#pragma unroll
      for (int t = 7; t >= 0; --t) {
        const bool bad0 = (u[t] & exponent) == exponent, bad1 = (u[t] >> 16 & exponent) == exponent;
        if (bad0) first0 = t0 + t;
        if (bad1) first1 = t0 + t;
        if (bad0 || bad1)
          *reinterpret_cast<uint32_t*>(at + tc::sw128_offset(t0 + t, (x & 63) >> 3)) =
              (bad0 ? 0u : u[t] & 0xffffu) | (bad1 ? 0u : u[t] & 0xffff0000u);
      }
    }
    first[x] = static_cast<unsigned char>(first0);
    first[x + 1] = static_cast<unsigned char>(first1);
  }
  tc::fence_proxy_async();
  __syncwarp();
}

// A thread with the row `row` of a tile of O: NaN in the columns that a value of that row
// or one before belongs to which is not finite.
__device__ __noinline__ void mark_row(unsigned char* tile, int row, int columns, const unsigned char* first) {
#pragma unroll 1
  for (int x0 = 0; x0 < columns; x0 += 8) {
    const uint2 f = *reinterpret_cast<const uint2*>(first + x0);
    uint16_t* o = reinterpret_cast<uint16_t*>(tile + (x0 >> 6) * kTile + tc::sw128_offset(row, (x0 & 63) >> 3));
#pragma unroll
    for (int x = 0; x < 8; ++x)
      if (row >= static_cast<int>((x < 4 ? f.x : f.y) >> (x & 3) * 8 & 0xffu)) o[x] = 0x7fff;
  }
}

// FULL: everything.  Else only what a piece adds to the state and its decay, from k,
// v and the gates; the tensor memory that is free then is a second place for V''.
template <int DK, int BV, typename IO, bool FULL>
__global__ void __launch_bounds__(kThreads, 1)
    lin_prefill_kernel(const __grid_constant__ PrefillParams p, const __grid_constant__ CUtensorMap map_q,
                       const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                       const __grid_constant__ CUtensorMap map_o) {
  constexpr bool BF16 = std::is_same<IO, __nv_bfloat16>::value;
  using L = Layout<DK, BV, BF16, FULL>;
  extern __shared__ __align__(1024) unsigned char smem[];
  Bars& bar = *reinterpret_cast<Bars*>(smem + L::kBars);
  const lin_prefill_args_t& a = p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int h = blockIdx.x / p.nvb, vb = blockIdx.x - h * p.nvb, hq = h / (a.Hv / a.Hqk);
  if (warp == kWarpMma) tc::tmem_alloc(&bar.tmem, 512);
  if (tid == 0) {
    for (int s = 0; s < 2; ++s) {
      for (int t = 0; t < 3; ++t) {
        mbar_init(&bar.full[t][s], 1);
        mbar_init(&bar.empty[t][s], t == kTileQ ? 4 : 1);
      }
      mbar_init(&bar.gfull[s], 1);
      mbar_init(&bar.gempty[s], FULL ? 16 : 12);
      mbar_init(&bar.v_ready[s], 4);
      mbar_init(&bar.v_free[s], 1);
    }
    mbar_init(&bar.sc_done, 1);
    mbar_init(&bar.q_ready, 4);
    mbar_init(&bar.q2_ready, 4);
    mbar_init(&bar.ds_free, 8);
    mbar_init(&bar.seen, 8);
    mbar_init(&bar.qs_done, 1);
    mbar_init(&bar.p_ready, 4);
    mbar_init(&bar.pv_done, FULL ? 2 : 1);
    mbar_init(&bar.ds_done, BF16 ? 1 : 2);
    mbar_init(&bar.s_ready, 8);
    mbar_init(&bar.o_free, 4);
    mbar_init(&bar.o_staged, 4);
    mbar_init(&bar.o_stored, 1);
    mbar_init(&bar.zeroed, 4);
    mbar_init(&bar.drain, 1);
    bar.bad = 0;
    fence_mbar_init();
  }
  if (tid < 4) prefetch_map(tid == 0 ? &map_q : tid == 1 ? &map_k : tid == 2 ? &map_v : &map_o);
  pdl_launch_dependents();
  pdl_wait();
  // (a CTA without work goes through the roles with no chunks and no state)
  const Item seq = find_item<FULL>(p, blockIdx.y, FULL && blockIdx.x == 0 && tid == 0,
                                   reinterpret_cast<uint32_t*>(smem + L::kO));
  const int chunks = seq.len > 0 ? (seq.len + kC - 1) / kC : 0;
  const int batch = a.cu_seqlens ? 0 : p.piece && static_cast<int>(blockIdx.y) < p.slots ? blockIdx.y / p.pieces
                                    : blockIdx.y - (p.piece ? p.slots : 0);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  constexpr uint32_t tmem = 0;
  const uint32_t sb = smem_u32(smem);
  uint32_t* const status = a.status;
  bool ok = true;

  if (FULL && warp < kWarpV) {
    // ------------------------------------------------ R: P, a row per thread
    const int row = tid;
    const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
    for (int c = 0; c < chunks; ++c) {
      const int st = c & 1;
      const float* G = reinterpret_cast<const float*>(smem + L::kGate + st * L::kGateStage);
      // Q into the columns that the last chunk's QS has read
      if (!(ok = wait(&bar.gfull[st], (c >> 1) & 1, &bar.full[kTileQ][0], c & 1, &bar.qs_done, (c & 1) ^ 1))) break;
      tc::fence_after_sync();
      const int form = bar.form[st];
      const float own = G[row];  // e^(-G_i) or e^(R - G_i) (bf16: 2^pow of it), or G_i
      const float Gi = form == kNearBlock ? bar.ref[st][warp] + (BF16 ? p.pow : 0.f) - __log2f(own) : own;  // (not kNear)
      float f = a.scale * (form == kNear ? __frcp_rn(own) : ex2(Gi));
      // SC takes Q as it is.  bf16, and not kFar: so does QS; O then lacks the row's
      // factor, and P leaves it out too: the epilogue applies it.  (kNearBlock: a factor
      // below 2^-kLeast is taken as that; P carries the rest of it, and of the state
      // before the chunk so little arrives that it makes no difference.)  Else P carries
      // the row's factor, and QS takes Q' = scale e^G Q written over Q: in bf16, whose
      // range it needs, and with f16 I/O in tf32, in part over the scores that P leaves
      // free; there the factor's power of two alone, which makes Q' exact, and the epilogue
      // and P take the rest of it.  f16 does not have P's range either: both are taken
      // times 2^-y, and the epilogue applies 2^y.  y comes from a bound of the row, its
      // largest score by the scale and the gates' growth: P 2^-y stays below 2^15 and is
      // lost 2^-39 below that, where the scores' fp32 sums are 2^-24 off.  (From P's own
      // largest 105 us at B = 4, T = 2048, d = 128; this 99.)
      const bool by_block = BF16 && form == kNearBlock, plain_q = BF16 && form != kFar;
      const auto queries = [&](bool scaled) {
#pragma unroll 1
        for (int b = 0; b < DK / 64; ++b) {
          uint32_t u[2][16];
#pragma unroll
          for (int e = 0; e < 8; ++e)
            lds128(smem + L::kQ + b * kTile + tc::sw128_offset(row, e), &u[e >> 2][(e & 3) * 4]);
          if (!BF16 && scaled) {
#pragma unroll
            for (int h4 = 0; h4 < 4; ++h4) {
              uint32_t x[16];
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const uint32_t w = u[h4 >> 1][(h4 & 1) * 8 + i];
                x[2 * i] = __float_as_uint(f * tc::unpack_lo<BF16>(w));
                x[2 * i + 1] = __float_as_uint(f * tc::unpack_hi<BF16>(w));
              }
              tc::tmem_st16(tmem + lanes + kTmV - DK + b * 64 + h4 * 16, x);
            }
            continue;
          }
          if (scaled) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              uint32_t& w = u[i >> 4][i & 15];
              w = tc::pack2<true>(f * tc::unpack_lo<BF16>(w), f * tc::unpack_hi<BF16>(w));
            }
          }
          tc::tmem_st16(tmem + lanes + kTmQ + b * 32, u[0]);
          tc::tmem_st16(tmem + lanes + kTmQ + b * 32 + 16, u[1]);
        }
      };
#pragma unroll 1
      for (int pass = 0; pass < (BF16 ? 2 : 1); ++pass) {
        if (pass && !(ok = wait(&bar.sc_done, c & 1))) break;
        tc::fence_after_sync();
        if (!pass || !plain_q) {
          queries(pass);
          tc::tmem_wait_st();
          tc::fence_before_sync();
          __syncwarp();
        }
        if (lane == 0) {
          mbar_arrive(pass ? &bar.q2_ready : &bar.q_ready);
          if (BF16 && pass != plain_q) mbar_arrive(&bar.empty[kTileQ][0]);  // read for the last time
        }
      }
      if (!BF16 && (ok = wait(&bar.sc_done, c & 1))) tc::fence_after_sync();
      if (!ok) break;
      float shrink = 1.f, f_pow2 = 1.f;  // scale 2^-y, without the rest of f; f's power of two 2^-y
      if (!BF16) {
        float most = 0.f;
#pragma unroll 1
        for (int b = 0; b <= warp; b += 2) {
          float x[4][16];
#pragma unroll
          for (int e = 0; e < 4; ++e) tc::tmem_ld16(tmem + lanes + kTmSC + b * 32 + e * 16, x[e]);
          tc::tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 64; ++e)
            if (e <= row - b * 32) most = fmaxf(most, fabsf(x[e >> 4][e & 15]));
        }
        const auto exponent = [](float x) { return static_cast<int>(__float_as_uint(fabsf(x)) >> 23) - 127; };
        // (a score that is not zero is 2^-48 at least.)  y >= -64 and f 2^-y <= 2^91 keep Q' S
        // and Q' within fp32; only rows of P that are zero come so low
        const int y = max(max(max(exponent(most), -48) + exponent(a.scale) + bar.grow[st] - 12, -64), exponent(f) - 90);
        shrink = __uint_as_float(static_cast<uint32_t>(127 - min(y, 115)) << 23);
        smem[L::kRow + st * 128 + row] = static_cast<unsigned char>(min(y, 115));
        f_pow2 = shrink * __uint_as_float(__float_as_uint(f) & 0x7f800000u);
        shrink *= a.scale * __frcp_rn(tc::significand(f));
      }
      // P in the I/O type over the scores: columns [32 b, 32 b + 32) go to [16 b, 16 b + 16)
#pragma unroll 1
      for (int b = 0; b < 4; ++b) {
        uint32_t u[16];
        if (b <= warp) {
          // the loads first: shared memory answers late while the products read it
          float x[2][16], d[32];
          tc::tmem_ld16(tmem + lanes + kTmSC + b * 32, x[0]);
          tc::tmem_ld16(tmem + lanes + kTmSC + b * 32 + 16, x[1]);
#pragma unroll
          for (int e = 0; e < 32; e += 4) lds128(G + b * 32 + e, d + e);
          if (form == kFar) {
#pragma unroll
            for (int e = 0; e < 32; ++e) d[e] = (BF16 ? a.scale : 1.f) * ex2(Gi - d[e]);
          } else if (by_block) {
            // the block's factor in two steps of at most 2^kSpan, or the row's as well
            // (its root, twice: the whole may pass the range of a float where d is small)
            const float r = ex2(0.5f * (Gi - fmaxf(Gi, -kLeast) - bar.ref[st][b]));
#pragma unroll
            for (int e = 0; e < 32; ++e) d[e] = d[e] * r * r;
          } else if (!BF16) {
            const float r = form == kNear ? __frcp_rn(own) : ex2(Gi - bar.ref[st][b]);
#pragma unroll
            for (int e = 0; e < 32; ++e) d[e] *= r;
          }
          tc::tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) d[e] *= BF16 ? x[e >> 4][e & 15] : x[e >> 4][e & 15] * shrink;
          if (b == warp) {  // on the diagonal
#pragma unroll
            for (int e = 0; e < 32; ++e) d[e] = e <= lane ? d[e] : 0.f;
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) u[e] = tc::pack2<BF16>(d[2 * e], d[2 * e + 1]);
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) u[e] = 0;
        }
        tc::tmem_st16(tmem + lanes + kTmSC + b * 16, u);
      }
      tc::tmem_wait_st();
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&bar.p_ready);
        mbar_arrive(&bar.gempty[st]);
      }
      if (!BF16) {
        f = f_pow2;
        queries(true);
        tc::tmem_wait_st();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bar.q2_ready);
          mbar_arrive(&bar.empty[kTileQ][0]);
        }
      }
    }
  } else if (warp >= kWarpV && warp < kWarpS) {
    // ------------------------------------------------ V: V'' parts, O
    const int quarter = warp - kWarpV, row = quarter * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const bool has_rows = quarter * 32 < BV;
    // Of this lane's tokens 2 l, 2 l + 1 and 2 l + 8, 2 l + 9 of each 16 of a half, l = lane % 4:
    // (hi, lo) of w for both tokens of a pair, or (f16) w of each
    const auto weights = [&](int st, int half, uint32_t (&ww)[4][4]) {
      const uint2* w = reinterpret_cast<const uint2*>(smem + L::kGate + st * L::kGateStage + kC * 4) + half * 32 + (lane & 3);
#pragma unroll
      for (int tb = 0; tb < 4; ++tb) {
        lds64(w + tb * 8, ww[tb]);
        lds64(w + tb * 8 + 4, ww[tb] + 2);
      }
    };
    // and of columns l / 4 (e even) and l / 4 + 8 of the i-th 16 of this warp, the values
    const auto values = [&](int st, int half, int i, uint32_t (&r)[4][4]) {
      const int dv = quarter * 32 + i * 16;
      const uint32_t block = sb + L::kV + st * L::kVTile + (dv >> 6) * kTile;
      const int chunk = ((dv & 63) >> 3) + ((lane >> 3) & 1);
#pragma unroll
      for (int tb = 0; tb < 4; ++tb)
        tc::ldsm_x4_trans(block + tc::sw128_offset(half * 64 + tb * 16 + (lane >> 4) * 8 + (lane & 7), chunk), r[tb]);
    };
    float shrink[2][2] = {};  // f16: 2^-x of those columns
    // x: the largest |w v| of a column times 2^-x lies in [2^13, 2^14)
    const auto find_shifts = [&](int st) {
      float most[2][2] = {};
#pragma unroll 1
      for (int half = 0; half < 2; ++half) {
        uint32_t ww[4][4], r[4][4];
        weights(st, half, ww);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          values(st, half, i, r);
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const uint32_t v = r[e >> 2][e & 3];
            float& m = most[i][e & 1];
            m = fmaxf(m, fabsf(__uint_as_float(ww[e >> 2][e & 2]) * tc::unpack_lo<BF16>(v)));
            m = fmaxf(m, fabsf(__uint_as_float(ww[e >> 2][(e & 2) + 1]) * tc::unpack_hi<BF16>(v)));
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float m = most[i >> 1][i & 1];
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
        // (below 2^-100 columns keep less; above, 2^115 for infinities)
        const int x = max(static_cast<int>(__float_as_uint(m) >> 23) - 127 - 13, -113);
        shrink[i >> 1][i & 1] = __uint_as_float(static_cast<uint32_t>(127 - x) << 23);
        if ((lane & 3) == 0)
          smem[L::kShift + st * 128 + quarter * 32 + i * 8 + (lane >> 2)] = static_cast<unsigned char>(x);
      }
    };
    // tokens [64 half, 64 half + 64) of chunk c: both parts
    const auto parts = [&](int c, int half) {
      const int st = c & 1;
      if (has_rows) {
        if (!BF16 && !FULL && !half) find_shifts(st);
        uint32_t ww[4][4], r[2][4][4];
        weights(st, half, ww);
        // all loads first (unrolled 98.2 against 99.5 us; at d = 64 37.9 against 40.7)
        values(st, half, 0, r[0]);
        values(st, half, 1, r[1]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t hi[16], lo[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const uint32_t v = r[i][e >> 2][e & 3], w0 = ww[e >> 2][e & 2], w1 = ww[e >> 2][(e & 2) + 1];
            if constexpr (BF16) {
              hi[e] = tc::fma2<BF16>(v, w0, tc::mul2<BF16>(v, w1));
              lo[e] = tc::fma2<BF16>(v, w1, tc::fma2<BF16>(v, w0, hi[e] ^ 0x80008000u));
            } else {
              const float x = __uint_as_float(w0) * tc::unpack_lo<BF16>(v) * shrink[i][e & 1];
              const float y = __uint_as_float(w1) * tc::unpack_hi<BF16>(v) * shrink[i][e & 1];
              hi[e] = tc::pack2<BF16>(x, y);
              lo[e] = tc::pack2<BF16>(x - tc::unpack_lo<BF16>(hi[e]), y - tc::unpack_hi<BF16>(hi[e]));
            }
          }
          const uint32_t to = tmem + lanes + (static_cast<uint32_t>(i * 16) << 16) + (FULL || half ? kTmV : kTmSC);
          tc::tmem_st_16x128b_x8(to, lo);
          tc::tmem_st_16x128b_x8(to + 32, hi);
        }
        tc::tmem_wait_st();
      }
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.v_ready[half]);
    };
    // O of chunk c: a token per thread, times the row's factor, packed into shared memory
    float factor = 1.f;
    const auto output = [&](int c) {
      unsigned char* o = smem + L::kO;
      if (!wait(&bar.pv_done, c & 1, &bar.o_stored, (c & 1) ^ 1)) return false;
      uint32_t bad;  // asked for early
      asm volatile("ld.shared.b32 %0, [%1];" : "=r"(bad) : "r"(smem_u32(&bar.bad)));
      tc::fence_after_sync();
      if (!BF16) {
        const int y = static_cast<signed char>(smem[L::kRow + (c & 1) * 128 + row]);
        factor *= __uint_as_float(static_cast<uint32_t>(127 + y) << 23);
      }
#pragma unroll 1
      for (int b = 0; b < BV / 32; ++b) {
        float x[2][16];
        tc::tmem_ld16(tmem + lanes + kTmO + b * 32, x[0]);
        tc::tmem_ld16(tmem + lanes + kTmO + b * 32 + 16, x[1]);
        tc::tmem_wait_ld();
        const uint32_t to = smem_u32(o) + (b >> 1) * kTile;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float* y = &x[e >> 1][(e & 1) * 8];
          tc::sts128(to + tc::sw128_offset(row, (b & 1) * 4 + e), tc::pack2<BF16>(factor * y[0], factor * y[1]),
                     tc::pack2<BF16>(factor * y[2], factor * y[3]), tc::pack2<BF16>(factor * y[4], factor * y[5]),
                     tc::pack2<BF16>(factor * y[6], factor * y[7]));
        }
      }
      if (bad == c + 1) mark_row(o, row, BV, smem + L::kFirst);
      tc::fence_before_sync();
      tc::fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&bar.o_staged);
        mbar_arrive(&bar.o_free);
      }
      const int rows = seq.len - c * kC;
      if (rows < kC) {  // the rows behind belong to another sequence, or to nobody
        if (!wait(&bar.o_staged, c & 1)) return false;
        IO* dst = static_cast<IO*>(a.o) + batch * a.o_sb + static_cast<int64_t>(seq.start + c * kC) * a.o_st + h * a.o_sh +
                  vb * BV;
        constexpr int kPer = BV / 8;  // 16-byte pieces of a row
        for (int i = row; i < rows * kPer; i += 128) {
          const int r = i / kPer, piece = i - r * kPer;
          const uint4 x = *reinterpret_cast<const uint4*>(o + (piece >> 3) * kTile + tc::sw128_offset(r, piece & 7));
          *reinterpret_cast<uint4*>(dst + r * a.o_st + piece * 8) = x;
        }
      }
      return true;
    };
    // Two steps a chunk, 64 tokens each, the last chunk's output between them.
    // One call site each keeps the kernel's code within the instruction cache.
#pragma unroll 1
    for (int step = 0; step < 2 * chunks + FULL; ++step) {
      const int c = step >> 1, half = step & 1, st = c & 1;
      if (c < chunks) {
        if (half == 0) {
          const uint32_t ph = (c >> 1) & 1;
          if (!(ok = wait(&bar.gfull[st], ph, &bar.full[kTileV][st], ph))) break;
          const int rows = seq.len - c * kC;
          if (rows < kC) {
            // rows of the next sequence, or outside: zero, whatever they hold, since
            // 0 x NaN would reach the sums over the chunk's tokens
            const int kst = c & (L::kKStages - 1);
            if (!(ok = wait(&bar.full[kTileK][kst], (c / L::kKStages) & 1))) break;
            for (int r = rows + quarter; r < kC; r += 4)
              for (int i = lane; i < (DK + BV) / 8; i += 32) {
                const int b = i >> 3;
                unsigned char* to = smem + (b < DK / 64 ? L::kK + kst * L::kKTile + b * kTile
                                                        : L::kV + st * L::kVTile + (b - DK / 64) * kTile);
                *reinterpret_cast<uint4*>(to + tc::sw128_offset(r, i & 7)) = make_uint4(0, 0, 0, 0);
              }
            tc::fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar.zeroed);
            if (!(ok = wait(&bar.zeroed, 0))) break;  // only the last chunk is short
          }
        }
        // meanwhile (S has read the shifts of the chunk before last: D0 of the last waited for it)
        if (!BF16 && FULL && !half && has_rows) find_shifts(st);
        // the columns' last user: the half before, or this half of the chunk before
        const int before = FULL ? step - 1 : step - 2;
        if (before >= 0 && !(ok = wait(&bar.v_free[before & 1], (before >> 1) & 1))) break;
        tc::fence_after_sync();
        parts(c, half);
        if (half) {
          if (FULL) {
            const float own = reinterpret_cast<const float*>(smem + L::kGate + st * L::kGateStage)[row];
            const int form = bar.form[st];
            factor = 1.f;
            if (!BF16) {  // as R has it
              const float Gi = form == kNearBlock ? bar.ref[st][quarter] - __log2f(own) : own;
              factor = tc::significand(a.scale * (form == kNear ? __frcp_rn(own) : ex2(Gi)));
            } else if (form == kNear) {
              factor = a.scale * __frcp_rn(own);
            } else if (form == kNearBlock) {
              const float Gi = bar.ref[st][quarter] + p.pow - __log2f(own);
              factor = p.rest * ex2(fmaxf(Gi, -kLeast));
            }
            __syncwarp();
          }
          if (lane == 0) mbar_arrive(&bar.gempty[st]);
        }
      }
      if (FULL && c && !half && !(ok = output(c - 1))) break;
    }
  } else if (warp >= kWarpS && warp < kWarpTma) {
    // ------------------------------------------------ S: the state, a value column per thread
    const int quarter = warp & 3, half = (warp - kWarpS) >> 2;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const int row = quarter * 32 + lane;  // value column of this CTA's block
    const bool has_rows = quarter * 32 < BV;
    constexpr int kN = DK / 2;            // d_k entries of this thread
    const int64_t at = (static_cast<int64_t>(h) * DK + half * kN) * a.dv + vb * BV + row;
    float S[kN];
    const float* from = seq.from + (seq.from ? at : 0);
#pragma unroll
    for (int i = 0; i < kN; ++i) S[i] = seq.from && has_rows ? from[static_cast<int64_t>(i) * a.dv] : 0.f;
    // the state before chunk 0, then after each chunk
#pragma unroll 1
    for (int c = FULL ? -1 : 0; c < chunks; ++c) {
      if (c >= 0) {
        const int st = c & 1;
        ok = wait(&bar.gfull[st], (c >> 1) & 1, &bar.ds_done, c & 1);
        if (!ok) break;
        tc::fence_after_sync();
        const float gamma = bar.gamma[st];
        if (has_rows) {
          const int x = BF16 ? 0 : static_cast<signed char>(smem[L::kShift + st * 128 + row]);
          const float grow = __uint_as_float(static_cast<uint32_t>(127 + x) << 23);
#pragma unroll
          for (int b = 0; b < kN / 16; ++b) {
            float d[16];
            tc::tmem_ld16(tmem + lanes + kTmDS + half * kN + b * 16, d);
            tc::tmem_wait_ld();
            if (FULL && b == 0) {  // at once: PV waits for it
              const bool bad = __any_sync(0xffffffffu, isnan(d[0]));
              if (lane == 0) {
                if (bad) bar.bad = c + 1;
                mbar_arrive(&bar.seen);
              }
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) S[b * 16 + e] = fmaf(gamma, S[b * 16 + e], BF16 ? d[e] : grow * d[e]);
          }
        } else if (FULL && lane == 0) {
          mbar_arrive(&bar.seen);
        }
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bar.gempty[st]);
          mbar_arrive(&bar.ds_free);
        }
      }
      if (!FULL || c + 1 == chunks) continue;
      float m = 1.f;
      if (BF16) {
        if (!(ok = wait(&bar.gfull[(c + 1) & 1], ((c + 1) >> 1) & 1))) break;
        m = bar.form[(c + 1) & 1] == kFar ? 1.f : p.pow2;
      } else if (c >= 0 && !(ok = wait(&bar.qs_done, c & 1))) {
        break;  // (in bf16 ds_done comes behind it)
      }
      if (has_rows && !BF16) {  // S^T rounded to tf32, the QS product's operand
#pragma unroll
        for (int i = 0; i < kN / 4; ++i) {
          const int piece = half * (kN / 4) + i;
          tc::sts128(sb + L::kS + (piece >> 3) * L::kSBlock + tc::sw128_offset(row, piece & 7), tc::to_tf32(S[4 * i]),
                     tc::to_tf32(S[4 * i + 1]), tc::to_tf32(S[4 * i + 2]), tc::to_tf32(S[4 * i + 3]));
        }
      } else if (has_rows) {  // or to bf16
#pragma unroll
        for (int i = 0; i < kN / 8; ++i) {
          const int piece = half * (kN / 8) + i;
          tc::sts128(sb + L::kS + (piece >> 3) * L::kSBlock + tc::sw128_offset(row, piece & 7),
                     tc::pack2<true>(m * S[8 * i], m * S[8 * i + 1]), tc::pack2<true>(m * S[8 * i + 2], m * S[8 * i + 3]),
                     tc::pack2<true>(m * S[8 * i + 4], m * S[8 * i + 5]), tc::pack2<true>(m * S[8 * i + 6], m * S[8 * i + 7]));
        }
      }
      tc::fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.s_ready);
    }
    if (ok && has_rows && seq.to) {
      float* to = seq.to + at;
#pragma unroll
      for (int i = 0; i < kN; ++i) to[static_cast<int64_t>(i) * a.dv] = S[i];
    }
  } else if (warp == kWarpTma) {
    if (tc::elect_one()) {
      // In the order in which the tiles come free (bf16: the second chunk's Q waits for the
      // first's; f16: R reads Q to its end); a tile's barrier is armed only then, its last
      // load being complete.
      constexpr int kStages[3] = {1, L::kKStages, 2};
      int armed[3] = {0, 0, 0};
      for (int c = 0; c < chunks && ok; ++c) {
        const int t = seq.start + c * kC;
#pragma unroll 1
        for (int i = 0; i < 3 && ok; ++i) {
          const int tile = !BF16 ? 2 - i : c == 1 ? (i + 1) % 3 : i;
          if (!FULL && tile == kTileQ) continue;
          const int stages = tile == kTileQ ? 1 : tile == kTileK ? L::kKStages : 2, st = c & (stages - 1);
          const int blocks = tile == kTileV ? BV / 64 : DK / 64;
          const int x = tile == kTileV ? vb * BV : 0, head = tile == kTileV ? h : hq;
          const CUtensorMap* map = tile == kTileQ ? &map_q : tile == kTileK ? &map_k : &map_v;
          unsigned char* to = smem + (tile == kTileQ ? L::kQ : tile == kTileK ? L::kK + st * L::kKTile : L::kV + st * L::kVTile);
          if (c >= stages && !(ok = wait1(&bar.empty[tile][st], (c / stages - 1) & 1))) break;
          mbar_arrive_expect_tx(&bar.full[tile][st], blocks * kTile);
          for (int b = 0; b < blocks; ++b) tc::tma_load_4d(to + b * kTile, map, x + b * 64, head, t, batch, &bar.full[tile][st]);
          armed[tile] = c + 1;
        }
      }
      // no copy may be in flight when the shared memory is released
#pragma unroll
      for (int tile = 0; tile < 3; ++tile) {
        const int stages = kStages[tile];
        for (int j = max(0, armed[tile] - stages); j < armed[tile]; ++j)
          if (!wait1(&bar.full[tile][j & (stages - 1)], (j / stages) & 1)) ok = false;
      }
    }
  } else if (warp == kWarpGate) {
    // ------------------------------------------------ gates: 4 tokens per lane
    const bool wide = a.g_dtype == GDN_DT_F32;
    const int64_t step = a.g_st * (wide ? 4 : 2);
    const char* at = static_cast<const char*>(a.g) + (batch * a.g_sb + h * a.g_sh) * (wide ? 4 : 2) +
                     (seq.start + lane * 4) * step;
    uint32_t next[4] = {0, 0, 0, 0};
    float x[4], sum = 0.f;
#pragma unroll 1
    for (int c = -1; c < chunks; ++c) {  // a chunk's gates are fetched while the one before is at work
#pragma unroll
      for (int e = 0; e < 4; ++e)
        x[e] = log2_gate(wide                         ? __uint_as_float(next[e])
                         : a.g_dtype == GDN_DT_BF16 ? __uint_as_float(next[e] << 16)
                                                      : __half2float(__ushort_as_half(static_cast<unsigned short>(next[e]))));
      const int left = seq.len - (c + 1) * kC - lane * 4;  // of this lane's tokens of the next chunk
      if (wide) {
#pragma unroll
        for (int e = 0; e < 4; ++e) next[e] = e < left ? __ldg(reinterpret_cast<const uint32_t*>(at + e * step)) : 0;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) next[e] = e < left ? __ldg(reinterpret_cast<const uint16_t*>(at + e * step)) : 0;
      }
      at += kC * step;
      if (c < 0) continue;
      const int st = c & 1;
      float* G = reinterpret_cast<float*>(smem + L::kGate + st * L::kGateStage);
      // G summed from the front; the weights' exponents from the back, so that those
      // near zero are sums of few small numbers and keep their precision
      float fwd[4], bwd[4];
      fwd[0] = x[0];
#pragma unroll
      for (int e = 1; e < 4; ++e) fwd[e] = fwd[e - 1] + x[e];
      bwd[3] = 0.f;
#pragma unroll
      for (int e = 2; e >= 0; --e) bwd[e] = bwd[e + 1] + x[e + 1];
      float before = fwd[3], after = fwd[3];
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const float y = __shfl_up_sync(0xffffffffu, before, off), z = __shfl_down_sync(0xffffffffu, after, off);
        if (lane >= off) before += y;
        if (lane + off < 32) after += z;
      }
      const float end = __shfl_sync(0xffffffffu, before, 31);
      sum += end;
      before = __shfl_up_sync(0xffffffffu, before, 1);
      after = __shfl_down_sync(0xffffffffu, after, 1);
      if (lane == 0) before = 0.f;
      if (lane == 31) after = 0.f;
      if (c >= 2 && !(ok = wait(&bar.gempty[st], ((c >> 1) & 1) ^ 1))) break;
      float gv[4], wv[4], lo = before + fwd[0], hi = lo;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        gv[e] = before + fwd[e];
        wv[e] = c * kC + lane * 4 + e < seq.len ? ex2(after + bwd[e]) : 0.f;
        lo = fminf(lo, gv[e]);
        hi = fmaxf(hi, gv[e]);
      }
      int form = kNear, grow = 0;
      float ref = 0.f;  // kNearBlock: R of this lane's block (8 lanes)
      if (FULL) {
#pragma unroll
        for (int off = 1; off < 8; off <<= 1) {
          lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, off));
          hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, off));
        }
        // (a NaN, which R_b would bring to the earlier rows of its block, fails this; a decay of
        // zero too: behind it nothing of the state may be left, not 2^-kLeast of it either)
        const auto falls = [](float x) { return x <= 0.f && x > kLowest; };
        const bool near_block = __all_sync(0xffffffffu, hi - lo <= kSpan && falls(x[0]) && falls(x[1]) && falls(x[2]) && falls(x[3]));
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, 8));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, 8));
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, 16));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, 16));
        const float end_of_block = __shfl_sync(0xffffffffu, gv[3], lane | 7);
        form = lo >= -kLeast && hi <= kMost ? kNear : near_block ? kNearBlock : kFar;
        if (form == kNearBlock) ref = end_of_block;
        const bool rises = x[0] > 0.f || x[1] > 0.f || x[2] > 0.f || x[3] > 0.f;
        if (!BF16 && __any_sync(0xffffffffu, rises)) {
          float low = fminf(fminf(gv[0], gv[1]), fminf(gv[2], gv[3])), up = 0.f;
#pragma unroll
          for (int off = 1; off < 32; off <<= 1) {
            const float y = __shfl_up_sync(0xffffffffu, low, off);
            if (lane >= off) low = fminf(low, y);
          }
          low = __shfl_up_sync(0xffffffffu, low, 1);
          if (lane == 0) low = gv[0];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            low = fminf(low, gv[e]);
            up = fmaxf(up, gv[e] - low);
          }
          grow = __reduce_max_sync(0xffffffffu, __float2int_ru(fminf(up, 200.f)));
        }
        if (form != kFar) {
#pragma unroll
          for (int e = 0; e < 4; ++e) gv[e] = ex2(ref - gv[e] + (BF16 ? p.pow : 0.f));
        }
      }
      *reinterpret_cast<float4*>(G + lane * 4) = make_float4(gv[0], gv[1], gv[2], gv[3]);
      uint32_t wp[4];
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        if (BF16) {  // the weights of two tokens in two parts: (hi, hi), (lo, lo)
          wp[e] = tc::pack2<BF16>(wv[e], wv[e + 1]);
          wp[e + 1] = tc::pack2<BF16>(wv[e] - tc::unpack_lo<BF16>(wp[e]), wv[e + 1] - tc::unpack_hi<BF16>(wp[e]));
        } else {
          wp[e] = __float_as_uint(wv[e]);
          wp[e + 1] = __float_as_uint(wv[e + 1]);
        }
      }
      *reinterpret_cast<uint4*>(G + kC + lane * 4) = make_uint4(wp[0], wp[1], wp[2], wp[3]);
      if (lane == 0) {
        bar.gamma[st] = ex2(end);
        bar.form[st] = form;
        if (FULL && !BF16) bar.grow[st] = grow;
      }
      if (FULL && (lane & 7) == 7) bar.ref[st][lane >> 3] = ref;
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.gfull[st]);
    }
    if (!FULL && lane == 0 && vb == 0 && chunks) p.decay[static_cast<int64_t>(blockIdx.y) * a.Hv + h] = ex2(sum);
  } else if (FULL && warp == kWarpStore) {
    if (tc::elect_one()) {  // whole chunks of O leave by TMA; V writes a short one
      for (int c = 0; c < chunks && seq.len - c * kC >= kC; ++c) {
        if (!(ok = wait1(&bar.o_staged, c & 1))) break;
        for (int b = 0; b < BV / 64; ++b)
          tc::tma_store_4d(&map_o, smem + L::kO + b * kTile, vb * BV + b * 64, h, seq.start + c * kC, batch);
        bulk_commit();
        bulk_wait_read();
        mbar_arrive(&bar.o_stored);
      }
      bulk_wait_all();
    }
  } else if (warp == kWarpMma && !tc::elect_one()) {
    // the other lanes, for which bar.call holds a chunk that wants clear_values, at last 0
    for (;;) {
      __syncwarp();
      const int c = *static_cast<volatile int*>(&bar.call) - 1;
      if (!FULL || c < 0) break;
      clear_values(smem + L::kV + (c & 1) * L::kVTile, BV, BF16 ? 0x7f80 : 0x7c00, smem + L::kFirst);
    }
  } else if (warp == kWarpMma) {
    // ------------------------------------------------ MMA: the elected lane
    constexpr uint32_t kIdSC = tc::idesc_f16(128, kC, false, false, BF16);
    constexpr uint32_t kIdDS = tc::idesc_f16(128, DK, false, true, BF16);
    constexpr uint32_t kIdQS = tc::idesc_f16(128, BV, false, false, true);
    constexpr uint32_t kIdPV = tc::idesc_f16(128, BV, false, true, BF16);
#pragma unroll 1
    for (int c = 0; c < chunks; ++c) {
      const int st = c & 1, kst = c & (L::kKStages - 1);
      const uint32_t kph = (c / L::kKStages) & 1;
      // step s of an operand lies a constant number of 16-byte units after step 0
      const uint32_t k_at = sb + L::kK + kst * L::kKTile;
      const uint64_t k = tc::kmajor_desc(k_at, kTile, 0);
      const uint64_t kt = tc::mnmajor_desc(k_at, kTile, 0), v = tc::mnmajor_desc(sb + L::kV + st * L::kVTile, kTile, 0);
      const uint64_t sT = tc::kmajor_desc(sb + L::kS, L::kSBlock, 0);
      const auto along = [](int s, int block) { return static_cast<uint64_t>(((s >> 2) * block + (s & 3) * 32) >> 4); };
      const auto add_ds = [&](int half) {  // 64 tokens: the small parts, then the large ones
#pragma unroll
        for (int s = 0; s < 8; ++s)
          tc::mma_tmem_a(kTmDS, (FULL || half ? kTmV : kTmSC) + s * 8, kt + half * 512 + (s & 3) * 128, kIdDS, half || s > 0);
      };
      if constexpr (FULL) {
        ok = wait1(&bar.full[kTileK][kst], kph, &bar.q_ready, c & 1, &bar.pv_done, (c & 1) ^ 1);
        if (!ok) break;
        tc::fence_after_sync();
#pragma unroll
        for (int s = 0; s < DK / 16; ++s)
          tc::mma_tmem_a(kTmSC, kTmQ + s * 8, k + along(s, kTile), kIdSC, s > 0);
        tc::commit(&bar.sc_done);
      }

      ok = wait1(&bar.full[kTileK][kst], kph, &bar.v_ready[0], c & 1, &bar.ds_free, (c & 1) ^ 1);
      if (!ok) break;
      tc::fence_after_sync();
      add_ds(0);
      tc::commit(&bar.v_free[0]);

      if constexpr (FULL && BF16) {
        ok = wait1(&bar.q2_ready, c & 1, &bar.s_ready, c & 1, &bar.o_free, (c & 1) ^ 1);
        if (!ok) break;
        tc::fence_after_sync();
#pragma unroll
        for (int s = 0; s < DK / 16; ++s)
          tc::mma_tmem_a(kTmO, kTmQ + s * 8, sT + along(s, L::kSBlock), kIdQS, s > 0);
        tc::commit(&bar.qs_done);
      }

      ok = wait1(&bar.v_ready[1], c & 1);
      if (!ok) break;
      tc::fence_after_sync();
      add_ds(1);
      tc::commit(&bar.v_free[1]);
      tc::commit(&bar.ds_done);
      if (!BF16) mbar_arrive(&bar.ds_done);  // (hands V's shifts on to S)
      tc::commit(&bar.empty[kTileK][kst]);

      if constexpr (FULL) {
        // seen: bar.bad says whether V holds only finite values
        ok = wait1(&bar.p_ready, c & 1, &bar.seen, c & 1, BF16 ? &bar.p_ready : &bar.o_free, BF16 ? c & 1 : (c & 1) ^ 1);
        if (!ok) break;
        if (*static_cast<volatile int*>(&bar.bad) == c + 1) {
          bar.call = c + 1;
          __syncwarp();
          clear_values(smem + L::kV + st * L::kVTile, BV, BF16 ? 0x7f80 : 0x7c00, smem + L::kFirst);
        }
        tc::fence_after_sync();
#pragma unroll
        for (int s = 0; s < kC / 16; ++s)
          tc::mma_tmem_a(kTmO, kTmSC + s * 8, v + s * 128, kIdPV, BF16 || s > 0);
        tc::commit(&bar.empty[kTileV][st]);
        if constexpr (!BF16) {
          if (!(ok = wait1(&bar.q2_ready, c & 1, &bar.s_ready, c & 1, &bar.s_ready, c & 1))) break;
          tc::fence_after_sync();
#pragma unroll
          for (int s = 0; s < DK / 8; ++s)
            tc::mma_tmem_a_tf32(kTmO, kTmV - DK + s * 8, sT + along(s, L::kSBlock), tc::idesc_tf32(128, BV), true);
          tc::commit(&bar.qs_done);
        }
        tc::commit(&bar.pv_done);
        mbar_arrive(&bar.pv_done);  // (hands kFirst, and in f16 R's shifts, on to V)
      } else {
        tc::commit(&bar.empty[kTileV][st]);
      }
    }
    if (!ok) {  // products in flight end before the tensor memory is released
      tc::commit(&bar.drain);
      wait1(&bar.drain, 0);
    }
    bar.call = 0;
    __syncwarp();
  }
  // a wait ran out: for a free slot, or for what the other warps do
  if (!ok) report(status, warp == kWarpTma || warp == kWarpGate ? GDN_DEVERR_EMPTY_TIMEOUT : GDN_DEVERR_MMA_TIMEOUT);
  __syncwarp();
  tc::fence_before_sync();
  __syncthreads();
  if (warp == kWarpMma) tc::tmem_dealloc(tmem, 512);
}

// The states that the pieces of cut sequences start from: slot j + 1 holds what
// piece j adds, and gets decay_j (slot j) + that; slot 0 the initial state.
__global__ void __launch_bounds__(256) lin_scan_kernel(const __grid_constant__ PrefillParams p) {
  const lin_prefill_args_t& a = p.a;
  pdl_launch_dependents();
  pdl_wait();
  int n = blockIdx.y;
  const int count = slots_of(p, n);
  if (!count) return;
  const int first = find_slot(p, -1, &n);
  if (first + count > p.slots) return;
  const Seq s = find_seq(a, n, false);
  const int64_t page = static_cast<int64_t>(a.Hv) * a.dk * a.dv;
  const int64_t e = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4;
  if (e >= page) return;
  const int h = static_cast<int>(e / (static_cast<int64_t>(a.dk) * a.dv));
  float4 S = make_float4(0.f, 0.f, 0.f, 0.f);
  if (s.page >= 0 && a.initial_state)
    S = *reinterpret_cast<const float4*>(a.initial_state + s.page * a.initial_sp + e);
  float* slot = p.slot_state + first * page + e;
  *reinterpret_cast<float4*>(slot) = S;
  // eight slots at a time: the loads do not wait for one another
  for (int j0 = 0; j0 + 1 < count; j0 += 8) {
    float4 x[8];
    float d[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int j = j0 + i;
      if (j + 1 >= count) break;
      x[i] = *reinterpret_cast<const float4*>(slot + (j + 1) * page);
      d[i] = p.decay[static_cast<int64_t>(first + j) * a.Hv + h];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int j = j0 + i;
      if (j + 1 >= count) break;
      S = make_float4(fmaf(d[i], S.x, x[i].x), fmaf(d[i], S.y, x[i].y), fmaf(d[i], S.z, x[i].z), fmaf(d[i], S.w, x[i].w));
      *reinterpret_cast<float4*>(slot + (j + 1) * page) = S;
    }
  }
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

// How the time axis is cut, and the workspace that takes.
struct Cut {
  int piece = 0, pieces = 0;
  int64_t slots = 0, state_bytes = 0, bytes = 0;
};

int block_cols(const lin_prefill_args_t& a) { return a.dv % 128 == 0 ? 128 : 64; }

Cut choose_cut(const lin_prefill_args_t& a, int sms) {
  Cut cut;
  const int64_t rows = static_cast<int64_t>(a.Hv) * (a.dv / block_cols(a));  // CTAs of one sequence
  const int64_t chunks = (static_cast<int64_t>(a.T) + kC - 1) / kC;
  if (a.cu_seqlens) {
    // Lengths are known on the device only: cut what would keep its CTAs busy for
    // more than half of the time that the whole work takes, and 2048 tokens at least.
    const int64_t share = (chunks * rows + 2 * sms - 1) / (2 * sms);
    const int64_t most = share > 16 ? share : 16;
    // (with many sequences a long one has others beside it)
    if (chunks < (rows * a.B < 4 * sms ? 4 : 8) * most) return cut;
    cut.piece = static_cast<int>(most * kC);
    cut.slots = 2 * (static_cast<int64_t>(a.T) / cut.piece);
  } else {
    // Cost in chunks of time (2.5 us), kStart of them to start a CTA, a piece's state
    // pass kState of a whole one, kScan for the scan and the launches.  Measured in bursts
    // (a call among others 10% more), d = 128, one sequence: 32 heads, 32768 tokens 700 us
    // whole, 317 in 9 pieces (345 in 4, 401 in 7); 8 heads 95 in 18 (146 in 9); 32 heads,
    // 4096 tokens 55 in 4 (70 in 9); two sequences of 8192 (64 CTAs) 172 to 185 in 2 and
    // 190 in 4.
    constexpr double kStart = 2.0, kState = 0.5, kScan = 3.0;
    const auto waves = [&](int64_t ctas) { return static_cast<double>((ctas + sms - 1) / sms); };
    double best = 0.95 * waves(rows * a.B) * (chunks + kStart);
    for (int m = 2; m <= 32 && m <= chunks / 4; ++m) {
      const int64_t len = (chunks + m - 1) / m, used = (chunks + len - 1) / len;
      const double cost = waves(rows * a.B * used) * (len + kStart) + waves(rows * a.B * (used - 1)) * (kState * len + kStart) + kScan;
      if (cost < best) {
        best = cost;
        cut.piece = static_cast<int>(len * kC);
        cut.pieces = static_cast<int>(used);
      }
    }
    cut.slots = static_cast<int64_t>(a.B) * cut.pieces;
  }
  if (!cut.slots || a.B + cut.slots > 65535) return Cut();
  const int64_t page = static_cast<int64_t>(a.Hv) * a.dk * a.dv;
  cut.state_bytes = cut.slots * page * 4;
  cut.bytes = cut.state_bytes + cut.slots * a.Hv * 4;
  return cut;
}

template <int DK, int BV, typename IO>
int launch(const lin_prefill_args_t& a, const Cut& cut, int sms, cudaStream_t stream) {
  constexpr bool bf = std::is_same<IO, __nv_bfloat16>::value;
  using L = Layout<DK, BV, bf, true>;
  using LState = Layout<DK, BV, bf, false>;
  static std::atomic<uint64_t> full_done{0}, state_done{0};
  PrefillParams p;
  p.a = a;
  const int pow = a.scale != 0.f ? ilogbf(a.scale) : 0;
  p.pow = static_cast<float>(pow < -32 ? -32 : pow > 32 ? 32 : pow);
  p.pow2 = exp2f(p.pow);
  p.rest = a.scale / p.pow2;
  p.nvb = a.dv / BV;
  p.piece = cut.piece;
  p.pieces = cut.pieces;
  p.slots = static_cast<int>(cut.slots);
  p.slot_state = static_cast<float*>(a.workspace);
  p.decay = reinterpret_cast<float*>(static_cast<char*>(a.workspace) + cut.state_bytes);
  const int B = a.cu_seqlens ? 1 : a.B;
  CUtensorMap mq, mk, mv, mo;
  int rc;
  if ((rc = io_map(&mq, bf, a.q, DK, a.Hqk, a.T, B, a.q_sh, a.q_st, a.q_sb)) ||
      (rc = io_map(&mk, bf, a.k, DK, a.Hqk, a.T, B, a.k_sh, a.k_st, a.k_sb)) ||
      (rc = io_map(&mv, bf, a.v, a.dv, a.Hv, a.T, B, a.v_sh, a.v_st, a.v_sb)) ||
      (rc = io_map(&mo, bf, a.o, a.dv, a.Hv, a.T, B, a.o_sh, a.o_st, a.o_sb)))
    return rc;
  p.ranked = a.cu_seqlens && a.B > 1 && a.B <= kRanked && static_cast<int64_t>(a.Hv) * p.nvb * a.B > sms;
  const unsigned rows = static_cast<unsigned>(a.Hv * p.nvb), slots = static_cast<unsigned>(cut.slots);
  if (slots) {
    const int64_t page = static_cast<int64_t>(a.Hv) * a.dk * a.dv;
    if ((rc = ensure_smem_attr(lin_prefill_kernel<DK, BV, IO, false>, LState::kBytes, state_done)) ||
        (rc = launch_pdl(lin_prefill_kernel<DK, BV, IO, false>, dim3(rows, slots), kThreads, LState::kBytes, stream, p, mq, mk, mv, mo)) ||
        (rc = launch_pdl(lin_scan_kernel, dim3(static_cast<unsigned>((page + 1023) / 1024), static_cast<unsigned>(a.B)), 256, 0,
                         stream, p)))
      return rc;
  }
  if ((rc = ensure_smem_attr(lin_prefill_kernel<DK, BV, IO, true>, L::kBytes, full_done))) return rc;
  // every sequence of a cut dense batch is cut: only slots then
  const unsigned items = slots + (slots && !a.cu_seqlens ? 0u : static_cast<unsigned>(a.B));
  return launch_pdl(lin_prefill_kernel<DK, BV, IO, true>, dim3(rows, items), kThreads, L::kBytes, stream, p, mq, mk, mv, mo);
}

template <typename IO>
int dispatch(const lin_prefill_args_t& a, const Cut& cut, int sms, cudaStream_t stream) {
  const bool wide = block_cols(a) == 128;
  if (a.dk == 64) return wide ? launch<64, 128, IO>(a, cut, sms, stream) : launch<64, 64, IO>(a, cut, sms, stream);
  return wide ? launch<128, 128, IO>(a, cut, sms, stream) : launch<128, 64, IO>(a, cut, sms, stream);
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
  const bool many = a->pages > 1;  // the stride of an axis of one is free
  if (page > INT32_MAX || (many && (a->final_sp < page || (a->initial_state && a->initial_sp < page)))) return GDN_ERR_SHAPE;
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
      if (size[j] == 1) continue;
      if (st[i][j] < 1 || st[i][j] >= (1ll << 38)) return GDN_ERR_SHAPE;
      if (!stride_ok(st[i][j], 2)) return GDN_ERR_ALIGN;
    }
  }
  if (many && (!stride_ok(a->final_sp, 4) || (a->initial_state && !stride_ok(a->initial_sp, 4)))) return GDN_ERR_ALIGN;
  if (a->initial_state && a->initial_state != a->final_state) {
    if (!pools_disjoint(a->initial_state, a->initial_sp, a->final_state, a->final_sp, page, a->pages)) return GDN_ERR_SHAPE;
  } else if (many && a->initial_state && a->initial_sp != a->final_sp) {
    return GDN_ERR_SHAPE;
  }
  return GDN_OK;
}

}  // namespace
}  // namespace gdn

extern "C" size_t lin_prefill_workspace_size(const lin_prefill_args_t* a) {
  if (gdn::validate(a)) return 0;
  gdn::DeviceInfo di;
  if (gdn::device_info(&di)) return 0;
  return static_cast<size_t>(gdn::choose_cut(*a, di.sm_count).bytes);
}

extern "C" int lin_prefill_launch(const lin_prefill_args_t* a, gdn_stream_t stream) {
  int rc = gdn::validate(a);
  if (rc) return rc;
  gdn::DeviceInfo di;
  if ((rc = gdn::device_info(&di))) return rc;
  const gdn::Cut cut = gdn::choose_cut(*a, di.sm_count);
  if (cut.bytes) {
    if (!a->workspace || a->workspace_bytes < static_cast<size_t>(cut.bytes)) return GDN_ERR_WORKSPACE;
    if (!gdn::aligned16(a->workspace)) return GDN_ERR_ALIGN;
  }
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return a->io_dtype == GDN_DT_BF16 ? gdn::dispatch<__nv_bfloat16>(*a, cut, di.sm_count, st) : gdn::dispatch<__half>(*a, cut, di.sm_count, st);
}
