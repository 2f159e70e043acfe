// flash_bwd_sm100.cu -- flashAttentionBackward (attention.metal:198-299) on
// sm_100a with tcgen05 UMMA, TMEM accumulators and TMA.
//
// Work unit, as in the reference (attention.metal:219-223): one 128-key tile
// of one (batch, head), walking the query tiles i from the diagonal to the end
// (causal: earlier queries never see these keys).  Per query tile (128
// queries):
//   S^T  = K Q_i^T                 UMMA 128x128xD  -> TMEM
//   dP^T = V dO_i^T                UMMA 128x128xD  -> TMEM
//   P^T  = exp2(S^T c - l_i log2e), 0 where key > query   (compute warps)
//   dS^T = P^T (dP^T - D_i) / sqrt(D)                       (compute warps)
//   dV  += P^T dO_i                UMMA 128xDx128  (TMEM-resident)
//   dK  += dS^T Q_i                UMMA 128xDx128  (TMEM-resident)
//   dQ_i = dS K                    UMMA 128xDx128  -> TMEM -> smem -> TMA
//                                  bulk reduce-add into fp32 dQ in global
// dS^T is written once to shared memory (bf16, K-major 128-byte swizzle); the
// dQ UMMA reads the same buffer as an MN-major operand.  At D=64, P^T goes to
// TMEM (bf16 pairs) and dV's UMMA takes it from there; at D=128 TMEM is full
// and P^T goes to shared memory like dS^T.  dK/dV are owned by the unit and
// stored once (bf16, straight from registers to global memory); dQ is
// accumulated in fp32 by the bulk reductions of every key tile into zeros:
// the launcher writes them first, unless the caller passes a dQ that already
// holds them (the accumulating entry point; the reference's host zeroes dQ,
// model.h:549).
//
// Scheduling: units are ordered in blocks of HB (batch, head) pairs, within
// a block by key tile (heaviest first), then head; HB = 1 is (batch,
// head)-major.  Short sequences at D=64 (PERSIST): one CTA per SM, HB = 1,
// units dealt in rounds of gridDim.x in alternating direction (CTA c takes
// position c in even rounds and gridDim.x-1-c in odd ones), so the units of
// a head start together and walk different query tiles, and the units in
// flight share a few heads' Q/dO in L2.  Longer sequences, whose units differ
// more in size: one CTA per unit; a running CTA takes its own unit and then,
// by cluster launch control, the units of CTAs that have not started yet, in
// launch order, so units go greedily to whichever SM is free.  Either way a
// unit's dK/dV epilogue runs after the next unit's first step has been handed
// to the tensor core.  At D=64 K/V are double-buffered, so the next unit's
// K/V, Q/dO tiles and first S^T/dP^T are fetched and computed while the
// current unit finishes; at D=128 (one K/V buffer) the next unit's K/V load
// and first S^T/dP^T wait for the current unit's last products.  (PERSIST,
// the template argument, selects the static schedule.)
//
// Roles (384 threads, three warpgroups):
//   warpgroup 0 (120 registers per thread after setmaxnreg):
//     warp 0   TMA producer: K/V per unit, Q_i/dO_i into a STAGES-deep ring
//     warp 1   TMEM owner; lane 0 issues every UMMA and commit
//     warp 2   statistics: -l_i*log2(e) and -D_i/sqrt(D) per query (strided
//              in global memory), loaded into registers a step ahead and
//              staged in shared memory for the compute warps
//     warp 3   lane 0 issues the dQ bulk reductions
//   warpgroups 1, 2 (192 registers): compute, thread = key row = TMEM lane;
//              warpgroup 1 takes query columns 0-63, warpgroup 2 columns
//              64-127; the dK/dV epilogue (each thread stores its key row's
//              slice of its part's columns) and, at D=128, the dQ drain into
//              the staging buffer.
// At D=64 a fourth warpgroup (warps 12-15, 64 registers) drains dQ, and the
// CTA has 512 threads (warpgroup 0 80 registers, compute 184).
// D=64 schedule ("early S"): S^T/dP^T of the next query tile are issued as
// soon as the compute warps have read the current one, so they run on the
// tensor core while the compute warps form P^T/dS^T; dV, dK and dQ follow, and
// dQ of a tile is drained after the next tile is handed over.  D=128 has no
// TMEM room for that (S^T, dP^T, dV, dK fill all 512 columns; dQ reuses the
// S^T columns) and runs the steps in order, draining dQ before the next S^T.
//
// Conventions as the reference: P = exp(S/sqrt(D) - l) with l read as stored,
// D read as stored (bf16), dS includes 1/sqrt(D).  The reference rounds S,
// dP, P, dS and the dQ tile to bf16 and accumulates dK/dV in bf16 memory;
// here S, dP, dQ and dK/dV stay fp32 until their single store, and P, dS are
// bf16 (the UMMA operand type).
//
// WIN: the same kernel for windowAttentionBackward (sliding window, sinks,
// grouped K/V heads, sequence lengths).  A unit is a key tile of a K/V head;
// its steps are the query tiles that can see it, for each query head of the
// group, so shared heads' gradients are summed in the accumulators.  A sink
// tile is seen by every later query: what lies past its window is cut into
// units of their own where that chain would be the longest (WinBwd), whose
// partial dK/dV the launcher's last kernel adds up in a fixed order.  The
// statistics come ready from a kernel before this one, [B][NH][T], and the
// warp that stages them also zeroes the padding rows of Q, dO, K and V tiles
// (their P is 0, but 0 * NaN is not).  A unit or chunk without a
// valid row runs one step in which everything is masked and so writes zeros.
//
// All mbarrier waits are bounded (about 2 s); on time-out the CTA winds down,
// frees its TMEM and sets STATUS_BWD_TIMEOUT.  Warps meet only at mbarriers
// (no named barriers), so a failed wait cannot leave a warp stuck at one.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "sm100.cuh"
#include "tmap.h"

namespace ma {
namespace {

using namespace sm100;

constexpr int BK = 128;  // keys per unit
constexpr int BQ = 128;  // queries per step
constexpr int PERSIST_MAX_NKT = 16;  // static schedule when T/128 <= this (D=64)
constexpr float LOG2E = 1.4426950408889634f;


template <int HD, bool PERSIST, bool WIN = false>
struct BwdCfg {
  static constexpr int KB = HD / 64;
  static constexpr bool D64 = HD == 64;
  // Compute warpgroups: each takes BQ / NPART query columns of every step.
  // D=64 with NPART=2: a fourth warpgroup drains dQ (register split per
  // thread after setmaxnreg: warpgroup 0 80, compute 184, drain 64).
  // Otherwise the compute warpgroups also drain dQ, each its share of the
  // columns: D=64 with NPART=4 (640 threads; 64 / 104; measured slower and
  // not used), D=128 (384 threads; 120 / 192).
  static constexpr int NPART = 2;
  static constexpr int CPP = BQ / NPART;       // query columns per part
  static constexpr int NCOMP = 128 * NPART;    // compute threads
  static constexpr bool DRAIN_WG = D64 && NPART == 2;
  static constexpr int NUM_THREADS = 128 + NCOMP + (DRAIN_WG ? 128 : 0);
  static constexpr int LAUNCH_REGS = (65536 / NUM_THREADS) & ~7;  // registers per thread at launch
  static constexpr int REGS_PRODUCER = NPART == 4 ? 64 : (DRAIN_WG ? 80 : 120);
  static constexpr int REGS_DRAIN = DRAIN_WG ? 64 : 0;
  static constexpr int REGS_COMPUTE =
      ((NUM_THREADS * LAUNCH_REGS - 128 * REGS_PRODUCER - 128 * REGS_DRAIN) / NCOMP) & ~7;
  static constexpr int NDRAIN = DRAIN_WG ? 128 : NCOMP;  // arrivals on DQE, DSF
  // The unit's dK/dV epilogue (TMEM -> bf16 -> global memory) is run by the
  // compute warps, each part its columns, once they have handed the next
  // unit's first step to the tensor core: they would otherwise wait there for
  // the step's products, and with all of them the accumulators are released
  // sooner than by the drain warpgroup alone.
  static constexpr bool EPI_COMPUTE = true;
  static_assert(EPI_COMPUTE, "the drain warpgroup drains dQ only");
  static constexpr int NACC = EPI_COMPUTE ? NCOMP : NDRAIN;  // arrivals on ACC
  static_assert(128 * REGS_PRODUCER + NCOMP * REGS_COMPUTE + 128 * REGS_DRAIN <=
                    NUM_THREADS * LAUNCH_REGS,
                "register split must fit the launch allocation");
  static_assert(CPP % 16 == 0 && (HD / NPART) % 16 == 0, "column split");
  // Q_i/dO_i stages and K/V buffers: at D=64 K/V are double-buffered to
  // prefetch the next unit (under launch control too, where a CTA also runs
  // many units: C4 backward 3.75 -> 3.64 ms against one K/V buffer and three
  // Q/dO stages); D=128 has room for one of each
  static constexpr int STAGES = D64 ? (WIN ? 3 : 2) : 1;
  static constexpr int KVB = D64 ? 2 : 1;
  static constexpr bool P_IN_TMEM = D64;         // P^T in TMEM (else smem)
  static constexpr bool EARLY_S = D64;           // next S^T before dV/dK/dQ
  static constexpr bool DQ_ALIAS = !D64;         // dQ accumulator reuses the S^T columns
  static constexpr bool DQS_ALIAS = !D64;        // dQ staging reuses the P^T/dS^T smem
  // dQ staging buffers (the code allows more than one; a second buffer was
  // measured slower: the extra shared-memory traffic in flight slows the
  // tensor core's operand reads more than the overlap gains).  Statistics
  // ring stages: the statistics warp loads a step's values into registers a
  // step ahead, so one stage suffices where the shared memory is tight.
  static constexpr int DQSB = 1;
  static constexpr int SSTG = D64 && (PERSIST || WIN) ? 1 : 8;
  // WIN at D=64 has the most code in flight, and fetching it stalls the warps
  // more than the UMMA issuer's loops do
  static constexpr int UMMA_UNROLL = WIN && D64 ? 1 : 8;
  static constexpr uint32_t KV_BYTES = BK * HD * 2;
  static constexpr uint32_t QD_BYTES = BQ * HD * 2;
  static constexpr uint32_t PT_BYTES = BK * BQ * 2;
  static constexpr uint32_t DQS_BYTES = BQ * HD * 4;
  static constexpr uint32_t STAT_BYTES = 2 * BQ * 4;  // -l*log2e[128], -D/sqrt(D)[128]
  static constexpr uint32_t OFF_K = 0;                                // [KVB]
  static constexpr uint32_t OFF_V = OFF_K + KVB * KV_BYTES;           // [KVB]
  static constexpr uint32_t OFF_Q = OFF_V + KVB * KV_BYTES;           // [STAGES]
  static constexpr uint32_t OFF_DO = OFF_Q + STAGES * QD_BYTES;       // [STAGES]
  static constexpr uint32_t OFF_PT = OFF_DO + STAGES * QD_BYTES;      // only without P_IN_TMEM
  static constexpr uint32_t OFF_DST = OFF_PT + (P_IN_TMEM ? 0 : PT_BYTES);
  static constexpr uint32_t OFF_DQS = DQS_ALIAS ? OFF_PT : OFF_DST + PT_BYTES;  // [DQSB]
  static constexpr uint32_t OFF_STAT = DQS_ALIAS ? OFF_DST + PT_BYTES : OFF_DQS + DQSB * DQS_BYTES;
  // the unit schedule: NSCHED 16-byte launch-control responses, read by the
  // producer, the UMMA issuer (twice: its look-ahead and current steps), the
  // statistics and reduce warps, and every compute and drain warp
  static constexpr bool DYN = !PERSIST;  // units taken by launch control
  // (batch, head) pairs per block of the unit order (measured: D=128 gains
  // from 16, D=64 at long sequences is fastest (batch, head)-major)
  static constexpr int HB = (DYN && !D64) ? 16 : 1;
  static constexpr int NSCHED = DYN ? (int)kSchedSlots : 0;
  static constexpr uint32_t SCHED_READERS = 5 + NCOMP / 32 + (DRAIN_WG ? 4 : 0);
  static constexpr uint32_t OFF_SCHED = OFF_STAT + SSTG * STAT_BYTES;
  // WIN: the units' descriptors (unit 0's after those of the responses' slots),
  // decoded once, by the producer
  static constexpr int NDESC = WIN ? NSCHED + 1 : 0;
  static constexpr uint32_t DESC_BYTES = 48;
  static constexpr uint32_t OFF_DESC = OFF_SCHED + NSCHED * 16;
  static constexpr uint32_t OFF_BAR = OFF_DESC + NDESC * DESC_BYTES;
  // kv_full/empty[KVB], qd_full/empty[S], st_full/empty[8], then s_full,
  // s_free, p_ready, p_free, dq_full, dq_free, dqs_full, dqs_free, done,
  // acc_free, never (nothing arrives: the time-out test hook), fin (the
  // UMMA issuer's wind-down), sched_full/empty[NSCHED] and, for WIN,
  // qd_fixed[S] (padding rows zeroed) and desc_full[NDESC]
  static constexpr int NBAR = 2 * KVB + 2 * STAGES + 2 * SSTG + 12 + 2 * (DQSB - 1) + 2 * NSCHED + (WIN ? STAGES : 0) + NDESC;
  static constexpr uint32_t OFF_TSLOT = OFF_BAR + NBAR * 8;
  static constexpr uint32_t SMEM_BYTES = OFF_TSLOT + 16 + 1024;
  static constexpr uint32_t TCOL_S = 0;
  static constexpr uint32_t TCOL_DP = 128;
  static constexpr uint32_t TCOL_DV = 256;
  static constexpr uint32_t TCOL_DK = 256 + HD;
  static constexpr uint32_t TCOL_DQ = DQ_ALIAS ? 0 : 256 + 2 * HD;
  static constexpr uint32_t TCOL_PT = 256 + 3 * HD;  // D=64 only: 64 columns of bf16 pairs
};

// What the window adds.  Sink tiles 0 .. nsplit-1 are split: their query
// tiles past the window go, far_tiles at a time, to nfar units each; unit
// `slot`s of part hold 2 x 128 x D fp32 partial sums (dV, dK), slot 0 of a
// tile its window's.
struct WinBwd {
  const int32_t* lens;
  int G, window, sinks;
  int nsplit, nfar, far_tiles;
  int nfar_units;              // nsplit * nfar * (batch, K/V head) pairs, dealt first
  int rows;                    // rows of a (batch, head) in the statistics
  const float *neg_l, *neg_d;  // -l*log2e, -D/sqrt(D)
  float* part;
};

struct BwdParams {
  int T, N, NH, bh_begin, nbh, nkt, nunits;
  float scale, scale_log2;
  const float* lse;
  const __nv_bfloat16* Dv;
  uint32_t* status;
  uint32_t expire_ns;  // time-out test hook (ma_debug_expire_next_wait), 0 = off
  WinBwd win;          // WIN only
};

// Unit k -> (batch, head, key tile); its query tiles are kt .. nkt-1.  Block
// k / (HB * nkt) holds the units of HB (batch, head) pairs (fewer in the last
// block), key tile-major; HB = 1 is (batch, head)-major.
struct BUnit {
  int b, h, kt, nq;
  __device__ int q_tile(int i) const { return kt + i; }
  __device__ int q_head(int) const { return h; }
};

// A unit under a window: nt query tiles from q0 on, for each query head.
// (48 bytes: it is passed on through shared memory.)
struct alignas(16) WinBUnit {
  int b, h, kt, nq;
  int q0, nt, head0;
  int n;     // valid rows; 0 where the unit has none: everything is masked
  int slot;  // partial sums go to this slot, or -1: straight to dK, dV
  int valid; // 0: no unit is left
  int pad[2];
  __device__ int q_tile(int i) const { return q0 + i % nt; }
  __device__ int q_head(int i) const { return head0 + i / nt; }
  // key `key` sees queries [*from, *to) of the query tile at row0
  __device__ void seen(const WinBwd& w, int key, int row0, int* from, int* to) const {
    *from = key - row0;
    *to = (key < w.sinks ? n : min(n, key + w.window)) - row0;
  }
};

template <int HB>
__device__ __forceinline__ BUnit bwd_unit(const BwdParams& prm, int k) {
  BUnit u;
  int bh;
  if constexpr (HB > 1) {
    const int per = HB * prm.nkt;
    const int blk = k / per, r = k % per;
    const int hb = min(HB, prm.nbh - blk * HB);
    bh = prm.bh_begin + blk * HB + r % hb;
    u.kt = r / hb;
  } else {
    bh = prm.bh_begin + k / prm.nkt;
    u.kt = k % prm.nkt;
  }
  u.b = bh / prm.NH;
  u.h = bh % prm.NH;
  u.nq = prm.nkt - u.kt;
  return u;
}

template <int HB>
__device__ __forceinline__ WinBUnit bwd_win_unit(const BwdParams& prm, int k) {
  const WinBwd& w = prm.win;
  WinBUnit u;
  const bool far = k < w.nfar_units;
  int c = 0;
  if (far) {
    const int bh = k % prm.nbh, r = k / prm.nbh;
    u.b = bh / prm.NH;
    u.h = bh % prm.NH;
    u.kt = r % w.nsplit;
    c = r / w.nsplit;
  } else {
    const BUnit p = bwd_unit<HB>(prm, k - w.nfar_units);
    u.b = p.b;
    u.h = p.h;
    u.kt = p.kt;
  }
  u.head0 = u.h * w.G;
  u.n = w.lens ? min(max(__ldg(w.lens + u.b), 0), prm.T) : prm.T;
  const bool split = u.kt < w.nsplit;
  u.slot = split ? ((u.b * prm.NH + u.h) * w.nsplit + u.kt) * (1 + w.nfar) + (far ? 1 + c : 0) : -1;
  const int k0 = u.kt * BK;
  const int last = (u.n - 1) / BQ;                     // the last query tile with a valid row
  const int win_last = (k0 + BK - 1 + w.window - 1) / BQ;  // and the last in the window
  u.q0 = far ? win_last + 1 + c * w.far_tiles : u.kt;
  int end = last;
  if (far) end = min(last, u.q0 + w.far_tiles - 1);
  else if (split || k0 >= w.sinks) end = min(last, win_last);
  u.nt = end - u.q0 + 1;
  u.nq = u.nt * w.G;
  if (u.nt <= 0 || u.n <= k0) {
    u.n = 0;
    u.q0 = u.kt;
    u.nt = u.nq = 1;
  }
  return u;
}

// The descriptors' ring: unit 0 in slot kSchedSlots, unit g in the slot of the
// response that named it, which the readers release together.
struct UnitRing {
  WinBUnit* desc;
  uint32_t full;  // slot 0's barrier
};

// Static schedule: the unit of this CTA in round g, -1 when rounds are
// exhausted, -2 when this CTA has none in round g (last, partial round).
__device__ __forceinline__ int bwd_unit_of_round(const BwdParams& prm, int g) {
  const int G = gridDim.x;
  if ((long long)g * G >= prm.nunits) return -1;
  const int c = blockIdx.x;
  const int k = g * G + ((g & 1) ? G - 1 - c : c);
  return k < prm.nunits ? k : -2;
}

// Walks this CTA's (unit, query tile) steps in order.  t counts steps over
// all units, uc counts units.
template <bool WIN>
struct StepIter {
  int g;        // dynamic: units fetched; static: next round to look at
  std::conditional_t<WIN, WinBUnit, BUnit> u;
  int i;        // step within the unit
  uint32_t t;   // global step
  uint32_t uc;  // unit counter
  bool valid;
};

// PUBLISH (WIN's producer): decodes the unit and passes it on; WIN's other
// roles read it (the code of twenty decodings would not fit the instruction
// cache).
template <bool DYN, int HB, bool WIN, bool WARP, bool PUBLISH = false>
__device__ __forceinline__ bool next_unit(const BwdParams& prm, StepIter<WIN>& s, const Sched& sc, const UnitRing& ur) {
  if constexpr (WIN && PUBLISH) {
    const uint32_t g = (uint32_t)s.g++;
    const int k = sched_unit<WARP>(sc, g);
    const bool some = k >= 0 && k < prm.nunits;
    if (some) s.u = bwd_win_unit<HB>(prm, k);
    s.u.valid = some;
    const uint32_t slot = g == 0 ? kSchedSlots : (g - 1) % kSchedSlots;
    ur.desc[slot] = s.u;
    mbar_arrive(ur.full + 8u * slot);
    return some;
  } else if constexpr (WIN) {
    const uint32_t g = (uint32_t)s.g++;
    const uint32_t slot = g == 0 ? kSchedSlots : (g - 1) % kSchedSlots;
    const uint32_t ph = g == 0 ? 0u : ((g - 1) / kSchedSlots) & 1u;
    if (!(WARP ? mbar_wait_warp(ur.full + 8u * slot, ph, sc.abort) : mbar_wait(ur.full + 8u * slot, ph, sc.abort)))
      return false;
    s.u = ur.desc[slot];
    if (g > 0) {
      if (WARP) __syncwarp();
      if (!WARP || (threadIdx.x & 31) == 0) mbar_arrive(sc.empty + 8u * slot);
    }
    return s.u.valid != 0;
  } else if constexpr (DYN) {
    const int k = sched_unit<WARP>(sc, (uint32_t)s.g++);
    if (k < 0 || k >= prm.nunits) return false;
    s.u = bwd_unit<HB>(prm, k);
    return true;
  } else {
    for (;;) {
      const int k = bwd_unit_of_round(prm, s.g);
      if (k == -1) return false;
      ++s.g;
      if (k >= 0) {
        s.u = bwd_unit<HB>(prm, k);
        return true;
      }
    }
  }
}

template <bool DYN, int HB, bool WIN, bool WARP, bool PUBLISH = false>
__device__ __forceinline__ StepIter<WIN> first_step(const BwdParams& prm, const Sched& sc, const UnitRing& ur) {
  StepIter<WIN> s;
  s.g = 0;
  s.i = 0;
  s.t = 0;
  s.uc = 0;
  s.valid = next_unit<DYN, HB, WIN, WARP, PUBLISH>(prm, s, sc, ur);
  return s;
}

template <bool DYN, int HB, bool WIN, bool WARP, bool PUBLISH = false>
__device__ __forceinline__ void advance(const BwdParams& prm, StepIter<WIN>& s, const Sched& sc, const UnitRing& ur) {
  ++s.t;
  if (s.i + 1 < s.u.nq) {
    ++s.i;
    return;
  }
  s.i = 0;
  ++s.uc;
  s.valid = next_unit<DYN, HB, WIN, WARP, PUBLISH>(prm, s, sc, ur);
}

// P^T and dS^T for N query columns of one key row.  s[] holds S^T on entry
// and P^T on exit; dp[] holds dP^T on entry and dS^T on exit.  nl = -l*log2e
// and nd = -D/sqrt(D) per query column (shared memory, broadcast reads).
// SEEN (a window's step): bit j of see[] says whether query column j is visible;
// else P and with it dS are 0 (padding rows hold zeros, so dP is finite).
template <bool DIAG, int N, bool SEEN = false>
__device__ __forceinline__ void p_ds_row(float (&s)[N], float (&dp)[N], const float* nl,
                                         const float* nd, float c, float sc, int krow, int qcol0,
                                         const uint32_t* see = nullptr) {
  const float2 c2 = make_float2(c, c), sc2 = make_float2(sc, sc);
#pragma unroll
  for (int j = 0; j < N; j += 4) {
    const float4 L = *reinterpret_cast<const float4*>(nl + j);
    const float4 Dn = *reinterpret_cast<const float4*>(nd + j);
    const float2 t0 = __ffma2_rn(make_float2(s[j], s[j + 1]), c2, make_float2(L.x, L.y));
    const float2 t1 = __ffma2_rn(make_float2(s[j + 2], s[j + 3]), c2, make_float2(L.z, L.w));
    float p0 = ex2(t0.x), p1 = ex2(t0.y), p2 = ex2(t1.x), p3 = ex2(t1.y);
    if constexpr (SEEN) {
      const uint32_t m = see[j / 32] >> (j % 32);
      if (!(m & 1u)) p0 = 0.0f;
      if (!(m & 2u)) p1 = 0.0f;
      if (!(m & 4u)) p2 = 0.0f;
      if (!(m & 8u)) p3 = 0.0f;
    }
    if (DIAG) {  // key after query: P = 0 (attention.metal:282)
      const int q = qcol0 + j;
      if (krow > q) p0 = 0.0f;
      if (krow > q + 1) p1 = 0.0f;
      if (krow > q + 2) p2 = 0.0f;
      if (krow > q + 3) p3 = 0.0f;
    }
    const float2 d0 = __ffma2_rn(make_float2(dp[j], dp[j + 1]), sc2, make_float2(Dn.x, Dn.y));
    const float2 d1 = __ffma2_rn(make_float2(dp[j + 2], dp[j + 3]), sc2, make_float2(Dn.z, Dn.w));
    const float2 r0 = __fmul2_rn(make_float2(p0, p1), d0);
    const float2 r1 = __fmul2_rn(make_float2(p2, p3), d1);
    s[j] = p0;
    s[j + 1] = p1;
    s[j + 2] = p2;
    s[j + 3] = p3;
    dp[j] = r0.x;
    dp[j + 1] = r0.y;
    dp[j + 2] = r1.x;
    dp[j + 3] = r1.y;
  }
}

// N bf16 values of one row as N/8 swizzled 16-byte chunks of a K-major SW128
// row, starting at chunk ch0 (row base `rowp`, swizzle phase `row & 7`).
template <int N>
__device__ __forceinline__ void store_row_sw128(uint8_t* rowp, int row, const float (&v)[N], int ch0) {
#pragma unroll
  for (int k = 0; k < N / 8; ++k) {
    const int c0 = k * 8, ch = ch0 + k;
    uint4 w;
    w.x = pack_bf16(v[c0 + 0], v[c0 + 1]);
    w.y = pack_bf16(v[c0 + 2], v[c0 + 3]);
    w.z = pack_bf16(v[c0 + 4], v[c0 + 5]);
    w.w = pack_bf16(v[c0 + 6], v[c0 + 7]);
    *reinterpret_cast<uint4*>(rowp + ((ch ^ (row & 7)) * 16)) = w;
  }
}

template <int HD, bool PERSIST, bool WIN>
__global__ void __launch_bounds__(BwdCfg<HD, PERSIST, WIN>::NUM_THREADS, 1)
    flash_bwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                     const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmdO,
                     const __grid_constant__ CUtensorMap tmdQ, __nv_bfloat16* __restrict__ dK,
                     __nv_bfloat16* __restrict__ dV, const BwdParams prm) {
  if constexpr (!WIN) pdl_wait_and_release();  // WIN: after the set-up below
  using C = BwdCfg<HD, PERSIST, WIN>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ int abort_flag;
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t sbase = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (sbase - raw);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  const uint32_t bar0 = sbase + C::OFF_BAR;
  auto BAR_KF = [&](int s) { return bar0 + 8u * s; };
  auto BAR_KE = [&](int s) { return bar0 + 8u * (C::KVB + s); };
  auto BAR_QF = [&](int s) { return bar0 + 8u * (2 * C::KVB + s); };
  auto BAR_QE = [&](int s) { return bar0 + 8u * (2 * C::KVB + C::STAGES + s); };
  auto BAR_TF = [&](int s) { return bar0 + 8u * (2 * C::KVB + 2 * C::STAGES + s); };
  auto BAR_TE = [&](int s) { return bar0 + 8u * (2 * C::KVB + 2 * C::STAGES + C::SSTG + s); };
  const uint32_t BAR_SF = bar0 + 8u * (2 * C::KVB + 2 * C::STAGES + 2 * C::SSTG);
  const uint32_t BAR_SE = BAR_SF + 8;
  const uint32_t BAR_PR = BAR_SF + 16;
  const uint32_t BAR_PE = BAR_SF + 24;
  const uint32_t BAR_DQF = BAR_SF + 32;
  const uint32_t BAR_DQE = BAR_SF + 40;
  // staging buffer b: BAR_DSF(b) written, BAR_DSE(b) read by its reduction
  auto BAR_DSF = [&](int b) { return b == 0 ? BAR_SF + 48 : BAR_SF + 96 + 16u * (b - 1); };
  auto BAR_DSE = [&](int b) { return b == 0 ? BAR_SF + 56 : BAR_SF + 104 + 16u * (b - 1); };
  const uint32_t BAR_DONE = BAR_SF + 64;  // a unit's last UMMA completed
  const uint32_t BAR_ACC = BAR_SF + 72;   // dK/dV TMEM read by the epilogue
  const uint32_t BAR_NEVER = BAR_SF + 80; // nothing arrives (time-out test hook)
  const uint32_t BAR_FIN = BAR_SF + 88;   // the UMMA issuer's last commit (wind-down)
  const uint32_t BAR_UF = BAR_SF + 96 + 16u * (C::DQSB - 1);  // sched_full[NSCHED], then sched_empty
  const uint32_t BAR_UE = BAR_UF + 8u * C::NSCHED;
  auto BAR_QZ = [&](int s) { return BAR_UE + 8u * (C::NSCHED + s); };  // WIN: padding rows of stage s zeroed
  const uint32_t tslot = sbase + C::OFF_TSLOT;
  float* stat_base = reinterpret_cast<float*>(gbase + C::OFF_STAT);

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < C::KVB; ++s) {
      mbar_init(BAR_KF(s), 1);
      mbar_init(BAR_KE(s), WIN ? 2 : 1);  // WIN: the warp that zeroes rows, too
    }
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(BAR_QF(s), 1);
      mbar_init(BAR_QE(s), WIN ? 2 : 1);
      if constexpr (WIN) mbar_init(BAR_QZ(s), 1);
    }
    for (int s = 0; s < C::SSTG; ++s) {
      mbar_init(BAR_TF(s), 32);
      mbar_init(BAR_TE(s), C::NCOMP);
    }
    mbar_init(BAR_SF, 1);
    mbar_init(BAR_SE, C::NCOMP);
    mbar_init(BAR_PR, C::NCOMP);
    mbar_init(BAR_PE, 1);
    mbar_init(BAR_DQF, 1);
    mbar_init(BAR_DQE, C::NDRAIN);
    for (int b = 0; b < C::DQSB; ++b) {
      mbar_init(BAR_DSF(b), C::NDRAIN);
      mbar_init(BAR_DSE(b), 1);
    }
    mbar_init(BAR_DONE, 1);
    mbar_init(BAR_ACC, C::NACC);
    mbar_init(BAR_NEVER, 1);
    mbar_init(BAR_FIN, 1);
    for (int u = 0; u < C::NSCHED; ++u) {
      mbar_init(BAR_UF + 8u * u, 1);
      mbar_init(BAR_UE + 8u * u, C::SCHED_READERS);
    }
    for (int u = 0; u < C::NDESC; ++u) mbar_init(BAR_QZ(C::STAGES + u), 1);  // desc_full
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tslot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // nothing before here touches global memory, so the barriers and TMEM are set
  // up while the kernel before is still draining
  if constexpr (WIN) pdl_wait_and_release();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(gbase + C::OFF_TSLOT);
  volatile int* abort_p = &abort_flag;
  const Sched sch{sbase + C::OFF_SCHED, BAR_UF, BAR_UE, abort_p};  // the unit schedule
  const UnitRing ring{reinterpret_cast<WinBUnit*>(gbase + C::OFF_DESC), BAR_QZ(C::STAGES)};

  // WIN: whether step s brings tiles with padding rows (a unit's first step:
  // its K tile too); past the tensor's end TMA has filled in zeros itself
  auto fix_q = [&](const StepIter<WIN>& s) {
    if constexpr (WIN) return s.u.n < prm.T && s.u.q_tile(s.i) * BQ + BQ > s.u.n;
    else return false;
  };
  auto fix_k = [&](const StepIter<WIN>& s) {
    if constexpr (WIN) return s.i == 0 && s.u.n < prm.T && s.u.kt * BK + BK > s.u.n;
    else return false;
  };

  if (warp < 4) {
    reg_dealloc<C::REGS_PRODUCER>();
    if (warp == 0) {
      // --------------------------------------------------------- producer
      if (lane == 0) {
        tma_prefetch_desc(&tmQ);
        tma_prefetch_desc(&tmdO);
        uint32_t kv_armed = 0, q_armed = 0;  // loads issued into each ring
        uint32_t nreq = 0;                   // launch-control requests issued
        for (StepIter<WIN> s = first_step<C::DYN, C::HB, WIN, false, true>(prm, sch, ring); s.valid; advance<C::DYN, C::HB, WIN, false, true>(prm, s, sch, ring)) {
          const int kv0 = s.u.h * HD, col0 = s.u.q_head(s.i) * HD;
          if (s.i == 0) {  // K/V of a new unit
            const int kvs = s.uc % C::KVB;
            if (s.uc >= C::KVB && !mbar_wait(BAR_KE(kvs), ((s.uc / C::KVB) - 1) & 1, abort_p)) break;
            mbar_arrive_expect_tx(BAR_KF(kvs), 2 * C::KV_BYTES);
            ++kv_armed;
            for (int kb = 0; kb < C::KB; ++kb) {
              tma_load_3d(sbase + C::OFF_K + kvs * C::KV_BYTES + kb * BK * 128, &tmK, BAR_KF(kvs),
                          kv0 + kb * 64, s.u.kt * BK, s.u.b);
              tma_load_3d(sbase + C::OFF_V + kvs * C::KV_BYTES + kb * BK * 128, &tmV, BAR_KF(kvs),
                          kv0 + kb * 64, s.u.kt * BK, s.u.b);
            }
          }
          const int st = s.t % C::STAGES;
          if (s.t >= C::STAGES && !mbar_wait(BAR_QE(st), ((s.t / C::STAGES) - 1) & 1, abort_p)) break;
          const int qt = s.u.q_tile(s.i);
          mbar_arrive_expect_tx(BAR_QF(st), 2 * C::QD_BYTES);
          ++q_armed;
          for (int kb = 0; kb < C::KB; ++kb) {
            tma_load_3d(sbase + C::OFF_Q + st * C::QD_BYTES + kb * BQ * 128, &tmQ, BAR_QF(st),
                        col0 + kb * 64, qt * BQ, s.u.b);
            tma_load_3d(sbase + C::OFF_DO + st * C::QD_BYTES + kb * BQ * 128, &tmdO, BAR_QF(st),
                        col0 + kb * 64, qt * BQ, s.u.b);
          }
          // three steps before the unit's end (or at its start), ask for the
          // next unit, so that every reader finds the answer when it gets there
          if (C::DYN && s.i == max(0, s.u.nq - 3)) {
            if (!sched_request(sch, nreq)) break;
            ++nreq;
          }
        }
        if (*abort_p) {  // wind-down: let the loads and the request still in flight land
          if (C::DYN) sched_drain(sch, nreq);
          drain_ring(BAR_KF, C::KVB, kv_armed);
          drain_ring(BAR_QF, C::STAGES, q_armed);
        }
      }
    } else if (warp == 1) {
      // -------------------------------------------------------------- MMA
      if (lane == 0) {
        constexpr uint32_t IDESC_S = idesc_bf16_f32(BK, BQ, 0, 0);   // S^T, dP^T
        constexpr uint32_t IDESC_KV = idesc_bf16_f32(BK, HD, 0, 1);  // dV, dK
        constexpr uint32_t IDESC_Q = idesc_bf16_f32(BQ, HD, 1, 1);   // dQ
        const uint32_t spt = sbase + C::OFF_PT, sdst = sbase + C::OFF_DST;
        uint32_t qzp = 0;  // WIN: bit s = parity of qd_fixed[s]'s next phase
        // S^T and dP^T of step s into their TMEM columns
        auto issue_s = [&](const StepIter<WIN>& s) -> bool {
          const int st = s.t % C::STAGES;
          const int kvs = s.uc % C::KVB;
          if (s.i == 0 && !mbar_wait(BAR_KF(kvs), (s.uc / C::KVB) & 1, abort_p)) return false;
          if (!mbar_wait(BAR_QF(st), (s.t / C::STAGES) & 1, abort_p)) return false;
          if constexpr (WIN) {
            if (fix_q(s) || fix_k(s)) {  // warp 2 has zeroed the padding rows
              if (!mbar_wait(BAR_QZ(st), (qzp >> st) & 1, abort_p)) return false;
              qzp ^= 1u << st;
            }
          }
          if (s.t >= 1 && !mbar_wait(BAR_SE, (s.t - 1) & 1, abort_p)) return false;
          if (C::DQ_ALIAS && s.t >= 1 && !mbar_wait(BAR_DQE, (s.t - 1) & 1, abort_p)) return false;
          tc_fence_after();
          const uint32_t sk = sbase + C::OFF_K + kvs * C::KV_BYTES;
          const uint32_t sv = sbase + C::OFF_V + kvs * C::KV_BYTES;
          const uint32_t sq = sbase + C::OFF_Q + st * C::QD_BYTES;
          const uint32_t sdo = sbase + C::OFF_DO + st * C::QD_BYTES;
          const uint64_t dk = smem_desc_sw128(sk, 16, 1024), dv = smem_desc_sw128(sv, 16, 1024);
          const uint64_t dq = smem_desc_sw128(sq, 16, 1024), ddo = smem_desc_sw128(sdo, 16, 1024);
#pragma unroll C::UMMA_UNROLL
          for (int kk = 0; kk < HD / 16; ++kk) {
            const uint32_t off = (kk >> 2) * (BK * 128) + (kk & 3) * 32;
            umma_bf16_ss(tmem + C::TCOL_S, desc_at(dk, off), desc_at(dq, off), IDESC_S, kk > 0 ? 1u : 0u);
          }
#pragma unroll C::UMMA_UNROLL
          for (int kk = 0; kk < HD / 16; ++kk) {
            const uint32_t off = (kk >> 2) * (BK * 128) + (kk & 3) * 32;
            umma_bf16_ss(tmem + C::TCOL_DP, desc_at(dv, off), desc_at(ddo, off), IDESC_S, kk > 0 ? 1u : 0u);
          }
          umma_commit(BAR_SF);
          return true;
        };
        StepIter<WIN> cur = first_step<C::DYN, C::HB, WIN, false>(prm, sch, ring);
        StepIter<WIN> la = cur;  // next step whose S^T/dP^T is to be issued
        bool ok = true;
        if (la.valid) {
          ok = issue_s(la);
          advance<C::DYN, C::HB, WIN, false>(prm, la, sch, ring);
        }
        // time-out test hook: with the first products in flight, wait on a
        // barrier nothing arrives at until the hook's limit runs out
        if (ok && prm.expire_ns) ok = mbar_wait(BAR_NEVER, 0, abort_p, prm.expire_ns);
        for (; ok && cur.valid; advance<C::DYN, C::HB, WIN, false>(prm, cur, sch, ring)) {
          // the next step's S^T/dP^T ahead of this step's products, except
          // where it starts a unit whose K/V can only be loaded into the
          // single K/V buffer once this step's products are done with it
          const bool early = C::EARLY_S && la.valid && (C::KVB > 1 || la.uc == cur.uc);
          if (early) {
            if (!issue_s(la)) break;
            advance<C::DYN, C::HB, WIN, false>(prm, la, sch, ring);
          }
          const int st = cur.t % C::STAGES;
          const int kvs = cur.uc % C::KVB;
          const uint32_t sk = sbase + C::OFF_K + kvs * C::KV_BYTES;
          const uint32_t sq = sbase + C::OFF_Q + st * C::QD_BYTES;
          const uint32_t sdo = sbase + C::OFF_DO + st * C::QD_BYTES;
          if (!mbar_wait(BAR_PR, cur.t & 1, abort_p)) break;
          // the previous unit's epilogue must have read dK/dV out of TMEM
          if (cur.i == 0 && cur.uc >= 1 && !mbar_wait(BAR_ACC, (cur.uc - 1) & 1, abort_p)) break;
          tc_fence_after();
          const uint64_t bdo = smem_desc_sw128(sdo, BQ * 128, 1024), bq = smem_desc_sw128(sq, BQ * 128, 1024);
          const uint64_t apt = smem_desc_sw128(spt, 16, 1024), adst = smem_desc_sw128(sdst, 16, 1024);
#pragma unroll C::UMMA_UNROLL
          for (int kk = 0; kk < BQ / 16; ++kk) {  // dV += P^T dO_i
            const uint32_t acc = (cur.i > 0 || kk > 0) ? 1u : 0u;
            if (C::P_IN_TMEM)
              umma_bf16_ts(tmem + C::TCOL_DV, tmem + C::TCOL_PT + kk * 8, desc_at(bdo, kk * 2048), IDESC_KV, acc);
            else
              umma_bf16_ss(tmem + C::TCOL_DV, desc_at(apt, (kk >> 2) * (BK * 128) + (kk & 3) * 32),
                           desc_at(bdo, kk * 2048), IDESC_KV, acc);
          }
#pragma unroll C::UMMA_UNROLL
          for (int kk = 0; kk < BQ / 16; ++kk) {  // dK += dS^T Q_i
            umma_bf16_ss(tmem + C::TCOL_DK, desc_at(adst, (kk >> 2) * (BK * 128) + (kk & 3) * 32),
                         desc_at(bq, kk * 2048), IDESC_KV, (cur.i > 0 || kk > 0) ? 1u : 0u);
          }
          umma_commit(BAR_QE(st));
          // the dQ columns must have been drained (previous step)
          if (cur.t >= 1 && !mbar_wait(BAR_DQE, (cur.t - 1) & 1, abort_p)) break;
          tc_fence_after();
          const uint64_t aq = smem_desc_sw128(sdst, BK * 128, 1024), bk = smem_desc_sw128(sk, BK * 128, 1024);
#pragma unroll C::UMMA_UNROLL
          for (int kk = 0; kk < BK / 16; ++kk)  // dQ_i = dS K (A = dS^T as MN-major)
            umma_bf16_ss(tmem + C::TCOL_DQ, desc_at(aq, kk * 2048), desc_at(bk, kk * 2048), IDESC_Q, kk > 0 ? 1u : 0u);
          umma_commit(BAR_DQF);
          umma_commit(BAR_PE);
          if (cur.i + 1 == cur.u.nq) {  // the unit's last UMMA
            umma_commit(BAR_KE(kvs));
            umma_commit(BAR_DONE);
          }
          // (after them: D=128, or a unit start with a single K/V buffer)
          if ((!C::EARLY_S || C::KVB == 1) && !early && la.valid) {
            if (!issue_s(la)) break;
            advance<C::DYN, C::HB, WIN, false>(prm, la, sch, ring);
          }
        }
        if (*abort_p) {  // wind-down: every UMMA issued must complete before TMEM is freed
          umma_commit(BAR_FIN);
          mbar_wait_for(BAR_FIN, 0, kDrainLimitNs);
        }
      }
    } else if (warp == 2) {
      // ------------------------------------------------------- statistics
      // A step's 128 (-l*log2e, -D/sqrt(D)) pairs, four queries per lane,
      // are loaded into registers one step ahead, so the ring slot is filled
      // as soon as the compute warps free it, whatever the load latency.
      float nl[4], nd[4];
      auto load_stats = [&](const StepIter<WIN>& s) {
        const int qt = s.u.q_tile(s.i);
        if constexpr (WIN) {  // prepared, padded to whole tiles
          const int heads = prm.NH * prm.win.G;
          const long long si = ((long long)s.u.b * heads + s.u.q_head(s.i)) * prm.win.rows + qt * BQ + lane * 4;
          const float4 L = __ldg(reinterpret_cast<const float4*>(prm.win.neg_l + si));
          const float4 D4 = __ldg(reinterpret_cast<const float4*>(prm.win.neg_d + si));
          nl[0] = L.x, nl[1] = L.y, nl[2] = L.z, nl[3] = L.w;
          nd[0] = D4.x, nd[1] = D4.y, nd[2] = D4.z, nd[3] = D4.w;
        } else {
          const long long rbase = (long long)s.u.b * prm.T;
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const int q = qt * BQ + lane * 4 + v;
            nl[v] = 0.0f;
            nd[v] = 0.0f;
            if (q < prm.T) {
              const long long si = (rbase + q) * prm.NH + s.u.h;
              nl[v] = -__ldg(prm.lse + si) * LOG2E;
              nd[v] = -__bfloat162float(prm.Dv[si]) * prm.scale;
            }
          }
        }
      };
      // WIN: rows [a, 128) of a tile are contiguous in each 64-column block
      // (the swizzle permutes the chunks of a row within its 128 bytes)
      auto zero_rows = [&](uint32_t off, int a) {
        for (int kb = 0; kb < C::KB; ++kb) {
          uint4* blk = reinterpret_cast<uint4*>(gbase + off + kb * BQ * 128);
          for (int i = a * 8 + lane; i < BQ * 8; i += 32) blk[i] = make_uint4(0u, 0u, 0u, 0u);
        }
      };
      StepIter<WIN> s = first_step<C::DYN, C::HB, WIN, true>(prm, sch, ring);
      if (s.valid) load_stats(s);
      while (s.valid) {
        const float cl[4] = {nl[0], nl[1], nl[2], nl[3]};
        const float cd[4] = {nd[0], nd[1], nd[2], nd[3]};
        StepIter<WIN> nx = s;
        advance<C::DYN, C::HB, WIN, true>(prm, nx, sch, ring);
        if (nx.valid) load_stats(nx);  // the next step's, in flight while this one waits
        if constexpr (WIN) {
          // every stage (and a unit's K/V) is waited for and released, so that
          // this warp stays within one phase of each slot's barriers
          const int qs = s.t % C::STAGES, kvs = s.uc % C::KVB;
          if (s.i == 0 && !mbar_wait_warp(BAR_KF(kvs), (s.uc / C::KVB) & 1, abort_p)) break;
          if (!mbar_wait_warp(BAR_QF(qs), (s.t / C::STAGES) & 1, abort_p)) break;
          const bool fq = fix_q(s), fk = fix_k(s);
          if (fk) {
            zero_rows(C::OFF_K + kvs * C::KV_BYTES, max(0, s.u.n - s.u.kt * BK));
            zero_rows(C::OFF_V + kvs * C::KV_BYTES, max(0, s.u.n - s.u.kt * BK));
          }
          if (fq) {
            const int a = max(0, s.u.n - s.u.q_tile(s.i) * BQ);
            zero_rows(C::OFF_Q + qs * C::QD_BYTES, a);
            zero_rows(C::OFF_DO + qs * C::QD_BYTES, a);
          }
          if (fq || fk) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(BAR_QZ(qs));
          }
          if (lane == 0) {
            mbar_arrive(BAR_QE(qs));
            if (s.i == 0) mbar_arrive(BAR_KE(kvs));
          }
        }
        const int st = s.t % C::SSTG;
        if (s.t >= C::SSTG && !mbar_wait_warp(BAR_TE(st), ((s.t / C::SSTG) - 1) & 1, abort_p)) break;
        float* stt = stat_base + st * (2 * BQ);
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          stt[lane * 4 + v] = cl[v];
          stt[BQ + lane * 4 + v] = cd[v];
        }
        mbar_arrive(BAR_TF(st));
        s = nx;
      }
    } else {
      // ------------------------------------------------- dQ reduce issuer
      if (lane == 0) {
        for (StepIter<WIN> s = first_step<C::DYN, C::HB, WIN, false>(prm, sch, ring); s.valid; advance<C::DYN, C::HB, WIN, false>(prm, s, sch, ring)) {
          const int b = s.t % C::DQSB;
          if (!mbar_wait(BAR_DSF(b), (s.t / C::DQSB) & 1, abort_p)) break;
          for (int box = 0; box < HD / 32; ++box)
            tma_reduce_add_3d(&tmdQ, sbase + C::OFF_DQS + b * C::DQS_BYTES + box * (BQ * 128),
                              s.u.q_head(s.i) * HD + box * 32, s.u.q_tile(s.i) * BQ, s.u.b);
          bulk_commit();
          // the reduction DQSB-1 steps back has read its buffer, which may
          // now be rewritten (with one buffer: this step's)
          bulk_wait_read<C::DQSB - 1>();
          if (s.t + 1 >= (uint32_t)C::DQSB) mbar_arrive(BAR_DSE((s.t + 1 - C::DQSB) % C::DQSB));
        }
        bulk_wait<0>();
      }
    }
  } else if (!C::DRAIN_WG || warp < 4 + C::NCOMP / 32) {
    reg_alloc<C::REGS_COMPUTE>();
    // ------------------------------------------------------------ compute
    constexpr int CPP = C::CPP;                // query columns per part
    const int cw = warp - 4;                   // 0 .. NCOMP/32 - 1
    const int quarter = warp & 3;              // TMEM lane quarter
    const int krow = quarter * 32 + lane;      // key row (and dQ query row) within the tile
    const int part = cw >> 2;                  // query columns part*CPP .. +CPP-1
    const uint32_t tl = tmem + ((uint32_t)(quarter * 32) << 16);
    const float c = prm.scale_log2, sc = prm.scale;
    bool ok = true;

    // dQ of global step t: TMEM -> fp32 staging (128-byte swizzle, 32-column
    // boxes); the reduce issuer (warp 3) sends it to global memory.  Each
    // part drains HD / NPART of the head dimension's columns.
    auto drain_dq = [&](uint32_t t) {
      const int b = t % C::DQSB;
      if (ok) ok = mbar_wait_warp(BAR_DQF, t & 1, abort_p);
      if (ok && t >= (uint32_t)C::DQSB) ok = mbar_wait_warp(BAR_DSE(b), ((t / C::DQSB) - 1) & 1, abort_p);
      if (!ok) return;
      tc_fence_after();
      constexpr int CPH = HD / C::NPART;  // dQ columns per part
      uint8_t* dqs = gbase + C::OFF_DQS + b * C::DQS_BYTES;
#pragma unroll
      for (int cc = 0; cc < CPH; cc += 16) {
        uint32_t r[16];
        tmem_ld16(tl + C::TCOL_DQ + part * CPH + cc, r);
        tmem_wait_ld_dep(r);
        const int col = part * CPH + cc;  // first column (fp32) of the 16
        uint8_t* rowp = dqs + (col / 32) * (BQ * 128) + krow * 128;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int ch = (col % 32) / 4 + q;
          uint4 v = make_uint4(r[q * 4 + 0], r[q * 4 + 1], r[q * 4 + 2], r[q * 4 + 3]);
          *reinterpret_cast<uint4*>(rowp + ((ch ^ (krow & 7)) * 16)) = v;
        }
      }
      tc_fence_before();
      mbar_arrive(BAR_DQE);
      fence_proxy_async_smem();
      mbar_arrive(BAR_DSF(b));
    };

    // dK/dV of unit v (its UMMAs complete, BAR_DONE phase vuc): TMEM ->
    // registers; frees the accumulators (BAR_ACC) for the next unit, then
    // converts to bf16 and stores this thread's row slice straight to global
    // memory (rows past T are not stored)
    auto epilogue = [&](const auto& v, uint32_t vuc) {
      if (ok) ok = mbar_wait_warp(BAR_DONE, vuc & 1, abort_p);
      if (!ok) return;
      tc_fence_after();
      constexpr int CPH = HD / C::NPART;  // dV, dK columns per part
      uint32_t acc[2][CPH];
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        const uint32_t tcol = which == 0 ? C::TCOL_DV : C::TCOL_DK;
#pragma unroll
        for (int cc = 0; cc < CPH; cc += 16) {
          uint32_t r[16];
          tmem_ld16(tl + tcol + part * CPH + cc, r);
          tmem_wait_ld_dep(r);
#pragma unroll
          for (int j = 0; j < 16; ++j) acc[which][cc + j] = r[j];
        }
      }
      tc_fence_before();
      mbar_arrive(BAR_ACC);  // the next unit may overwrite dK/dV in TMEM
      const int key = v.kt * BK + krow;
      if constexpr (WIN) {
        if (v.slot >= 0) {  // partial sums, fp32
#pragma unroll
          for (int which = 0; which < 2; ++which) {
            float4* dst = reinterpret_cast<float4*>(
                prm.win.part + (((long long)v.slot * 2 + which) * BK + krow) * HD + part * CPH);
#pragma unroll
            for (int cc = 0; cc < CPH; cc += 4)
              dst[cc / 4] = make_float4(__uint_as_float(acc[which][cc + 0]), __uint_as_float(acc[which][cc + 1]),
                                        __uint_as_float(acc[which][cc + 2]), __uint_as_float(acc[which][cc + 3]));
          }
          return;
        }
      }
      if (key < prm.T) {
        const long long off = ((long long)v.b * prm.T + key) * prm.N + v.h * HD + part * CPH;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
          uint4* dst = reinterpret_cast<uint4*>((which == 0 ? dV : dK) + off);
#pragma unroll
          for (int cc = 0; cc < CPH; cc += 8) {
            uint4 w;
            w.x = pack_bf16(__uint_as_float(acc[which][cc + 0]), __uint_as_float(acc[which][cc + 1]));
            w.y = pack_bf16(__uint_as_float(acc[which][cc + 2]), __uint_as_float(acc[which][cc + 3]));
            w.z = pack_bf16(__uint_as_float(acc[which][cc + 4]), __uint_as_float(acc[which][cc + 5]));
            w.w = pack_bf16(__uint_as_float(acc[which][cc + 6]), __uint_as_float(acc[which][cc + 7]));
            dst[cc / 8] = w;
          }
        }
      }
    };

    // A unit's last dQ drain and its dK/dV epilogue run after the first step
    // of the next unit has been handed to the tensor core (or after the last
    // step of the last unit), so they overlap the next unit's UMMAs.
    decltype(StepIter<WIN>::u) prev{};
    bool have_prev = false;
    // Step st: P^T and dS^T formed and handed to the UMMA issuer.
    auto form = [&](const StepIter<WIN>& st_it) {
      const auto& u = st_it.u;
      const int i = st_it.i;
      const uint32_t t = st_it.t;
      const int ss = t % C::SSTG;
      ok = mbar_wait_warp(BAR_SF, t & 1, abort_p);
      if (!ok) return;
      tc_fence_after();
      float s[CPP], dp[CPP];
      if constexpr (CPP == 64) {
        uint32_t ra[32], rb[32];
        tmem_ld32(tl + C::TCOL_S + part * 64, ra);
        tmem_ld32(tl + C::TCOL_S + part * 64 + 32, rb);
        tmem_wait_ld_dep(ra, rb);
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          s[j] = __uint_as_float(ra[j]);
          s[32 + j] = __uint_as_float(rb[j]);
        }
        tmem_ld32(tl + C::TCOL_DP + part * 64, ra);
        tmem_ld32(tl + C::TCOL_DP + part * 64 + 32, rb);
        tmem_wait_ld_dep(ra, rb);
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          dp[j] = __uint_as_float(ra[j]);
          dp[32 + j] = __uint_as_float(rb[j]);
        }
      } else {
        static_assert(CPP == 32, "column split");
        uint32_t ra[32], rb[32];
        tmem_ld32(tl + C::TCOL_S + part * 32, ra);
        tmem_ld32(tl + C::TCOL_DP + part * 32, rb);
        tmem_wait_ld_dep(ra, rb);
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          s[j] = __uint_as_float(ra[j]);
          dp[j] = __uint_as_float(rb[j]);
        }
      }
      tc_fence_before();
      mbar_arrive(BAR_SE);
      ok = mbar_wait_warp(BAR_TF(ss), (t / C::SSTG) & 1, abort_p);
      if (!ok) return;
      const float* stt = stat_base + ss * (2 * BQ) + part * CPP;
      if constexpr (WIN) {
        const int row0 = u.q_tile(i) * BQ;
        // one form for masked and whole steps (a second would cost more in
        // instruction fetches than it saves)
        int from, to;
        u.seen(prm.win, u.kt * BK + krow, row0 + part * CPP, &from, &to);
        uint32_t see[CPP / 32];
#pragma unroll
        for (int w = 0; w < CPP / 32; ++w) see[w] = bits_below(to - 32 * w) & ~bits_below(from - 32 * w);
        p_ds_row<false, CPP, true>(s, dp, stt, stt + BQ, c, sc, krow, part * CPP, see);
      } else if (i == 0) {
        p_ds_row<true, CPP>(s, dp, stt, stt + BQ, c, sc, krow, part * CPP);
      } else {
        p_ds_row<false, CPP>(s, dp, stt, stt + BQ, c, sc, krow, part * CPP);
      }
      mbar_arrive(BAR_TE(ss));
      // the previous step's UMMAs must be done with P^T/dS^T, and when the dQ
      // staging shares their smem its reduction must have read it
      if (t >= 1) ok = mbar_wait_warp(BAR_PE, (t - 1) & 1, abort_p);
      if (ok && C::DQS_ALIAS && t >= 1) ok = mbar_wait_warp(BAR_DSE(0), (t - 1) & 1, abort_p);
      if (!ok) return;
      // this part's columns of the key row: P^T (bf16 pairs in TMEM, or smem),
      // dS^T (smem); chunk (part*CPP % 64) / 8 of 64-column block part*CPP / 64
      const int blk = (part * CPP) / 64, ch0 = ((part * CPP) % 64) / 8;
      if constexpr (C::P_IN_TMEM) {
        uint32_t pk[CPP / 2];
#pragma unroll
        for (int j = 0; j < CPP / 2; ++j) pk[j] = pack_bf16(s[2 * j], s[2 * j + 1]);
        if constexpr (CPP == 64) tmem_st32(tl + C::TCOL_PT + part * 32, pk);
        else tmem_st16(tl + C::TCOL_PT + part * 16, pk);
        tmem_wait_st();
      } else {
        store_row_sw128<CPP>(gbase + C::OFF_PT + blk * (BK * 128) + krow * 128, krow, s, ch0);
      }
      store_row_sw128<CPP>(gbase + C::OFF_DST + blk * (BK * 128) + krow * 128, krow, dp, ch0);
      fence_proxy_async_smem();
      tc_fence_before();
      mbar_arrive(BAR_PR);
    };
    for (StepIter<WIN> st_it = first_step<C::DYN, C::HB, WIN, true>(prm, sch, ring); ok;
         advance<C::DYN, C::HB, WIN, true>(prm, st_it, sch, ring)) {
      if (st_it.valid) form(st_it);
      if (!ok) break;
      // on a unit's first step the previous unit's dK/dV epilogue comes
      // first: the UMMA issuer waits for it before this step's products,
      // the dQ product that drain_dq(t) waits for among them.  The last
      // unit's follows its last step.
      if constexpr (C::EPI_COMPUTE) {
        if (have_prev && (!st_it.valid || st_it.i == 0)) {
          if constexpr (!C::DRAIN_WG && C::EARLY_S)
            if (!st_it.valid) drain_dq(st_it.t - 1);
          epilogue(prev, st_it.uc - 1);
        }
        if (!st_it.valid) break;
        prev = st_it.u;
        have_prev = true;
      }
      if constexpr (!C::DRAIN_WG) {
        if (C::EARLY_S) {
          if (st_it.t >= 1) drain_dq(st_it.t - 1);
        } else {
          drain_dq(st_it.t);
        }
      }
    }
  } else {
    reg_dealloc<C::REGS_DRAIN>();
    // ---------------------------------------------------------- dQ drain
    // (D=64, warps 12-15): thread = TMEM lane = dQ query row
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t tl = tmem + ((uint32_t)(quarter * 32) << 16);
    bool ok = true;
    for (StepIter<WIN> s = first_step<C::DYN, C::HB, WIN, true>(prm, sch, ring); ok && s.valid; advance<C::DYN, C::HB, WIN, true>(prm, s, sch, ring)) {
      const uint32_t t = s.t;
      const int b = t % C::DQSB;
      uint8_t* dqs = gbase + C::OFF_DQS + b * C::DQS_BYTES;
      // dQ of step t: TMEM -> fp32 staging b (128-byte swizzle, 32-column
      // boxes); the reduce issuer (warp 3) adds it into global dQ
      ok = mbar_wait_warp(BAR_DQF, t & 1, abort_p);
      if (ok && t >= (uint32_t)C::DQSB) ok = mbar_wait_warp(BAR_DSE(b), ((t / C::DQSB) - 1) & 1, abort_p);
      if (!ok) break;
      tc_fence_after();
#pragma unroll
      for (int cc = 0; cc < HD; cc += 16) {
        uint32_t r[16];
        tmem_ld16(tl + C::TCOL_DQ + cc, r);
        tmem_wait_ld_dep(r);
        uint8_t* rowp = dqs + (cc / 32) * (BQ * 128) + row * 128;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int ch = (cc % 32) / 4 + q;
          const uint4 v = make_uint4(r[q * 4 + 0], r[q * 4 + 1], r[q * 4 + 2], r[q * 4 + 3]);
          *reinterpret_cast<uint4*>(rowp + ((ch ^ (row & 7)) * 16)) = v;
        }
      }
      tc_fence_before();
      mbar_arrive(BAR_DQE);
      fence_proxy_async_smem();
      mbar_arrive(BAR_DSF(b));
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (threadIdx.x == 0 && abort_flag) atomicOr(prm.status, STATUS_BWD_TIMEOUT);
}

// Zeroes the dQ columns of the (batch, head) shard range.
__global__ void zero_dq_shard_kernel(float4* __restrict__ dQ, int T, int N, int D, int NH,
                                     int bh_begin, int bh_end) {
  pdl_wait_and_release();
  const long long per_bh = (long long)T * (D / 4);
  const long long total = (long long)(bh_end - bh_begin) * per_bh;
  for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < total;
       i += (long long)gridDim.x * blockDim.x) {
    const long long bh = bh_begin + i / per_bh;
    const long long rem = i % per_bh;
    const long long t = rem / (D / 4), c4 = rem % (D / 4);
    const long long bb = bh / NH, hh = bh % NH;
    dQ[((bb * T + t) * N + hh * D) / 4 + c4] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
}

// T rows of queries and keys, nq and nkv columns.
template <int HD, bool PERSIST, bool WIN = false>
cudaError_t launch_bwd_kernel(const __nv_bfloat16* dO, const __nv_bfloat16* q,
                              const __nv_bfloat16* k, const __nv_bfloat16* v, float* dQ,
                              __nv_bfloat16* dK, __nv_bfloat16* dV, int T, int B, uint64_t nq, uint64_t nkv,
                              const BwdParams& prm, int grid, cudaStream_t st) {
  using C = BwdCfg<HD, PERSIST, WIN>;
  // The setmaxnreg split assumes the kernel was compiled to exactly
  // LAUNCH_REGS registers per thread; refuse to launch otherwise.
  static const cudaError_t reg_check = [] {
    cudaFuncAttributes a;
    cudaError_t e = cudaFuncGetAttributes(&a, flash_bwd_kernel<HD, PERSIST, WIN>);
    if (e != cudaSuccess) return e;
    return a.numRegs == C::LAUNCH_REGS ? cudaSuccess : cudaErrorInvalidKernelImage;
  }();
  if (reg_check != cudaSuccess) return reg_check;
  CUtensorMap tq, tk, tv, tdo, tdq;
  const CUtensorMapDataType bf = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUtensorMapSwizzle sw = CU_TENSOR_MAP_SWIZZLE_128B;
  if (!make_tmap_3d(&tq, q, bf, 2, nq, T, B, 64, BQ, sw) ||
      !make_tmap_3d(&tk, k, bf, 2, nkv, T, B, 64, BK, sw) ||
      !make_tmap_3d(&tv, v, bf, 2, nkv, T, B, 64, BK, sw) ||
      !make_tmap_3d(&tdo, dO, bf, 2, nq, T, B, 64, BQ, sw) ||
      !make_tmap_3d(&tdq, dQ, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, nq, T, B, 32, BQ, sw))
    return cudaErrorInvalidValue;
  cudaError_t e = cudaFuncSetAttribute(flash_bwd_kernel<HD, PERSIST, WIN>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES);
  if (e != cudaSuccess) return e;
  launch_pdl(flash_bwd_kernel<HD, PERSIST, WIN>, grid, C::NUM_THREADS, C::SMEM_BYTES, st, tq, tk, tv, tdo, tdq, dK,
             dV, prm);
  count_launches(1);
  return cudaGetLastError();
}

template <int HD>
cudaError_t launch_bwd(const __nv_bfloat16* dO, const __nv_bfloat16* Dv, const float* lse,
                       const __nv_bfloat16* q, const __nv_bfloat16* k, const __nv_bfloat16* v,
                       float* dQ, __nv_bfloat16* dK, __nv_bfloat16* dV, const AttnShape& s,
                       uint32_t* status, cudaStream_t st, bool accumulate_dq) {
  // dQ is accumulated by bulk reductions: zero the shard's columns first,
  // unless the caller asks for dQ += (it holds zeros or partial sums)
  const int nbh = s.bh_end - s.bh_begin;
  if (!accumulate_dq) {
    const cudaError_t e = launch_zero_dq(dQ, s, st);
    if (e != cudaSuccess) return e;
  }
  BwdParams prm{};
  prm.T = s.T;
  prm.N = s.N;
  prm.NH = s.NH;
  prm.bh_begin = s.bh_begin;
  prm.nbh = nbh;
  prm.nkt = (s.T + BK - 1) / BK;
  prm.nunits = prm.nkt * nbh;
  prm.scale = 1.0f / sqrtf((float)HD);
  prm.scale_log2 = LOG2E / sqrtf((float)HD);
  prm.lse = lse;
  prm.Dv = Dv;
  prm.status = status;
  prm.expire_ns = take_expire_request(STATUS_BWD_TIMEOUT);
  // short sequences at D=64: static rounds over one CTA per SM, (batch,
  // head)-major; otherwise one CTA per unit, the running CTAs taking over the
  // rest (see bwd_unit)
  if (HD == 64 && prm.nkt <= PERSIST_MAX_NKT) {
    int dev = 0, sms = 148;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    const int grid = prm.nunits < sms ? prm.nunits : sms;
    return launch_bwd_kernel<HD, true>(dO, q, k, v, dQ, dK, dV, s.T, s.B, s.N, s.N, prm, grid, st);
  }
  return launch_bwd_kernel<HD, false>(dO, q, k, v, dQ, dK, dV, s.T, s.B, s.N, s.N, prm, prm.nunits, st);
}

// ------------------------------------------------------- windowed backward
// How a call's workspace is laid out, and how its sink tiles are split.
struct WinPlan {
  int nqt, rows, nsplit, nfar, far_tiles;
  size_t stat, part, dq;  // bytes: one statistic, the partial sums, dQ in fp32
  size_t total() const { return 2 * stat + part + dq; }
};

WinPlan win_plan(const WindowArgs& a, bool dq_f32) {
  WinPlan p{};
  p.nqt = (a.M + BQ - 1) / BQ;
  p.rows = p.nqt * BQ;
  const int nbh = a.B * a.NKV;
  const int ns = (int)std::min<long long>(((long long)a.sinks + BK - 1) / BK, p.nqt);
  const int window = std::min(a.window, 1 << 25);
  const int near = (BK - 1 + window - 1) / BQ + 1;  // query tiles of tile 0's window
  const int far = p.nqt - near;
  // A sink tile's far queries are a chain of `far` steps a head where other
  // units have `near`.  Where the sink tiles alone would not keep the GPU busy
  // twice over, the chain is cut into pieces of a window's length, of 8 tiles
  // at least (a piece costs 2 x 128 x D fp32 written and read) and 16 at most.
  if (far > near && far > 8 && (long long)ns * nbh < 2 * 148) {
    p.nsplit = ns;
    p.far_tiles = std::max({near, 8, (far + 15) / 16});
    p.nfar = ns > 0 ? (far + p.far_tiles - 1) / p.far_tiles : 0;
  }
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  p.stat = up((size_t)a.B * a.NH * p.rows * sizeof(float));
  p.part = up((size_t)nbh * p.nsplit * (1 + p.nfar) * 2 * BK * a.D * sizeof(float));
  p.dq = dq_f32 ? 0 : up((size_t)a.B * a.M * a.NH * a.D * sizeof(float));
  return p;
}

__device__ __forceinline__ float dot8(uint4 a, uint4 b) {
  const __nv_bfloat162* x = reinterpret_cast<const __nv_bfloat162*>(&a);
  const __nv_bfloat162* y = reinterpret_cast<const __nv_bfloat162*>(&b);
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 u = __bfloat1622float2(x[i]), v = __bfloat1622float2(y[i]);
    s = fmaf(u.x, v.x, s);
    s = fmaf(u.y, v.y, s);
  }
  return s;
}

// The statistics -l*log2e and -(dO . O)/sqrt(D), [B][NH][rows] (0 for padding
// and past the end), and zeros for dQ.  HBM-bound: dO, O read and dQ written
// once.  A warp takes 32 rows of a head, D/8 lanes a row with 16-byte loads,
// and writes 32 neighbouring statistics.
template <int HD>
__global__ void __launch_bounds__(256) window_stats_kernel(const WindowArgs a, const __nv_bfloat16* __restrict__ dO,
                                                           float* __restrict__ neg_l, float* __restrict__ neg_d,
                                                           float* __restrict__ dQ, int rows) {
  pdl_wait_and_release();
  constexpr int G = HD / 8, RPI = 32 / G;  // lanes a row, rows an instruction
  const int lane = threadIdx.x % 32;
  const int tiles = rows / 32;
  const long long items = (long long)a.B * tiles * a.NH;
  for (long long it = blockIdx.x * 8ll + threadIdx.x / 32; it < items; it += gridDim.x * 8ll) {
    const int h = (int)(it % a.NH);
    const long long r = it / a.NH;
    const int b = (int)(r / tiles), row0 = (int)(r % tiles) * 32;
    const int n = a.len(b);
    float mine = 0.0f;  // of row row0 + lane
    // loads before stores: 8 rows of a lane in flight at once
#pragma unroll
    for (int i0 = 0; i0 < 32; i0 += 8 * RPI < 32 ? 8 * RPI : 32) {
      constexpr int N = 8 * RPI < 32 ? 8 : 32 / RPI;
      uint4 x[N], y[N];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int row = row0 + i0 + k * RPI + lane / G;
        const long long off = (((long long)b * a.M + row) * a.NH + h) * HD;
        x[k] = y[k] = make_uint4(0u, 0u, 0u, 0u);
        if (row < n) {
          x[k] = __ldcs(reinterpret_cast<const uint4*>(dO + off) + lane % G);
          y[k] = __ldcs(reinterpret_cast<const uint4*>(a.out + off) + lane % G);
        }
      }
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int i = i0 + k * RPI;
        float s = dot8(x[k], y[k]);
#pragma unroll
        for (int m = G / 2; m >= 1; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
        const float got = __shfl_sync(0xffffffffu, s, (lane - i) * G & 31);
        if (lane >= i && lane < i + RPI) mine = got;
      }
    }
#pragma unroll
    for (int i = 0; i < 32; i += RPI) {
      const int row = row0 + i + lane / G;
      if (row < a.M) {
        float4* z = reinterpret_cast<float4*>(dQ + (((long long)b * a.M + row) * a.NH + h) * HD) + lane % G;
        z[0] = z[G] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
    }
    const int row = row0 + lane;
    const bool valid = row < n;
    const long long at = ((long long)b * a.NH + h) * rows + row;
    neg_l[at] = valid ? -a.l[((long long)b * a.M + row) * a.NH + h] * LOG2E : 0.0f;
    neg_d[at] = valid ? -mine * a.scale : 0.0f;
  }
}

// dQ rounded to bf16, and the split sink tiles' partial dV, dK added up in
// slot order and rounded.
__global__ void __launch_bounds__(256) window_finish_kernel(const float* __restrict__ dQ, __nv_bfloat16* __restrict__ dQ16,
                                                            long long nq4, const float* __restrict__ part, int slots,
                                                            int nsplit, int D, int NKV, int T, long long npart4,
                                                            __nv_bfloat16* __restrict__ dK, __nv_bfloat16* __restrict__ dV) {
  pdl_wait_and_release();
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < nq4 + npart4; i += gridDim.x * 256ll) {
    if (i < npart4) {
      const int d4 = D / 4;
      const int c = (int)(i % d4);
      long long r = i / d4;
      const int row = (int)(r % BK);
      r /= BK;
      const int which = (int)(r % 2);
      r /= 2;  // (batch, K/V head, sink tile)
      const int tile = (int)(r % nsplit);
      const long long bh = r / nsplit;
      const int key = tile * BK + row;
      if (key >= T) continue;
      float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int k = 0; k < slots; ++k) {
        const float4 x = __ldg(reinterpret_cast<const float4*>(part) + (((r * slots + k) * 2 + which) * BK + row) * d4 + c);
        s.x += x.x, s.y += x.y, s.z += x.z, s.w += x.w;
      }
      __nv_bfloat16* to = (which == 0 ? dV : dK) + ((bh / NKV * T + key) * NKV + bh % NKV) * D + c * 4;
      *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16(s.x, s.y), pack_bf16(s.z, s.w));
    } else {
      const long long j = i - npart4;
      const float4 x = __ldcs(reinterpret_cast<const float4*>(dQ) + j);
      reinterpret_cast<uint2*>(dQ16)[j] = make_uint2(pack_bf16(x.x, x.y), pack_bf16(x.z, x.w));
    }
  }
}

template <int HD>
cudaError_t launch_win_bwd(const WindowArgs& a, const WindowGrads& g, cudaStream_t st) {
  const WinPlan p = win_plan(a, g.dq_f32);
  char* ws = static_cast<char*>(g.workspace);
  float* neg_l = reinterpret_cast<float*>(ws);
  float* neg_d = reinterpret_cast<float*>(ws + p.stat);
  float* part = reinterpret_cast<float*>(ws + 2 * p.stat);
  float* dQ = g.dq_f32 ? static_cast<float*>(g.dQ) : reinterpret_cast<float*>(ws + 2 * p.stat + p.part);
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  auto blocks = [&](long long n, int per) { return (unsigned)std::min<long long>((n + per - 1) / per, sms * 16ll); };
  launch_pdl(window_stats_kernel<HD>, blocks((long long)a.B * a.NH * (p.rows / 32), 8), 256, 0, st, a, g.dO, neg_l,
             neg_d, dQ, p.rows);
  count_launches(1);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  BwdParams prm{};
  prm.T = a.M;
  prm.N = a.NKV * HD;
  prm.NH = a.NKV;
  prm.nbh = a.B * a.NKV;
  prm.nkt = p.nqt;
  prm.scale = 1.0f / sqrtf((float)HD);
  prm.scale_log2 = LOG2E / sqrtf((float)HD);
  prm.status = a.status;
  WinBwd& w = prm.win;
  w.lens = a.lens;
  w.G = a.NH / a.NKV;
  w.window = std::min(a.window, 1 << 25);  // M <= 2^24: the same mask, and sums of positions stay in range
  w.sinks = a.sinks;
  w.nsplit = p.nsplit;
  w.nfar = p.nfar;
  w.far_tiles = p.far_tiles;
  w.nfar_units = p.nsplit * p.nfar * prm.nbh;
  w.rows = p.rows;
  w.neg_l = neg_l;
  w.neg_d = neg_d;
  w.part = part;
  prm.nunits = w.nfar_units + prm.nkt * prm.nbh;
  e = launch_bwd_kernel<HD, false, true>(g.dO, a.q, a.k, a.v, dQ, g.dK, g.dV, a.M, a.B, (uint64_t)a.NH * HD,
                                         (uint64_t)a.NKV * HD, prm, prm.nunits, st);
  if (e != cudaSuccess) return e;
  const long long nq4 = g.dq_f32 ? 0 : (long long)a.B * a.M * a.NH * HD / 4;
  const long long npart4 = (long long)prm.nbh * p.nsplit * 2 * BK * HD / 4;
  if (nq4 + npart4 == 0) return cudaSuccess;
  launch_pdl(window_finish_kernel, blocks(nq4 + npart4, 256), 256, 0, st, dQ,
             static_cast<__nv_bfloat16*>(g.dQ), nq4, part, 1 + p.nfar, p.nsplit, HD, a.NKV, a.M, npart4, g.dK, g.dV);
  count_launches(1);
  return cudaGetLastError();
}

}  // namespace

size_t window_bwd_workspace(const WindowArgs& a, bool dq_f32) { return win_plan(a, dq_f32).total(); }

cudaError_t launch_window_bwd(const WindowArgs& a, const WindowGrads& g, cudaStream_t st) {
  return a.D == 64 ? launch_win_bwd<64>(a, g, st) : launch_win_bwd<128>(a, g, st);
}

cudaError_t launch_zero_dq(float* dQ, const AttnShape& s, cudaStream_t st) {
  if (s.bh_begin == 0 && s.bh_end == s.B * s.NH)
    return cudaMemsetAsync(dQ, 0, (size_t)s.B * s.T * s.N * sizeof(float), st);
  launch_pdl(zero_dq_shard_kernel, 1184, 256, 0, st, reinterpret_cast<float4*>(dQ), s.T, s.N, s.D, s.NH,
             s.bh_begin, s.bh_end);
  count_launches(1);
  return cudaGetLastError();
}

cudaError_t launch_flash_bwd(const __nv_bfloat16* dO, const __nv_bfloat16* Dv,
                             const float* lse, const __nv_bfloat16* q,
                             const __nv_bfloat16* k, const __nv_bfloat16* v, float* dQ,
                             __nv_bfloat16* dK, __nv_bfloat16* dV, const AttnShape& s,
                             uint32_t* status, cudaStream_t st, bool accumulate_dq) {
  if (s.bh_end <= s.bh_begin) return cudaSuccess;
  return s.D == 64 ? launch_bwd<64>(dO, Dv, lse, q, k, v, dQ, dK, dV, s, status, st, accumulate_dq)
                   : launch_bwd<128>(dO, Dv, lse, q, k, v, dQ, dK, dV, s, status, st, accumulate_dq);
}

}  // namespace ma
