// window_fwd_sm100.cu -- windowAttentionForward, and windowAttentionCached for
// many query rows (sliding window, sinks, grouped K/V heads, sequence lengths,
// queries that start inside a cache), on sm_100a: the causal forward's pipeline
// (flash_fwd_sm100.cu: TMA producer, UMMA issue, two softmax warpgroups with a
// 128-row query tile each, S, P and O in TMEM, lazy rescaling of O), a kernel of
// its own so that neither carries the other's code.
//
// A unit visits the sink tiles and the tiles from the first row's window on, the
// tiles that every row sees whole carry no masking code, and a tile in which
// some row sees nothing is allowed.  Warp 2
// zeroes the rows of a V tile that no query may see (padding, a cache's rows
// past the end or out of the window): P is 0 there, but 0 * NaN is not.  Warp 1
// issues S and warp 3 PV.  SINGLE: a unit is one query tile, not a pair, and the
// two softmax warpgroups share its key tiles (few units, long windows).
// Measured: 8192 tokens, 32 / 8 heads of 128, window 1024, 16 sinks 200 us, 653
// TFLOP/s, bound like the causal form by the chain of a tile's scores,
// exponentials and product; 500 tokens over a cache, 16 heads of 64, window 2048
// 26 us (SINGLE; in pairs 33).
//
// Every mbarrier wait is bounded (mbar_poll, about 2 s); on time-out the CTA sets an
// abort flag that all roles poll, winds down, frees its TMEM and sets
// STATUS_FWD_TIMEOUT in the device status word.
#include <type_traits>

#include "common.cuh"
#include "sm100.cuh"
#include "tmap.h"

namespace ma {
namespace {

using namespace sm100;

constexpr int BM = 128;  // query rows per tile
constexpr int BN = 128;  // keys per tile
constexpr int NARROW = 32;  // columns of a sink tile with at most that many sinks
constexpr int NUM_THREADS = 384;
constexpr int LAUNCH_REGS = 168;    // 65536 / 384, rounded down to a multiple of 8
constexpr int REGS_PRODUCER = 120;  // warpgroup 0 after setmaxnreg.dec
constexpr int REGS_SOFTMAX = 192;  // warpgroups 1, 2 after setmaxnreg.inc
static_assert(128 * REGS_PRODUCER + 256 * REGS_SOFTMAX == NUM_THREADS * LAUNCH_REGS,
              "register split must equal the launch allocation");
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr float RESCALE_THRESHOLD = 8.0f;  // log2 units

template <int HD>
struct FwdCfg {
  static constexpr int KB = HD / 64;  // 64-column blocks per row
  static constexpr int QST = HD == 64 ? 2 : 1;  // Q-pair stages
  static constexpr int KST = HD == 64 ? 3 : 2;  // K tile stages
  static constexpr int VST = HD == 64 ? 3 : 1;  // V tile stages
  // D=64: P_X lives in TMEM (bf16 pairs) and PV_X reads it from there, which
  // halves the shared-memory traffic of the tensor core.  At D=128 S and O of both
  // tiles fill TMEM, and P is staged in shared memory, so that S_X(j+1) need not
  // wait for PV_X(j) as it would with P over S_X's own columns; its 64 KB leave
  // two stages for K and one for V
  static constexpr bool P_TMEM = HD == 64;
  static constexpr uint32_t QT_BYTES = BM * HD * 2;  // one query tile
  static constexpr uint32_t KV_BYTES = BN * HD * 2;
  static constexpr uint32_t P_BYTES = BM * BN * 2;
  // per tile X: P (shared-memory P) or only the epilogue's O staging
  static constexpr uint32_t STG_BYTES = P_TMEM ? BM * HD * 2 : P_BYTES;
  // shared memory map (offsets from a 1024-aligned base)
  static constexpr uint32_t OFF_Q = 0;                          // [QST][2 tiles]
  static constexpr uint32_t OFF_K = OFF_Q + QST * 2 * QT_BYTES;  // [KST]
  static constexpr uint32_t OFF_V = OFF_K + KST * KV_BYTES;      // [VST]
  static constexpr uint32_t OFF_P = OFF_V + VST * KV_BYTES;      // [2 tiles] P / O staging
  // the unit schedule: NSCHED 16-byte launch-control responses
  static constexpr int NSCHED = (int)kSchedSlots;
  // unit order: blocks of HB (batch, head) pairs at D=128, whose query tiles share
  // K/V in L2, one block at D=64 (blocks of 16 at 64 x 1024, 12 heads of 64, window
  // 250: 258 us against 216)
  static constexpr int HB = HD == 128 ? 16 : 0;
  // SINGLE: B's maximum and sum of each row, for A to join
  static constexpr uint32_t OFF_ML = OFF_P + 2 * STG_BYTES;
  static constexpr uint32_t ML_BYTES = BM * 8;
  static constexpr uint32_t OFF_SCHED = OFF_ML + ML_BYTES;
  static constexpr uint32_t OFF_BAR = OFF_SCHED + NSCHED * 16;
  // q_full/empty[QST], k_full/empty[KST], v_full/empty[VST], per tile X:
  // s_full, s_free, p_full, pv_done, o_free; then fin (the S issuer's wind-down),
  // sched_full/empty[NSCHED], v_fixed[VST], fin of the PV issuer and b_done
  static constexpr int NBAR = 2 * QST + 2 * KST + 2 * VST + 2 * 5 + 1 + 2 * NSCHED + VST + 2;
  static constexpr uint32_t OFF_TSLOT = OFF_BAR + NBAR * 8;
  static constexpr uint32_t SMEM_BYTES = OFF_TSLOT + 16 + 1024;  // + alignment slack
  static constexpr uint32_t TCOL_S = 0;     // S_A, S_B at columns 0, 128
  static constexpr uint32_t TCOL_O = 256;   // O_A, O_B at 256, 256+HD
  static constexpr uint32_t TCOL_P = 256 + 2 * HD;  // P_A, P_B (D=64): 64 columns each
  static_assert(!P_TMEM || TCOL_P + 2 * (BN / 2) <= 512, "TMEM columns");
  static_assert(OFF_BAR + NBAR * 8 + 16 + 1024 <= 232448, "shared memory");
};

struct FwdParams {
  int T, NH, nbh, npairs, nqt;
  int nunits;
  float scale_log2;
  float* lse;
  uint32_t* status;
  uint32_t expire_ns;  // time-out test hook (ma_debug_expire_next_wait), 0 = off
  WindowArgs win;
};

// Work units, one CTA each, later queries first: k -> (pair = npairs-1 - k / nbh,
// bh = k % nbh).  A running CTA takes its own unit (k = blockIdx.x) and then, by
// cluster launch control, the units of CTAs that have not started yet, in launch
// order, so units go greedily to whichever SM is free.  With HB > 0 the order is
// blocked: block k / (HB*npairs) holds HB (batch, head) pairs (fewer in the last
// block), whose units in flight share their heads' K/V tiles in L2.
struct Unit {
  int pair, b, h, nA, nB, nkv;
};

template <int HB>
__device__ __forceinline__ Unit decode_unit(const FwdParams& prm, int k) {
  Unit x;
  int bh;
  if constexpr (HB > 0) {  // blocks of HB (batch, head) pairs, heaviest pair first in each
    const int per = HB * prm.npairs;
    const int blk = k / per, r = k % per;
    const int hb = min(HB, prm.nbh - blk * HB);
    x.pair = prm.npairs - 1 - r / hb;
    bh = blk * HB + r % hb;
  } else {
    x.pair = prm.npairs - 1 - k / prm.nbh;
    bh = k % prm.nbh;
  }
  x.b = bh / prm.NH;
  x.h = bh % prm.NH;
  return x;
}

// A unit under a window.  The key tiles it visits, by list index j: the sink
// tiles 0 .. ns-1 before the window, then lo, lo+1, ...; tile A is active for
// j < nA, tile B for j < nB except j == skip (the one tile that A's window
// reaches and B's does not).  A unit of one query tile (single) works on it
// with both: A takes the even list indices, B the odd ones, and A joins them.
struct WinUnit : Unit {
  bool single;
  int tile0; // query tile of A; B's is the next
  int n;     // valid rows of the sequence
  int ns, lo, skip;
  int t0A, t1A, t0B, t1B;  // positions of the first and the last valid row of A and B
  int end;   // keys of the sequence: rows from here on are padding
  bool cached;

  __device__ int key_tile(int j) const { return j < ns ? j : lo + (j - ns); }
  __device__ bool active(int x, int j) const {
    if (single) return (j & 1) == x && j < nkv;
    return x == 0 ? j < nA : j < nB && j != skip;
  }
  // the first list index of a tile: its PV starts the sum
  __device__ int first(int x) const { return x == 1 && (single || skip == 0) ? 1 : 0; }
  // only the sinks of this tile are visible, and they fill a quarter at most:
  // its products and exponentials stop there
  __device__ bool narrow(const WindowArgs& w, int j) const { return j < ns && w.sinks - j * BN <= NARROW; }
  // every valid row of tile x sees every key of the tile at k0
  __device__ bool whole(const WindowArgs& w, int x, int k0) const {
    return k0 + BN - 1 <= (x == 0 ? t0A : t0B) &&
           (k0 > (x == 0 ? t1A : t1B) - w.window || k0 + BN - 1 < w.sinks);
  }
  // rows [*a, *b) of the tile at k0 that no query sees: past the end
  __device__ bool past_end(const WindowArgs& w, int k0, int* a) const {
    *a = max(0, end - k0);
    return k0 + BN > end && end < w.K && *a < BN;
  }
  // and, in a cache, between the sinks and the first row's window
  __device__ bool out_of_window(const WindowArgs& w, int k0, int* a, int* b) const {
    *a = min(max(w.sinks, k0) - k0, BN);
    *b = min(max(0, t0A - w.window + 1) - k0, BN);
    return cached && *a < *b;
  }
  __device__ bool fix(const WindowArgs& w, int k0) const {
    int a, b;
    return past_end(w, k0, &a) || out_of_window(w, k0, &a, &b);
  }
};

template <int HB, bool SINGLE>
__device__ __forceinline__ WinUnit decode_win_unit(const FwdParams& prm, int k) {
  const WindowArgs& w = prm.win;
  WinUnit x;
  static_cast<Unit&>(x) = decode_unit<HB>(prm, k);
  x.single = SINGLE;
  x.tile0 = SINGLE ? x.pair : 2 * x.pair;
  x.n = w.len(x.b);
  x.cached = w.start != nullptr;
  x.nA = x.nB = x.nkv = x.ns = x.lo = 0;
  x.t0A = x.t1A = x.t0B = x.t1B = 0;
  x.skip = -1;
  x.end = x.n > 0 ? w.pos(x.b, x.n - 1) + 1 : 0;
  const int r0 = x.tile0 * BM;
  if (r0 >= x.n) return x;
  const int nS = w.sinks / BN + (w.sinks % BN != 0);
  const bool b = !SINGLE && r0 + BM < x.n;
  const int rB = SINGLE ? r0 : min(r0 + BM, x.n - 1);  // one tile: B's rows are A's
  x.t0A = w.pos(x.b, r0);
  x.t1A = w.pos(x.b, min(r0 + BM - 1, x.n - 1));
  x.t0B = w.pos(x.b, rB);
  x.t1B = w.pos(x.b, min(rB + BM - 1, x.n - 1));
  const int loB = max(0, x.t0B - w.window + 1) / BN;
  x.lo = max(0, x.t0A - w.window + 1) / BN;
  x.ns = min(nS, x.lo);
  x.nA = x.ns + x.t1A / BN - x.lo + 1;
  x.nB = b ? x.ns + x.t1B / BN - x.lo + 1 : 0;
  x.skip = b && loB > x.lo && x.lo >= nS ? x.ns : -1;
  x.nkv = b ? x.nB : x.nA;
  if (SINGLE && x.nkv > 1) x.nB = x.nkv;
  return x;
}

template <int HD, bool SINGLE>
__global__ void __launch_bounds__(NUM_THREADS, 1)
    window_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                     const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmO,
                     const FwdParams prm) {
  using C = FwdCfg<HD>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ int abort_flag;
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t sbase = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (sbase - raw);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  const uint32_t bar0 = sbase + C::OFF_BAR;
  auto BAR_QF = [&](int s) { return bar0 + 8u * s; };
  auto BAR_QE = [&](int s) { return bar0 + 8u * (C::QST + s); };
  auto BAR_KF = [&](int s) { return bar0 + 8u * (2 * C::QST + s); };
  auto BAR_KE = [&](int s) { return bar0 + 8u * (2 * C::QST + C::KST + s); };
  auto BAR_VF = [&](int s) { return bar0 + 8u * (2 * C::QST + 2 * C::KST + s); };
  auto BAR_VE = [&](int s) { return bar0 + 8u * (2 * C::QST + 2 * C::KST + C::VST + s); };
  const uint32_t barX = bar0 + 8u * (2 * C::QST + 2 * C::KST + 2 * C::VST);
  // per tile X in {0: A, 1: B}
  auto BAR_SF = [&](int x) { return barX + 8u * (0 * 2 + x); };
  auto BAR_SE = [&](int x) { return barX + 8u * (1 * 2 + x); };
  auto BAR_PF = [&](int x) { return barX + 8u * (2 * 2 + x); };
  auto BAR_PV = [&](int x) { return barX + 8u * (3 * 2 + x); };
  auto BAR_OE = [&](int x) { return barX + 8u * (4 * 2 + x); };
  const uint32_t BAR_FIN = barX + 8u * 10;    // the S issuer's last commit (wind-down)
  auto BAR_UF = [&](int s) { return barX + 8u * (11 + s); };              // response s landed
  auto BAR_UE = [&](int s) { return barX + 8u * (11 + C::NSCHED + s); };  // response s read by all
  auto BAR_VZ = [&](int s) { return barX + 8u * (11 + 2 * C::NSCHED + s); };  // V slot s zeroed where it must be
  const uint32_t BAR_FIN2 = barX + 8u * (11 + 2 * C::NSCHED + C::VST);  // the PV issuer's wind-down
  const uint32_t BAR_MG = BAR_FIN2 + 8;  // B's part of a shared tile is complete
  // unit g >= 1 of this CTA is the one launch-control response g-1 names
  // (requested by the TMA producer when it starts unit g-1); readers: the
  // producer, both issuers, the warp that zeroes V rows and the 8 softmax warps
  constexpr uint32_t SCHED_READERS = 12;
  auto unit = [&](int k) { return decode_win_unit<C::HB, SINGLE>(prm, k); };
  const uint32_t tslot = sbase + C::OFF_TSLOT;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < C::QST; ++s) {
      mbar_init(BAR_QF(s), 1);
      mbar_init(BAR_QE(s), 1);
    }
    for (int s = 0; s < C::KST; ++s) {
      mbar_init(BAR_KF(s), 1);
      mbar_init(BAR_KE(s), 1);
    }
    for (int s = 0; s < C::VST; ++s) {
      mbar_init(BAR_VF(s), 1);
      mbar_init(BAR_VE(s), 2);  // PV, and the warp that zeroes rows
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(BAR_SF(x), 1);
      mbar_init(BAR_SE(x), 128);
      mbar_init(BAR_PF(x), 128);
      mbar_init(BAR_PV(x), 1);
      mbar_init(BAR_OE(x), 128);
    }
    mbar_init(BAR_FIN, 1);
    for (int u = 0; u < C::NSCHED; ++u) {
      mbar_init(BAR_UF(u), 1);
      mbar_init(BAR_UE(u), SCHED_READERS);
    }
    for (int s = 0; s <= C::VST; ++s) mbar_init(BAR_VZ(s), 1);  // and BAR_FIN2
    mbar_init(BAR_MG, 128);
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
  pdl_wait_and_release();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(gbase + C::OFF_TSLOT);
  volatile int* abort_p = &abort_flag;
  const Sched sch{sbase + C::OFF_SCHED, BAR_UF(0), BAR_UE(0), abort_p};

  if (warp < 4) {
    reg_dealloc<REGS_PRODUCER>();
    if (warp == 0 && lane == 0) {
      // ---------------------------------------------------- TMA producer
      tma_prefetch_desc(&tmQ);
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
      uint32_t qc = 0, kc = 0, vc = 0;
      uint32_t nreq = 0;  // launch-control requests issued (request r names unit r+1)
      bool ok = true;
      for (int g = 0; ok; ++g) {
        const int k = sched_unit<false>(sch, g);
        if (k < 0) break;
        // request unit g+1 now, a unit ahead of every reader
        if (!sched_request(sch, nreq)) break;
        ++nreq;
        const auto un = unit(k);
        const int col0 = un.h * HD;
        const int kv0 = un.h / (prm.win.NH / prm.win.NKV) * HD;  // columns of the K/V head
        if (un.nkv == 0) continue;  // only padding
        const int qs = qc % C::QST;
        if (qc >= C::QST && !mbar_poll(BAR_QE(qs), ((qc / C::QST) - 1) & 1, abort_p)) break;
        const int ntile = !SINGLE && un.nB > 0 ? 2 : 1;
        mbar_arrive_expect_tx(BAR_QF(qs), ntile * C::QT_BYTES);
        for (int x = 0; x < ntile; ++x)
          for (int kb = 0; kb < C::KB; ++kb)
            tma_load_3d(sbase + C::OFF_Q + (qs * 2 + x) * C::QT_BYTES + kb * BM * 128, &tmQ,
                        BAR_QF(qs), col0 + kb * 64, (un.tile0 + x) * BM, un.b);
        ++qc;
        for (int j = 0; j < un.nkv; ++j) {
          const int kt = un.key_tile(j);
          const int ks = kc % C::KST;
          if (kc >= C::KST && !mbar_poll(BAR_KE(ks), ((kc / C::KST) - 1) & 1, abort_p)) { ok = false; break; }
          mbar_arrive_expect_tx(BAR_KF(ks), C::KV_BYTES);
          for (int kb = 0; kb < C::KB; ++kb)
            tma_load_3d(sbase + C::OFF_K + ks * C::KV_BYTES + kb * BN * 128, &tmK, BAR_KF(ks),
                        kv0 + kb * 64, kt * BN, un.b);
          ++kc;
          const int vs = vc % C::VST;
          if (vc >= C::VST && !mbar_poll(BAR_VE(vs), ((vc / C::VST) - 1) & 1, abort_p)) { ok = false; break; }
          mbar_arrive_expect_tx(BAR_VF(vs), C::KV_BYTES);
          for (int kb = 0; kb < C::KB; ++kb)
            tma_load_3d(sbase + C::OFF_V + vs * C::KV_BYTES + kb * BN * 128, &tmV, BAR_VF(vs),
                        kv0 + kb * 64, kt * BN, un.b);
          ++vc;
        }
      }
      if (*abort_p) {  // wind-down: let the loads and the request still in flight land
        sched_drain(sch, nreq);
        drain_ring(BAR_QF, C::QST, qc);
        drain_ring(BAR_KF, C::KST, kc);
        drain_ring(BAR_VF, C::VST, vc);
      }
    } else if (warp == 1 && lane == 0) {
      // ---------------------------------------------------- S, under a window
      // S_X(j) = Q_X K_j^T, as soon as softmax X has read S_X(j-1).  Another
      // warp issues the products with V, so neither waits for the other's tile.
      constexpr uint32_t IDESC_S = idesc_bf16_f32(BM, BN, 0, 0);
      constexpr uint32_t IDESC_SN = idesc_bf16_f32(BM, NARROW, 0, 0);
      uint32_t qc = 0, kc = 0, sc[2] = {0, 0};
      bool ok = true;
      for (int g = 0; ok; ++g) {
        const int k = sched_unit<false>(sch, g);
        if (k < 0) break;
        const auto un = unit(k);
        if (un.nkv == 0) continue;  // only padding
        const int qs = qc % C::QST;
        if (!mbar_poll(BAR_QF(qs), (qc / C::QST) & 1, abort_p)) break;
        for (int j = 0; ok && j < un.nkv; ++j, ++kc) {
          const int ks = kc % C::KST;
          ok = mbar_poll(BAR_KF(ks), (kc / C::KST) & 1, abort_p);
          const uint32_t idesc = un.narrow(prm.win, j) ? IDESC_SN : IDESC_S;
          const uint32_t dk = desc_lo(sbase + C::OFF_K + ks * C::KV_BYTES, 16);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            if (!ok || !un.active(x, j)) continue;
            if (sc[x] >= 1 && !mbar_poll(BAR_SE(x), (sc[x] - 1) & 1, abort_p)) {
              ok = false;
              continue;
            }
            tc_fence_after();
            const uint32_t dq = desc_lo(sbase + C::OFF_Q + (qs * 2 + (SINGLE ? 0 : x)) * C::QT_BYTES, 16);
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk) {
              const uint32_t off = ((kk >> 2) * (BM * 128) + (kk & 3) * 32) >> 4;
              umma_bf16_ss_lo(tmem + C::TCOL_S + x * BN, dq + off, dk + off, idesc, kk > 0 ? 1u : 0u);
            }
            umma_commit(BAR_SF(x));
            ++sc[x];
          }
          if (ok) umma_commit(BAR_KE(ks));
        }
        if (ok) umma_commit(BAR_QE(qs));
        ++qc;
      }
      if (*abort_p) {  // wind-down: every UMMA issued must complete before TMEM is freed
        umma_commit(BAR_FIN);
        mbar_wait_for(BAR_FIN, 0, kDrainLimitNs);
      }
    } else if (warp == 3 && lane == 0) {
      // --------------------------------------------------- PV, under a window
      // O_X += P_X V_j, once softmax X has written P_X(j)
      constexpr uint32_t IDESC_O = idesc_bf16_f32(BM, HD, 0, 1);
      uint32_t vc = 0, pvc[2] = {0, 0}, uc[2] = {0, 0};
      uint32_t vzp = 0;  // bit s = parity of v_fixed[s]'s next phase
      // time-out test hook: while the first scores are formed, wait until its limit
      // runs out on the barrier that nothing arrives at before the wind-down
      if (prm.expire_ns) mbar_wait(BAR_FIN2, 0, abort_p, prm.expire_ns);
      bool ok = true;
      for (int g = 0; ok; ++g) {
        const int k = sched_unit<false>(sch, g);
        if (k < 0) break;
        const auto un = unit(k);
        for (int j = 0; ok && j < un.nkv; ++j, ++vc) {
          const int vs = vc % C::VST;
          ok = mbar_poll(BAR_VF(vs), (vc / C::VST) & 1, abort_p);
          if (ok && un.fix(prm.win, un.key_tile(j) * BN)) {  // warp 2 has zeroed its unseen rows
            ok = mbar_poll(BAR_VZ(vs), (vzp >> vs) & 1, abort_p);
            vzp ^= 1u << vs;
          }
          const bool narrow = un.narrow(prm.win, j);
          const uint32_t dv = desc_lo(sbase + C::OFF_V + vs * C::KV_BYTES, BN * 128);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            if (!ok || !un.active(x, j)) continue;
            const bool first = j == un.first(x);
            ok = mbar_poll(BAR_PF(x), pvc[x] & 1, abort_p);
            // the tile's previous unit has been read out of O_X
            if (ok && first && uc[x] >= 1) ok = mbar_poll(BAR_OE(x), (uc[x] - 1) & 1, abort_p);
            if (!ok) continue;
            tc_fence_after();
            const uint32_t dp = desc_lo(sbase + C::OFF_P + x * C::STG_BYTES, 16);
#pragma unroll
            for (int kk = 0; kk < BN / 16; ++kk) {
              if (narrow && kk >= NARROW / 16) break;
              const uint32_t acc = !first || kk > 0 ? 1u : 0u;
              if (C::P_TMEM)  // A = P_X from TMEM: 8 columns per 16 keys
                umma_bf16_ts_lo(tmem + C::TCOL_O + x * HD, tmem + C::TCOL_P + x * (BN / 2) + kk * 8,
                                dv + kk * (2048 >> 4), IDESC_O, acc);
              else
                umma_bf16_ss_lo(tmem + C::TCOL_O + x * HD, dp + (((kk >> 2) * (BM * 128) + (kk & 3) * 32) >> 4),
                                dv + kk * (2048 >> 4), IDESC_O, acc);
            }
            umma_commit(BAR_PV(x));
            ++pvc[x];
          }
          if (ok) umma_commit(BAR_VE(vs));
        }
        if (un.nA > 0) ++uc[0];
        if (un.nB > 0) ++uc[1];
      }
      if (*abort_p) {
        umma_commit(BAR_FIN2);
        mbar_wait_for(BAR_FIN2, 0, kDrainLimitNs);
      }
    } else if (warp == 2) {
      // ------------------------------------------------ unseen rows of V
      uint32_t vc = 0;
      bool ok = true;
      for (int g = 0; ok; ++g) {
        const int k = sched_unit<true>(sch, g);
        if (k < 0) break;
        const auto un = unit(k);
        for (int j = 0; ok && j < un.nkv; ++j) {
          // every tile is waited for and released, so that this warp stays
          // within one phase of each slot's barriers
          const int k0 = un.key_tile(j) * BN;
          const uint32_t v = vc + j, vs = v % C::VST;
          ok = mbar_poll_warp(BAR_VF(vs), (v / C::VST) & 1, abort_p);
          if (!ok) break;
          if (!un.fix(prm.win, k0)) {
            if (lane == 0) mbar_arrive(BAR_VE(vs));
            continue;
          }
          // rows [a, b) are contiguous in each 64-column block (the swizzle
          // permutes the chunks of a row within its 128 bytes)
          auto zero = [&](int a, int b) {
            for (int kb = 0; kb < C::KB; ++kb) {
              uint4* blk = reinterpret_cast<uint4*>(gbase + C::OFF_V + vs * C::KV_BYTES + kb * BN * 128);
              for (int i = a * 8 + lane; i < b * 8; i += 32) blk[i] = make_uint4(0u, 0u, 0u, 0u);
            }
          };
          int a, b;
          if (un.past_end(prm.win, k0, &a)) zero(a, BN);
          if (un.out_of_window(prm.win, k0, &a, &b)) zero(a, b);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(BAR_VZ(vs));
            mbar_arrive(BAR_VE(vs));
          }
        }
        vc += un.nkv;
      }
    }
  } else {
    reg_alloc<REGS_SOFTMAX>();
    // --------------------------------------------------------- softmax
    const int x = (warp - 4) >> 2;               // 0: tile A (warps 4-7), 1: tile B (8-11)
    const uint32_t wg_bar = 1 + x;               // named barrier of this warpgroup
    const int quarter = warp & 3;                // TMEM lane quarter of this warp
    const int row = quarter * 32 + lane;         // query row within the tile
    const uint32_t trow = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t tcol_s = C::TCOL_S + x * BN, tcol_o = C::TCOL_O + x * HD;
    const float c = prm.scale_log2;
    const bool wg_leader = (warp == 4 + 4 * x) && lane == 0;
    uint8_t* pbuf = gbase + C::OFF_P + x * C::STG_BYTES;
    uint32_t sc = 0;  // S_X consumed so far (== P_X produced)
    uint32_t nmg = 0;       // A: shared tiles joined so far
    uint32_t scb = 0;       // A: key tiles B has worked on in them
    int k = sched_unit<true>(sch, 0);
    for (uint32_t g = 1; k >= 0; ++g) {
      const auto un = unit(k);
      const int nt = x == 0 ? un.nA : un.nB;
      const int qtile = un.tile0 + (SINGLE ? 0 : x);
      const int grow = qtile * BM + row;
      bool ok = true, store = true;
      // The last store (of O, or of a padding unit's zeros) must have read the
      // staging before it is written again: at D=128 it holds P from a unit's first
      // tile on, so wait here; at D=64 (P in TMEM) only the epilogue writes it and
      // waits, so a unit's first tiles overlap the store.
      if (!C::P_TMEM || nt == 0) {
        if (wg_leader) bulk_wait_read<0>();
        bar_sync_named(wg_bar, 128);
      }
      if (nt == 0) {  // only padding: O = 0, l = -inf (rows past T are clipped)
        store = !(SINGLE && x == 1) && qtile * BM < prm.T;
        for (int kb = 0; kb < C::KB; ++kb)
#pragma unroll
          for (int ch = 0; ch < 8; ++ch)
            *reinterpret_cast<uint4*>(pbuf + kb * (BM * 128) + row * 128 + ch * 16) = make_uint4(0u, 0u, 0u, 0u);
        fence_proxy_async_smem();
        if (store && grow < prm.T) prm.lse[((long long)un.b * prm.T + grow) * prm.NH + un.h] = -INFINITY;
      } else {
        float m_used = -INFINITY, l_sum = 0.0f;
        // one key tile; DIAG: some key of it is hidden from some row (past the
        // diagonal, out of the window, not a sink).  NC: the tile's first columns that
        // matter (all 128, or a sink tile's 32).  Three instances, so that the tiles
        // which every row sees whole carry no masking code.
        auto tile = [&](auto diag_tag, auto nc_tag, int j) -> bool {
          constexpr bool DIAG = decltype(diag_tag)::value;
          constexpr int NC = decltype(nc_tag)::value;
          if (!mbar_poll_warp(BAR_SF(x), sc & 1, abort_p)) return false;
          tc_fence_after();
          float s[NC];
          if constexpr (NC == 32) {
            uint32_t ra[32];
            tmem_ld32(trow + tcol_s, ra);
            tmem_wait_ld_dep(ra);
#pragma unroll
            for (int i = 0; i < 32; ++i) s[i] = __uint_as_float(ra[i]);
          } else {
#pragma unroll
            for (int cc = 0; cc < NC; cc += 64) {
              uint32_t ra[32], rb[32];
              tmem_ld32(trow + tcol_s + cc, ra);
              tmem_ld32(trow + tcol_s + cc + 32, rb);
              tmem_wait_ld_dep(ra, rb);
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                s[cc + i] = __uint_as_float(ra[i]);
                s[cc + 32 + i] = __uint_as_float(rb[i]);
              }
            }
          }
          tc_fence_before();
          mbar_arrive(BAR_SE(x));
          if constexpr (DIAG) {
            // key k0 + i is visible up to the row's own position, and from its
            // window's first key on or among the sinks; 32 keys to a word of
            // bits, one test and one select a key
            const int k0 = un.key_tile(j) * BN;
            const int t = prm.win.pos(un.b, qtile * BM + row);
            const int up = t - k0, from = t - prm.win.window + 1 - k0, sink = prm.win.sinks - k0;
#pragma unroll
            for (int w = 0; w < NC; w += 32) {
              const uint32_t see = bits_below(up + 1 - w) & (~bits_below(from - w) | bits_below(sink - w));
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (!(see & (1u << i))) s[w + i] = -INFINITY;
            }
          }
          // row maximum: 8 independent partial maxima, 3-input max (short chains)
          float pm[8];
#pragma unroll
          for (int q = 0; q < 8; ++q) pm[q] = fmaxf(s[q], s[8 + q]);
#pragma unroll
          for (int i = 16; i < NC; i += 16)
#pragma unroll
            for (int q = 0; q < 8; ++q) pm[q] = fmax3(pm[q], s[i + q], s[i + 8 + q]);
          const float mx = fmax3(fmax3(pm[0], pm[1], pm[2]), fmax3(pm[3], pm[4], pm[5]),
                                 fmaxf(pm[6], pm[7]));
          const float m_new = fmaxf(m_used, mx * c);
          // lazy rescaling: only rows whose maximum grew by more than 2^8 move
          // m_used; O_X is rescaled below, once PV_X(j-1) has completed
          bool rescale = false;
          float alpha = 1.0f;
          const bool first = j == un.first(x);
          if (first) {
            m_used = m_new;
          } else {
            const bool need = m_new > m_used + RESCALE_THRESHOLD;
            rescale = __any_sync(0xffffffffu, need);
            if (need) {
              alpha = ex2(m_used - m_new);
              l_sum *= alpha;
              m_used = m_new;
            }
          }
          // P = 2^(S*c - m) with packed fp32x2 FMAs; row sum in 4 packed partials
          // (a row that has seen no key yet has m = -inf and P = 2^-inf = 0)
          const float base = m_used == -INFINITY ? 0.0f : m_used;
          const float2 c2 = make_float2(c, c), nm2 = make_float2(-base, -base);
          float2 ps[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f),
                          make_float2(0.f, 0.f)};
          uint32_t pk[NC / 2];  // P as bf16 pairs, even key in the low half
#pragma unroll
          for (int i = 0; i < NC; i += 2) {
            const float2 t = __ffma2_rn(make_float2(s[i], s[i + 1]), c2, nm2);
            const float e0 = ex2(t.x), e1 = ex2(t.y);
            ps[(i >> 1) & 3] = __fadd2_rn(ps[(i >> 1) & 3], make_float2(e0, e1));
            pk[i / 2] = pack_bf16(e0, e1);
          }
          l_sum += (ps[0].x + ps[0].y) + (ps[1].x + ps[1].y) + (ps[2].x + ps[2].y) +
                   (ps[3].x + ps[3].y);
          // PV_X(j-1) must be complete before O_X is rescaled and before P_X(j)
          // overwrites P_X (waited for only now, so the exponentials overlap it)
          if (!first) {
            if (!mbar_poll_warp(BAR_PV(x), (sc - 1) & 1, abort_p)) return false;
            tc_fence_after();
          }
          if (rescale) {
#pragma unroll
            for (int cc = 0; cc < HD; cc += 16) {
              uint32_t r[16];
              tmem_ld16(trow + tcol_o + cc, r);
              tmem_wait_ld_dep(r);
#pragma unroll
              for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
              tmem_st16(trow + tcol_o + cc, r);
            }
            tmem_wait_st();
          }
          if constexpr (C::P_TMEM) {
            // this lane's P row into P_X
#pragma unroll
            for (int q = 0; q < NC / 32; ++q) {
              uint32_t r[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) r[i] = pk[q * 16 + i];
              tmem_st16(trow + C::TCOL_P + x * (BN / 2) + q * 16, r);
            }
            tmem_wait_st();
          } else {
#pragma unroll
            for (int kb = 0; kb < (NC + 63) / 64; ++kb) {
#pragma unroll
              for (int ch = 0; ch < (NC < 64 ? NC / 8 : 8); ++ch) {
                const int c0 = (kb * 64 + ch * 8) / 2;
                const uint4 v = make_uint4(pk[c0], pk[c0 + 1], pk[c0 + 2], pk[c0 + 3]);
                *reinterpret_cast<uint4*>(pbuf + kb * (BM * 128) + row * 128 + ((ch ^ (row & 7)) * 16)) = v;
              }
            }
            fence_proxy_async_smem();
          }
          tc_fence_before();
          mbar_arrive(BAR_PF(x));
          ++sc;
          return true;
        };
        using All = std::integral_constant<int, BN>;
        for (int j = 0; ok && j < nt; ++j) {
          if (!un.active(x, j)) continue;
          if (un.narrow(prm.win, j)) ok = tile(std::true_type{}, std::integral_constant<int, NARROW>{}, j);
          else if (un.whole(prm.win, x, un.key_tile(j) * BN)) ok = tile(std::false_type{}, All{}, j);
          else ok = tile(std::true_type{}, All{}, j);
        }
        // --------------------------------------------- epilogue of tile X
        ok = ok && mbar_poll_warp(BAR_PV(x), (sc - 1) & 1, abort_p);
        if constexpr (C::P_TMEM) {
          // the epilogue is the staging's first writer in this unit
          if (wg_leader) bulk_wait_read<0>();
          bar_sync_named(wg_bar, 128);
        }
        const bool joined = SINGLE && un.nB > 0;
        if (joined && x == 1) {
          // this half's maximum and sum; O_B stays in TMEM, where A reads it
          if (ok) {
            reinterpret_cast<float2*>(gbase + C::OFF_ML)[row] = make_float2(m_used, l_sum);
            tc_fence_before();
            mbar_arrive(BAR_MG);
          }
          store = false;
        }
        float fa = 1.0f, fb = 0.0f;  // factors of O_A and O_B
        if (joined && x == 0) {
          scb += un.nkv / 2;
          ok = ok && mbar_poll_warp(BAR_MG, nmg++ & 1, abort_p) &&
                mbar_poll_warp(BAR_PV(1), (scb - 1) & 1, abort_p);
          if (ok) {
            const float2 ml = reinterpret_cast<const float2*>(gbase + C::OFF_ML)[row];
            const float top = fmaxf(m_used, ml.x), base = top == -INFINITY ? 0.0f : top;
            fa = ex2(m_used - base);
            fb = ex2(ml.x - base);
            l_sum = l_sum * fa + ml.y * fb;
            m_used = top;
          }
        }
        if (ok && store) {
          tc_fence_after();
          const float inv = 1.0f / l_sum;
          const bool valid = grow < un.n;
          // stage O (bf16) in this tile's P buffer (free: its last PV is done);
          // O is read from TMEM 64 columns (two loads, one wait) at a time
#pragma unroll
          for (int c64 = 0; c64 < HD; c64 += 64) {
            uint32_t ra[32], rb[32];
            tmem_ld32(trow + tcol_o + c64, ra);
            tmem_ld32(trow + tcol_o + c64 + 32, rb);
            tmem_wait_ld_dep(ra, rb);
            if (joined) {
              uint32_t rc[32], rd[32];
              tmem_ld32(trow + C::TCOL_O + HD + c64, rc);
              tmem_ld32(trow + C::TCOL_O + HD + c64 + 32, rd);
              tmem_wait_ld_dep(rc, rd);
              auto join = [&](uint32_t a, uint32_t b) {
                return __float_as_uint(__uint_as_float(a) * fa + __uint_as_float(b) * fb);
              };
#pragma unroll
              for (int i = 0; i < 32; ++i) ra[i] = join(ra[i], rc[i]), rb[i] = join(rb[i], rd[i]);
            }
#pragma unroll
            for (int c16 = 0; c16 < 64; c16 += 16) {
              const uint32_t* r = c16 < 32 ? ra + c16 : rb + (c16 - 32);
              const int cc = c64 + c16;
              uint4 v0, v1;
              v0.x = pack_bf16(__uint_as_float(r[0]) * inv, __uint_as_float(r[1]) * inv);
              v0.y = pack_bf16(__uint_as_float(r[2]) * inv, __uint_as_float(r[3]) * inv);
              v0.z = pack_bf16(__uint_as_float(r[4]) * inv, __uint_as_float(r[5]) * inv);
              v0.w = pack_bf16(__uint_as_float(r[6]) * inv, __uint_as_float(r[7]) * inv);
              v1.x = pack_bf16(__uint_as_float(r[8]) * inv, __uint_as_float(r[9]) * inv);
              v1.y = pack_bf16(__uint_as_float(r[10]) * inv, __uint_as_float(r[11]) * inv);
              v1.z = pack_bf16(__uint_as_float(r[12]) * inv, __uint_as_float(r[13]) * inv);
              v1.w = pack_bf16(__uint_as_float(r[14]) * inv, __uint_as_float(r[15]) * inv);
              if (!valid) v0 = v1 = make_uint4(0u, 0u, 0u, 0u);  // a padding row, whatever it computed
              const int kb = cc / 64, ch = (cc % 64) / 8;
              uint8_t* blk = pbuf + kb * (BM * 128) + row * 128;
              uint4* p0 = reinterpret_cast<uint4*>(blk + ((ch ^ (row & 7)) * 16));
              uint4* p1 = reinterpret_cast<uint4*>(blk + (((ch + 1) ^ (row & 7)) * 16));
              *p0 = v0;
              *p1 = v1;
            }
          }
          tc_fence_before();
          mbar_arrive(BAR_OE(x));  // O_X may be overwritten by the next unit
          if (joined) mbar_arrive(BAR_OE(1));
          fence_proxy_async_smem();
          if (grow < prm.T) {
            const long long ri = ((long long)un.b * prm.T + grow) * prm.NH + un.h;
            prm.lse[ri] = !valid ? -INFINITY : (m_used + log2f(l_sum)) * LN2;
          }
        }
      }
      // One verdict for the warpgroup, on this unit and on the wait for the next (after
      // a time-out one warp's wait may have given up where another's found the
      // response): the barriers above wait for all four warps.
      k = sched_unit<true>(sch, g);
      __syncwarp();
      if (!bar_red_and(wg_bar, 128, ok && k != -2)) break;
      if (store && wg_leader) {
        for (int kb = 0; kb < C::KB; ++kb)
          tma_store_3d(&tmO, sbase + C::OFF_P + x * C::STG_BYTES + kb * BM * 128, un.h * HD + kb * 64,
                       qtile * BM, un.b);
        bulk_commit();
      }
    }
    if (wg_leader) bulk_wait<0>();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (threadIdx.x == 0 && abort_flag) atomicOr(prm.status, STATUS_FWD_TIMEOUT);
}

template <int HD, bool SINGLE>
cudaError_t launch_fwd_kernel(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                              const CUtensorMap& to, const FwdParams& prm, cudaStream_t st) {
  using C = FwdCfg<HD>;
  // The setmaxnreg split assumes the kernel was compiled to exactly
  // LAUNCH_REGS registers per thread; refuse to launch otherwise.
  static const cudaError_t reg_check = [] {
    cudaFuncAttributes a;
    cudaError_t e = cudaFuncGetAttributes(&a, window_fwd_kernel<HD, SINGLE>);
    if (e != cudaSuccess) return e;
    return a.numRegs == LAUNCH_REGS ? cudaSuccess : cudaErrorInvalidKernelImage;
  }();
  if (reg_check != cudaSuccess) return reg_check;
  cudaError_t e = cudaFuncSetAttribute(window_fwd_kernel<HD, SINGLE>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES);
  if (e != cudaSuccess) return e;
  launch_pdl(window_fwd_kernel<HD, SINGLE>, prm.nunits, NUM_THREADS, C::SMEM_BYTES, st, tq, tk, tv, to, prm);
  count_launches(1);
  return cudaGetLastError();
}

template <int HD>
cudaError_t launch_win(const WindowArgs& a, cudaStream_t st) {
  CUtensorMap tq, tk, tv, to;
  const CUtensorMapDataType bf = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUtensorMapSwizzle sw = CU_TENSOR_MAP_SWIZZLE_128B;
  const uint64_t n = (uint64_t)a.NH * HD, nkv = (uint64_t)a.NKV * HD;
  if (!make_tmap_3d(&tq, a.q, bf, 2, n, a.M, a.B, 64, BM, sw) ||
      !make_tmap_3d(&tk, a.k, bf, 2, nkv, a.K, a.B, 64, BN, sw) ||
      !make_tmap_3d(&tv, a.v, bf, 2, nkv, a.K, a.B, 64, BN, sw) ||
      !make_tmap_3d(&to, a.out, bf, 2, n, a.M, a.B, 64, BM, sw))
    return cudaErrorInvalidValue;
  FwdParams prm{};
  prm.T = a.M;
  prm.NH = a.NH;
  prm.nbh = a.B * a.NH;
  prm.nqt = (a.M + BM - 1) / BM;
  // pairs share their K/V tiles, but a few of them leave most SMs idle: then a
  // unit is one tile, its keys shared by the two softmax warpgroups (2 x 500
  // queries of 16 heads over a cache: 64 pairs or 128 tiles for 148 SMs)
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const bool single = (long long)prm.nqt * prm.nbh <= sms;
  prm.npairs = single ? prm.nqt : (prm.nqt + 1) / 2;
  prm.nunits = prm.npairs * prm.nbh;
  prm.scale_log2 = LOG2E / sqrtf((float)HD);
  prm.lse = a.l;
  prm.status = a.status;
  prm.expire_ns = take_expire_request(STATUS_FWD_TIMEOUT);
  prm.win = a;
  return single ? launch_fwd_kernel<HD, true>(tq, tk, tv, to, prm, st)
                : launch_fwd_kernel<HD, false>(tq, tk, tv, to, prm, st);
}

}  // namespace

cudaError_t launch_window_fwd(const WindowArgs& a, cudaStream_t st) {
  return a.D == 64 ? launch_win<64>(a, st) : launch_win<128>(a, st);
}

}  // namespace ma
