// window_bwd_sm100.cu -- windowAttentionBackward on sm_100a: tcgen05 UMMA with
// TMEM accumulators, TMA-staged tiles, units dealt by cluster launch control.
//
//   P_ij  = exp(q_i k_j / sqrt(D) - l_i) where query i sees key j, else 0
//   dS_ij = P_ij (dO_i v_j - delta_i) / sqrt(D),  delta_i = dO_i . O_i
//   dV_j  = sum_i P_ij dO_i,  dK_j = sum_i dS_ij q_i  (over the group's heads)
//   dQ_i  = sum_j dS_ij k_j
//
// Two passes of one kernel, each of which owns what it sums and keeps it in
// TMEM until its single store, so nothing is added up in global memory and the
// result does not depend on the order in which units run:
//   dK/dV pass  unit = 128 keys of a K/V head; steps = the query tiles that see
//               them, for each query head of the group.  Rows are keys.
//   dQ pass     unit = 128 queries of a head; steps = the key tiles that they
//               see (sinks, window).  Rows are queries.
// Both have a resident pair of tiles (R1, R2) = (K, V) or (Q, dO) and a streamed
// pair (X1, X2) = (Q, dO) or (K, V); a step is
//   S  = R1 X1^T, dP = R2 X2^T       UMMA 128x128xD -> TMEM
//   P  = exp2(S c - l log2e), dS = P (dP - delta) / sqrt(D)   compute warps
//   dK/dV: dV += P X2, dK += dS X1   dQ: dQ += dS X1          UMMA 128xDx128
// P and dS go back to TMEM as bf16 pairs, over the dP columns they came from, and
// the products take them from there (a tile in shared memory would cost its
// write, its reads and the room for the rings).  (The form that computes all
// three gradients in one pass and adds dQ up in global memory spends 5 products
// a step where these spend 4 + 3, but it had to zero dQ, add 64 KB a step into
// L2 and convert the sums: at B=2, 4096 tokens, 16 / 4 heads of 128, window 1000
// it took 384 us, at up to 64 x 1024, 12 heads of 64, window 250 605 us; these
// passes take 272 (571 TFLOP/s; the tensor pipe is busy 56 % of the time) and 420
// (units of three steps).  The chain from a step's scores over the row math to
// its products bounds them, at D=64 the row math's instructions.)
//
// Pipeline: S of the next step is issued as soon as this step's has been read,
// and with two dP buffers (all but dK/dV at D=128) dP ahead of this step's
// products too, so the tensor core works on the next step while the compute
// warps form this one's P and dS.
//
// Roles (512 threads): warpgroup 0 (72 registers): warp 0 TMA producer, which
// also decodes the units and passes them on through shared memory (each role
// decoding for itself is more code than the instruction cache holds); warp 1
// issues S and dP, warp 3 the products (one thread for both spent more on waits
// and addresses than the tensor core on the work: a step 2.9 us); warp 2
// brings the statistics of the dK/dV pass and zeroes padding rows of streamed
// tiles (their P is 0, but 0 * NaN is not), and passes the step on (Cfg::ONE).  Warpgroups 1, 2 (184
// registers) compute: thread = row = TMEM lane, 64 columns each.  Warpgroup 3
// (72 registers) stores a unit's sums while the next unit is under way.
//
// A sink tile is seen by every later query, a chain of steps far longer than
// any other unit's; what lies past its window is cut into units of their own
// whose partial dV, dK a last kernel adds up in slot order (win_plan).
//
// All mbarrier waits are bounded (mbar_poll, about 2 s); on time-out the CTA winds down,
// frees its TMEM and sets STATUS_BWD_TIMEOUT.
#include <algorithm>

#include "common.cuh"
#include "sm100.cuh"
#include "tmap.h"

namespace ma {
namespace {

using namespace sm100;

constexpr int BT = 128;  // rows of every tile
constexpr int NUM_THREADS = 512;
constexpr int LAUNCH_REGS = 128;
constexpr int REGS_PRODUCER = 72;
constexpr int REGS_COMPUTE = 184;
constexpr int REGS_STORE = 72;
constexpr int NCOMP = 256;
static_assert(128 * (REGS_PRODUCER + REGS_STORE) + NCOMP * REGS_COMPUTE == NUM_THREADS * LAUNCH_REGS,
              "register split must equal the launch allocation");
constexpr float LOG2E = 1.4426950408889634f;

template <int HD, bool DQ>
struct Cfg {
  static constexpr int KB = HD / 64;  // 64-column blocks of a row
  static constexpr uint32_t TILE = BT * HD * 2;
  // resident buffers, streamed stages (X1 is held until this step's products,
  // X2 too in the dK/dV pass) and dP buffers: what shared memory and TMEM hold
  static constexpr int RST = HD == 64 ? 2 : 1;
  static constexpr int X1ST = HD == 64 ? 4 : 3;
  static constexpr int X2ST = HD == 64 ? 4 : 2;
  static constexpr int DPB = !DQ && HD == 128 ? 1 : 2;
  // the dK/dV pass's statistics: at D=64 added by the tensor core (see EXT in
  // the kernel), else a ring of fp32 rows
  static constexpr bool EXT = !DQ && HD == 64;
  // warp 2 passes a step on to the issuer of S and dP when all of it is ready
  // (tiles, zeroed rows, statistics): one wait for five.  Not where S must not
  // wait for X2, whose two stages are held until the products.
  static constexpr bool ONE = DPB == 2;
  static constexpr int SSTG = DQ ? 0 : EXT ? 2 : 1;
  static constexpr uint32_t STAT = EXT ? BT * 128 / 2 : 2 * BT * 4;  // EXT: one tile in all
  static constexpr int NDESC = (int)kSchedSlots + 1;
  static constexpr uint32_t DESC = 48;
  static constexpr uint32_t OFF_R = 0;                              // [RST][2]
  static constexpr uint32_t OFF_X1 = OFF_R + RST * 2 * TILE;        // [X1ST]
  static constexpr uint32_t OFF_X2 = OFF_X1 + X1ST * TILE;          // [X2ST]
  static constexpr uint32_t OFF_STAT = OFF_X2 + X2ST * TILE;        // [SSTG]
  static constexpr uint32_t OFF_SCHED = OFF_STAT + SSTG * STAT;     // 16-byte responses
  static constexpr uint32_t OFF_DESC = OFF_SCHED + kSchedSlots * 16;
  static constexpr uint32_t OFF_BAR = OFF_DESC + NDESC * DESC;
  // full and empty of R, X1, X2, stat (EXT: its full is not used, X2 fixed says it
  // too); X1/X2 fixed; dp_full[DPB],
  // p_ready[DPB], p_free[DPB]; s_full, s_free, done, acc_free, fin[2]; sched
  // full/empty, desc_full
  static constexpr int NBAR = 2 * (RST + X1ST + X2ST + SSTG) + X1ST + X2ST + 3 * DPB + 6 + 2 * (int)kSchedSlots + NDESC;
  static constexpr uint32_t OFF_TSLOT = OFF_BAR + NBAR * 8;
  static constexpr uint32_t SMEM = OFF_TSLOT + 16 + 1024;  // + alignment slack
  static_assert(SMEM <= 232448, "shared memory");
  static constexpr uint32_t TCOL_ACC = 0;  // dV, dK or dQ
  static constexpr uint32_t TCOL_S = !DQ && HD == 128 ? 256 : 128;
  static constexpr uint32_t TCOL_DP = TCOL_S + 128;  // [DPB]
  static_assert(TCOL_DP + DPB * 128 <= 512, "TMEM columns");
};

struct Params {
  int T, NH, NKV, G, B;
  int nunits, ntiles;
  int window, sinks;
  const int32_t* lens;
  float scale, scale_log2;
  int rows;                    // rows of a (batch, head) in the statistics
  const float *neg_l, *neg_d;  // -l*log2e, -delta/sqrt(D), [B][NH][rows]
  const uint4* ext;            // D=64: -l*sqrt(D) and -delta as three bf16 each, and two zeros
  uint32_t* status;
  uint32_t expire_ns;          // time-out test hook (ma_debug_expire_next_wait), 0 = off
  // dK/dV pass: sink tiles 0 .. nsplit-1 are split: their query tiles past the
  // window go, far_tiles at a time, to nfar units each, dealt first; unit
  // `slot`s of part hold 2 x 128 x D fp32 partial sums (dV, dK), slot 0 of a
  // tile its window's
  int nsplit, nfar, far_tiles, nfar_units;
  float* part;
  __nv_bfloat16 *dK, *dV;
  void* dQ;
  bool dq_f32;
};

// What one unit does.  (48 bytes: passed on through shared memory.)
struct alignas(16) Unit {
  int b, tile, head;  // the resident tiles: rows tile*128.., head `head`
  int nq;             // steps; 0: no valid row, zeros are stored
  int n;              // valid rows of the sequence
  int first, count;   // dK/dV: query tiles first .. first+count-1, for each head
                      // dQ: list index j < count is sink tile j, else tile first + j - count
  int head0;          // head of the streamed tiles at step 0
  int slot;           // dK/dV: partial sums' slot, or -1
  int valid;          // 0: no unit is left
  int pad[2];
  template <bool DQ>
  __device__ int x_tile(int i) const {
    if constexpr (DQ) return i < count ? i : first + i - count;
    else return first + i % count;
  }
  template <bool DQ>
  __device__ int x_head(int i) const {
    if constexpr (DQ) return head0;
    else return head0 + i / count;
  }
};

__device__ __forceinline__ int length(const Params& p, int b) {
  return p.lens ? min(max(__ldg(p.lens + b), 0), p.T) : p.T;
}

// dK/dV pass: unit k.  The split sink tiles' far units first (they are as long
// as any other), then key tiles in order, (batch, K/V head)s side by side in
// blocks of 16, whose units share their heads' Q and dO in L2.
__device__ __forceinline__ Unit decode_dkv(const Params& p, int k) {
  constexpr int HB = 16;
  Unit u;
  const int nbh = p.B * p.NKV;
  const bool far = k < p.nfar_units;
  int c = 0, bh;
  if (far) {
    bh = k % nbh;
    const int r = k / nbh;
    u.tile = r % p.nsplit;
    c = r / p.nsplit;
  } else {
    k -= p.nfar_units;
    const int per = HB * p.ntiles, blk = k / per, r = k % per;
    const int hb = min(HB, nbh - blk * HB);
    bh = blk * HB + r % hb;
    u.tile = r / hb;
  }
  u.b = bh / p.NKV;
  u.head = bh % p.NKV;
  u.head0 = u.head * p.G;
  u.n = length(p, u.b);
  const bool split = u.tile < p.nsplit;
  u.slot = split ? (bh * p.nsplit + u.tile) * (1 + p.nfar) + (far ? 1 + c : 0) : -1;
  const int k0 = u.tile * BT;
  const int last = (u.n - 1) / BT;                    // the last query tile with a valid row
  const int win_last = (k0 + BT - 1 + p.window - 1) / BT;  // and the last in the window
  u.first = far ? win_last + 1 + c * p.far_tiles : u.tile;
  int end = last;
  if (far) end = min(last, u.first + p.far_tiles - 1);
  else if (split || k0 >= p.sinks) end = min(last, win_last);
  u.count = end - u.first + 1;
  u.nq = u.count * p.G;
  if (u.count <= 0 || u.n <= k0) u.n = u.nq = 0;  // no valid row
  return u;
}

// dQ pass: unit k, in blocks of (batch, head)s as above, the longest windows
// of a block first.
__device__ __forceinline__ Unit decode_dq(const Params& p, int k) {
  constexpr int HB = 16;
  Unit u;
  const int nbh = p.B * p.NH, per = HB * p.ntiles;
  const int blk = k / per, r = k % per, hb = min(HB, nbh - blk * HB);
  const int bh = blk * HB + r % hb;
  u.tile = p.ntiles - 1 - r / hb;
  u.b = bh / p.NH;
  u.head = bh % p.NH;
  u.head0 = u.head / p.G;
  u.n = length(p, u.b);
  u.slot = -1;
  const int q0 = u.tile * BT;
  u.first = max(0, q0 - p.window + 1) / BT;
  u.count = min(p.sinks / BT + (p.sinks % BT != 0), u.first);
  u.nq = u.count + u.tile - u.first + 1;
  if (q0 >= u.n) u.n = u.nq = 0;  // only padding
  return u;
}

struct Step {
  int g;       // units fetched
  Unit u;
  int i;       // step within the unit
  uint32_t t;  // step over all units
  uint32_t uc; // unit with steps
  bool valid;
  uint32_t nreq;  // the producer: launch-control requests issued (request r names unit r + 1)
};

// The units of a CTA as its producer passes them on: unit 0 in descriptor slot
// kSchedSlots, unit g in the slot of the launch-control response that named it,
// which all readers release together.
struct Ring {
  Sched sched;
  Unit* desc;
  uint32_t full;  // slot 0's barrier
};

// PUBLISH (the producer): decodes the unit and passes it on; else reads it.
template <bool DQ, bool WARP, bool PUBLISH>
__device__ __forceinline__ bool next_unit(const Params& p, Step& s, const Ring& ring) {
  const uint32_t g = (uint32_t)s.g++;
  const uint32_t slot = g == 0 ? kSchedSlots : (g - 1) % kSchedSlots;
  if constexpr (PUBLISH) {
    const int k = sched_unit<WARP>(ring.sched, g);
    const bool some = k >= 0 && k < p.nunits;
    if (some) s.u = DQ ? decode_dq(p, k) : decode_dkv(p, k);
    s.u.valid = some;
    ring.desc[slot] = s.u;
    mbar_arrive(ring.full + 8u * slot);
    return some;
  } else {
    const uint32_t ph = g == 0 ? 0u : ((g - 1) / kSchedSlots) & 1u;
    volatile int* abort = ring.sched.abort;
    if (!(WARP ? mbar_poll_warp(ring.full + 8u * slot, ph, abort) : mbar_poll(ring.full + 8u * slot, ph, abort)))
      return false;
    s.u = ring.desc[slot];
    if (g > 0) {
      __threadfence_block();  // read, before the slot is released
      if (WARP) __syncwarp();
      if (!WARP || (threadIdx.x & 31) == 0) mbar_arrive(ring.sched.empty + 8u * slot);
    }
    return s.u.valid != 0;
  }
}

// A role's loop is `for (Step s = before_first(); advance<...>(prm, s, ring);)`:
// one copy of the code that goes on to the next unit.
__device__ __forceinline__ Step before_first() {
  Step s;
  s.g = s.i = 0;
  s.u.nq = 1;
  s.t = s.uc = ~0u;
  s.valid = false;
  s.nreq = 0;
  return s;
}

template <bool DQ, bool WARP, bool PUBLISH = false>
__device__ __forceinline__ bool advance(const Params& p, Step& s, const Ring& ring) {
  ++s.t;
  if (s.i + 1 < s.u.nq) {
    ++s.i;
    return true;
  }
  s.i = 0;
  ++s.uc;
  for (;;) {  // past units that only store zeros
    s.valid = next_unit<DQ, WARP, PUBLISH>(p, s, ring);
    if (!s.valid || s.u.nq > 0) return s.valid;
    if (PUBLISH && !sched_request(ring.sched, s.nreq++)) return false;
  }
}

// 64 fp32 columns of this lane's TMEM row
__device__ __forceinline__ void load_row64(uint32_t taddr, float (&v)[64]) {
  uint32_t ra[32], rb[32];
  tmem_ld32(taddr, ra);
  tmem_ld32(taddr + 32, rb);
  tmem_wait_ld_dep(ra, rb);
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    v[j] = __uint_as_float(ra[j]);
    v[32 + j] = __uint_as_float(rb[j]);
  }
}

// and 64 values into 32 columns as bf16 pairs, the UMMA operand type
__device__ __forceinline__ void store_row64(uint32_t taddr, const float (&v)[64]) {
  uint32_t r[32];
#pragma unroll
  for (int j = 0; j < 32; ++j) r[j] = pack_bf16(v[2 * j], v[2 * j + 1]);
  tmem_st32(taddr, r);
}

template <int HD, bool DQ>
__global__ void __launch_bounds__(NUM_THREADS, 1)
    window_bwd_kernel(const __grid_constant__ CUtensorMap tmR1, const __grid_constant__ CUtensorMap tmR2,
                      const __grid_constant__ CUtensorMap tmX1, const __grid_constant__ CUtensorMap tmX2,
                      const Params prm) {
  using C = Cfg<HD, DQ>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ int abort_flag;
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t sbase = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (sbase - raw);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  const uint32_t bar0 = sbase + C::OFF_BAR;
  auto BAR = [&](int n) { return bar0 + 8u * n; };
  constexpr int B_X1 = 2 * C::RST, B_X2 = B_X1 + 3 * C::X1ST, B_T = B_X2 + 3 * C::X2ST, B_DP = B_T + 2 * C::SSTG,
                B_PR = B_DP + C::DPB, B_PE = B_PR + C::DPB, B_1 = B_PE + C::DPB;
  auto BAR_RF = [&](int s) { return BAR(s); };
  auto BAR_RE = [&](int s) { return BAR(C::RST + s); };
  auto BAR_X1F = [&](int s) { return BAR(B_X1 + s); };
  auto BAR_X1E = [&](int s) { return BAR(B_X1 + C::X1ST + s); };
  auto BAR_X1Z = [&](int s) { return BAR(B_X1 + 2 * C::X1ST + s); };  // padding rows zeroed
  auto BAR_X2F = [&](int s) { return BAR(B_X2 + s); };
  auto BAR_X2E = [&](int s) { return BAR(B_X2 + C::X2ST + s); };
  auto BAR_X2Z = [&](int s) { return BAR(B_X2 + 2 * C::X2ST + s); };
  auto BAR_TF = [&](int s) { return BAR(B_T + s); };
  auto BAR_TE = [&](int s) { return BAR(B_T + C::SSTG + s); };
  auto BAR_DPF = [&](int s) { return BAR(B_DP + s); };
  // P and dS written, and read by the products: one barrier each a dP buffer,
  // since with two buffers the next step's may come before a waiter has looked
  auto BAR_PR = [&](int s) { return BAR(B_PR + s); };
  auto BAR_PE = [&](int s) { return BAR(B_PE + s); };
  const uint32_t BAR_SF = BAR(B_1), BAR_SE = BAR(B_1 + 1);  // S ready, S read
  const uint32_t BAR_DONE = BAR(B_1 + 2);                   // a unit's last product completed
  const uint32_t BAR_ACC = BAR(B_1 + 3);                    // its sums read
  const uint32_t BAR_FIN = BAR(B_1 + 4);                    // wind-down, one for each issuer
  const uint32_t BAR_U = BAR(B_1 + 6);                      // sched full, empty, desc_full
  float* stat_base = reinterpret_cast<float*>(gbase + C::OFF_STAT);
  // readers of a unit: the producer, the issuers, warp 2, the 8 compute and the
  // 4 storing warps
  constexpr uint32_t READERS = 4 + NCOMP / 32 + 4;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < C::NBAR; ++i) {
      uint32_t n = 1;
      if (i >= B_X1 + C::X1ST && i < B_X1 + 2 * C::X1ST) n = 2;  // the products, and warp 2
      if (i >= B_X2 + C::X2ST && i < B_X2 + 2 * C::X2ST) n = 2;
      if (i >= B_T && i < B_T + C::SSTG) n = 32;
      if (i >= B_T + C::SSTG && i < B_DP) n = C::EXT ? 1 : NCOMP;
      if ((i >= B_PR && i < B_PE) || i == B_1 + 1) n = NCOMP;
      if (i == B_1 + 3) n = 128;
      if (i >= B_1 + 6 + (int)kSchedSlots && i < B_1 + 6 + 2 * (int)kSchedSlots) n = READERS;
      mbar_init(BAR(i), n);
    }
    fence_mbar_init();
  }
  // EXT: S - l sqrt(D) and dP - delta come from one more product of 16 columns.  A
  // tile's rows of 128 bytes hold four operands of 16: ones in columns 0-2, ones
  // in 3-5, and two stages of statistics, each value as three bf16 (24 bits).
  // (As fp32 in shared memory they cost the compute warps a broadcast load for
  // every two scores.)
  if constexpr (C::EXT) {
    for (int i = threadIdx.x; i < BT * 8; i += NUM_THREADS) {
      const int r = i / 8, ch = i % 8;
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (ch == 0) v.x = 0x3f803f80u, v.y = 0x3f80u;
      if (ch == 2) v.y = 0x3f800000u, v.z = 0x3f803f80u;
      *reinterpret_cast<uint4*>(gbase + C::OFF_STAT + r * 128 + ((ch ^ (r & 7)) * 16)) = v;
    }
    fence_proxy_async_smem();
  }
  if (warp == 1) {
    tmem_alloc(sbase + C::OFF_TSLOT, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // nothing before here touches global memory, so the barriers and TMEM are set
  // up while the kernel before is still draining.  The dQ pass does not wait
  // for the dK/dV pass before it at all, which shares nothing with it but
  // inputs: it may start once that pass's last blocks have, each of which has
  // waited for the statistics, and fills the SMs that they leave idle.
  if constexpr (DQ) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  else pdl_wait_and_release();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(gbase + C::OFF_TSLOT);
  volatile int* abort_p = &abort_flag;
  const Ring ring{Sched{sbase + C::OFF_SCHED, BAR_U, BAR_U + 8u * kSchedSlots, abort_p},
                  reinterpret_cast<Unit*>(gbase + C::OFF_DESC), BAR_U + 16u * kSchedSlots};
  // whether step s streams padding rows in (past the tensor's end TMA itself
  // fills in zeros)
  auto padded = [&](const Step& s) { return s.u.n < prm.T && s.u.x_tile<DQ>(s.i) * BT + BT > s.u.n; };

  if (warp < 4) {
    reg_dealloc<REGS_PRODUCER>();
    if (warp == 0) {
      // --------------------------------------------------------- producer
      if (lane == 0) {
        tma_prefetch_desc(&tmR1);
        tma_prefetch_desc(&tmR2);
        tma_prefetch_desc(&tmX1);
        tma_prefetch_desc(&tmX2);
        uint32_t r_armed = 0, x1_armed = 0, x2_armed = 0;
        Step s = before_first();
        while (advance<DQ, false, true>(prm, s, ring)) {
          if (s.i == 0) {
            const int rs = s.uc % C::RST, col = s.u.head * HD;
            if (s.uc >= C::RST && !mbar_poll(BAR_RE(rs), ((s.uc / C::RST) - 1) & 1, abort_p)) break;
            mbar_arrive_expect_tx(BAR_RF(rs), 2 * C::TILE);
            ++r_armed;
            for (int kb = 0; kb < C::KB; ++kb) {
              const uint32_t to = sbase + C::OFF_R + rs * 2 * C::TILE + kb * BT * 128;
              tma_load_3d(to, &tmR1, BAR_RF(rs), col + kb * 64, s.u.tile * BT, s.u.b);
              tma_load_3d(to + C::TILE, &tmR2, BAR_RF(rs), col + kb * 64, s.u.tile * BT, s.u.b);
            }
          }
          const int s1 = s.t % C::X1ST, s2 = s.t % C::X2ST;
          const int col = s.u.x_head<DQ>(s.i) * HD, row = s.u.x_tile<DQ>(s.i) * BT;
          if (s.t >= C::X1ST && !mbar_poll(BAR_X1E(s1), ((s.t / C::X1ST) - 1) & 1, abort_p)) break;
          mbar_arrive_expect_tx(BAR_X1F(s1), C::TILE);
          ++x1_armed;
          for (int kb = 0; kb < C::KB; ++kb)
            tma_load_3d(sbase + C::OFF_X1 + s1 * C::TILE + kb * BT * 128, &tmX1, BAR_X1F(s1), col + kb * 64, row, s.u.b);
          if (s.t >= C::X2ST && !mbar_poll(BAR_X2E(s2), ((s.t / C::X2ST) - 1) & 1, abort_p)) break;
          mbar_arrive_expect_tx(BAR_X2F(s2), C::TILE);
          ++x2_armed;
          for (int kb = 0; kb < C::KB; ++kb)
            tma_load_3d(sbase + C::OFF_X2 + s2 * C::TILE + kb * BT * 128, &tmX2, BAR_X2F(s2), col + kb * 64, row, s.u.b);
          // three steps before the unit's end (or at its start), ask for the
          // next unit
          if (s.i == max(0, s.u.nq - 3) && !sched_request(ring.sched, s.nreq++)) break;
        }
        if (*abort_p) {  // wind-down: let the loads and the request still in flight land
          sched_drain(ring.sched, s.nreq);
          drain_ring(BAR_RF, C::RST, r_armed);
          drain_ring(BAR_X1F, C::X1ST, x1_armed);
          drain_ring(BAR_X2F, C::X2ST, x2_armed);
        }
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------- S and dP
      if (lane == 0) {
        constexpr uint32_t IDESC_S = idesc_bf16_f32(BT, BT, 0, 0);
        uint32_t z1 = 0, z2 = 0;  // bit s: parity of the next phase of X1Z(s), X2Z(s)
        // 128 x 128 scores: both operands K-major
        auto scores = [&](uint32_t d, uint32_t a, uint32_t b) {
          const uint32_t da = desc_lo(a, 16), db = desc_lo(b, 16);
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            const uint32_t off = ((kk >> 2) * (BT * 128) + (kk & 3) * 32) >> 4;
            umma_bf16_ss_lo(d, da + off, db + off, IDESC_S, kk > 0 ? 1u : 0u);
          }
        };
        for (Step s = before_first(); advance<DQ, false>(prm, s, ring);) {
          const uint32_t t = s.t, rs = s.uc % C::RST, s1 = t % C::X1ST, s2 = t % C::X2ST, b = t % C::DPB;
          const bool pad = padded(s);
          if (s.i == 0 && !mbar_poll(BAR_RF(rs), (s.uc / C::RST) & 1, abort_p)) break;
          const uint32_t st = C::EXT ? t % C::SSTG : 0;
          if constexpr (C::ONE) {
            if (!mbar_poll(BAR_X2Z(s2), (t / C::X2ST) & 1, abort_p)) break;
          } else {
            if (!mbar_poll(BAR_X1F(s1), (t / C::X1ST) & 1, abort_p)) break;
            if (pad) {
              if (!mbar_poll(BAR_X1Z(s1), (z1 >> s1) & 1, abort_p)) break;
              z1 ^= 1u << s1;
            }
          }
          if (t >= 1 && !mbar_poll(BAR_SE, (t - 1) & 1, abort_p)) break;
          tc_fence_after();
          const uint32_t de = desc_lo(sbase + C::OFF_STAT, 16);  // 32 bytes an operand
          scores(tmem + C::TCOL_S, sbase + C::OFF_R + rs * 2 * C::TILE, sbase + C::OFF_X1 + s1 * C::TILE);
          if (C::EXT) umma_bf16_ss_lo(tmem + C::TCOL_S, de, de + 4 + 2 * st, IDESC_S, 1u);
          umma_commit(BAR_SF);
          if constexpr (!C::ONE) {
            if (!mbar_poll(BAR_X2F(s2), (t / C::X2ST) & 1, abort_p)) break;
            if (pad) {
              if (!mbar_poll(BAR_X2Z(s2), (z2 >> s2) & 1, abort_p)) break;
              z2 ^= 1u << s2;
            }
          }
          // the products that read P and dS out of its columns have completed
          if (t >= C::DPB && !mbar_poll(BAR_PE(b), ((t / C::DPB) - 1) & 1, abort_p)) break;
          tc_fence_after();
          scores(tmem + C::TCOL_DP + b * 128, sbase + C::OFF_R + (rs * 2 + 1) * C::TILE,
                 sbase + C::OFF_X2 + s2 * C::TILE);
          if (C::EXT) umma_bf16_ss_lo(tmem + C::TCOL_DP + b * 128, de + 2, de + 4 + 2 * st, IDESC_S, 1u);
          umma_commit(BAR_DPF(b));
          if (C::EXT) umma_commit(BAR_TE(st));
          if (DQ) umma_commit(BAR_X2E(s2));
          if (s.i + 1 == s.u.nq) umma_commit(BAR_RE(rs));  // the resident tiles' last use
        }
        if (*abort_p) {  // wind-down: every UMMA issued must complete before TMEM is freed
          umma_commit(BAR_FIN);
          mbar_wait_for(BAR_FIN, 0, kDrainLimitNs);
        }
      }
    } else if (warp == 3) {
      // ----------------------------------------------------------- products
      if (lane == 0) {
        constexpr uint32_t IDESC_ACC = idesc_bf16_f32(BT, HD, 0, 1);
        // A = P or dS in TMEM (each half of the columns over its half of dP),
        // B = a streamed tile, MN-major
        auto product = [&](uint32_t d, uint32_t a, uint32_t b, bool start) {
          const uint32_t db = desc_lo(b, BT * 128);
#pragma unroll
          for (int kk = 0; kk < BT / 16; ++kk)
            umma_bf16_ts_lo(d, a + (kk >> 2) * 64 + (kk & 3) * 8, db + kk * (2048 >> 4), IDESC_ACC,
                            start && kk == 0 ? 0u : 1u);
        };
        // time-out test hook: while the first scores are formed, wait until its limit
        // runs out on the barrier that nothing arrives at before the wind-down
        if (prm.expire_ns) mbar_wait(BAR_FIN + 8, 0, abort_p, prm.expire_ns);
        for (Step s = before_first(); advance<DQ, false>(prm, s, ring);) {
          const uint32_t t = s.t, s1 = t % C::X1ST, s2 = t % C::X2ST, b = t % C::DPB;
          const uint32_t p = tmem + C::TCOL_DP + b * 128, ds = p + 32;
          if (!mbar_poll(BAR_PR(b), (t / C::DPB) & 1, abort_p)) break;
          // the unit before has been read out of the sums' columns
          if (s.i == 0 && s.uc >= 1 && !mbar_poll(BAR_ACC, (s.uc - 1) & 1, abort_p)) break;
          tc_fence_after();
          if constexpr (!DQ) {
            product(tmem + C::TCOL_ACC, p, sbase + C::OFF_X2 + s2 * C::TILE, s.i == 0);  // dV += P dO
            umma_commit(BAR_X2E(s2));
          }
          // dK += dS Q, dQ += dS K
          product(tmem + C::TCOL_ACC + (DQ ? 0 : HD), ds, sbase + C::OFF_X1 + s1 * C::TILE, s.i == 0);
          umma_commit(BAR_PE(b));
          umma_commit(BAR_X1E(s1));
          if (s.i + 1 == s.u.nq) umma_commit(BAR_DONE);
        }
        if (*abort_p) {
          umma_commit(BAR_FIN + 8);
          mbar_wait_for(BAR_FIN + 8, 0, kDrainLimitNs);
        }
      }
    } else if (warp == 2) {
      // ------------------------------- statistics, padding rows of X1 and X2
      // rows [a, 128) of a tile are contiguous in each 64-column block (the
      // swizzle permutes the chunks of a row within its 128 bytes)
      auto zero_rows = [&](uint32_t off, int a) {
        for (int kb = 0; kb < C::KB; ++kb) {
          uint4* blk = reinterpret_cast<uint4*>(gbase + off + kb * BT * 128);
          for (int i = a * 8 + lane; i < BT * 8; i += 32) blk[i] = make_uint4(0u, 0u, 0u, 0u);
        }
        fence_proxy_async_smem();
        __syncwarp();
      };
      // every stage is waited for and released, so that this warp stays within
      // one phase of each slot's barriers
      for (Step s = before_first(); advance<DQ, true>(prm, s, ring);) {
        const int s1 = s.t % C::X1ST, s2 = s.t % C::X2ST;
        const bool pad = padded(s);
        const int a = max(0, s.u.n - s.u.x_tile<DQ>(s.i) * BT);
        float4 L, D4;
        uint4 x4[4];
        if constexpr (!DQ) {  // in flight while the tiles land
          const long long at = ((long long)s.u.b * prm.NH + s.u.x_head<DQ>(s.i)) * prm.rows + s.u.x_tile<DQ>(s.i) * BT;
          // (not __ldg: this grid was on the GPU before they were written)
          if constexpr (C::EXT) {
#pragma unroll
            for (int j = 0; j < 4; ++j) x4[j] = __ldcg(prm.ext + at + lane + 32 * j);
          } else {
            L = __ldcg(reinterpret_cast<const float4*>(prm.neg_l + at) + lane);
            D4 = __ldcg(reinterpret_cast<const float4*>(prm.neg_d + at) + lane);
          }
        }
        if (!mbar_poll_warp(BAR_X1F(s1), (s.t / C::X1ST) & 1, abort_p)) break;
        if (pad) zero_rows(C::OFF_X1 + s1 * C::TILE, a);
        if (lane == 0) {
          if (pad && !C::ONE) mbar_arrive(BAR_X1Z(s1));
          mbar_arrive(BAR_X1E(s1));
        }
        if constexpr (!DQ) {
          const int st = s.t % C::SSTG;
          if (s.t >= C::SSTG && !mbar_poll_warp(BAR_TE(st), ((s.t / C::SSTG) - 1) & 1, abort_p)) break;
          if constexpr (C::EXT) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {  // lane + 32 j: its 16 bytes of the stage
              const int r = lane + 32 * j;
              *reinterpret_cast<uint4*>(gbase + C::OFF_STAT + r * 128 + (((4 + 2 * st) ^ (r & 7)) * 16)) = x4[j];
            }
          } else {
            float* stt = stat_base + st * (2 * BT);
            reinterpret_cast<float4*>(stt)[lane] = L;
            reinterpret_cast<float4*>(stt + BT)[lane] = D4;
          }
          if constexpr (!C::EXT) mbar_arrive(BAR_TF(st));
        }
        if (!mbar_poll_warp(BAR_X2F(s2), (s.t / C::X2ST) & 1, abort_p)) break;
        if (pad) zero_rows(C::OFF_X2 + s2 * C::TILE, a);
        if constexpr (C::ONE) {
          fence_proxy_async_smem();
          __syncwarp();
        }
        if (lane == 0) {
          if (pad || C::ONE) mbar_arrive(BAR_X2Z(s2));
          mbar_arrive(BAR_X2E(s2));
        }
      }
    }
  } else if (warp < 12) {
    reg_alloc<REGS_COMPUTE>();
    // ------------------------------------------------------------ compute
    const int quarter = warp & 3, part = (warp - 4) >> 2;  // columns part*64 .. +63
    const int row = quarter * 32 + lane;
    const uint32_t tl = tmem + ((uint32_t)(quarter * 32) << 16);
    const float2 c2 = make_float2(prm.scale_log2, prm.scale_log2), sc2 = make_float2(prm.scale, prm.scale);
    bool ok = true;
    float nl = 0.0f, nd = 0.0f;  // dQ: the row's statistics

    // P and dS of step s, handed to the UMMA issuer
    auto form = [&](const Step& s) {
      const uint32_t t = s.t;
      const int r = s.u.tile * BT + row;                        // the thread's row
      const int x0 = s.u.x_tile<DQ>(s.i) * BT + part * 64;      // its first column
      if constexpr (DQ) {
        if (s.i == 0) {
          const long long at = ((long long)s.u.b * prm.NH + s.u.head) * prm.rows + r;
          nl = __ldcg(prm.neg_l + at);
          nd = __ldcg(prm.neg_d + at);
        }
      }
      uint32_t see[2];
      if constexpr (DQ) {  // query r: its window's keys and the sinks
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const int k0 = x0 + 32 * w;
          see[w] = r < s.u.n ? bits_below(r + 1 - k0) & (~bits_below(r - prm.window + 1 - k0) | bits_below(prm.sinks - k0))
                             : 0u;
        }
      } else {  // key r: the queries from itself to its window's end, a sink's to the sequence's
        const int to = (r < prm.sinks ? s.u.n : min(s.u.n, r + prm.window)) - x0, from = r - x0;
#pragma unroll
        for (int w = 0; w < 2; ++w) see[w] = bits_below(to - 32 * w) & ~bits_below(from - 32 * w);
      }
      ok = mbar_poll_warp(BAR_SF, t & 1, abort_p);
      if (!ok) return;
      tc_fence_after();
      float p[64];
      load_row64(tl + C::TCOL_S + part * 64, p);
      tc_fence_before();
      mbar_arrive(BAR_SE);
      const float* stt = stat_base;
      if constexpr (!DQ && !C::EXT) {
        const int st = t % C::SSTG;
        ok = mbar_poll_warp(BAR_TF(st), (t / C::SSTG) & 1, abort_p);
        if (!ok) return;
        stt += st * (2 * BT) + part * 64;
      }
#pragma unroll
      for (int j = 0; j < 64; j += 4) {
        float4 L = make_float4(nl, nl, nl, nl);
        if constexpr (!DQ && !C::EXT) L = *reinterpret_cast<const float4*>(stt + j);
        const float2 t0 = __ffma2_rn(make_float2(p[j], p[j + 1]), c2, make_float2(L.x, L.y));
        const float2 t1 = __ffma2_rn(make_float2(p[j + 2], p[j + 3]), c2, make_float2(L.z, L.w));
        const uint32_t m = see[j / 32] >> (j % 32);
        p[j] = m & 1u ? ex2(t0.x) : 0.0f;
        p[j + 1] = m & 2u ? ex2(t0.y) : 0.0f;
        p[j + 2] = m & 4u ? ex2(t1.x) : 0.0f;
        p[j + 3] = m & 8u ? ex2(t1.y) : 0.0f;
      }
      ok = mbar_poll_warp(BAR_DPF(t % C::DPB), (t / C::DPB) & 1, abort_p);
      if (!ok) return;
      tc_fence_after();
      const uint32_t tdp = tl + C::TCOL_DP + t % C::DPB * 128 + part * 64;
      float d[64];
      load_row64(tdp, d);
      if constexpr (!DQ) store_row64(tdp, p);  // over this thread's own dP, now in registers
#pragma unroll
      for (int j = 0; j < 64; j += 4) {
        float4 Dn = make_float4(nd, nd, nd, nd);
        if constexpr (!DQ && !C::EXT) Dn = *reinterpret_cast<const float4*>(stt + BT + j);
        float2 d0 = make_float2(d[j], d[j + 1]), d1 = make_float2(d[j + 2], d[j + 3]);
        if constexpr (!C::EXT) {  // EXT: dK is multiplied by 1/sqrt(D) as it is stored
          d0 = __ffma2_rn(d0, sc2, make_float2(Dn.x, Dn.y));
          d1 = __ffma2_rn(d1, sc2, make_float2(Dn.z, Dn.w));
        }
        const float2 r0 = __fmul2_rn(make_float2(p[j], p[j + 1]), d0);
        const float2 r1 = __fmul2_rn(make_float2(p[j + 2], p[j + 3]), d1);
        d[j] = r0.x;
        d[j + 1] = r0.y;
        d[j + 2] = r1.x;
        d[j + 3] = r1.y;
      }
      store_row64(tdp + 32, d);
      tmem_wait_st();
      if constexpr (!DQ && !C::EXT) mbar_arrive(BAR_TE(t % C::SSTG));  // all read: dS is stored
      tc_fence_before();
      mbar_arrive(BAR_PR(t % C::DPB));
    };

    for (Step s = before_first(); ok && advance<DQ, true>(prm, s, ring);) form(s);
  } else {
    reg_dealloc<REGS_STORE>();
    // ------------------------------------------------------- a unit's sums
    // thread = row = TMEM lane; 32 columns at a time, TMEM -> registers ->
    // global memory
    const int row = (warp & 3) * 32 + lane;
    const uint32_t tl = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    Step s = before_first();
    while (next_unit<DQ, true, false>(prm, s, ring)) {
      const bool some = s.u.nq > 0;
      if (some) {
        if (!mbar_poll_warp(BAR_DONE, ++s.uc & 1, abort_p)) break;
        tc_fence_after();
      }
      const Unit& v = s.u;
      const int at = v.tile * BT + row;
      const bool valid = at < v.n;  // a padding row's sums are 0, whatever its own tile held
      constexpr int COLS = (DQ ? 1 : 2) * HD;
#pragma unroll 1
      for (int cc = 0; cc < COLS; cc += 32) {
        uint32_t r[32] = {};
        if (some) {
          tmem_ld32(tl + C::TCOL_ACC + cc, r);
          tmem_wait_ld_dep(r);
          if (cc + 32 == COLS) {  // all read: the next unit may overwrite them
            tc_fence_before();
            mbar_arrive(BAR_ACC);
          }
#pragma unroll
          for (int j = 0; j < 32; ++j) r[j] = valid ? r[j] : 0u;
        }
        const int which = cc / HD, col = cc % HD;
        if (C::EXT && which == 1) {
#pragma unroll
          for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * prm.scale);
        }
        float* f32 = nullptr;
        __nv_bfloat16* b16 = nullptr;
        if constexpr (DQ) {
          const long long off = (((long long)v.b * prm.T + at) * prm.NH + v.head) * HD + col;
          if (prm.dq_f32) f32 = static_cast<float*>(prm.dQ) + off;
          else b16 = static_cast<__nv_bfloat16*>(prm.dQ) + off;
        } else if (v.slot >= 0) {
          f32 = prm.part + (((long long)v.slot * 2 + which) * BT + row) * HD + col;
        } else {
          b16 = (which == 0 ? prm.dV : prm.dK) + (((long long)v.b * prm.T + at) * prm.NKV + v.head) * HD + col;
        }
        if (at >= prm.T && (DQ || v.slot < 0)) continue;
        if (f32) {
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            *reinterpret_cast<uint4*>(f32 + j) = make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]);
        } else {
          auto pair = [&](int j) { return pack_bf16(__uint_as_float(r[j]), __uint_as_float(r[j + 1])); };
#pragma unroll
          for (int j = 0; j < 32; j += 8)
            *reinterpret_cast<uint4*>(b16 + j) = make_uint4(pair(j), pair(j + 2), pair(j + 4), pair(j + 6));
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  // what follows the dQ pass waits for it, and so must not find the dK/dV pass
  // still running
  if constexpr (DQ) asm volatile("griddepcontrol.wait;" ::: "memory");
  if (threadIdx.x == 0 && abort_flag) atomicOr(prm.status, STATUS_BWD_TIMEOUT);
}

// How a call's workspace is laid out, and how its sink tiles are split.
struct Plan {
  int ntiles, rows, nsplit, nfar, far_tiles;
  size_t stat, ext, part;  // bytes: one statistic, both as bf16, the partial sums
  size_t total() const { return 2 * stat + ext + part; }
};

Plan win_plan(const WindowArgs& a) {
  Plan p{};
  p.ntiles = (a.M + BT - 1) / BT;
  p.rows = p.ntiles * BT;
  const int nbh = a.B * a.NKV;
  const int ns = (int)std::min<long long>(((long long)a.sinks + BT - 1) / BT, p.ntiles);
  const int window = std::min(a.window, 1 << 25);
  const int near = (BT - 1 + window - 1) / BT + 1;  // query tiles of tile 0's window
  const int far = p.ntiles - near;
  // A sink tile's far queries are a chain of `far` steps a head where other
  // units have `near`.  Where the sink tiles alone would not keep the GPU busy
  // twice over, the chain is cut into pieces of a window's length, of 8 tiles
  // at least (a piece costs 2 x 128 x D fp32 written and read) and 16 at most.
  if (ns > 0 && far > near && far > 8 && (long long)ns * nbh < 2 * 148) {
    p.nsplit = ns;
    p.far_tiles = std::max({near, 8, (far + 15) / 16});
    p.nfar = (far + p.far_tiles - 1) / p.far_tiles;
  }
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  p.stat = up((size_t)a.B * a.NH * p.rows * sizeof(float));
  p.ext = a.D == 64 ? 4 * p.stat : 0;
  p.part = up((size_t)nbh * p.nsplit * (1 + p.nfar) * 2 * BT * a.D * sizeof(float));
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
// and past the end).  HBM-bound: dO and O read once.  A warp takes 8 * 32 / (D/8)
// rows of a head, D/8 lanes a row with 16-byte loads, all of them in flight, and
// writes neighbouring statistics.
template <int HD>
__global__ void __launch_bounds__(256, 2) window_stats_kernel(const WindowArgs a, const __nv_bfloat16* __restrict__ dO,
                                                              float* __restrict__ neg_l, float* __restrict__ neg_d,
                                                              uint4* __restrict__ ext, int rows) {
  pdl_wait_and_release();
  constexpr int G = HD / 8, RPI = 32 / G, N = 8, ROWS = N * RPI;  // lanes a row, rows an instruction, loads in flight
  const int lane = threadIdx.x % 32;
  const int tiles = rows / ROWS;
  const long long items = (long long)a.B * tiles * a.NH;
  for (long long it = blockIdx.x * 8ll + threadIdx.x / 32; it < items; it += gridDim.x * 8ll) {
    const int h = (int)(it % a.NH);
    const long long r = it / a.NH;
    const int b = (int)(r / tiles), row0 = (int)(r % tiles) * ROWS;
    const int n = a.len(b);
    uint4 x[N], y[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int row = row0 + k * RPI + lane / G;
      const long long off = (((long long)b * a.M + row) * a.NH + h) * HD;
      x[k] = y[k] = make_uint4(0u, 0u, 0u, 0u);
      if (row < n) {
        x[k] = __ldcs(reinterpret_cast<const uint4*>(dO + off) + lane % G);
        y[k] = __ldcs(reinterpret_cast<const uint4*>(a.out + off) + lane % G);
      }
    }
    float mine = 0.0f;  // of row row0 + lane
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int i = k * RPI;
      float s = dot8(x[k], y[k]);
#pragma unroll
      for (int m = G / 2; m >= 1; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
      const float got = __shfl_sync(0xffffffffu, s, (lane - i) * G & 31);
      if (lane >= i && lane < i + RPI) mine = got;
    }
    if (lane < ROWS) {
      const int row = row0 + lane;
      const bool valid = row < n;
      const long long at = ((long long)b * a.NH + h) * rows + row;
      const float l = valid ? -a.l[((long long)b * a.M + row) * a.NH + h] : 0.0f, d = valid ? -mine : 0.0f;
      neg_l[at] = l * LOG2E;
      neg_d[at] = d * a.scale;
      if constexpr (HD == 64) {  // 24 bits each, as three operands of the tensor core
        uint32_t x[6];
        auto three = [&](float v, uint32_t* to) {
#pragma unroll
          for (int i = 0; i < 3; ++i) {
            to[i] = sm100::pack_bf16(v, 0.0f) & 0xffffu;
            v -= __uint_as_float(to[i] << 16);
          }
        };
        three(l * 8.0f, x);  // sqrt(D) = 8
        three(d, x + 3);
        ext[at] = make_uint4(x[0] | x[1] << 16, x[2] | x[3] << 16, x[4] | x[5] << 16, 0u);
      }
    }
  }
}

// The split sink tiles' partial dV, dK added up in slot order and rounded.
__global__ void __launch_bounds__(256) window_join_sinks_kernel(const float* __restrict__ part, int slots, int nsplit,
                                                                int D, int NKV, int T, long long n4,
                                                                __nv_bfloat16* __restrict__ dK,
                                                                __nv_bfloat16* __restrict__ dV) {
  pdl_wait_and_release();
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n4; i += gridDim.x * 256ll) {
    const int d4 = D / 4;
    const int c = (int)(i % d4);
    long long r = i / d4;
    const int row = (int)(r % BT);
    r /= BT;
    const int which = (int)(r % 2);
    r /= 2;  // (batch, K/V head, sink tile)
    const int tile = (int)(r % nsplit);
    const long long bh = r / nsplit;
    const int key = tile * BT + row;
    if (key >= T) continue;
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int k = 0; k < slots; ++k) {
      const float4 x = __ldcg(reinterpret_cast<const float4*>(part) + (((r * slots + k) * 2 + which) * BT + row) * d4 + c);
      s.x += x.x, s.y += x.y, s.z += x.z, s.w += x.w;
    }
    __nv_bfloat16* to = (which == 0 ? dV : dK) + ((bh / NKV * T + key) * NKV + bh % NKV) * D + c * 4;
    *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16(s.x, s.y), pack_bf16(s.z, s.w));
  }
}

template <int HD, bool DQ>
cudaError_t launch_pass(const CUtensorMap& r1, const CUtensorMap& r2, const CUtensorMap& x1, const CUtensorMap& x2,
                        const Params& prm, cudaStream_t st) {
  using C = Cfg<HD, DQ>;
  // The setmaxnreg split assumes the kernel was compiled to exactly
  // LAUNCH_REGS registers per thread; refuse to launch otherwise.
  static const cudaError_t reg_check = [] {
    cudaFuncAttributes a;
    cudaError_t e = cudaFuncGetAttributes(&a, window_bwd_kernel<HD, DQ>);
    if (e != cudaSuccess) return e;
    return a.numRegs == LAUNCH_REGS ? cudaSuccess : cudaErrorInvalidKernelImage;
  }();
  if (reg_check != cudaSuccess) return reg_check;
  cudaError_t e = cudaFuncSetAttribute(window_bwd_kernel<HD, DQ>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  if (e != cudaSuccess) return e;
  launch_pdl(window_bwd_kernel<HD, DQ>, prm.nunits, NUM_THREADS, C::SMEM, st, r1, r2, x1, x2, prm);
  count_launches(1);
  return cudaGetLastError();
}

template <int HD>
cudaError_t launch_all(const WindowArgs& a, const WindowGrads& g, cudaStream_t st) {
  const Plan p = win_plan(a);
  char* ws = static_cast<char*>(g.workspace);
  float* neg_l = reinterpret_cast<float*>(ws);
  float* neg_d = reinterpret_cast<float*>(ws + p.stat);
  uint4* ext = reinterpret_cast<uint4*>(ws + 2 * p.stat);
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  auto blocks = [&](long long n, int per) { return (unsigned)std::min<long long>((n + per - 1) / per, sms * 16ll); };
  launch_pdl(window_stats_kernel<HD>, blocks((long long)a.B * a.NH * p.rows / (2048 / HD), 8), 256, 0, st, a, g.dO, neg_l,
             neg_d, ext, p.rows);
  count_launches(1);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  CUtensorMap tq, tk, tv, tdo;
  const CUtensorMapDataType bf = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUtensorMapSwizzle sw = CU_TENSOR_MAP_SWIZZLE_128B;
  const uint64_t nq = (uint64_t)a.NH * HD, nkv = (uint64_t)a.NKV * HD;
  if (!make_tmap_3d(&tq, a.q, bf, 2, nq, a.M, a.B, 64, BT, sw) ||
      !make_tmap_3d(&tk, a.k, bf, 2, nkv, a.M, a.B, 64, BT, sw) ||
      !make_tmap_3d(&tv, a.v, bf, 2, nkv, a.M, a.B, 64, BT, sw) ||
      !make_tmap_3d(&tdo, g.dO, bf, 2, nq, a.M, a.B, 64, BT, sw))
    return cudaErrorInvalidValue;
  Params prm{};
  prm.T = a.M;
  prm.NH = a.NH;
  prm.NKV = a.NKV;
  prm.G = a.NH / a.NKV;
  prm.B = a.B;
  prm.ntiles = p.ntiles;
  prm.window = std::min(a.window, 1 << 25);  // M <= 2^24: the same mask, and sums of positions stay in range
  prm.sinks = a.sinks;
  prm.lens = a.lens;
  prm.scale = a.scale;
  prm.scale_log2 = a.scale * LOG2E;
  prm.rows = p.rows;
  prm.neg_l = neg_l;
  prm.neg_d = neg_d;
  prm.status = a.status;
  prm.expire_ns = take_expire_request(STATUS_BWD_TIMEOUT);  // of both passes
  prm.nsplit = p.nsplit;
  prm.nfar = p.nfar;
  prm.far_tiles = p.far_tiles;
  prm.nfar_units = p.nsplit * p.nfar * a.B * a.NKV;
  prm.ext = ext;
  prm.part = reinterpret_cast<float*>(ws + 2 * p.stat + p.ext);
  prm.dK = g.dK;
  prm.dV = g.dV;
  prm.dQ = g.dQ;
  prm.dq_f32 = g.dq_f32;
  prm.nunits = prm.nfar_units + p.ntiles * a.B * a.NKV;
  // The order of the two is fixed, with nothing between them: the dQ pass reads the
  // statistics without a wait of its own, and may because every block of the dK/dV
  // pass has waited for them before it lets the dQ pass start.
  e = launch_pass<HD, false>(tk, tv, tq, tdo, prm, st);
  if (e != cudaSuccess) return e;
  prm.nunits = p.ntiles * a.B * a.NH;
  e = launch_pass<HD, true>(tq, tdo, tk, tv, prm, st);
  if (e != cudaSuccess || p.nsplit == 0) return e;
  const long long n4 = (long long)a.B * a.NKV * p.nsplit * 2 * BT * HD / 4;
  launch_pdl(window_join_sinks_kernel, blocks(n4, 256), 256, 0, st, prm.part, 1 + p.nfar, p.nsplit, HD, a.NKV, a.M, n4,
             g.dK, g.dV);
  count_launches(1);
  return cudaGetLastError();
}

}  // namespace

size_t window_bwd_workspace(const WindowArgs& a) { return win_plan(a).total(); }

cudaError_t launch_window_bwd(const WindowArgs& a, const WindowGrads& g, cudaStream_t st) {
  return a.D == 64 ? launch_all<64>(a, g, st) : launch_all<128>(a, g, st);
}

}  // namespace ma
