// window_attn.cu -- windowAttentionCached: the windowed attention of new tokens
// over a K/V cache.
//
// For each sequence and K/V head the R = M * G query rows (M new tokens, G
// query heads a K/V head; row r is token r / G, head r % G) share one pass over
// the visible cache rows: the sinks before the window and the union of the
// rows' windows, in blocks of 64 keys,
//   S = Q K^T / sqrt(D),  P = exp(S - m),  O += P V,  l += sum P
// with a running maximum m, so each visible K/V row is read once a 16-row
// group.
//
// HBM-bound: G * M multiply-adds an element read, far below the tensor cores'
// rate even on mma.sync, whose 16-row tile fits the few rows (a tcgen05 tile
// has 64 at least, and its operands are shared-memory tiles either way).  What
// counts is bytes in flight: a producer thread keeps a ring of K/V blocks
// filled by TMA (96 KB a CTA, two CTAs a SM) and four warps consume it, each
// 16 keys of every block with its own m, l and O in registers, joined at the
// end.  Few rows on a long axis leave most SMs idle, so the blocks are split
// over CTAs until the GPU is full, and a second kernel joins the splits'
// (m, l, O) in a fixed order.  Measured: 64 requests, 32 / 8 heads of 128, window
// 4096: 166 us, 6.5 TB/s; one request over 131072 keys: 93 us, 83 of them the
// splits at 6.5 TB/s.
//
// Cache rows that no query sees may hold anything: their scores are replaced
// by -inf and their V rows zeroed in shared memory, since 0 * NaN is NaN.
#include <algorithm>

#include "common.cuh"
#include "sm100.cuh"
#include "tmap.h"

namespace ma {
namespace {

using namespace sm100;

constexpr int KEYS = 64;       // keys of a block
constexpr int ROWS = 16;       // query rows of a CTA
constexpr int WARPS = 4;       // consumers: KEYS / WARPS = 16 keys each
constexpr int THREADS = 32 * WARPS + 32;
constexpr int CTAS_PER_SM = 2;
constexpr int SMS = 148;
constexpr int MIN_BLOCKS = 4;  // a split has this many blocks at least
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr float RESCALE_THRESHOLD = 8.0f;  // log2 units

template <int HD>
struct DecodeCfg {
  static constexpr int KB = HD / 64;
  static constexpr uint32_t TILE = KEYS * HD * 2;          // K or V of a block
  static constexpr int STAGES = 96 * 1024 / (2 * (int)TILE);
  static constexpr uint32_t OFF_BAR = STAGES * 2 * TILE;
  // full and empty of each stage, and one that nothing arrives at (the time-out hook's)
  static constexpr uint32_t SMEM = OFF_BAR + (2 * STAGES + 1) * 8 + 1024;  // + alignment slack
  static_assert(WARPS * ROWS * HD * 4 + WARPS * ROWS * 8 <= OFF_BAR, "the join reuses the ring");
};

struct DecodeParams {
  WindowArgs a;
  int groups, nsplit;  // 16-row groups a K/V head, splits of the key axis
  float scale_log2;
  uint32_t expire_ns;  // time-out test hook (ma_debug_expire_next_wait), 0 = off
  float *part_o, *part_ml;  // nsplit > 1: [unit][split][16][D], [unit][split][16][2]
};

// What a 16-row group visits: sink blocks [0, ns), then window blocks from lo.
struct Span {
  int rows, n0;           // rows of the group, its first row
  int t0, t1;             // positions of its first and last valid row
  int sink_end, lo;       // sinks before the window, the window's first key
  int sink_blocks, blocks;
  __device__ int first_key(int blk) const { return blk < sink_blocks ? blk * KEYS : lo + (blk - sink_blocks) * KEYS; }
};

__device__ __forceinline__ Span span_of(const WindowArgs& a, int b, int grp) {
  Span s;
  const int G = a.NH / a.NKV;
  s.n0 = grp * ROWS;
  s.rows = min(ROWS, a.M * G - s.n0);
  const int i0 = s.n0 / G, i1 = min((s.n0 + s.rows - 1) / G, a.len(b) - 1);
  s.blocks = s.sink_blocks = s.sink_end = s.lo = s.t0 = s.t1 = 0;
  if (i1 < i0) return s;  // only padding
  s.t0 = a.pos(b, i0);
  s.t1 = a.pos(b, i1);
  s.lo = max(0, s.t0 - a.window + 1);
  s.sink_end = min(a.sinks, s.lo);
  s.sink_blocks = (s.sink_end + KEYS - 1) / KEYS;
  s.blocks = s.sink_blocks + (s.t1 - s.lo) / KEYS + 1;
  return s;
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int HD>
__global__ void __launch_bounds__(THREADS, CTAS_PER_SM)
    window_decode_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                         const DecodeParams prm) {
  pdl_wait_and_release();
  using C = DecodeCfg<HD>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ int abort_flag;
  const WindowArgs& a = prm.a;
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t sbase = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (sbase - raw);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  auto BAR_F = [&](int s) { return sbase + C::OFF_BAR + 8u * s; };
  auto BAR_E = [&](int s) { return sbase + C::OFF_BAR + 8u * (C::STAGES + s); };
  const uint32_t BAR_NEVER = sbase + C::OFF_BAR + 16u * C::STAGES;

  const int split = blockIdx.x % prm.nsplit;
  const int unit = blockIdx.x / prm.nsplit;  // (batch, K/V head, row group)
  const int grp = unit % prm.groups;
  const int kh = unit / prm.groups % a.NKV, b = unit / prm.groups / a.NKV;
  const Span sp = span_of(a, b, grp);
  const int blk0 = (int)((long long)sp.blocks * split / prm.nsplit);
  const int blk1 = (int)((long long)sp.blocks * (split + 1) / prm.nsplit);

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(BAR_F(s), 1);
      mbar_init(BAR_E(s), WARPS);
    }
    mbar_init(BAR_NEVER, 1);
    fence_mbar_init();
  }
  __syncthreads();
  volatile int* abort_p = &abort_flag;

  const int G = a.NH / a.NKV;
  const int g = lane / 4, c = lane % 4;  // a thread's rows g and g + 8, its column pair
  float o[HD / 8][4];
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
  if (warp == WARPS) {
    // ------------------------------------------------------- TMA producer
    if (lane == 0) {
      uint32_t n = 0;
      for (int blk = blk0; blk < blk1; ++blk, ++n) {
        const int st = n % C::STAGES;
        // time-out test hook: with the first block's loads in flight, wait until its
        // limit runs out
        if (n == 1 && prm.expire_ns && !mbar_wait(BAR_NEVER, 0, abort_p, prm.expire_ns)) break;
        if (n >= C::STAGES && !mbar_wait(BAR_E(st), ((n / C::STAGES) - 1) & 1, abort_p)) break;
        mbar_arrive_expect_tx(BAR_F(st), 2 * C::TILE);
        const int k0 = sp.first_key(blk);
        const uint32_t dst = sbase + st * 2 * C::TILE;
        for (int kb = 0; kb < C::KB; ++kb) {
          tma_load_3d(dst + kb * KEYS * 128, &tmK, BAR_F(st), kh * HD + kb * 64, k0, b);
          tma_load_3d(dst + C::TILE + kb * KEYS * 128, &tmV, BAR_F(st), kh * HD + kb * 64, k0, b);
        }
      }
      drain_ring(BAR_F, C::STAGES, n);  // every load has landed before the ring is reused, after a time-out too
    }
  } else {
    // ---------------------------------------------------------- consumers
    // Q as MMA fragments: rows g and g + 8 of the group (padding: zeros).  Not
    // __ldg: this grid may be on the GPU before the one that writes q has ended.
    uint32_t q[HD / 16][4];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int r = sp.n0 + g + 8 * half;
      const bool in = g + 8 * half < sp.rows && r / G < a.len(b);
      const uint32_t* p = reinterpret_cast<const uint32_t*>(
          a.q + (((long long)b * a.M + r / G) * a.NH + kh * G + r % G) * HD);
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk) {
        q[kk][half] = in ? __ldcg(p + kk * 8 + c) : 0u;
        q[kk][half + 2] = in ? __ldcg(p + kk * 8 + 4 + c) : 0u;
      }
    }
    // position of each of the two rows (of the last valid one, for padding)
    const int t[2] = {a.pos(b, min((sp.n0 + g) / G, max(a.len(b) - 1, 0))),
                      a.pos(b, min((sp.n0 + g + 8) / G, max(a.len(b) - 1, 0)))};
#pragma unroll
    for (int i = 0; i < HD / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    const int key_w = warp * 16;  // this warp's keys within a block
    uint32_t n = 0;
    for (int blk = blk0; blk < blk1; ++blk, ++n) {
      const int st = n % C::STAGES;
      if (!mbar_wait_warp(BAR_F(st), (n / C::STAGES) & 1, abort_p)) break;
      const uint32_t sk = sbase + st * 2 * C::TILE, sv = sk + C::TILE;
      // S: keys 0-7 and 8-15 of the warp
      float s[2][4] = {};
      {
        // ldmatrix lane -> row (key) and 16-byte chunk of a 16 x 16 piece
        const int row = key_w + (lane & 7) + ((lane >> 4) << 3), half = (lane >> 3) & 1;
        const uint32_t base = sk + row * 128;
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          const int ch = (kk % 4) * 2 + half;
          uint32_t k4[4];
          ldsm4(base + (kk / 4) * (KEYS * 128) + ((ch ^ (row & 7)) * 16), k4);
          mma16816(s[0], q[kk], k4[0], k4[1]);
          mma16816(s[1], q[kk], k4[2], k4[3]);
        }
      }
      const bool sink = blk < sp.sink_blocks;
      const int k0 = sp.first_key(blk) + key_w;  // the warp's first key
      // which keys some row sees: [k0, seen) of this warp's 16
      const int seen = sink ? sp.sink_end : sp.t1 + 1;
      if (k0 + 16 > seen || (!sink && (k0 + 15 > sp.t0 || k0 <= sp.t1 - a.window))) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = k0 + x * 8 + c * 2 + (e & 1), tt = t[e >> 1];
            const bool see = sink ? key < sp.sink_end
                                  : key <= tt && (tt - key < a.window || key < a.sinks);
            if (!see) s[x][e] = -INFINITY;
          }
        if (k0 + 16 > seen) {  // unseen V rows to zero
          const int from = max(0, seen - k0);
          for (int i = lane; i < (16 - from) * C::KB * 8; i += 32) {
            const int row = key_w + from + i / (C::KB * 8), ch = i % (C::KB * 8);
            *reinterpret_cast<uint4*>(gbase + (sv - sbase) + (ch / 8) * (KEYS * 128) + row * 128 + (ch % 8) * 16) =
                make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async_smem();  // before TMA fills the slot again
          __syncwarp();
        }
      }
      // P as two bf16 operands, hi + lo: 16 bits of it, so that the output's own
      // rounding is all that is lost (one operand: 1.4 times that).  The tensor
      // cores have the time: a step of 64 requests takes 165 us, with one 162.
      uint32_t p4[4], r4[4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float mx = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float m_new = fmaxf(m[h], mx * prm.scale_log2);
        // O and l move to the new maximum only when it grew by more than 2^8
        const bool need = m_new > m[h] + RESCALE_THRESHOLD;
        if (__any_sync(0xffffffffu, need)) {
          const float alpha = need ? ex2(m[h] - m_new) : 1.0f;
          if (need) m[h] = m_new;
          l[h] *= alpha;
#pragma unroll
          for (int i = 0; i < HD / 8; ++i) {
            o[i][2 * h] *= alpha;
            o[i][2 * h + 1] *= alpha;
          }
        }
        const float base = m[h] == -INFINITY ? 0.0f : m[h];  // no key seen yet: P = 2^-inf = 0
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) p[e] = ex2(fmaf(s[e / 2][2 * h + (e & 1)], prm.scale_log2, -base));
        l[h] += (p[0] + p[1]) + (p[2] + p[3]);
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const uint32_t hi = pack_bf16(p[e], p[e + 1]);
          p4[h + e] = hi;
          r4[h + e] = pack_bf16(p[e] - __uint_as_float(hi << 16), p[e + 1] - __uint_as_float(hi & 0xffff0000u));
        }
      }
      {
        const int row = key_w + (lane & 15), half = lane >> 4;
        const uint32_t base = sv + row * 128;
#pragma unroll
        for (int d = 0; d < HD / 16; ++d) {
          const int ch = (d % 4) * 2 + half;
          uint32_t v4[4];
          ldsm4_t(base + (d / 4) * (KEYS * 128) + ((ch ^ (row & 7)) * 16), v4);
          mma16816(o[2 * d], p4, v4[0], v4[1]);
          mma16816(o[2 * d + 1], p4, v4[2], v4[3]);
          mma16816(o[2 * d], r4, v4[0], v4[1]);
          mma16816(o[2 * d + 1], r4, v4[2], v4[3]);
        }
      }
      // V has been read.  (Without the fence the last ldmatrix of a block could
      // still be to come at the arrival, and a warp held up there read the next
      // block's rows: one unit in a few hundred.)
      __threadfence_block();
      __syncwarp();
      if (lane == 0) mbar_arrive(BAR_E(st));
    }
  }
  __syncthreads();  // every block loaded has been consumed (or a wait ran out): the ring is free

  // -------------------------------------- join the warps, each its own keys
  float* jo = reinterpret_cast<float*>(gbase);                         // [WARPS][ROWS][HD]
  float* jm = jo + WARPS * ROWS * HD;                                  // [WARPS][ROWS][2]
  if (warp < WARPS) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float sum = l[h];
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      const int r = warp * ROWS + g + 8 * h;
      if (c == 0) jm[2 * r] = m[h], jm[2 * r + 1] = sum;
#pragma unroll
      for (int i = 0; i < HD / 8; ++i)
        *reinterpret_cast<float2*>(jo + r * HD + i * 8 + c * 2) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < sp.rows * (HD / 4); i += THREADS) {
    const int r = i / (HD / 4), d = i % (HD / 4) * 4;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, jm[2 * (w * ROWS + r)]);
    const float base = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float f = ex2(jm[2 * (w * ROWS + r)] - base);
      const float4 y = *reinterpret_cast<const float4*>(jo + (w * ROWS + r) * HD + d);
      sum = fmaf(f, jm[2 * (w * ROWS + r) + 1], sum);
      x.x = fmaf(f, y.x, x.x), x.y = fmaf(f, y.y, x.y), x.z = fmaf(f, y.z, x.z), x.w = fmaf(f, y.w, x.w);
    }
    if (prm.nsplit > 1) {
      const long long at = (long long)blockIdx.x * ROWS + r;  // [unit][split][row]
      *reinterpret_cast<float4*>(prm.part_o + at * HD + d) = x;
      if (d == 0) *reinterpret_cast<float2*>(prm.part_ml + at * 2) = make_float2(top, sum);
    } else {
      const int row = sp.n0 + r;
      const bool valid = row / G < a.len(b);
      const float inv = valid ? 1.0f / sum : 0.0f;
      const long long item = ((long long)b * a.M + row / G) * a.NH + kh * G + row % G;
      *reinterpret_cast<uint2*>(a.out + item * HD + d) =
          valid ? make_uint2(pack_bf16(x.x * inv, x.y * inv), pack_bf16(x.z * inv, x.w * inv)) : make_uint2(0u, 0u);
      if (d == 0) a.l[item] = valid ? (top + log2f(sum)) * LN2 : -INFINITY;
    }
  }
  if (threadIdx.x == 0 && abort_flag) atomicOr(a.status, STATUS_FWD_TIMEOUT);
}

// Joins the splits of a row.  A block a row: D/4 threads across the columns,
// JOIN / (D/4) slices of the splits, each slice in split order and then the
// slices in theirs, so the order of the sums is fixed.  Latency-bound (a few
// hundred KB in all), so the slices' loads go out together.
constexpr int JOIN = 256;

template <int HD>
__global__ void __launch_bounds__(JOIN) window_join_kernel(const DecodeParams prm) {
  constexpr int LANES = HD / 4, SLICES = JOIN / LANES;
  __shared__ float4 so[SLICES][LANES];
  __shared__ float2 sml[SLICES];
  pdl_wait_and_release();
  const WindowArgs& a = prm.a;
  const int G = a.NH / a.NKV, R = a.M * G;
  const int row = blockIdx.x % R;
  const int bk = blockIdx.x / R;
  const int b = bk / a.NKV, kh = bk % a.NKV;
  const int lane = threadIdx.x % LANES, slice = threadIdx.x / LANES;
  const long long at0 = (((long long)bk * prm.groups + row / ROWS) * prm.nsplit) * ROWS + row % ROWS;
  float top = -INFINITY, sum = 0.0f;
  float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  auto add = [&](float2 ml, float4 y) {
    const float m = fmaxf(top, ml.x), base = m == -INFINITY ? 0.0f : m;
    const float f = ex2(top - base), h = ex2(ml.x - base);
    top = m;
    sum = sum * f + ml.y * h;
    x.x = x.x * f + y.x * h, x.y = x.y * f + y.y * h, x.z = x.z * f + y.z * h, x.w = x.w * f + y.w * h;
  };
#pragma unroll 4
  for (int s = slice; s < prm.nsplit; s += SLICES) {
    const long long at = at0 + (long long)s * ROWS;
    add(__ldcg(reinterpret_cast<const float2*>(prm.part_ml) + at),
        __ldcg(reinterpret_cast<const float4*>(prm.part_o + at * HD) + lane));
  }
  so[slice][lane] = x;
  if (lane == 0) sml[slice] = make_float2(top, sum);
  __syncthreads();
  if (slice > 0) return;
#pragma unroll
  for (int s = 1; s < SLICES; ++s) add(sml[s], so[s][lane]);
  const bool valid = row / G < a.len(b);
  const float inv = valid ? 1.0f / sum : 0.0f;
  const long long item = ((long long)b * a.M + row / G) * a.NH + kh * G + row % G;
  *reinterpret_cast<uint2*>(a.out + item * HD + lane * 4) =
      valid ? make_uint2(pack_bf16(x.x * inv, x.y * inv), pack_bf16(x.z * inv, x.w * inv)) : make_uint2(0u, 0u);
  if (lane == 0) a.l[item] = valid ? (top + log2f(sum)) * LN2 : -INFINITY;
}

// Few query rows a K/V head take the kernel of this file, more the tiled forward,
// whose tiles hold 128 rows of one head: this one's time goes by the rows and the
// other's by the heads.  Measured (us, this kernel / tiled, heads of 64, window
// 4096): 8 requests, 32 / 8 heads: 16 rows 29 / 104, 64 rows 51 / 106, 68 rows
// 88 / 106, 128 rows 96 / 106, 256 rows 182 / 106; 16 requests, 16 / 16 heads: 32
// rows 98 / 104, 64 rows 184 / 104.  The times meet at about 32 new tokens whatever
// the heads of a group; 64 rows are on the safe side of that from 2 heads a group on.
// (The two also differ in P: hi + lo here, one bf16 operand there.)
bool few_rows(const WindowArgs& a) { return (long long)a.M * (a.NH / a.NKV) <= 4 * ROWS; }

struct DecodePlan {
  int groups, nsplit;
  long long units;
};

DecodePlan decode_plan(const WindowArgs& a) {
  DecodePlan p;
  p.groups = (a.M * (a.NH / a.NKV) + ROWS - 1) / ROWS;
  p.units = (long long)a.B * a.NKV * p.groups;
  // the blocks a group can have at most; the host does not know the lengths
  const long long keys = std::min<long long>(a.K, (long long)a.window + a.M - 1 + std::min(a.sinks, a.K));
  const long long blocks = keys / KEYS + 2;
  const long long fill = SMS * CTAS_PER_SM / p.units;  // splits that fill the GPU once
  p.nsplit = (int)std::max<long long>(1, std::min(fill, blocks / MIN_BLOCKS));
  return p;
}

template <int HD>
cudaError_t launch_decode(const WindowArgs& a, void* workspace, cudaStream_t st) {
  using C = DecodeCfg<HD>;
  const DecodePlan p = decode_plan(a);
  CUtensorMap tk, tv;
  const CUtensorMapDataType bf = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  if (!make_tmap_3d(&tk, a.k, bf, 2, (uint64_t)a.NKV * HD, a.K, a.B, 64, KEYS, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !make_tmap_3d(&tv, a.v, bf, 2, (uint64_t)a.NKV * HD, a.K, a.B, 64, KEYS, CU_TENSOR_MAP_SWIZZLE_128B))
    return cudaErrorInvalidValue;
  DecodeParams prm;
  prm.a = a;
  prm.groups = p.groups;
  prm.nsplit = p.nsplit;
  prm.scale_log2 = a.scale * LOG2E;
  prm.expire_ns = take_expire_request(STATUS_FWD_TIMEOUT);
  prm.part_o = static_cast<float*>(workspace);
  prm.part_ml = prm.part_o + p.units * p.nsplit * ROWS * HD;
  cudaError_t e = cudaFuncSetAttribute(window_decode_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  if (e != cudaSuccess) return e;
  launch_pdl(window_decode_kernel<HD>, (unsigned)(p.units * p.nsplit), THREADS, C::SMEM, st, tk, tv, prm);
  count_launches(1);
  e = cudaGetLastError();
  if (e != cudaSuccess || p.nsplit == 1) return e;
  launch_pdl(window_join_kernel<HD>, (unsigned)(a.B * a.M * a.NH), JOIN, 0, st, prm);
  count_launches(1);
  return cudaGetLastError();
}

}  // namespace

size_t window_cached_workspace(const WindowArgs& a) {
  if (!few_rows(a)) return 0;
  const DecodePlan p = decode_plan(a);
  return p.nsplit == 1 ? 0 : (size_t)p.units * p.nsplit * ROWS * (a.D + 2) * sizeof(float);
}

cudaError_t launch_window_cached(const WindowArgs& a, void* workspace, cudaStream_t st) {
  if (!few_rows(a)) return launch_window_fwd(a, st);
  return a.D == 64 ? launch_decode<64>(a, workspace, st) : launch_decode<128>(a, workspace, st);
}

}  // namespace ma
