// window_attn.cu -- attention with a sliding window and sinks.
//
// Query i of a sequence sits at position pos = start + i and sees key j when
//   j <= pos  and  (pos - j < window  or  j < sinks)
// (a row i past the sequence's length sees nothing: O = 0, l = -inf, and it
// adds nothing to any gradient).  Over the visible keys
//   l_i = ln sum_j exp(q_i k_j / sqrt(D)),  O_i = sum_j exp(q_i k_j / sqrt(D) - l_i) v_j
//   delta_i = dO_i . O_i,  dS_ij = P_ij (dO_i v_j - delta_i) / sqrt(D)
//   dQ_i = sum_j dS_ij k_j,  dK_j = sum_i dS_ij q_i,  dV_j = sum_i P_ij dO_i
// where the sums over i run over every query head that shares the K/V head.
//
// One warp a row, CUDA cores, fp32 throughout.
#include "common.cuh"

namespace ma {
namespace {

constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) x += __shfl_xor_sync(0xffffffffu, x, m);
  return x;
}

template <int E>
__device__ __forceinline__ void load_row(const __nv_bfloat16* p, int lane, float (&x)[E]) {
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = __bfloat162float(p[lane + 32 * e]);
}

template <int E>
__device__ __forceinline__ float dot(const float (&a)[E], const float (&b)[E]) {
  float s = 0.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) s = fmaf(a[e], b[e], s);
  return warp_sum(s);
}

// delta and dQ of a row
template <int HD>
__global__ void __launch_bounds__(256) window_bwd_dq_rows(const WindowArgs a, const WindowGrads g) {
  pdl_wait_and_release();
  constexpr int E = HD / 32;
  const int lane = threadIdx.x % 32;
  const long long items = (long long)a.B * a.M * a.NH;
  for (long long it = blockIdx.x * 8ll + threadIdx.x / 32; it < items; it += gridDim.x * 8ll) {
    const int h = (int)(it % a.NH);
    const long long row = it / a.NH;
    const int b = (int)(row / a.M), i = (int)(row % a.M);
    const int kh = h / (a.NH / a.NKV);
    float q[E], d[E], o[E], dq[E] = {};
    load_row<E>(a.q + it * HD, lane, q);
    load_row<E>(g.dO + it * HD, lane, d);
    load_row<E>(a.out + it * HD, lane, o);
    const float delta = dot<E>(d, o);
    if (lane == 0) static_cast<float*>(g.workspace)[it] = delta;
    if (i < a.len(b)) {
      const float l = a.l[it];
      const int low = max(0, i - a.window + 1), ns = min(a.sinks, low);
      for (int n = 0; n < ns + i + 1 - low; ++n) {
        const int j = n < ns ? n : low + n - ns;
        const long long off = (((long long)b * a.K + j) * a.NKV + kh) * HD;
        float k[E], v[E];
        load_row<E>(a.k + off, lane, k);
        load_row<E>(a.v + off, lane, v);
        const float p = exp2f((dot<E>(q, k) * a.scale - l) * LOG2E);
        const float ds = p * (dot<E>(d, v) - delta) * a.scale;
#pragma unroll
        for (int e = 0; e < E; ++e) dq[e] = fmaf(ds, k[e], dq[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (g.dq_f32) static_cast<float*>(g.dQ)[it * HD + lane + 32 * e] = dq[e];
      else static_cast<__nv_bfloat16*>(g.dQ)[it * HD + lane + 32 * e] = __float2bfloat16_rn(dq[e]);
    }
  }
}

// dK and dV of a key row
template <int HD>
__global__ void __launch_bounds__(256) window_bwd_dkv_rows(const WindowArgs a, const WindowGrads g) {
  pdl_wait_and_release();
  constexpr int E = HD / 32;
  const int lane = threadIdx.x % 32;
  const long long items = (long long)a.B * a.K * a.NKV;
  for (long long it = blockIdx.x * 8ll + threadIdx.x / 32; it < items; it += gridDim.x * 8ll) {
    const int kh = (int)(it % a.NKV);
    const long long row = it / a.NKV;
    const int b = (int)(row / a.K), j = (int)(row % a.K);
    const int G = a.NH / a.NKV;
    float k[E], v[E], dk[E] = {}, dv[E] = {};
    load_row<E>(a.k + it * HD, lane, k);
    load_row<E>(a.v + it * HD, lane, v);
    const int n = a.len(b);
    const int end = j < a.sinks ? n : (int)min((long long)n, (long long)j + a.window);
    for (int i = j; i < end; ++i) {
      for (int h = kh * G; h < kh * G + G; ++h) {
        const long long qi = ((long long)b * a.M + i) * a.NH + h;
        float q[E], d[E];
        load_row<E>(a.q + qi * HD, lane, q);
        load_row<E>(g.dO + qi * HD, lane, d);
        const float p = exp2f((dot<E>(q, k) * a.scale - a.l[qi]) * LOG2E);
        const float ds = p * (dot<E>(d, v) - static_cast<const float*>(g.workspace)[qi]) * a.scale;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          dk[e] = fmaf(ds, q[e], dk[e]);
          dv[e] = fmaf(p, d[e], dv[e]);
        }
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      g.dK[it * HD + lane + 32 * e] = __float2bfloat16_rn(dk[e]);
      g.dV[it * HD + lane + 32 * e] = __float2bfloat16_rn(dv[e]);
    }
  }
}

unsigned row_blocks(long long items) {
  const long long b = (items + 7) / 8;
  return (unsigned)(b < (1ll << 30) ? b : (1ll << 30));
}

}  // namespace

size_t window_cached_workspace(const WindowArgs&) { return 0; }

cudaError_t launch_window_cached(const WindowArgs& a, void*, cudaStream_t st) { return launch_window_fwd(a, st); }

// delta per (row, head)
size_t window_bwd_workspace(const WindowArgs& a, bool) { return (size_t)a.B * a.M * a.NH * sizeof(float); }

cudaError_t launch_window_bwd(const WindowArgs& a, const WindowGrads& g, cudaStream_t st) {
  launch_pdl(a.D == 64 ? window_bwd_dq_rows<64> : window_bwd_dq_rows<128>, row_blocks((long long)a.B * a.M * a.NH),
             256, 0, st, a, g);
  launch_pdl(a.D == 64 ? window_bwd_dkv_rows<64> : window_bwd_dkv_rows<128>, row_blocks((long long)a.B * a.K * a.NKV),
             256, 0, st, a, g);
  count_launches(2);
  return cudaGetLastError();
}

}  // namespace ma
