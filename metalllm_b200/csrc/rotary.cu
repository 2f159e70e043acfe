// rotary.cu -- rotary positions: rotaryForward, rotaryBackward and
// rotaryCacheAppend.
//
// A pair (a, b) of a head's first `rot` columns at position t turns by the
// angle t * f_i of its frequency:
//   forward   (a cos - b sin, a sin + b cos) * amplitude
//   backward  the transpose: (a cos + b sin, b cos - a sin) * amplitude
// Half layout pairs column i with i + rot/2, interleaved 2i with 2i + 1; the
// columns from `rot` on pass through.  The products are fp32 and each output
// rounds once.
//
// The angle is the only place where fp32 would lose: at position 10^6 an fp32
// product is off by 0.03 rad.  It is formed in fp64 in whole turns, the whole
// turns are dropped, and the rest (at most half a turn, 2^-25 exact) goes to
// sincospif in fp32.
//
// HBM-bound: each element is read and written once.  A thread owns one unit
// of a row's rotation (8 pairs of the half layout = two 16-byte vectors, 4
// pairs of the interleaved one = one vector, or fewer where `rot` does not
// allow that) and walks heads with it, so a sine is computed once
// for the heads of a thread and not once for each head.  Neighbouring lanes
// take the units of one head and then the next head, so a warp reads whole
// rows.  A thread loads BATCH heads before it turns the first.  Heads are dealt
// to as many threads as fill half of the GPU: at few rows every thread has one
// head (latency), at many rows the sines are shared.  Measured: 16384 rows of
// 32 + 8 heads of 128 57.5 us, 5.8 TB/s.
#include "common.cuh"
#include "sm100.cuh"

namespace ma {
namespace {

constexpr int THREADS = 128;
constexpr int BATCH = 2;

// What the kernel turns and copies.  Heads 0 .. hq-1 are q's, the next hk k's.
struct RotArgs {
  const void* q;
  const __nv_bfloat16* k;
  const __nv_bfloat16* v;  // append only: copied to the cache
  void* q_out;
  __nv_bfloat16* k_out;  // [B][T][hk*D], or the caches [B][cap][hk*D]
  __nv_bfloat16* v_out;
  const double* inv_freq;
  const int32_t* positions;  // [B][T] or null (row index)
  const int32_t* start;      // append: [B], position of a sequence's first new row
  const int32_t* lens;       // append: [B] valid rows, or null
  long long rows;
  int T, cap;
  int hq, hk, D, rot;
  int hsplit;     // threads a row's heads are dealt to
  int units;      // rotation units of one head
  int cunits;     // copied units of one head: q's and k's columns from rot on,
  int edge;       // `edge` pairs up to a multiple of 8, then vectors of 8
  int vunits;     // append: copied units of one head of v
  bool copy_q, copy_k;  // out of place, so the columns from rot on move too
  float amp, sign;      // sign -1: the backward's negative angle
};

// N elements as they lie in memory: 16-byte vectors where N fills them, kept
// packed in registers (a bf16 element of its own would take a whole one).
template <typename T, int N>
struct Piece;

template <int N>
struct Piece<float, N> {
  float x[N];
  __device__ __forceinline__ void load(const float* p) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      if constexpr (N % 4 == 0) *reinterpret_cast<float4*>(x + i) = *reinterpret_cast<const float4*>(p + i);
      else if constexpr (N == 2) *reinterpret_cast<float2*>(x) = *reinterpret_cast<const float2*>(p);
      else x[0] = p[0];
    }
  }
  __device__ __forceinline__ void store(float* p) const {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      if constexpr (N % 4 == 0) *reinterpret_cast<float4*>(p + i) = *reinterpret_cast<const float4*>(x + i);
      else if constexpr (N == 2) *reinterpret_cast<float2*>(p) = *reinterpret_cast<const float2*>(x);
      else p[0] = x[0];
    }
  }
  __device__ __forceinline__ float get(int i) const { return x[i]; }
  __device__ __forceinline__ void set2(int i, float u, float v) { x[i] = u, x[i + 1] = v; }  // i even
  __device__ __forceinline__ void set(float u) { x[0] = u; }                                 // N = 1
};

template <int N>
struct Piece<__nv_bfloat16, N> {
  static constexpr int W = N < 2 ? 1 : N / 2;
  uint32_t w[W];
  __device__ __forceinline__ void load(const __nv_bfloat16* p) {
    if constexpr (N == 8) {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else if constexpr (N == 4) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[0] = v.x, w[1] = v.y;
    } else if constexpr (N == 2) {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
      w[0] = *reinterpret_cast<const uint16_t*>(p);
    }
  }
  __device__ __forceinline__ void store(__nv_bfloat16* p) const {
    if constexpr (N == 8) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else if constexpr (N == 4) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else if constexpr (N == 2) *reinterpret_cast<uint32_t*>(p) = w[0];
    else *reinterpret_cast<uint16_t*>(p) = (uint16_t)w[0];
  }
  __device__ __forceinline__ float get(int i) const {
    return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
  }
  __device__ __forceinline__ void set2(int i, float u, float v) { w[i / 2] = sm100::pack_bf16(u, v); }
  __device__ __forceinline__ void set(float u) { w[0] = sm100::pack_bf16(u, 0.0f) & 0xffffu; }
};

// The two pieces of a unit turned: half layout, pair i is (x[i], y[i]);
// interleaved, (x[2i], x[2i + 1]) and y is empty.
template <bool INTER, typename T, int P>
__device__ __forceinline__ void turn_unit(Piece<T, INTER ? 2 * P : P>& x, Piece<T, P>& y, const float (&c)[P],
                                          const float (&s)[P], bool zero) {
  auto one = [&](float a, float b, int i, float& u, float& v) {
    u = zero ? 0.0f : a * c[i] - b * s[i];
    v = zero ? 0.0f : a * s[i] + b * c[i];
  };
  if constexpr (INTER) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      float u, v;
      one(x.get(2 * i), x.get(2 * i + 1), i, u, v);
      x.set2(2 * i, u, v);
    }
  } else if constexpr (P == 1) {
    float u, v;
    one(x.get(0), y.get(0), 0, u, v);
    x.set(u);
    y.set(v);
  } else {
#pragma unroll
    for (int i = 0; i < P; i += 2) {
      float u0, v0, u1, v1;
      one(x.get(i), y.get(i), i, u0, v0);
      one(x.get(i + 1), y.get(i + 1), i + 1, u1, v1);
      x.set2(i, u0, u1);
      y.set2(i, v0, v1);
    }
  }
}

// One unit (P pairs) of heads h0, h0 + step, ... below `heads`; in and out are
// the row's first head.  zero: a row past its sequence's length.
template <typename T, bool INTER, int P>
__device__ __forceinline__ void turn(const T* in, T* out, int h0, int step, int heads, int D, int unit, int half,
                                     const float (&c)[P], const float (&s)[P], bool zero) {
  const int at = INTER ? unit * 2 * P : unit * P;
  for (int h = h0; h < heads; h += BATCH * step) {
    Piece<T, INTER ? 2 * P : P> x[BATCH];
    Piece<T, P> y[BATCH];
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      const int g = h + j * step;
      if (g < heads) {
        x[j].load(in + (long long)g * D + at);
        if constexpr (!INTER) y[j].load(in + (long long)g * D + at + half);
      }
    }
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      const int g = h + j * step;
      if (g < heads) {
        turn_unit<INTER, T, P>(x[j], y[j], c, s, zero);
        x[j].store(out + (long long)g * D + at);
        if constexpr (!INTER) y[j].store(out + (long long)g * D + at + half);
      }
    }
  }
}

// Where row `row` of the new tokens goes in a cache: its row there, or -1.
__device__ __forceinline__ long long cache_row(const RotArgs& a, int b, int t, bool valid) {
  const long long pos = (long long)a.start[b] + t;
  return valid && pos >= 0 && pos < a.cap ? (long long)b * a.cap + pos : -1;
}

// N columns from `in` to `out`, or zeros.
template <int N, typename T>
__device__ __forceinline__ void copy(const T* in, T* out, bool zero) {
  Piece<T, N> x;
  x.load(in);
  if (zero) {
#pragma unroll
    for (int i = 0; i < N; i += 2) x.set2(i, 0.0f, 0.0f);
  }
  x.store(out);
}

// P pairs a unit.
template <typename TQ, bool INTER, int P, bool APPEND>
__global__ void __launch_bounds__(THREADS) rotary_kernel(const RotArgs a) {
  pdl_wait_and_release();
  const int heads = a.hq + a.hk, D = a.D, half = a.rot / 2;
  const long long nrot = a.rows * a.units * a.hsplit;
  const int copies = heads * a.cunits + (APPEND ? a.hk * a.vunits : 0);
  const long long total = nrot + a.rows * copies;
  for (long long g = blockIdx.x * (long long)THREADS + threadIdx.x; g < total;
       g += (long long)gridDim.x * THREADS) {
    if (g < nrot) {
      const int unit = (int)(g % a.units);
      const long long r = g / a.units;
      const int h0 = (int)(r % a.hsplit);
      const long long row = r / a.hsplit;
      const int b = (int)(row / a.T), t = (int)(row % a.T);
      const bool valid = !APPEND || !a.lens || t < a.lens[b];
      const long long pos = APPEND ? (long long)a.start[b] + t : a.positions ? a.positions[row] : t;
      float c[P], s[P];
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const double turns = (double)pos * (a.inv_freq[unit * P + i] * 0.15915494309189533577);
        sincospif(2.0f * (float)(turns - rint(turns)), &s[i], &c[i]);
        c[i] *= a.amp;
        s[i] *= a.amp * a.sign;
      }
      const long long krow = APPEND ? cache_row(a, b, t, valid) : row;
      const long long qoff = row * a.hq * D;
      turn<TQ, INTER, P>(static_cast<const TQ*>(a.q) + qoff, static_cast<TQ*>(a.q_out) + qoff, h0, a.hsplit, a.hq, D,
                         unit, half, c, s, !valid);
      if (krow >= 0) {
        // k's heads go on where q's ended
        const int k0 = a.hq <= h0 ? h0 - a.hq : (a.hsplit - (a.hq - h0) % a.hsplit) % a.hsplit;
        turn<__nv_bfloat16, INTER, P>(a.k + row * a.hk * D, a.k_out + krow * a.hk * D, k0, a.hsplit, a.hk, D, unit, half,
                                      c, s, false);
      }
      continue;
    }
    // the columns that only move: q's and k's from rot on, and v
    const long long r = g - nrot;
    const long long row = r / copies;
    int u = (int)(r % copies);
    const int b = (int)(row / a.T), t = (int)(row % a.T);
    const bool valid = !APPEND || !a.lens || t < a.lens[b];
    if (u < heads * a.cunits) {
      const int h = u / a.cunits, c = u % a.cunits;
      const bool pair = c < a.edge;
      const int at = pair ? a.rot + 2 * c : a.rot + 2 * a.edge + 8 * (c - a.edge);
      if (h < a.hq) {
        if (!a.copy_q && valid) continue;
        const long long off = (row * a.hq + h) * D + at;
        const TQ* in = static_cast<const TQ*>(a.q) + off;
        TQ* out = static_cast<TQ*>(a.q_out) + off;
        if (pair) copy<2>(in, out, !valid);
        else copy<8>(in, out, !valid);
      } else if (a.copy_k) {
        const long long krow = APPEND ? cache_row(a, b, t, valid) : row;
        if (krow < 0) continue;
        const int kh = h - a.hq;
        const __nv_bfloat16* in = a.k + (row * a.hk + kh) * D + at;
        __nv_bfloat16* out = a.k_out + (krow * a.hk + kh) * D + at;
        if (pair) copy<2>(in, out, false);
        else copy<8>(in, out, false);
      }
    } else if constexpr (APPEND) {  // v, always in 16-byte pieces
      u -= heads * a.cunits;
      const long long krow = cache_row(a, b, t, valid);
      if (krow < 0) continue;
      const int at = u * 8;  // within the row's hk*D columns
      Piece<__nv_bfloat16, 8> x;
      x.load(a.v + row * a.hk * D + at);
      x.store(a.v_out + krow * a.hk * D + at);
    }
  }
}

template <typename TQ, bool INTER, int P, bool APPEND>
cudaError_t launch_as(RotArgs a, cudaStream_t st) {
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int heads = a.hq + a.hk;
  a.units = a.rot / 2 / P;
  const bool copied = APPEND || a.copy_q || a.copy_k;
  a.edge = copied ? (8 - a.rot % 8) % 8 / 2 : 0;
  a.cunits = copied ? a.edge + (a.D - a.rot) / 8 : 0;
  a.vunits = APPEND ? a.D / 8 : 0;
  // threads enough for half of what a SM holds, each at least one head (at
  // 16384 rows of 40 heads 57.5 us against 58.5 for all it holds and 63 for a
  // third; at 16000 rows of 16 narrow heads 19.4 against 22.6 and 17.3)
  const long long fill = (long long)sms * 1024;
  long long split = fill / (a.rows * a.units) + 1;
  a.hsplit = (int)(split < heads ? split : heads);
  const long long total = a.rows * a.units * a.hsplit +
                          a.rows * ((long long)heads * a.cunits + (APPEND ? a.hk * a.vunits : 0));
  const long long blocks = (total + THREADS - 1) / THREADS;
  const long long most = 1ll << 30;
  launch_pdl(rotary_kernel<TQ, INTER, P, APPEND>, (unsigned)(blocks < most ? blocks : most), THREADS, 0, st, a);
  count_launches(1);
  return cudaGetLastError();
}

// The widest vectors that `rot` is a whole number of.
template <typename TQ, bool APPEND>
cudaError_t launch_type(const RotArgs& a, bool inter, cudaStream_t st) {
  if (inter) {
    if (a.rot % 8 == 0) return launch_as<TQ, true, 4, APPEND>(a, st);
    return a.rot % 4 == 0 ? launch_as<TQ, true, 2, APPEND>(a, st) : launch_as<TQ, true, 1, APPEND>(a, st);
  }
  if (a.rot % 16 == 0) return launch_as<TQ, false, 8, APPEND>(a, st);
  if (a.rot % 8 == 0) return launch_as<TQ, false, 4, APPEND>(a, st);
  return a.rot % 4 == 0 ? launch_as<TQ, false, 2, APPEND>(a, st) : launch_as<TQ, false, 1, APPEND>(a, st);
}

RotArgs rot_args(const AttnShape& s, int NKV, const MaRotary& r, bool back) {
  RotArgs a{};
  a.rows = (long long)s.B * s.T;
  a.T = s.T;
  a.hq = s.NH;
  a.hk = NKV;
  a.D = s.D;
  a.rot = (int)r.rot;
  a.inv_freq = r.inv_freq;
  a.amp = r.amplitude;
  a.sign = back ? -1.0f : 1.0f;
  return a;
}

}  // namespace

cudaError_t launch_rotary(const void* q, bool q_f32, const __nv_bfloat16* k, void* q_out, __nv_bfloat16* k_out,
                          const MaRotary& r, const int32_t* positions, const AttnShape& s, int NKV, bool back,
                          cudaStream_t st) {
  RotArgs a = rot_args(s, NKV, r, back);
  a.q = q;
  a.k = k;
  a.q_out = q_out;
  a.k_out = k_out;
  a.positions = positions;
  a.copy_q = q != q_out;
  a.copy_k = k != k_out;
  return q_f32 ? launch_type<float, false>(a, r.interleaved, st)
               : launch_type<__nv_bfloat16, false>(a, r.interleaved, st);
}

cudaError_t launch_rotary_append(const __nv_bfloat16* q, const __nv_bfloat16* k, const __nv_bfloat16* v,
                                 __nv_bfloat16* q_out, __nv_bfloat16* k_cache, __nv_bfloat16* v_cache,
                                 const int32_t* start, const int32_t* lens, const MaRotary& r, const AttnShape& s,
                                 int NKV, int cap, cudaStream_t st) {
  RotArgs a = rot_args(s, NKV, r, false);
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_out = q_out;
  a.k_out = k_cache;
  a.v_out = v_cache;
  a.start = start;
  a.lens = lens;
  a.cap = cap;
  a.copy_q = q != q_out;
  a.copy_k = true;
  return launch_type<__nv_bfloat16, true>(a, r.interleaved, st);
}

}  // namespace ma
