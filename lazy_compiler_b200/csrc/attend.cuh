// Shared pieces of the serving attention kernels (window_attention.cu,
// paged_decode.cu): which keys a query sees, 16-bit element conversion, and
// the plain row form (one key at a time, any head size up to 256) that covers
// what the tensor-core kernels do not.
//
// A query at position p sees key j when j <= p and (window == 0, or
// j > p - window, or j < sinks): two intervals, [0, sink_end) and [lo, p].
// Scores are kept in units of log2 (s * scale * log2 e), so a weight is
// 2^(s - m); m, l and the output sums are f32.  m is the row's reference: its maximum so far
// less a constant, which keeps the weights where the operand type and the sums hold them.
#pragma once

#include "common.cuh"

namespace lc {
namespace attend {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kMaxHead = 256;

template <class T>
struct Elem;
template <>
struct Elem<__half> {
  static __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
};
template <>
struct Elem<__nv_bfloat16> {
  static __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
};

// The keys position p sees: [0, sink_end) and [lo, p + 1).
struct Visible {
  int sink_end, lo;
};
__host__ __device__ __forceinline__ Visible visible(int p, int window, int sinks) {
  const int first = p - window + 1;  // window >= 1 here
  const int lo = window == 0 || first < 0 ? 0 : first;
  return {sinks < lo ? sinks : lo, lo};
}

// bf16 values reach f32's largest number, which the sum of two of them passes: the weights
// of bf16 rows are at most 2^-40 (2^-32 where the prompt form's maximum lags), so that the sum
// of 2^30 does not.  They end at f32's smallest number, 2^-86 of the largest weight.
constexpr float kLiftBf16 = -40.f;
// What the weights of the plain row form, whose operands are f32, are lifted by.
template <class T>
constexpr float kRowLift = kLiftBf16;
template <>
constexpr float kRowLift<__half> = 0.f;

// The log-sum-exp of a row with the reference m: its maximum again plus a small logarithm,
// since log2 of a lifted l alone would be rounded like a number of the lift's size.
template <int LIFT>
__device__ __forceinline__ float lse_of(float m, float l) {
  constexpr float kBack = LIFT < 0 ? (float)(1ll << (-LIFT & 63)) : 1.f / (float)(1ll << (LIFT & 63));
  return ((m + LIFT) + log2f(l * kBack)) * kLn2;
}

// Running softmax of one query row of up to 32 NC columns spread over the lanes of a
// warp: lane c holds output elements c, c + 32, ...
template <int NC>
struct RowState {
  float m = -INFINITY, l = 0.f;
  float acc[NC];
  __device__ __forceinline__ RowState() {
#pragma unroll
    for (int i = 0; i < NC; ++i) acc[i] = 0.f;
  }
};

template <class T, int NC>
__device__ __forceinline__ void load_row(float (&q)[NC], const T *src, int d, int lane, float factor) {
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = lane + 32 * i;
    q[i] = c < d ? Elem<T>::to_float(src[c]) * factor : 0.f;
  }
}

// Takes the keys j = begin, begin + step, ... < end into the row; `at(j, k, v)` sets
// the rows of key j, or readable ones in their place, and says whether key j counts.
// Four keys at a time, and every load unconditional in the key, so that the loads
// and the lanes' sums overlap.
template <class T, int NC, class At>
__device__ __forceinline__ void attend_keys(RowState<NC> &st, const float (&q)[NC], int d, int lane, int begin, int end, int step,
                                            const At &at) {
  constexpr int U = 4;
  for (int j = begin; j < end; j += U * step) {
    bool real[U];
    const T *kr[U], *vr[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int key = j + u * step;
      real[u] = at(key < end ? key : j, kr[u], vr[u]) && key < end;
    }
    T kv[U][NC], vv[U][NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = lane + 32 * i;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        kv[u][i] = vv[u][i] = Elem<T>::from_float(0.f);
        if (c < d) {
          kv[u][i] = kr[u][c];
          vv[u][i] = vr[u][c];
        }
      }
    }
    float s[U], v[U][NC];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      s[u] = 0.f;
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        s[u] = fmaf(q[i], Elem<T>::to_float(kv[u][i]), s[u]);
        v[u][i] = Elem<T>::to_float(vv[u][i]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) s[u] = warp_sum(s[u]);
    float m_new = st.m;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (real[u]) m_new = fmaxf(m_new, s[u] - kRowLift<T>);
    const float base = m_new == -INFINITY ? 0.f : m_new;  // a row of -inf scores so far
    const float alpha = exp2f(st.m - base);
    st.m = m_new;
    st.l *= alpha;
#pragma unroll
    for (int i = 0; i < NC; ++i) st.acc[i] *= alpha;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!real[u]) continue;
      const float w = exp2f(s[u] - base);
      st.l += w;
#pragma unroll
      for (int i = 0; i < NC; ++i) st.acc[i] = fmaf(w, v[u][i], st.acc[i]);
    }
  }
}

// Writes a row whose sums are complete: O / l, and the log-sum-exp.  A row
// that saw nothing (or only scores of -inf) is 0 and -inf.
template <class T, int NC>
__device__ __forceinline__ void store_row(const RowState<NC> &st, T *o, float *lse, int d, int lane) {
  const float inv = st.l == 0.f ? 0.f : 1.f / st.l;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = lane + 32 * i;
    if (c < d) o[c] = Elem<T>::from_float(st.acc[i] * inv);
  }
  if (lse && lane == 0) *lse = st.l == 0.f ? -INFINITY : lse_of<(int)kRowLift<T>>(st.m, st.l);
}

// The same row for a kernel whose own sums came out infinite or NaN in some
// columns: those alone are written, the others keep their bits.
template <class T, int NC>
__device__ __forceinline__ void mend_row(const RowState<NC> &st, T *o, int d, int lane) {
  const float inv = st.l == 0.f ? 0.f : 1.f / st.l;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = lane + 32 * i;
    if (c < d && !isfinite(Elem<T>::to_float(o[c]))) o[c] = Elem<T>::from_float(st.acc[i] * inv);
  }
}

// Joins the states of the WARPS warps of a CTA, which each took a share of one
// row's keys, in warp order; warp 0 receives the row.
template <int WARPS, int NC>
__device__ __forceinline__ void join_warps(RowState<NC> &st, float *scratch /* WARPS * (32 * NC + 2) */) {
  constexpr int kWide = 32 * NC;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float *mine = scratch + warp * (kWide + 2);
#pragma unroll
  for (int i = 0; i < NC; ++i) mine[lane + 32 * i] = st.acc[i];
  if (lane == 0) {
    mine[kWide] = st.m;
    mine[kWide + 1] = st.l;
  }
  __syncthreads();
  if (warp != 0) return;
  float m = -INFINITY;
  for (int w = 0; w < WARPS; ++w) m = fmaxf(m, scratch[w * (kWide + 2) + kWide]);
  RowState<NC> sum;
  sum.m = m;
  for (int w = 0; w < WARPS; ++w) {
    const float *s = scratch + w * (kWide + 2);
    if (s[kWide + 1] == 0.f) continue;  // no keys: its sums are zero
    const float a = exp2f(s[kWide] - (m == -INFINITY ? 0.f : m));
    sum.l = fmaf(s[kWide + 1], a, sum.l);
#pragma unroll
    for (int i = 0; i < NC; ++i) sum.acc[i] = fmaf(s[lane + 32 * i], a, sum.acc[i]);
  }
  st = sum;
}

}  // namespace attend
}  // namespace lc
