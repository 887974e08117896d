// Shared pieces of the serving attention kernels (window_attention.cu,
// paged_decode.cu): which keys a query sees, 16-bit element conversion, and
// the plain row form (one key at a time, any head size up to 256) that covers
// what the tensor-core kernels do not.
//
// A query at position p sees key j when j <= p and (window == 0, or
// j > p - window, or j < sinks): two intervals, [0, sink_end) and [lo, p].
// Scores are kept in units of log2 (s * scale * log2 e), so a weight is
// 2^(s - m); m, l and the output sums are f32.
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

// Running softmax of one query row spread over the lanes of a warp: lane c
// holds output elements c, c + 32, ...
struct RowState {
  float m = -INFINITY, l = 0.f;
  float acc[kMaxHead / 32];
  __device__ __forceinline__ RowState() {
#pragma unroll
    for (int i = 0; i < kMaxHead / 32; ++i) acc[i] = 0.f;
  }
};

template <class T>
__device__ __forceinline__ void load_row(float (&q)[kMaxHead / 32], const T *src, int d, int lane, float factor) {
#pragma unroll
  for (int i = 0; i < kMaxHead / 32; ++i) {
    const int c = lane + 32 * i;
    q[i] = c < d ? Elem<T>::to_float(src[c]) * factor : 0.f;
  }
}

// Takes the keys j = begin, begin + step, ... < end into the row; `at(j, k, v)`
// sets the rows of key j, or returns false where there is none.
template <class T, class At>
__device__ __forceinline__ void attend_keys(RowState &st, const float (&q)[kMaxHead / 32], int d, int lane, int begin,
                                            int end, int step, const At &at) {
  for (int j = begin; j < end; j += step) {
    const T *k, *v;
    if (!at(j, k, v)) continue;
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < kMaxHead / 32; ++i) {
      const int c = lane + 32 * i;
      if (c < d) dot = fmaf(q[i], Elem<T>::to_float(k[c]), dot);
    }
    dot = warp_sum(dot);
    const float m_new = fmaxf(st.m, dot);
    const float base = m_new == -INFINITY ? 0.f : m_new;  // a row of -inf scores so far
    const float alpha = exp2f(st.m - base), w = exp2f(dot - base);
    st.m = m_new;
    st.l = st.l * alpha + w;
#pragma unroll
    for (int i = 0; i < kMaxHead / 32; ++i) {
      const int c = lane + 32 * i;
      if (c < d) st.acc[i] = fmaf(w, Elem<T>::to_float(v[c]), st.acc[i] * alpha);
    }
  }
}

// Writes a row whose sums are complete: O / l, and the log-sum-exp.  A row
// that saw nothing (or only scores of -inf) is 0 and -inf.
template <class T>
__device__ __forceinline__ void store_row(const RowState &st, T *o, float *lse, int d, int lane) {
  const float inv = st.l == 0.f ? 0.f : 1.f / st.l;
#pragma unroll
  for (int i = 0; i < kMaxHead / 32; ++i) {
    const int c = lane + 32 * i;
    if (c < d) o[c] = Elem<T>::from_float(st.acc[i] * inv);
  }
  if (lse && lane == 0) *lse = st.l == 0.f ? -INFINITY : (st.m + log2f(st.l)) * kLn2;
}

// The same row for a kernel whose own sums came out infinite or NaN in some
// columns: those alone are written, the others keep their bits.
template <class T>
__device__ __forceinline__ void mend_row(const RowState &st, T *o, int d, int lane) {
  const float inv = st.l == 0.f ? 0.f : 1.f / st.l;
#pragma unroll
  for (int i = 0; i < kMaxHead / 32; ++i) {
    const int c = lane + 32 * i;
    if (c < d && !isfinite(Elem<T>::to_float(o[c]))) o[c] = Elem<T>::from_float(st.acc[i] * inv);
  }
}

// Joins the states of the WARPS warps of a CTA, which each took a share of one
// row's keys, in warp order; warp 0 receives the row.
template <int WARPS>
__device__ __forceinline__ void join_warps(RowState &st, float *scratch /* WARPS * (kMaxHead + 2) */) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float *mine = scratch + warp * (kMaxHead + 2);
#pragma unroll
  for (int i = 0; i < kMaxHead / 32; ++i) mine[lane + 32 * i] = st.acc[i];
  if (lane == 0) {
    mine[kMaxHead] = st.m;
    mine[kMaxHead + 1] = st.l;
  }
  __syncthreads();
  if (warp != 0) return;
  float m = -INFINITY;
  bool nan = false;
  for (int w = 0; w < WARPS; ++w) {
    m = fmaxf(m, scratch[w * (kMaxHead + 2) + kMaxHead]);
    nan |= isnan(scratch[w * (kMaxHead + 2) + kMaxHead + 1]);
  }
  RowState sum;
  sum.m = m;
  if (nan || m != -INFINITY) {
    for (int w = 0; w < WARPS; ++w) {
      const float *s = scratch + w * (kMaxHead + 2);
      if (s[kMaxHead + 1] == 0.f) continue;  // no keys: its sums are zero
      const float a = exp2f(s[kMaxHead] - (m == -INFINITY ? 0.f : m));
      sum.l = fmaf(s[kMaxHead + 1], a, sum.l);
#pragma unroll
      for (int i = 0; i < kMaxHead / 32; ++i) sum.acc[i] = fmaf(s[lane + 32 * i], a, sum.acc[i]);
    }
  }
  st = sum;
}

}  // namespace attend
}  // namespace lc
