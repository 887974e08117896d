// Attention of a prompt over its keys, causal, with an optional sliding window
// and a few first tokens that stay visible:
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j   over the keys j that query i sees
// (attend.cuh says which), lse_i = log sum_j exp(scale q_i . k_j).  Grouped
// heads: query head h reads key-value head h / (q_heads / kv_heads).
#include "attend.cuh"

namespace lc {
namespace {

using namespace attend;

struct WindowParams {
  const void *q, *k, *v;
  void *o;
  float *lse;
  const int *q_lens, *kv_lens;
  int batch, s_q, s_kv, q_heads, kv_heads, d;
  int64_t qs[3], ks[3], vs[3], os[3];  // element strides: batch, token, head
  int window, sinks;
  float scale_log2;
};

// How many of a sequence's rows exist (the lengths are data: clamped to the buffers).
__device__ __forceinline__ int length_of(const int *lens, int b, int most) {
  return lens ? min(max(lens[b], 0), most) : most;
}

// ---------------------------------------------------------------- plain form
// One CTA of four warps per (row, query head), the row's keys dealt to the
// warps: any head size up to 256, any strides.
constexpr int kRowWarps = 4;

template <class T>
__global__ void __launch_bounds__(kRowWarps * 32) window_row_kernel(WindowParams p) {
  __shared__ float scratch[kRowWarps * (kMaxHead + 2)];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int i = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int hk = h / (p.q_heads / p.kv_heads);
  const int n_q = length_of(p.q_lens, b, p.s_q), n_kv = length_of(p.kv_lens, b, p.s_kv);
  const int pos = n_kv - n_q + i;
  RowState st;
  if (i < n_q && pos >= 0) {
    float q[kMaxHead / 32];
    load_row(q, static_cast<const T *>(p.q) + b * p.qs[0] + i * p.qs[1] + h * p.qs[2], p.d, lane, p.scale_log2);
    const T *k0 = static_cast<const T *>(p.k) + b * p.ks[0] + hk * p.ks[2];
    const T *v0 = static_cast<const T *>(p.v) + b * p.vs[0] + hk * p.vs[2];
    auto at = [&](int j, const T *&k, const T *&v) {
      k = k0 + j * p.ks[1];
      v = v0 + j * p.vs[1];
      return true;
    };
    const Visible see = visible(pos, p.window, p.sinks);
    attend_keys<T>(st, q, p.d, lane, warp, see.sink_end, kRowWarps, at);
    attend_keys<T>(st, q, p.d, lane, see.lo + warp, pos + 1, kRowWarps, at);
  }
  join_warps<kRowWarps>(st, scratch);
  if (warp == 0)
    store_row(st, static_cast<T *>(p.o) + b * p.os[0] + i * p.os[1] + h * p.os[2],
              p.lse ? p.lse + ((int64_t)b * p.q_heads + h) * p.s_q + i : nullptr, p.d, lane);
}

}  // namespace
}  // namespace lc

extern "C" int lc_window_attention(int dtype, const void *q, const void *k, const void *v, void *o, float *lse,
                                   const int32_t *q_lens, const int32_t *kv_lens, int64_t batch, int64_t s_q,
                                   int64_t s_kv, int64_t q_heads, int64_t kv_heads, int64_t d, const int64_t *strides,
                                   int64_t window, int64_t sinks, float scale, void *stream) {
  using namespace lc;
  const char *me = "lc_window_attention";
  if (dtype != LC_F16 && dtype != LC_BF16) return fail(LC_ERR_INVALID, "%s: dtype %d is not f16 or bf16", me, dtype);
  if (batch < 0 || s_q < 0 || s_kv < 0 || q_heads < 1 || kv_heads < 1 || d < 1 || window < 0 || sinks < 0)
    return fail(LC_ERR_INVALID, "%s: negative or zero size", me);
  if (q_heads % kv_heads) return fail(LC_ERR_INVALID, "%s: %lld query heads over %lld key-value heads", me, (long long)q_heads, (long long)kv_heads);
  if (!strides) return fail(LC_ERR_INVALID, "%s: null strides", me);
  if (!(scale > 0.f) || scale > 3e38f) return fail(LC_ERR_INVALID, "%s: scale must be positive and finite", me);
  if (d > attend::kMaxHead) return fail(LC_ERR_UNSUPPORTED, "%s: head size %lld is over 256", me, (long long)d);
  if (batch > 65535 || q_heads > 65535 || s_q > (1 << 30) || s_kv > (1 << 30) || batch * s_q > INT32_MAX)
    return fail(LC_ERR_UNSUPPORTED, "%s: shape too large", me);
  if (batch == 0 || s_q == 0) return LC_OK;
  if (!q || !o || (s_kv > 0 && (!k || !v))) return fail(LC_ERR_INVALID, "%s: null buffer", me);
  if (!aligned(q, 2) || !aligned(k, 2) || !aligned(v, 2) || !aligned(o, 2)) return fail(LC_ERR_ALIGN, "%s: elements are two bytes", me);
  WindowParams p;
  p.q = q, p.k = k, p.v = v, p.o = o, p.lse = lse, p.q_lens = q_lens, p.kv_lens = kv_lens;
  p.batch = (int)batch, p.s_q = (int)s_q, p.s_kv = (int)s_kv;
  p.q_heads = (int)q_heads, p.kv_heads = (int)kv_heads, p.d = (int)d;
  for (int i = 0; i < 3; ++i) p.qs[i] = strides[i], p.ks[i] = strides[3 + i], p.vs[i] = strides[6 + i], p.os[i] = strides[9 + i];
  // a window no query can reach past is no window
  p.window = window >= s_kv ? 0 : (int)window;
  p.sinks = (int)(sinks < s_kv ? sinks : s_kv);
  p.scale_log2 = scale * attend::kLog2e;
  cudaStream_t s = as_stream(stream);
  const dim3 grid((unsigned)s_q, (unsigned)q_heads, (unsigned)batch);
  if (dtype == LC_F16)
    window_row_kernel<__half><<<grid, kRowWarps * 32, 0, s>>>(p);
  else
    window_row_kernel<__nv_bfloat16><<<grid, kRowWarps * 32, 0, s>>>(p);
  return check_launch(me);
}
