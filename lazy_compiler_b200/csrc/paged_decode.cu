// Attention of one new token of every sequence over its paged key-value cache
// (the single-token form of window_attention.cu): slot s has lens[s] cached
// tokens, its query is the last of them, and token j is row j % page_size of
// page table[s][j / page_size].
#include "attend.cuh"

namespace lc {
namespace {

using namespace attend;

struct DecodeParams {
  const void *q, *k, *v;
  void *o;
  float *lse;
  const int *table, *lens;
  int slots, width, pages, page_size, q_heads, kv_heads, d;
  int64_t qs[2], ks[3], vs[3], os[2], ts;  // element strides: q, o slot and head; k, v page, head, token; table slot
  int window, sinks;
  float scale_log2;
};

__device__ __forceinline__ int cached_tokens(const DecodeParams &p, int slot) {
  const int64_t most = (int64_t)p.width * p.page_size;
  const int n = max(p.lens[slot], 0);
  return n < most ? n : (int)most;
}

// ---------------------------------------------------------------- plain form
// One CTA of eight warps per (slot, query head), the keys dealt to the warps.
constexpr int kRowWarps = 8;

template <class T>
__global__ void __launch_bounds__(kRowWarps * 32) decode_row_kernel(DecodeParams p) {
  __shared__ float scratch[kRowWarps * (kMaxHead + 2)];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slot = blockIdx.x, h = blockIdx.y;
  const int hk = h / (p.q_heads / p.kv_heads);
  const int n = cached_tokens(p, slot);
  RowState st;
  if (n > 0) {
    float q[kMaxHead / 32];
    load_row(q, static_cast<const T *>(p.q) + slot * p.qs[0] + h * p.qs[1], p.d, lane, p.scale_log2);
    const int *row = p.table + slot * p.ts;
    auto at = [&](int j, const T *&k, const T *&v) {
      const int page = row[j / p.page_size], r = j % p.page_size;
      if ((unsigned)page >= (unsigned)p.pages) return false;
      k = static_cast<const T *>(p.k) + page * p.ks[0] + hk * p.ks[1] + r * p.ks[2];
      v = static_cast<const T *>(p.v) + page * p.vs[0] + hk * p.vs[1] + r * p.vs[2];
      return true;
    };
    const Visible see = visible(n - 1, p.window, p.sinks);
    attend_keys<T>(st, q, p.d, lane, warp, see.sink_end, kRowWarps, at);
    attend_keys<T>(st, q, p.d, lane, see.lo + warp, n, kRowWarps, at);
  }
  join_warps<kRowWarps>(st, scratch);
  if (warp == 0)
    store_row(st, static_cast<T *>(p.o) + slot * p.os[0] + h * p.os[1],
              p.lse ? p.lse + (int64_t)slot * p.q_heads + h : nullptr, p.d, lane);
}

}  // namespace
}  // namespace lc

extern "C" int lc_paged_decode(int dtype, const void *q, const void *k, const void *v, void *o, float *lse,
                               const int32_t *table, const int32_t *lens, int64_t slots, int64_t width, int64_t pages,
                               int64_t page_size, int64_t q_heads, int64_t kv_heads, int64_t d, const int64_t *strides,
                               int64_t window, int64_t sinks, float scale, void *stream) {
  using namespace lc;
  const char *me = "lc_paged_decode";
  if (dtype != LC_F16 && dtype != LC_BF16) return fail(LC_ERR_INVALID, "%s: dtype %d is not f16 or bf16", me, dtype);
  if (slots < 0 || width < 0 || pages < 0 || page_size < 1 || q_heads < 1 || kv_heads < 1 || d < 1 || window < 0 || sinks < 0)
    return fail(LC_ERR_INVALID, "%s: negative or zero size", me);
  if (q_heads % kv_heads) return fail(LC_ERR_INVALID, "%s: %lld query heads over %lld key-value heads", me, (long long)q_heads, (long long)kv_heads);
  if (!strides) return fail(LC_ERR_INVALID, "%s: null strides", me);
  if (!(scale > 0.f) || scale > 3e38f) return fail(LC_ERR_INVALID, "%s: scale must be positive and finite", me);
  if (d > attend::kMaxHead) return fail(LC_ERR_UNSUPPORTED, "%s: head size %lld is over 256", me, (long long)d);
  if (slots > (1 << 20) || q_heads > 65535 || pages > INT32_MAX || page_size > (1 << 20) || width * page_size > (1ll << 30))
    return fail(LC_ERR_UNSUPPORTED, "%s: shape too large", me);
  if (slots == 0) return LC_OK;
  if (!q || !o || !lens || (width > 0 && !table) || (pages > 0 && (!k || !v))) return fail(LC_ERR_INVALID, "%s: null buffer", me);
  if (!aligned(q, 2) || !aligned(k, 2) || !aligned(v, 2) || !aligned(o, 2)) return fail(LC_ERR_ALIGN, "%s: elements are two bytes", me);
  DecodeParams p;
  p.q = q, p.k = k, p.v = v, p.o = o, p.lse = lse, p.table = table, p.lens = lens;
  p.slots = (int)slots, p.width = (int)width, p.pages = (int)pages, p.page_size = (int)page_size;
  p.q_heads = (int)q_heads, p.kv_heads = (int)kv_heads, p.d = (int)d;
  for (int i = 0; i < 2; ++i) p.qs[i] = strides[i], p.os[i] = strides[8 + i];
  for (int i = 0; i < 3; ++i) p.ks[i] = strides[2 + i], p.vs[i] = strides[5 + i];
  p.ts = strides[10];
  const int64_t most = width * page_size;
  p.window = window >= most ? 0 : (int)window;  // a window the cache cannot outgrow is no window
  p.sinks = (int)(sinks < most ? sinks : most);
  p.scale_log2 = scale * attend::kLog2e;
  cudaStream_t s = as_stream(stream);
  const dim3 grid((unsigned)slots, (unsigned)q_heads);
  if (dtype == LC_F16)
    decode_row_kernel<__half><<<grid, kRowWarps * 32, 0, s>>>(p);
  else
    decode_row_kernel<__nv_bfloat16><<<grid, kRowWarps * 32, 0, s>>>(p);
  return check_launch(me);
}
