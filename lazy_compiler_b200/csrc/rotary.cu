// Positions as rotations: pair i of a head, (x[i], x[i + rot / 2]) or interleaved
// (x[2 i], x[2 i + 1]), turns by the angle position * f_i; what lies behind the
// first `rot` elements passes.  lc_rotate does this to a tensor; lc_cache_append to
// the newest queries and keys of a paged cache on their way: the keys, and the
// values unturned, go to their pages, the queries to `out`.
//
// Angles: a frequency is a 64-bit fraction of a turn, so position * frequency modulo
// 2^64 is the angle modulo a turn, exact at any position (an f32 product is off by 0.06
// rad at a million); what the fraction's own rounding adds is 2^-33 of a turn at the
// farthest position there is.  The nearest quarter turn comes off in integers too, and
// sincospif sees at most an eighth of a turn: off by 2^-25 or so.
//
// Bound by HBM, each element read and written once.  An angle belongs to all heads of a
// token, so a CTA works out the rotations of its tokens once, in shared memory, and a
// thread then takes units of V pairs (16 bytes of each half) of any head.  Measured, bf16,
// 40 heads of 128: 4 x 8191 tokens in 108 us, 6.2 TB/s; f32: 203 us, 6.6 TB/s; into the cache,
// f16, 32/8 heads, 16 prompts of 1023 to 4095 tokens: 206 us, 5.9 TB/s; 64 x 1 token: 3.1 and 4.2 us.
#include <algorithm>

#include "common.cuh"
#include "softmax.cuh"

namespace lc {
namespace {

constexpr int kThreads = 256;
constexpr int kMostTokens = 32;    // of a CTA
constexpr int kMostRotations = 2048;  // of a CTA's tokens, in shared memory
constexpr int kMostHead = 1024;

// A division by a number known at the launch: (x * multiplier) >> shift, exact for x below 2^26 (the products stay
// below 2^64, the multiplier's rounding below x's last part).
struct Divisor {
  unsigned multiplier, shift;
};
inline Divisor divisor_of(unsigned n) {
  unsigned shift = 26;
  while ((1u << (shift - 26)) < n) ++shift;  // 2^shift / n is below 2^26 + 1, and off by less than 2^(shift - 26) / n <= 1 in 2^26
  return {(unsigned)(((1ull << shift) + n - 1) / n), shift};
}
__device__ __forceinline__ unsigned by(int x, const Divisor &d) { return (unsigned)((unsigned long long)(unsigned)x * d.multiplier >> d.shift); }

struct RotaryParams {
  const int64_t *turns;  // rot / 2 of them, in 2^-64 of a turn
  int rot, interleaved;
  float magnitude;
};

struct RotateParams {
  RotaryParams rotary;
  const void *x[3];       // queries (or the one tensor), keys, values
  int64_t xs[3][3];       // batch, token, head, in elements
  void *out;              // of x[0]
  int64_t os[3];
  const int *positions;   // lc_rotate
  int64_t ps[2];
  // lc_cache_append
  void *pages[2];         // keys, values
  int64_t kp[2][3];       // page, head, token
  const int *table, *lens, *add, *refused;
  int width, page_count, page_size, zero_rest;
  Divisor per_token, per_row;  // units of a token, of a head
  int tokens, tiles, tile, heads[2], rows, d, units, turned;  // tile: tokens of a CTA; rows: of a token
};

template <class T>
__device__ __forceinline__ float widen(T v);
template <>
__device__ __forceinline__ float widen(float v) { return v; }
template <>
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ float narrow(float v) { return v; }
template <>
__device__ __forceinline__ __half narrow(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow(float v) { return __float2bfloat16_rn(v); }

template <class T, int V>
struct alignas(sizeof(T) * V) Piece {
  T v[V];
};

// Whole pieces by streaming stores: what is written here leaves L2 before what is read (4 x 8191 tokens of 40 heads:
// 114 -> 108 us).
template <class T, int V>
__device__ __forceinline__ void put(T *to, const Piece<T, V> &x) {
  if constexpr (sizeof(x) == 16)
    st_stream_u4(to, *reinterpret_cast<const uint4 *>(&x));
  else
    *reinterpret_cast<Piece<T, V> *>(to) = x;
}

// (cos, sin) of position * frequency, times the magnitude.
__device__ __forceinline__ float2 rotation(int64_t turns, int64_t position, float magnitude) {
  const uint64_t angle = (uint64_t)turns * (uint64_t)position;  // of 2^64 a turn
  const uint64_t quarter = (angle + (1ull << 61)) >> 62;
  const int rest = (int)((int64_t)(angle - (quarter << 62)) >> 32);  // at most an eighth of a turn: 2^29
  float s, c;
  sincospif((float)rest * 0x1p-31f, &s, &c);
  if (quarter & 1) {
    const float t = c;
    c = -s;
    s = t;
  }
  if (quarter & 2) {
    c = -c;
    s = -s;
  }
  return make_float2(c * magnitude, s * magnitude);
}

// Pairs (f, g) turned, two by two in Blackwell's paired f32 form.
template <int V>
__device__ __forceinline__ void turn_pairs(float (&f)[V], float (&g)[V], const float *cosines, const float *sines) {
  using namespace softmax;
  if constexpr (V == 1) {
    const float c = cosines[0], s = sines[0], u = f[0], v = g[0];
    f[0] = u * c - v * s;
    g[0] = u * s + v * c;
  } else {
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      const uint64_t u = pack2(f[e], f[e + 1]), v = pack2(g[e], g[e + 1]);
      const uint64_t c = *reinterpret_cast<const uint64_t *>(cosines + e), s = *reinterpret_cast<const uint64_t *>(sines + e);
      const float2 x = unpack2(fsub2(ffma2(u, c, 0ull), ffma2(v, s, 0ull))), y = unpack2(ffma2(u, s, ffma2(v, c, 0ull)));
      f[e] = x.x, f[e + 1] = x.y;
      g[e] = y.x, g[e + 1] = y.y;
    }
  }
}

template <class T, int V, bool APPEND>
__global__ void __launch_bounds__(kThreads) rotate_kernel(const __grid_constant__ RotateParams p) {
  __shared__ __align__(16) float cosines[kMostRotations], sines[kMostRotations];
  __shared__ int64_t to[2][kMostTokens];  // where a token's key and value go, -1: nowhere
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, b = blockIdx.x / p.tiles, first = (blockIdx.x - b * p.tiles) * p.tile;
  int count = min(p.tile, p.tokens - first), real = count;  // tokens of the tile, and those that are turned
  int64_t start = 0;
  if (APPEND) {
    const int add = p.add[b];
    start = (int64_t)p.lens[b] - add;
    const bool none = (p.refused && *p.refused) || start < 0;
    real = none ? 0 : min(count, max(0, add - first));
    if (!p.zero_rest) count = real;
    if (count == 0) return;
    if (tid < real) {
      const int64_t pos = start + first + tid, entry = pos / p.page_size, r = pos - entry * p.page_size;
      const int page = entry < p.width ? p.table[(int64_t)b * p.width + entry] : -1;
      const bool held = (unsigned)page < (unsigned)p.page_count;
      to[0][tid] = held ? page * p.kp[0][0] + r * p.kp[0][2] : -1;
      to[1][tid] = held ? page * p.kp[1][0] + r * p.kp[1][2] : -1;
    }
  }
  const int half = p.rotary.rot / 2;
  for (int i = tid; i < real * half; i += kThreads) {
    const int t = i / half, pair = i - t * half;
    const int64_t pos = APPEND ? start + first + t : p.positions[b * p.ps[0] + (first + t) * p.ps[1]];
    const float2 cs = rotation(p.rotary.turns[pair], pos, p.rotary.magnitude);
    cosines[i] = cs.x;
    sines[i] = cs.y;
  }
  __syncthreads();

  using P = Piece<T, V>;
  const int per_token = p.rows * p.units, inner = p.rotary.interleaved ? V : half;  // from a unit's first piece to its second
  // (Two or four units a thread with their loads together: 134 and 198 us for 4 x 8191 tokens of 40 heads, since fewer
  // CTAs fit an SM then, against 120 one by one, all before the streaming stores.)
#pragma unroll 1
  for (int i = tid; i < count * per_token; i += kThreads) {
    const int t = (int)by(i, p.per_token), in_token = i - t * per_token;
    const int row = (int)by(in_token, p.per_row), unit = in_token - row * p.units;
    // whose row: queries, keys, values
    const int which = !APPEND || row < p.heads[0] ? 0 : row < p.heads[0] + p.heads[1] ? 1 : 2;
    const int head = which == 0 ? row : which == 1 ? row - p.heads[0] : row - p.heads[0] - p.heads[1];
    const bool turn = which != 2 && unit < p.turned;
    // the unit's two pieces; behind the turned ones they lie side by side
    const int a = turn ? (p.rotary.interleaved ? 2 * V : V) * unit : which == 2 ? 2 * V * unit : p.rotary.rot + 2 * V * (unit - p.turned);
    const int c = a + (turn ? inner : V);
    if (a >= p.d) continue;
    T *dst;
    if (which == 0) {
      dst = static_cast<T *>(p.out) + b * p.os[0] + (first + t) * p.os[1] + head * p.os[2];
    } else {
      if (t >= real || to[which - 1][t] < 0) continue;
      dst = static_cast<T *>(p.pages[which - 1]) + to[which - 1][t] + head * p.kp[which - 1][1];
    }
    P x, y;
    if (APPEND && t >= real) {  // a query behind the last: zero
#pragma unroll
      for (int e = 0; e < V; ++e) x.v[e] = y.v[e] = narrow<T>(0.f);
    } else {
      const T *src = static_cast<const T *>(p.x[which]) + b * p.xs[which][0] + (first + t) * p.xs[which][1] + head * p.xs[which][2];
      x = *reinterpret_cast<const P *>(src + a);
      if (c < p.d) y = *reinterpret_cast<const P *>(src + c);
      if (turn) {
        float f[V], g[V];  // the pairs
#pragma unroll
        for (int e = 0; e < V; ++e) {
          if (p.rotary.interleaved) {
            f[e] = widen<T>(2 * e < V ? x.v[2 * e % V] : y.v[2 * e % V]);
            g[e] = widen<T>(2 * e < V ? x.v[(2 * e + 1) % V] : y.v[(2 * e + 1) % V]);
          } else {
            f[e] = widen<T>(x.v[e]);
            g[e] = widen<T>(y.v[e]);
          }
        }
        if (V == 1 && p.rotary.interleaved) f[0] = widen<T>(x.v[0]), g[0] = widen<T>(y.v[0]);
        turn_pairs<V>(f, g, cosines + t * half + V * unit, sines + t * half + V * unit);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          if (p.rotary.interleaved && V > 1) {
            (2 * e < V ? x : y).v[2 * e % V] = narrow<T>(f[e]);
            (2 * e < V ? x : y).v[(2 * e + 1) % V] = narrow<T>(g[e]);
          } else {
            x.v[e] = narrow<T>(f[e]);
            y.v[e] = narrow<T>(g[e]);
          }
        }
      }
    }
    put(dst + a, x);
    if (c < p.d) put(dst + c, y);
  }
}

// Whether pieces of `bytes` divide everything: addresses, strides (of axes longer than one), heads and halves.
struct Fit {
  int64_t all = 0;
  void address(const void *p) { all |= (int64_t)reinterpret_cast<uintptr_t>(p); }
  void strides(const int64_t *s, const int64_t *extent, int n, int64_t size) {
    for (int i = 0; i < n; ++i)
      if (extent[i] > 1) all |= s[i] * size;
  }
  bool by(int64_t bytes) const { return (all & (bytes - 1)) == 0; }
};

int check_rotary(const char *me, int dtype, const int64_t *turns, int64_t d, int64_t rot, float magnitude) {
  if (dtype != LC_F32 && dtype != LC_F16 && dtype != LC_BF16) return fail(LC_ERR_INVALID, "%s: dtype %d is not f32, f16 or bf16", me, dtype);
  if (d < 1 || rot < 0 || rot % 2 || rot > d) return fail(LC_ERR_INVALID, "%s: %lld of %lld elements cannot turn in pairs", me, (long long)rot, (long long)d);
  if (d > kMostHead) return fail(LC_ERR_UNSUPPORTED, "%s: head size %lld is over %d", me, (long long)d, kMostHead);
  if (rot && !turns) return fail(LC_ERR_INVALID, "%s: null frequencies", me);
  if (!(magnitude > 0.f) || magnitude > 3e38f) return fail(LC_ERR_INVALID, "%s: magnitude must be positive and finite", me);
  return LC_OK;
}

// The largest pieces that fit, and the launch.
template <bool APPEND>
int launch_rotate(const char *me, int dtype, RotateParams &p, int64_t batch, const Fit &fit, cudaStream_t s) {
  const int size = dtype == LC_F32 ? 4 : 2, rot = p.rotary.rot;
  auto fits = [&](int v) {
    return fit.by((int64_t)v * size) && p.d % v == 0 && (p.rotary.interleaved ? rot % (2 * v) == 0 : rot / 2 % v == 0);
  };
  int v = 1;
  for (int x = 16 / size; x > 1 && v == 1; x /= 2)
    if (x * size >= 8 && fits(x)) v = x;
  p.turned = rot / (2 * v);
  p.units = p.turned + (p.d - rot + 2 * v - 1) / (2 * v);
  p.per_token = divisor_of((unsigned)p.rows * p.units), p.per_row = divisor_of(p.units);
  // Tokens of a CTA: eight units a thread (four: 124 us, 16: 120), but no fewer than two CTAs an SM for the sake of it.
  const int64_t all = batch * p.tokens, per_token = (int64_t)p.rows * p.units;
  int64_t tile = std::min<int64_t>(8 * kThreads / per_token, kMostTokens);
  tile = std::min<int64_t>(tile, kMostRotations / std::max(1, rot / 2));
  tile = std::max<int64_t>(1, std::min<int64_t>(tile, std::min<int64_t>(p.tokens, all / (2 * sm_count()))));
  p.tile = (int)tile;
  p.tiles = (int)((p.tokens + tile - 1) / tile);
  if (batch * p.tiles > INT32_MAX) return fail(LC_ERR_UNSUPPORTED, "%s: shape too large", me);
  const dim3 grid((unsigned)(batch * p.tiles)), block(kThreads);
  auto go = [&](auto kernel) { return check_cuda(launch_pdl(kernel, grid, block, 0, s, p), me); };
  if (dtype == LC_F32) return v == 4 ? go(rotate_kernel<float, 4, APPEND>) : v == 2 ? go(rotate_kernel<float, 2, APPEND>) : go(rotate_kernel<float, 1, APPEND>);
  if (dtype == LC_F16) return v == 8 ? go(rotate_kernel<__half, 8, APPEND>) : v == 4 ? go(rotate_kernel<__half, 4, APPEND>) : go(rotate_kernel<__half, 1, APPEND>);
  return v == 8   ? go(rotate_kernel<__nv_bfloat16, 8, APPEND>)
         : v == 4 ? go(rotate_kernel<__nv_bfloat16, 4, APPEND>)
                  : go(rotate_kernel<__nv_bfloat16, 1, APPEND>);
}

}  // namespace
}  // namespace lc

extern "C" int lc_rotate(int dtype, const void *x, void *out, const int32_t *positions, const int64_t *turns, int64_t batch,
                         int64_t tokens, int64_t heads, int64_t d, int64_t rot, int interleaved, float magnitude,
                         const int64_t *strides, void *stream) {
  using namespace lc;
  const char *me = "lc_rotate";
  if (int rc = check_rotary(me, dtype, turns, d, rot, magnitude)) return rc;
  if (batch < 0 || tokens < 0 || heads < 0) return fail(LC_ERR_INVALID, "%s: negative size", me);
  if (!strides) return fail(LC_ERR_INVALID, "%s: null strides", me);
  if (batch > INT32_MAX || tokens > INT32_MAX / 2 || heads > (1 << 22) || heads * d > (1 << 22)) return fail(LC_ERR_UNSUPPORTED, "%s: shape too large", me);
  if (batch == 0 || tokens == 0 || heads == 0) return LC_OK;
  if (!x || !out || !positions) return fail(LC_ERR_INVALID, "%s: null buffer", me);
  const int64_t size = dtype == LC_F32 ? 4 : 2, extent[3] = {batch, tokens, heads};
  if (!aligned(x, size) || !aligned(out, size)) return fail(LC_ERR_ALIGN, "%s: an element's address", me);
  RotateParams p = {};
  p.rotary = {turns, (int)rot, interleaved != 0, magnitude};
  p.x[0] = x, p.out = out, p.positions = positions;
  for (int i = 0; i < 3; ++i) p.xs[0][i] = strides[i], p.os[i] = strides[3 + i];
  p.ps[0] = strides[6], p.ps[1] = strides[7];
  p.tokens = (int)tokens, p.heads[0] = p.rows = (int)heads, p.d = (int)d;
  Fit fit;
  fit.address(x), fit.address(out);
  fit.strides(p.xs[0], extent, 3, size), fit.strides(p.os, extent, 3, size);
  return launch_rotate<false>(me, dtype, p, batch, fit, as_stream(stream));
}

extern "C" int lc_cache_append(int dtype, const void *q, const void *k, const void *v, void *out, void *k_pages, void *v_pages,
                               const int32_t *table, const int32_t *lens, const int32_t *add, const int32_t *refused,
                               const int64_t *turns, int64_t slots, int64_t most, int64_t width, int64_t pages, int64_t page_size,
                               int64_t q_heads, int64_t kv_heads, int64_t d, int64_t rot, int interleaved, float magnitude,
                               int zero_rest, const int64_t *strides, void *stream) {
  using namespace lc;
  const char *me = "lc_cache_append";
  if (int rc = check_rotary(me, dtype, turns, d, rot, magnitude)) return rc;
  if (slots < 0 || most < 0 || width < 0 || pages < 0 || page_size < 1 || q_heads < 0 || kv_heads < 1)
    return fail(LC_ERR_INVALID, "%s: negative or zero size", me);
  if (!strides) return fail(LC_ERR_INVALID, "%s: null strides", me);
  if (slots > (1 << 20) || most > (1 << 30) || pages > (1 << 30) || page_size > (1 << 20) || width > (1 << 24) ||
      width * page_size > (1ll << 30) || q_heads > (1 << 22) || kv_heads > (1 << 22) || (q_heads + 2 * kv_heads) * d > (1 << 22))
    return fail(LC_ERR_UNSUPPORTED, "%s: shape too large", me);
  if (slots == 0 || most == 0) return LC_OK;
  if (!k || !v || !lens || !add || (q_heads > 0 && (!q || !out)) || (width > 0 && !table) || (pages > 0 && (!k_pages || !v_pages)))
    return fail(LC_ERR_INVALID, "%s: null buffer", me);
  const int64_t size = dtype == LC_F32 ? 4 : 2;
  const void *addresses[6] = {q, k, v, out, k_pages, v_pages};
  RotateParams p = {};
  Fit fit;
  for (int x = 0; x < 6; ++x) {
    if (q_heads == 0 && (x == 0 || x == 3)) continue;
    if (!aligned(addresses[x], size)) return fail(LC_ERR_ALIGN, "%s: an element's address", me);
    // slot, token, head of the tensors; page, head, token of the planes
    const int64_t heads = x == 0 || x == 3 ? q_heads : kv_heads;
    const int64_t tensor[3] = {slots, most, heads}, plane[3] = {pages, kv_heads, page_size};
    fit.address(addresses[x]);
    fit.strides(strides + 3 * x, x < 4 ? tensor : plane, 3, size);
  }
  p.rotary = {turns, (int)rot, interleaved != 0, magnitude};
  p.x[0] = q, p.x[1] = k, p.x[2] = v, p.out = out, p.pages[0] = k_pages, p.pages[1] = v_pages;
  for (int i = 0; i < 3; ++i) {
    for (int x = 0; x < 3; ++x) p.xs[x][i] = strides[3 * x + i];
    p.os[i] = strides[9 + i], p.kp[0][i] = strides[12 + i], p.kp[1][i] = strides[15 + i];
  }
  p.table = table, p.lens = lens, p.add = add, p.refused = refused;
  p.width = (int)width, p.page_count = (int)pages, p.page_size = (int)page_size, p.zero_rest = zero_rest && q_heads > 0;
  p.tokens = (int)most, p.heads[0] = (int)q_heads, p.heads[1] = (int)kv_heads, p.rows = (int)(q_heads + 2 * kv_heads), p.d = (int)d;
  return launch_rotate<true>(me, dtype, p, slots, fit, as_stream(stream));
}
