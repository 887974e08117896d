// Attention of a prompt over its keys, causal, with an optional sliding window
// and a few first tokens that stay visible:
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j   over the keys j that query i sees
// (attend.cuh says which), lse_i = log sum_j exp(scale q_i . k_j).  Grouped
// heads: query head h reads key-value head h / (q_heads / kv_heads).
#include <cudaTypedefs.h>

#include <type_traits>

#include "attend.cuh"
#include "sm100.cuh"
#include "softmax.cuh"

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
// warps: what the tensor-core form does not take (head sizes over 128 or not a
// multiple of 8, odd alignments, groups of over 128 heads).
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

// ---------------------------------------------------------------- tensor-core form
// Flash attention on tcgen05, the schedule of sdpa.cu: per CTA two query tiles of
// 128 rows share every block of 128 keys; warp 0 loads (TMA), one thread of warp 1
// issues the products (S = Q K^T and O += P V, P from tensor memory), and a
// warpgroup per tile does the softmax, one row per thread.  What is different:
//   rows    a tile's 128 rows are G heads of a group x 128 / G tokens (one 5-D TMA
//           box), so a key block is loaded once for the whole group, and a tile spans
//           few tokens: the keys that two tiles see are the window plus 2 x 128 / G,
//           against the window plus 256 with one head per tile;
//   keys    an item (two tiles of one sequence and key-value head) visits the blocks
//           of the sinks and then blocks from the first key that its first token
//           sees on (a TMA box may start at any row), nothing else; only blocks that
//           cross a bound of some row are masked, by four 32-bit words per row;
//   bounds  lengths come from the device; items run longest first, so that the causal
//           triangle's tail is made of short ones;
//   values  0 x infinity is NaN, so the rows of V beyond a sequence's end are cleared
//           in shared memory, and a row whose sums come out infinite or NaN is
//           computed again key by key (it may hold a value that its mask hides).
// P is rounded to the storage type for the second product: beside the output's own
// rounding its error averages out over the keys.
using namespace sm100;
using namespace softmax;

constexpr int kRows = 128;     // of a query tile
constexpr int kTiles = 2;      // per CTA
constexpr int kKeys = 128;     // of a block
constexpr int kStages = 2;
constexpr int kThreads = 64 + kTiles * 128;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kOCol = 256;             // O of tile t at kOCol + t * DP; S of tile t at t * 128
constexpr float kRescale = 8.0f;            // log2 units a row's maximum may lag behind
constexpr int kChunkBytes = 128 * 64 * 2;   // 128 rows x 64 columns, one swizzle span

template <int DP>
struct WindowLayout {
  static constexpr int kTileBytes = DP / 64 * kChunkBytes;
  static constexpr int kQBytes = kTiles * kTileBytes;
  static constexpr int kBytes = kQBytes + kStages * 2 * kTileBytes + 1024;
};

struct TensorParams {
  int group, tokens;        // heads per key-value head, tokens of a tile
  int q_blocks, items;      // items = q_blocks x batch x kv_heads
  int k_head, k_batch, v_head, v_batch;  // 0 where the axis is broadcast (stride 0), else 1
  int o_vec;                // output rows by 32-byte (2) or 16-byte (1) stores
  int *err;
};

// One item: its tokens and the key blocks that they see.
struct Item {
  int b, hk, i0;            // first token of tile 0
  int n_q, n_kv, base;      // token i is at position base + i
  int n, n_sink, start, sinks;  // blocks; the first n_sink hold keys 0 .. sinks - 1, the others start at key `start`
};

__device__ __forceinline__ int first_seen(int p, int window) { return window == 0 ? 0 : max(0, p - window + 1); }

__device__ __forceinline__ Item item_of(const WindowParams &p, const TensorParams &t, int index) {
  Item it;
  const int heads = p.batch * p.kv_heads;
  const int qb = t.q_blocks - 1 - index / heads, bh = index % heads;
  it.b = bh / p.kv_heads;
  it.hk = bh - it.b * p.kv_heads;
  it.i0 = qb * kTiles * t.tokens;
  it.n_q = length_of(p.q_lens, it.b, p.s_q);
  it.n_kv = length_of(p.kv_lens, it.b, p.s_kv);
  it.base = it.n_kv - it.n_q;
  const int last = min(it.i0 + kTiles * t.tokens, it.n_q) - 1;  // the last token that exists
  const int p_first = max(0, it.base + it.i0), p_last = it.base + last;
  it.n = it.n_sink = it.start = 0;
  it.sinks = p.sinks;
  if (last < it.i0 || p_last < 0) return it;
  const int lo = first_seen(p_first, p.window);
  if (lo > p.sinks) {  // a gap, or nothing, between the sinks and the windows
    it.n_sink = (p.sinks + kKeys - 1) / kKeys;
    it.start = lo;
  }
  it.n = it.n_sink + (p_last + 1 - it.start + kKeys - 1) / kKeys;
  return it;
}
__device__ __forceinline__ int block_key(const Item &it, int j) {
  return j < it.n_sink ? j * kKeys : it.start + (j - it.n_sink) * kKeys;
}

// 5-D and 4-D tiled TMA loads (c0 innermost).
__device__ __forceinline__ void tma_load_5d(void *dst, const CUtensorMap *map, uint64_t *bar, int32_t c0, int32_t c1,
                                            int32_t c2, int32_t c3, int32_t c4) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tma_load_4d(void *dst, const CUtensorMap *map, uint64_t *bar, int32_t c0, int32_t c1,
                                            int32_t c2, int32_t c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Bits [lo, hi) of a 32-bit word (either bound may lie outside it).
__device__ __forceinline__ uint32_t bits_between(int lo, int hi) {
  const uint32_t below_hi = hi >= 32 ? 0xffffffffu : hi <= 0 ? 0u : (1u << hi) - 1;
  const uint32_t below_lo = lo >= 32 ? 0xffffffffu : lo <= 0 ? 0u : (1u << lo) - 1;
  return below_hi & ~below_lo;
}

template <class T>
__device__ __forceinline__ uint32_t pack16(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack16<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}

__device__ __forceinline__ void give_up(const TensorParams &t, volatile int *abort, int code) {
  *abort = 1;
  atomicCAS(t.err, 0, code);
}
// Every lane waits, and the warp agrees on the outcome.
__device__ __forceinline__ bool wait_all(uint64_t *bar, uint32_t parity, volatile int *abort, const TensorParams &t, int code) {
  const int ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, abort) ? 1 : 0);
  if (!ok && (threadIdx.x & 31) == 0) give_up(t, abort, code);
  return ok != 0;
}

// Rows of this warp (a lane each, `odd` where it holds one) whose output came out
// infinite or NaN, key by key; the columns that came out finite keep their bits.
template <class T>
__device__ __noinline__ void mend_rows(const WindowParams &p, bool odd, int b, int hk, int pos, int i, int h) {
  const int lane = threadIdx.x & 31;
  __syncwarp();
  for (unsigned left = __ballot_sync(0xffffffffu, odd); left; left &= left - 1) {
    const int from = __ffs(left) - 1;
    const int row_pos = __shfl_sync(0xffffffffu, pos, from), row_i = __shfl_sync(0xffffffffu, i, from),
              row_h = __shfl_sync(0xffffffffu, h, from);
    RowState st;
    float q[kMaxHead / 32];
    load_row(q, static_cast<const T *>(p.q) + b * p.qs[0] + row_i * p.qs[1] + row_h * p.qs[2], p.d, lane, p.scale_log2);
    const T *k0 = static_cast<const T *>(p.k) + b * p.ks[0] + hk * p.ks[2];
    const T *v0 = static_cast<const T *>(p.v) + b * p.vs[0] + hk * p.vs[2];
    auto at = [&](int j, const T *&k, const T *&v) {
      k = k0 + j * p.ks[1];
      v = v0 + j * p.vs[1];
      return true;
    };
    const Visible see = visible(row_pos, p.window, p.sinks);
    attend_keys<T>(st, q, p.d, lane, 0, see.sink_end, 1, at);
    attend_keys<T>(st, q, p.d, lane, see.lo, row_pos + 1, 1, at);
    mend_row(st, static_cast<T *>(p.o) + b * p.os[0] + row_i * p.os[1] + row_h * p.os[2], p.d, lane);
  }
}

// POLY: of sixteen pairs of exponentials, how many go to the FMA pipe.
template <class T, int DP, int POLY>
__global__ void __launch_bounds__(kThreads, 1)
    window_kernel(const __grid_constant__ CUtensorMap tma_q, const __grid_constant__ CUtensorMap tma_k,
                  const __grid_constant__ CUtensorMap tma_v, const __grid_constant__ WindowParams p,
                  const __grid_constant__ TensorParams tp) {
  using L = WindowLayout<DP>;
  constexpr int kTile = L::kTileBytes;
  constexpr bool kBf16 = sizeof(T) == 2 && !std::is_same<T, __half>::value;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t *q_s = smem;
  uint8_t *kv_s = smem + L::kQBytes;
  __shared__ __align__(8) uint64_t q_full, q_empty;
  __shared__ __align__(8) uint64_t k_full[kStages], v_full[kStages], k_empty[kStages], v_empty[kStages];
  __shared__ __align__(8) uint64_t s_full[kTiles], p_full[kTiles], o_done[kTiles], o_empty[kTiles];
  __shared__ uint32_t tmem_base;
  __shared__ int abort_flag;
  volatile int *abort = &abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(&q_full, 1);
    mbar_init(&q_empty, 1);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int t = 0; t < kTiles; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], 4);
      mbar_init(&o_done[t], 1);
      mbar_init(&o_empty[t], 4);
    }
    abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&tma_q);
    prefetch_tmap(&tma_k);
    prefetch_tmap(&tma_v);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base;
  pdl_wait();
  pdl_trigger();
  // Every barrier phase counts over all blocks of the CTA's items: block g (over all
  // items) uses stage g & 1, and s_full / p_full / o_done complete once per block.

  if (warp == 0) {
    if (lane == 0) {
      int g = 0, local = 0;
      bool ok = true;
      const uint32_t q_bytes = kTiles * DP / 64 * tp.group * tp.tokens * 128;
      for (int index = blockIdx.x; ok && index < tp.items; index += gridDim.x) {
        const Item it = item_of(p, tp, index);
        if (it.n == 0) continue;
        // Q of the previous item is free once its last S products completed
        if (local > 0 && !mbar_wait(&q_empty, (local - 1) & 1, abort)) {
          give_up(tp, abort, kErrTimeoutProducer);
          break;
        }
        ++local;
        mbar_expect_tx(&q_full, q_bytes);
        for (int t = 0; t < kTiles; ++t)
          for (int c = 0; c < DP / 64; ++c)
            tma_load_5d(q_s + t * kTile + c * kChunkBytes, &tma_q, &q_full, c * 64, 0, it.i0 + t * tp.tokens, it.hk, it.b);
        for (int j = 0; j < it.n; ++j, ++g) {
          const int st = g & 1, key = block_key(it, j);
          const uint32_t ph = (g >> 1) & 1;
          uint8_t *k_s = kv_s + st * 2 * kTile, *v_s = k_s + kTile;
          if (!mbar_wait(&k_empty[st], ph ^ 1, abort)) {
            give_up(tp, abort, kErrTimeoutProducer);
            ok = false;
            break;
          }
          mbar_expect_tx(&k_full[st], kTile);
          for (int c = 0; c < DP / 64; ++c)
            tma_load_4d(k_s + c * kChunkBytes, &tma_k, &k_full[st], c * 64, key, it.hk * tp.k_head, it.b * tp.k_batch);
          if (!mbar_wait(&v_empty[st], ph ^ 1, abort)) {
            give_up(tp, abort, kErrTimeoutProducer);
            ok = false;
            break;
          }
          mbar_expect_tx(&v_full[st], kTile);
          for (int c = 0; c < DP / 64; ++c)
            tma_load_4d(v_s + c * kChunkBytes, &tma_v, &v_full[st], c * 64, key, it.hk * tp.v_head, it.b * tp.v_batch);
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc_s = idesc_f16(kBf16, false, false, kRows, kKeys);
      constexpr uint32_t idesc_o = idesc_f16(kBf16, false, true, kRows, DP);
      const uint64_t q_desc = smem_desc_sw128(smem_u32(q_s), 16, 1024);
      const uint64_t k_desc = smem_desc_sw128(smem_u32(kv_s), 16, 1024);
      const uint64_t v_desc = smem_desc_sw128(smem_u32(kv_s) + kTile, kChunkBytes, 1024);
      constexpr uint32_t kStageStep = 2 * kTile / 16;
      auto issue_s = [&](int t, int g) {  // S_t = Q_t K(block g)^T
        const uint64_t qd = q_desc + (uint64_t)(t * kTile / 16);
        const uint64_t kd = k_desc + (uint64_t)((g & 1) * kStageStep);
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
          const uint32_t off = ((k >> 2) * kChunkBytes + (k & 3) * 32) / 16;
          mma_f16(tmem + t * kKeys, qd + off, kd + off, idesc_s, k > 0);
        }
        mma_commit(&s_full[t]);
      };
      auto issue_pv = [&](int t, int g, bool first) {  // O_t (+)= P_t V(block g), P_t over S_t
        const uint64_t vd = v_desc + (uint64_t)((g & 1) * kStageStep);
#pragma unroll
        for (int k = 0; k < kKeys / 16; ++k)
          mma_f16_tmem_a(tmem + kOCol + t * DP, tmem + t * kKeys + k * 8, vd + (uint64_t)(k * 2048 / 16), idesc_o, !(first && k == 0));
        mma_commit(&o_done[t]);
      };
      int g0 = 0, local = 0;
      bool ok = true;
      for (int index = blockIdx.x; ok && index < tp.items; index += gridDim.x) {
        const int n = item_of(p, tp, index).n;
        if (n == 0) continue;
        ok = mbar_wait(&q_full, local & 1, abort) && mbar_wait(&k_full[g0 & 1], (g0 >> 1) & 1, abort);
        if (!ok) break;
        tc_fence_after();
        for (int t = 0; t < kTiles; ++t) issue_s(t, g0);
        mma_commit(&k_empty[g0 & 1]);
        if (n == 1) mma_commit(&q_empty);
        for (int j = 0; ok && j < n; ++j) {
          const int g = g0 + j, st = g & 1;
          const uint32_t ph = (g >> 1) & 1;
          const bool next = j + 1 < n;
          for (int t = 0; t < kTiles; ++t) {
            if ((t == 0 && !mbar_wait(&v_full[st], ph, abort)) ||
                (t == 0 && next && !mbar_wait(&k_full[(g + 1) & 1], ((g + 1) >> 1) & 1, abort)) ||
                (j == 0 && local > 0 && !mbar_wait(&o_empty[t], (local - 1) & 1, abort)) ||
                !mbar_wait(&p_full[t], g & 1, abort)) {
              ok = false;
              break;
            }
            tc_fence_after();
            issue_pv(t, g, j == 0);
            if (t == kTiles - 1) mma_commit(&v_empty[st]);
            if (next) {
              issue_s(t, g + 1);
              if (t == kTiles - 1) {
                mma_commit(&k_empty[(g + 1) & 1]);
                if (j + 2 == n) mma_commit(&q_empty);  // the item's last S products
              }
            }
          }
        }
        ++local;
        g0 += n;
      }
      if (!ok) give_up(tp, abort, kErrTimeoutMma);
    }
  } else {
    const int t = (warp - 2) >> 2;  // query tile of this warpgroup
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_at = tmem + lane_base + t * kKeys, o_at = tmem + lane_base + kOCol + t * DP;
    const bool in_tile = row < tp.group * tp.tokens;
    const int token = row / tp.group, head = row - token * tp.group;
    int g0 = 0;
    bool ok = true;
    for (int index = blockIdx.x; ok && index < tp.items; index += gridDim.x) {
      const Item it = item_of(p, tp, index);
      const int i = it.i0 + t * tp.tokens + token, h = it.hk * tp.group + head;
      const int pos = it.base + i;
      const int p_low = it.base + it.i0 + t * tp.tokens, p_high = p_low + tp.tokens - 1;
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < it.n; ++j) {
        const int g = g0 + j, key = block_key(it, j);
        if (!wait_all(&s_full[t], g & 1, abort, tp, kErrTimeoutSoftmax)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t sr[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(s_at + c * 32, sr[c]);
        tmem_wait_ld();
        // the block's keys that this row sees: [from, to) and [0, sunk)
        int from, to, sunk;
        bool whole;  // every row of the tile sees every key
        if (j < it.n_sink) {
          from = to = 0;
          sunk = it.sinks - key;
          whole = sunk >= kKeys;
        } else {
          from = first_seen(pos, p.window) - key;
          to = pos + 1 - key;
          sunk = min(it.sinks - key, to);
          whole = key + kKeys - 1 <= p_low && key >= first_seen(p_high, p.window);
        }
        if (!whole) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t sees = bits_between(from - c * 32, to - c * 32) | bits_between(0, sunk - c * 32);
#pragma unroll
            for (int x = 0; x < 32; ++x)
              if (!(sees >> x & 1)) sr[c][x] = __float_as_uint(-INFINITY);
          }
        }
        if (key + kKeys > it.n_kv && it.n_kv < p.s_kv) {
          // the buffer goes on behind the sequence's end: clear those rows of V
          if (!wait_all(&v_full[g & 1], (g >> 1) & 1, abort, tp, kErrTimeoutSoftmax)) {
            ok = false;
            break;
          }
          if (key + row >= it.n_kv) {
            uint8_t *v_row = kv_s + (g & 1) * 2 * kTile + kTile + row * 128;
            for (int c = 0; c < DP / 64; ++c)
              for (int x = 0; x < 8; ++x) *reinterpret_cast<uint4 *>(v_row + c * kChunkBytes + x * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_async_shared();
        }
        // max of the raw scores, as 8 independent chains
        float mx8[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) mx8[k] = -INFINITY;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int x = 0; x < 32; x += 2)
            mx8[(x >> 1) & 7] = max3(mx8[(x >> 1) & 7], __uint_as_float(sr[c][x]), __uint_as_float(sr[c][x + 1]));
        const float mx = max3(max3(mx8[0], mx8[1], mx8[2]), max3(mx8[3], mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7])) * p.scale_log2;
        const float m_new = fmaxf(m, mx);
        const bool need = m_new > m + kRescale;
        if (__any_sync(0xffffffffu, need)) {
          const float alpha = need ? ex2(m - m_new) : 1.0f;
          if (need) {
            l *= alpha;
            m = m_new;
          }
          if (j > 0) {
            if (!wait_all(&o_done[t], (g - 1) & 1, abort, tp, kErrTimeoutCorrection)) {
              ok = false;
              break;
            }
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < DP / 16; ++c) {
              uint32_t o[16];
              tmem_ld16(o_at + c * 16, o);
              tmem_wait_ld();
#pragma unroll
              for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * alpha);
              tmem_st16(o_at + c * 16, o);
            }
            tmem_wait_st();
          }
        }
        uint64_t part2[4] = {0ull, 0ull, 0ull, 0ull};
        const uint64_t scale2 = pack2(p.scale_log2, p.scale_log2);
        const float base = m == -INFINITY ? 0.f : -m;  // nothing seen so far: all weights are 2^-inf
        const uint64_t base2 = pack2(base, base);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t packed[16];
#pragma unroll
          for (int x = 0; x < 16; ++x) {
            const uint64_t x2 = ffma2(pack2(__uint_as_float(sr[c][2 * x]), __uint_as_float(sr[c][2 * x + 1])), scale2, base2);
            uint64_t p2;
            if ((x + 1) * POLY / 16 > x * POLY / 16) {
              p2 = ex2_poly2<true>(x2);
            } else {
              const float2 xx = unpack2(x2);
              p2 = pack2(ex2(xx.x), ex2(xx.y));
            }
            part2[x & 3] = fadd2(part2[x & 3], p2);
            const float2 pp = unpack2(p2);
            packed[x] = pack16<T>(pp.x, pp.y);
          }
          tmem_st16(s_at + c * 16, packed);
        }
        tmem_wait_st();
        const float2 sum = unpack2(fadd2(fadd2(part2[0], part2[1]), fadd2(part2[2], part2[3])));
        l += sum.x + sum.y;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);
      }
      if (!ok) break;
      const bool stored = in_tile && i < p.s_q;
      const bool live = stored && i < it.n_q && pos >= 0 && m != -INFINITY;  // sees something
      T *out = static_cast<T *>(p.o) + it.b * p.os[0] + i * p.os[1] + h * p.os[2];
      if (p.lse && stored)
        p.lse[((int64_t)it.b * p.q_heads + h) * p.s_q + i] = live || isnan(l) && i < it.n_q ? (m + log2f(l)) * kLn2 : -INFINITY;
      if (it.n > 0) {
        if (!wait_all(&o_done[t], (g0 + it.n - 1) & 1, abort, tp, kErrTimeoutSoftmax)) break;
        tc_fence_after();
      }
      const bool some = live || (stored && i < it.n_q && isnan(l));
      const float inv = some ? 1.0f / l : 0.f;
      bool odd = false;
#pragma unroll 1
      for (int c = 0; c < DP / 32; ++c) {
        uint32_t o[32];
        if (it.n > 0) {
          tmem_ld32(o_at + c * 32, o);
          tmem_wait_ld();
          if (c == DP / 32 - 1) {  // O may now be overwritten by the next item's first product
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&o_empty[t]);
          }
        }
        if (stored) {
          uint32_t packed[16];
          float top = 0.f;
#pragma unroll
          for (int x = 0; x < 16; ++x) {
            const float a = some ? __uint_as_float(o[2 * x]) * inv : 0.f, b = some ? __uint_as_float(o[2 * x + 1]) * inv : 0.f;
            top = max_nan(top, max_nan(fabsf(a), fabsf(b)));
            packed[x] = pack16<T>(a, b);
          }
          odd |= !isfinite(top) && c * 32 < p.d;
          T *to = out + c * 32;
          if (tp.o_vec == 2) {
            if (c * 32 + 16 <= p.d) st_global_v8_b32(to, packed);
            if (c * 32 + 32 <= p.d) st_global_v8_b32(to + 16, packed + 8);
          } else {
#pragma unroll
            for (int x = 0; x < 4; ++x)
              if (c * 32 + x * 8 + 8 <= p.d)
                reinterpret_cast<uint4 *>(to)[x] = make_uint4(packed[4 * x], packed[4 * x + 1], packed[4 * x + 2], packed[4 * x + 3]);
          }
        }
        __syncwarp();
      }
      if (__any_sync(0xffffffffu, odd)) mend_rows<T>(p, odd, it.b, it.hk, pos, i, h);
      g0 += it.n;
    }
  }

  __syncthreads();
  if (abort_flag) drain_delay();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// ---------------------------------------------------------------- host side

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    cudaDriverEntryPointQueryResult found;
    void *ptr = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      ptr = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  }();
  return fn;
}

// A map of 16-bit elements, dims[0] contiguous; strides in elements from dims[1] on
// (an axis of one entry has any).
int make_map(CUtensorMap *map, bool bf16, const void *base, int rank, const int64_t *sizes, const int64_t *strides, const int *boxes) {
  auto fn = encode_fn();
  if (!fn) return fail(LC_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  cuuint64_t dims[5], bytes[4];
  cuuint32_t box[5], one[5];
  for (int i = 0; i < rank; ++i) {
    dims[i] = (cuuint64_t)sizes[i];
    box[i] = (cuuint32_t)boxes[i];
    one[i] = 1;
    if (i > 0) bytes[i - 1] = sizes[i] == 1 ? 16 : (cuuint64_t)strides[i] * 2;
  }
  const CUresult r = fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank, const_cast<void *>(base),
                        dims, bytes, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(LC_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return LC_OK;
}

// What the TMA loads and the row stores take: head sizes up to 128 in pieces of 8,
// a group that fits a tile, 16-byte alignment, strides that a tensor map holds (a
// broadcast batch or head of K and V becomes an axis of one).
bool window_tensor(const WindowParams &p) {
  const int group = p.q_heads / p.kv_heads;
  bool ok = p.d <= 128 && p.d % 8 == 0 && group <= kRows && p.s_kv > 0 && aligned(p.q, 16) && aligned(p.k, 16) &&
            aligned(p.v, 16) && aligned(p.o, 16);
  const int sizes[4][3] = {{p.batch, p.s_q, p.q_heads}, {p.batch, p.s_kv, p.kv_heads}, {p.batch, p.s_kv, p.kv_heads}, {p.batch, p.s_q, p.q_heads}};
  const int64_t *strides[4] = {p.qs, p.ks, p.vs, p.os};
  for (int x = 0; x < 4; ++x)
    for (int a = 0; a < 3; ++a) {
      const bool repeats = (x == 1 || x == 2) && a != 1;  // may have a stride of zero
      const int64_t s = strides[x][a];
      ok = ok && (sizes[x][a] == 1 || (s % 8 == 0 && (s > 0 || (s == 0 && repeats)) && s < (1ll << 38)));
    }
  return ok;
}

template <class T, int DP, int POLY>
int launch_window(const WindowParams &p, cudaStream_t s) {
  using L = WindowLayout<DP>;
  constexpr bool kBf16 = !std::is_same<T, __half>::value;
  auto *kernel = window_kernel<T, DP, POLY>;
  TensorParams t;
  t.group = p.q_heads / p.kv_heads;
  t.tokens = kRows / t.group;
  CUtensorMap tq, tk, tv;
  const int64_t q_sizes[5] = {p.d, t.group, p.s_q, p.kv_heads, p.batch};
  const int64_t q_strides[5] = {1, p.qs[2], p.qs[1], p.qs[2] * t.group, p.qs[0]};
  const int q_box[5] = {64, t.group, t.tokens, 1, 1};
  if (int rc = make_map(&tq, kBf16, p.q, 5, q_sizes, q_strides, q_box)) return rc;
  const int kv_box[4] = {64, kKeys, 1, 1};
  auto keys_map = [&](CUtensorMap *map, const void *base, const int64_t *st, int *head, int *batch) {
    *head = st[2] != 0;
    *batch = st[0] != 0;
    const int64_t sizes[4] = {p.d, p.s_kv, *head ? p.kv_heads : 1, *batch ? p.batch : 1};
    const int64_t strides[4] = {1, st[1], st[2], st[0]};
    return make_map(map, kBf16, base, 4, sizes, strides, kv_box);
  };
  if (int rc = keys_map(&tk, p.k, p.ks, &t.k_head, &t.k_batch)) return rc;
  if (int rc = keys_map(&tv, p.v, p.vs, &t.v_head, &t.v_batch)) return rc;
  t.q_blocks = (p.s_q + kTiles * t.tokens - 1) / (kTiles * t.tokens);
  const int64_t items = (int64_t)t.q_blocks * p.batch * p.kv_heads;
  if (items > INT32_MAX) return fail(LC_ERR_UNSUPPORTED, "lc_window_attention: shape too large");
  t.items = (int)items;
  bool by32 = aligned(p.o, 32) && p.d % 16 == 0;
  for (int a = 0; a < 3; ++a) by32 = by32 && p.os[a] % 16 == 0;
  t.o_vec = by32 ? 2 : 1;
  if (int rc = device_error_word(&t.err)) return rc;
  static bool configured[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    if (int rc = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes), "window shared memory"))
      return rc;
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  const int grid = t.items < sm_count() ? t.items : sm_count();
  return check_cuda(launch_pdl(kernel, dim3(grid), dim3(kThreads), L::kBytes, s, tq, tk, tv, p, t), "lc_window_attention");
}

template <class T>
int window_sized(const WindowParams &p, cudaStream_t s) {
  return p.d <= 64 ? launch_window<T, 64, 1>(p, s) : launch_window<T, 128, 1>(p, s);
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
  if (window_tensor(p)) return dtype == LC_F16 ? window_sized<__half>(p, s) : window_sized<__nv_bfloat16>(p, s);
  const dim3 grid((unsigned)s_q, (unsigned)q_heads, (unsigned)batch);
  if (dtype == LC_F16)
    window_row_kernel<__half><<<grid, kRowWarps * 32, 0, s>>>(p);
  else
    window_row_kernel<__nv_bfloat16><<<grid, kRowWarps * 32, 0, s>>>(p);
  return check_launch(me);
}
