// Attention of a prompt over its keys, causal, with an optional sliding window
// and a few first tokens that stay visible:
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j   over the keys j that query i sees
// (attend.cuh says which), lse_i = log sum_j exp(scale q_i . k_j).  Grouped
// heads: query head h reads key-value head h / (q_heads / kv_heads).
#include <cudaTypedefs.h>

#include <algorithm>
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
// warps: few rows of few keys, and what the tensor-core form does not take (head
// sizes over 128 or not a multiple of 8, odd alignments, groups of over 128 heads).
constexpr int kRowWarps = 4;

template <class T, int NC>
__global__ void __launch_bounds__(kRowWarps * 32) window_row_kernel(WindowParams p) {
  __shared__ float scratch[kRowWarps * (32 * NC + 2)];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int i = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int hk = h / (p.q_heads / p.kv_heads);
  const int n_q = length_of(p.q_lens, b, p.s_q), n_kv = length_of(p.kv_lens, b, p.s_kv);
  const int pos = n_kv - n_q + i;
  RowState<NC> st;
  if (i < n_q && pos >= 0) {
    float q[NC];
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
// Attention with a running softmax on tcgen05, the schedule of sdpa.cu: per CTA two query tiles of
// 128 rows share every block of 128 keys; warp 0 loads (TMA), one thread of warp 1
// issues the products (S = Q K^T and O += P V, P from tensor memory), a warpgroup per
// tile does the softmax, one row per thread.  Under a window an item is only a few
// blocks long, so its end must not stop the others: warp 2 works out the coming items
// and leaves them in a ring, and a fourth warpgroup divides and stores the finished
// tiles while the softmax is at the next item.  What else is different:
//   rows    a tile's 128 rows are G heads of a group x 128 / G tokens (one 5-D TMA
//           box), so a key block is loaded once for the whole group, and a tile spans
//           few tokens: the keys that two tiles see are the window plus 2 x 128 / G,
//           against the window plus 256 with one head per tile;
//   keys    an item (two tiles of one sequence and key-value head) visits the blocks
//           of the sinks and then blocks from the first key that its first token
//           sees on (a TMA box may start at any row), nothing else; where the last of
//           them is half empty, its second half takes the sinks instead; only blocks
//           that cross a bound of some row are masked, by four 32-bit words per row;
//   cuts    lengths come from the device.  With many items each CTA takes every
//           gridDim-th one, longest first, so that the causal triangle's tail is made
//           of short ones.  With few, or ragged ones, all items' blocks are laid end to
//           end and each CTA takes an equal run of them: of whole items where that is
//           nearly as even, else cut anywhere; then what a run holds of an item without
//           holding it all goes to the workspace in f32, and join_kernel adds it up in
//           CTA order;
//   values  0 x infinity is NaN, so the rows of V beyond a sequence's end are cleared
//           in shared memory, and a row whose sums come out infinite or NaN is
//           computed again key by key (it may hold a value that its mask hides).
// P is rounded to the storage type for the second product: an error of the size of the
// output's own rounding (and kLift's, where a row's weights are many and small).
// Bound by a tile's chain of softmax and products (3500 cycles a block of 128 keys, of
// which the tensor pipe needs 2080 for both tiles), in long runs by the power cap.
// Measured, f16, 32/8 heads of 128: 32768 tokens, window 4096: 1.77 ms, 1170 TFLOP/s;
// bf16, 4 ragged chunks of up to 777 over 4001 keys, window 1024: 51 us, 685 TFLOP/s.
using namespace sm100;
using namespace softmax;

constexpr int kRows = 128;     // of a query tile
constexpr int kTiles = 2;      // per CTA
constexpr int kKeys = 128;     // of a block
constexpr int kStages = 2;
constexpr int kMinRun = 6;     // units of a run: a shorter one costs more to join than it saves
// Units that cutting costs: few items (deep: 64 queries of 8 key-value heads over 1024 keys,
// 4 units saved: 20.8 us whole, 23.3 cut; over 1500, 8 saved: 28.0, 23.6) or shares of the
// first and last item of every CTA (2 x 2048 tokens, 9 saved: 83, 92; 4096, 13: 148, 140);
// and what whole items may take beyond a CTA's share before the kernel cuts them.
constexpr int kDeepCut = 6, kWideCut = 11, kDeepSlack = 3, kWideSlack = 5;
constexpr int kMostCtas = 256;
constexpr int kMaxCutItems = 2048;
constexpr int kSpansSlot = 43, kSumsSlot = 44, kStatsSlot = 45;  // scratch_buffer slots
constexpr int kThreads = 128 + kTiles * 128 + 128;  // loads and products, softmax, output
// Registers per thread after the split: the softmax warpgroups' rows of 128 scores
// need more than the 128 that 512 threads are launched with, the others less;
// 72 x 256 + 184 x 256 = 128 x 512.
constexpr int kLaunchRegs = 128, kFewRegs = 72, kManyRegs = 184;
constexpr int kLensHeld = 256;  // sequences whose lengths are kept in shared memory
constexpr int kRing = 4;        // pieces of work known ahead
constexpr int kReaders = 2 + 8 + 4;  // of a piece: loads, products, the softmax's and the output's warps
constexpr uint32_t kTmemCols = 512;
// Tensor memory: S of tile t at t * 128, P over it, O of tile t at kOCol + t * DP.  (P of its
// own, which a head size of 64 has room for, takes the products off the softmax's chain and
// was slower, 8 x 4096 tokens of 16 heads: 590 against 483 us: both tiles' exponentials then
// run at once.)
constexpr uint32_t kOCol = 256;
constexpr float kRescale = 8.0f;            // log2 units a row's maximum may lag behind
// A row's reference is its maximum less kLift, so that with the lag f16 weights reach 2^15 (its
// largest number is just under 2^16).  They end at 2^-25, and a row's largest weight is 2^7 or more:
// what is lost is 2^-32 of it a key, 2^-25 without the lift.  bf16 has f32's range, and is kept down.
template <class T>
constexpr float kLift = kLiftBf16;
template <>
constexpr float kLift<__half> = 7.f;
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
  // runs of blocks (cut): the item that began in a CTA and goes on after it, or -1, and that
  // item's last CTA; a CTA's shares of the item that began before it, and of that one
  int cut, deep, ctas;
  int2 *spans;
  float *sums;              // [CTA][2][tile][DP / 8][row][8]: 8 columns of a warp's rows lie together
  float2 *stats;            // [CTA][2][tile][row]: m and l
};

// One item: its tokens and the key blocks that they see.
struct Item {
  int b, hk, i0;            // first token of tile 0
  int n_q, n_kv, base;      // token i is at position base + i
  int n, n_sink, start, sinks;  // blocks; the first n_sink hold keys 0 .. sinks - 1, the others start at key `start`
  bool sink_half;               // the last block's rows from 64 on hold the keys from 0 on
};

__device__ __forceinline__ int first_seen(int p, int window) { return window == 0 ? 0 : max(0, p - window + 1); }

// The lengths, from shared memory where they fit.
struct Lens {
  const int *q, *kv;
};

__device__ __forceinline__ Item item_of(const WindowParams &p, const TensorParams &t, const Lens &lens, int index) {
  Item it;
  const int heads = p.batch * p.kv_heads;
  const int qb = t.q_blocks - 1 - index / heads, bh = index % heads;
  it.b = bh / p.kv_heads;
  it.hk = bh - it.b * p.kv_heads;
  it.i0 = qb * kTiles * t.tokens;
  it.n_q = length_of(lens.q, it.b, p.s_q);
  it.n_kv = length_of(lens.kv, it.b, p.s_kv);
  it.base = it.n_kv - it.n_q;
  const int last = min(it.i0 + kTiles * t.tokens, it.n_q) - 1;  // the last token that exists
  const int p_first = max(0, it.base + it.i0), p_last = it.base + last;
  it.n = it.n_sink = it.start = 0;
  it.sinks = p.sinks;
  it.sink_half = false;
  if (last < it.i0 || p_last < 0) return it;
  const int lo = first_seen(p_first, p.window);
  int keys = p_last + 1;
  if (lo > p.sinks) {  // a gap, or nothing, between the sinks and the windows
    it.start = lo;
    keys -= lo;
    const int rest = keys % kKeys;
    it.sink_half = p.sinks > 0 && p.sinks <= kKeys / 2 && rest > 0 && rest <= kKeys / 2;
    it.n_sink = it.sink_half ? 0 : (p.sinks + kKeys - 1) / kKeys;
  }
  it.n = it.n_sink + (keys + kKeys - 1) / kKeys;
  return it;
}
__device__ __forceinline__ int block_key(const Item &it, int j) {
  return j < it.n_sink ? j * kKeys : it.start + (j - it.n_sink) * kKeys;
}

// What a CTA works on: blocks [j0, j1) of an item after the other.  A run is measured
// in units of a block's time; beginning and ending an item costs some more of them,
// which count as lying before its first block.
constexpr int kItemUnits = 2;
__host__ __device__ __forceinline__ int units_of(int blocks) { return blocks > 0 ? blocks + kItemUnits : 0; }

struct Piece {
  Item it;
  int index, j0, j1;
};
struct Pieces {
  int index, skip, left;  // skip: units of the first item that lie before the run; left: the run's units (cut)
  __device__ __forceinline__ bool next(const WindowParams &p, const TensorParams &t, const Lens &lens, Piece &out) {
    for (;;) {
      if (index >= t.items || (t.cut && left <= 0)) return false;
      out.it = item_of(p, t, lens, index);
      out.index = index;
      out.j0 = 0;
      out.j1 = out.it.n;
      index += t.cut ? 1 : gridDim.x;
      if (t.cut) {
        const int end = min(units_of(out.it.n), skip + left);
        out.j0 = max(0, skip - kItemUnits);
        out.j1 = max(0, end - kItemUnits);
        left -= end - skip;
        skip = 0;
      }
      if (out.j1 > out.j0) return true;
    }
  }
};

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
template <class T, int NC>
__device__ __noinline__ void mend_rows(const WindowParams &p, bool odd, int b, int hk, int pos, int i, int h) {
  const int lane = threadIdx.x & 31;
  __syncwarp();
  for (unsigned left = __ballot_sync(0xffffffffu, odd); left; left &= left - 1) {
    const int from = __ffs(left) - 1;
    const int row_pos = __shfl_sync(0xffffffffu, pos, from), row_i = __shfl_sync(0xffffffffu, i, from),
              row_h = __shfl_sync(0xffffffffu, h, from);
    RowState<NC> st;
    float q[NC];
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

// The rows of a finished item, a lane each (row 0 .. 255 of its two tiles).
template <class T, int NC>
__device__ __noinline__ void mend_piece(const WindowParams &p, const TensorParams &tp, const Item &it, int tile_row) {
  const int t = tile_row / kRows, row = tile_row % kRows;
  const int token = row / tp.group, h = it.hk * tp.group + row - token * tp.group;
  const int i = it.i0 + t * tp.tokens + token, pos = it.base + i;
  bool odd = false;
  if (row < tp.group * tp.tokens && i < it.n_q && pos >= 0) {
    const T *out = static_cast<const T *>(p.o) + it.b * p.os[0] + i * p.os[1] + h * p.os[2];
    for (int c = 0; c < p.d; ++c) odd |= !isfinite(Elem<T>::to_float(out[c]));
  }
  __syncwarp();
  if (__any_sync(0xffffffffu, odd)) mend_rows<T, NC>(p, odd, it.b, it.hk, pos, i, h);
}

template <class T, int DP>
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
  __shared__ __align__(8) uint64_t s_full[kTiles], p_half[kTiles], p_full[kTiles], o_done[kTiles], o_empty[kTiles], stat_full[kTiles];
  __shared__ float2 stat[kTiles][kRows];  // m and l of a tile's rows, from the softmax to the output warps
  __shared__ int held_lens[2][kLensHeld];
  __shared__ uint32_t tmem_base;
  __shared__ int abort_flag, any_odd;
  __shared__ int warp_blocks[kThreads / 32];
  __shared__ Pieces run;
  __shared__ int run_end, run_total, run_ctas, first_item;
  __shared__ int load[kMostCtas];  // units of each CTA, with whole items
  __shared__ Piece ring[kRing];
  __shared__ __align__(8) uint64_t piece_full[kRing], piece_empty[kRing];
  volatile int *abort = &abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int r = 0; r < kRing; ++r) {
      mbar_init(&piece_full[r], 1);
      mbar_init(&piece_empty[r], kReaders);
    }
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
      mbar_init(&p_half[t], 4);
      mbar_init(&p_full[t], 4);
      mbar_init(&o_done[t], 1);
      mbar_init(&o_empty[t], 4);
      mbar_init(&stat_full[t], 4);
    }
    abort_flag = 0;
    any_odd = 0;
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
  Lens lens = {p.q_lens, p.kv_lens};
  if (p.batch <= kLensHeld && (lens.q || lens.kv)) {
    for (int b = threadIdx.x; b < p.batch; b += kThreads) {
      held_lens[0][b] = length_of(p.q_lens, b, p.s_q);
      held_lens[1][b] = length_of(p.kv_lens, b, p.s_kv);
    }
    lens = {held_lens[0], held_lens[1]};
    __syncthreads();
  }
  if (!tp.cut) {
    if (threadIdx.x == 0) run = {(int)blockIdx.x, 0, 0};
  } else {
    // this CTA's run: unit blockIdx.x * total / ctas of all items' units on
    constexpr int kPer = kMaxCutItems / kThreads;  // a thread's items, or fewer
    const int per = (tp.items + kThreads - 1) / kThreads, first = threadIdx.x * per;
    int units[kPer], own = 0;
#pragma unroll
    for (int x = 0; x < kPer; ++x) {
      units[x] = x < per && first + x < tp.items ? units_of(item_of(p, tp, lens, first + x).n) : 0;
      own += units[x];
    }
    int inc = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    if (lane == 31) warp_blocks[warp] = inc;
    for (int i = threadIdx.x; i < (int)gridDim.x; i += kThreads) load[i] = 0;
    if (threadIdx.x == 0) {
      run = {tp.items, 0, 0};
      first_item = tp.items;
    }
    __syncthreads();
    int before = inc - own, total = 0;
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) before += warp_blocks[w];
      total += warp_blocks[w];
    }
    const int ctas = min((int)gridDim.x, (total + kMinRun - 1) / kMinRun);
    // Whole items, each in the run that its middle falls in, where no CTA gets much more than
    // its share by that: shares of items are 128 KB a tile to write and to read again.
    int at = before;
#pragma unroll
    for (int x = 0; x < kPer; ++x) {
      if (units[x] > 0) {
        const int cta = (int)((int64_t)(at + units[x] / 2) * ctas / total);
        atomicAdd(load + cta, units[x]);
        if (cta == (int)blockIdx.x) atomicMin(&first_item, first + x);
      }
      at += units[x];
    }
    __syncthreads();
    int heaviest = 0;
    for (int i = threadIdx.x; i < ctas; i += kThreads) heaviest = max(heaviest, load[i]);
    const bool whole = !__syncthreads_or(heaviest > total / max(1, ctas) + (tp.deep ? kDeepSlack : kWideSlack));
    const int begin = ctas ? (int)((int64_t)blockIdx.x * total / ctas) : 0;
    const int end = ctas ? (int)((int64_t)(blockIdx.x + 1) * total / ctas) : 0;
    if (whole) {
      if (threadIdx.x == 0 && (int)blockIdx.x < ctas && load[blockIdx.x] > 0) run = {first_item, 0, load[blockIdx.x]};
    } else if ((int)blockIdx.x < ctas && begin >= before && begin < before + own) {
      at = before;
#pragma unroll
      for (int x = 0; x < kPer; ++x) {
        if (begin >= at && begin < at + units[x]) run = {first + x, begin - at, end - begin};
        at += units[x];
      }
    }
    if (threadIdx.x == 0) {
      run_end = end;
      run_total = total;
      run_ctas = ctas;
      tp.spans[blockIdx.x] = make_int2(-1, -1);
    }
  }
  __syncthreads();
  // Every barrier phase counts over all blocks of the CTA's items: block g (over all
  // items) uses stage g & 1, and s_full / p_full / o_done complete once per block.

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegs));
    if (warp == 2 && lane == 0) {
      Pieces pieces = run;
      Piece piece;
      for (int k = 0;; ++k) {
        const int r = k % kRing;
        const bool more = pieces.next(p, tp, lens, piece);
        if (!more) piece.j0 = piece.j1 = 0;  // the end
        if (k >= kRing && !mbar_wait(&piece_empty[r], (k / kRing - 1) & 1, abort)) {
          give_up(tp, abort, kErrTimeoutProducer);
          break;
        }
        ring[r] = piece;
        mbar_arrive(&piece_full[r]);
        if (!more) break;
      }
    } else if (warp == 0 && lane == 0) {
      int g = 0, local = 0;
      bool ok = true;
      const uint32_t q_bytes = kTiles * DP / 64 * tp.group * tp.tokens * 128;
      while (ok) {
        const int r = local % kRing;
        if (!mbar_wait(&piece_full[r], local / kRing & 1, abort)) {
          give_up(tp, abort, kErrTimeoutProducer);
          break;
        }
        const Piece piece = ring[r];
        const Item &it = piece.it;
        mbar_arrive(&piece_empty[r]);
        if (piece.j1 == 0) break;
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
        for (int j = piece.j0; j < piece.j1; ++j, ++g) {
          const int st = g & 1, key = block_key(it, j);
          const int half_key = it.sink_half && j + 1 == it.n ? 0 : key + kKeys / 2;
          const uint32_t ph = (g >> 1) & 1;
          uint8_t *k_s = kv_s + st * 2 * kTile, *v_s = k_s + kTile;
          if (!mbar_wait(&k_empty[st], ph ^ 1, abort)) {
            give_up(tp, abort, kErrTimeoutProducer);
            ok = false;
            break;
          }
          mbar_expect_tx(&k_full[st], kTile);
          for (int c = 0; c < DP / 64; ++c) {
            tma_load_4d(k_s + c * kChunkBytes, &tma_k, &k_full[st], c * 64, key, it.hk * tp.k_head, it.b * tp.k_batch);
            tma_load_4d(k_s + c * kChunkBytes + kChunkBytes / 2, &tma_k, &k_full[st], c * 64, half_key, it.hk * tp.k_head, it.b * tp.k_batch);
          }
          if (!mbar_wait(&v_empty[st], ph ^ 1, abort)) {
            give_up(tp, abort, kErrTimeoutProducer);
            ok = false;
            break;
          }
          mbar_expect_tx(&v_full[st], kTile);
          for (int c = 0; c < DP / 64; ++c) {
            tma_load_4d(v_s + c * kChunkBytes, &tma_v, &v_full[st], c * 64, key, it.hk * tp.v_head, it.b * tp.v_batch);
            tma_load_4d(v_s + c * kChunkBytes + kChunkBytes / 2, &tma_v, &v_full[st], c * 64, half_key, it.hk * tp.v_head, it.b * tp.v_batch);
          }
        }
      }
    } else if (warp == 1) {
      const uint32_t leader = elect_one();
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
          warp_mma(leader, tmem + t * kKeys, qd + off, kd + off, idesc_s, k > 0);
        }
        warp_commit(leader, &s_full[t]);
      };
      auto issue_pv = [&](int t, int g, bool first, int half) {  // O_t (+)= P_t V(block g), P_t over S_t
        const uint64_t vd = v_desc + (uint64_t)((g & 1) * kStageStep);
#pragma unroll
        for (int k = half * kKeys / 32; k < (half + 1) * kKeys / 32; ++k)
          warp_mma_tmem_a(leader, tmem + kOCol + t * DP, tmem + t * kKeys + k * 8, vd + (uint64_t)(k * 2048 / 16), idesc_o, !(first && k == 0));
        if (half) warp_commit(leader, &o_done[t]);
      };
      // PV_0(g), S_0(g + 1), PV_1(g), S_1(g + 1): block g + 1 may be the next piece's first.
      bool ok = true;
      auto blocks = [&](int k) {  // of the k-th piece; 0: there is none
        if (!mbar_wait(&piece_full[k % kRing], k / kRing & 1, abort)) {
          ok = false;
          return 0;
        }
        return ring[k % kRing].j1 - ring[k % kRing].j0;
      };
      auto leave = [&](int k) {  // its entry may be overwritten
        __syncwarp();
        if (lane == 0) mbar_arrive(&piece_empty[k % kRing]);
      };
      auto products_pv = [&](int t, int g, bool first, int piece) {  // once P_t(g), V(g) and O_t are there
        if (!mbar_wait(&v_full[g & 1], (g >> 1) & 1, abort) ||
            (first && piece > 0 && !mbar_wait(&o_empty[t], (piece - 1) & 1, abort)) || !mbar_wait(&p_half[t], g & 1, abort))
          return false;
        tc_fence_after();
        issue_pv(t, g, first, 0);
        if (!mbar_wait(&p_full[t], g & 1, abort)) return false;
        tc_fence_after();
        issue_pv(t, g, false, 1);
        if (t == kTiles - 1) warp_commit(leader, &v_empty[g & 1]);
        return true;
      };
      const int n_first = blocks(0);
      if (n_first > 0) {
        ok = mbar_wait(&q_full, 0, abort) && mbar_wait(&k_full[0], 0, abort);
        if (ok) {
          tc_fence_after();
          for (int t = 0; t < kTiles; ++t) issue_s(t, 0);
          warp_commit(leader, &k_empty[0]);
          if (n_first == 1) warp_commit(leader, &q_empty);
        }
      }
      struct Place {
        int k, j, n;  // block j of the n blocks of piece k; n = 0: there is none
      };
      auto after = [&](const Place &a) { return a.j + 1 < a.n ? Place{a.k, a.j + 1, a.n} : Place{a.k + 1, 0, blocks(a.k + 1)}; };
      auto products_s = [&](int t, int g, const Place &a) {
        if ((t == 0 && a.j == 0 && !mbar_wait(&q_full, a.k & 1, abort)) || (t == 0 && !mbar_wait(&k_full[g & 1], (g >> 1) & 1, abort)))
          return false;
        tc_fence_after();
        issue_s(t, g);
        if (t == kTiles - 1) {
          warp_commit(leader, &k_empty[g & 1]);
          if (a.j + 1 == a.n) warp_commit(leader, &q_empty);  // a piece's last S products
        }
        return true;
      };
      Place now = {0, 0, n_first};
      for (int g = 0; ok && now.n > 0; ++g) {
        const Place next = after(now);
        const bool more = next.n > 0;
        if (!ok) break;
        for (int t = 0; ok && t < kTiles; ++t) ok = products_pv(t, g, now.j == 0, now.k) && (!more || products_s(t, g + 1, next));
        if (now.j + 1 == now.n) leave(now.k);
        now = next;
      }
      if (!ok && lane == 0) give_up(tp, abort, kErrTimeoutMma);
    }
  } else if (warp < 12) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManyRegs));
    const int t = (warp - 4) >> 2;  // query tile of this warpgroup
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_at = tmem + lane_base + t * kKeys, o_at = tmem + lane_base + kOCol + t * DP;
    const int token = row / tp.group;
    int g0 = 0, local = 0;
    bool ok = true;
    while (ok) {
      if (!wait_all(&piece_full[local % kRing], local / kRing & 1, abort, tp, kErrTimeoutSoftmax)) break;
      const Piece piece = ring[local % kRing];
      const Item &it = piece.it;
      const int n = piece.j1 - piece.j0;
      __syncwarp();
      if (lane == 0) mbar_arrive(&piece_empty[local % kRing]);
      if (n == 0) break;
      const int pos = it.base + it.i0 + t * tp.tokens + token;
      const int p_low = it.base + it.i0 + t * tp.tokens, p_high = p_low + tp.tokens - 1;
      float m = -INFINITY, l = 0.f;
      for (int x = 0; x < n; ++x) {
        const int g = g0 + x, j = piece.j0 + x, key = block_key(it, j);
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
        const bool sink_half = it.sink_half && j + 1 == it.n;
        int sunk_from = 0;
        if (sink_half) {  // keys 0 .. sinks - 1 are rows 64 on
          whole = false;
          to = min(to, kKeys / 2);
          sunk_from = kKeys / 2;
          sunk = kKeys / 2 + it.sinks;
        }
        if (!wait_all(&s_full[t], g & 1, abort, tp, kErrTimeoutSoftmax)) {
          ok = false;
          break;
        }
        tc_fence_after();
        // The row's scores, the second half's load under the first half's mask and maximum
        // (of the raw scores, as 8 independent chains).
        uint32_t sr[4][32];
        float mx8[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) mx8[k] = -INFINITY;
        tmem_ld32(s_at, sr[0]);
        tmem_ld32(s_at + 32, sr[1]);
        tmem_wait_ld();
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (half == 0) {
            tmem_ld32(s_at + 64, sr[2]);
            tmem_ld32(s_at + 96, sr[3]);
          } else {
            tmem_wait_ld();
          }
#pragma unroll
          for (int c = half * 2; c < half * 2 + 2; ++c) {
            if (!whole) {
              const uint32_t sees = bits_between(from - c * 32, to - c * 32) | bits_between(sunk_from - c * 32, sunk - c * 32);
              if (sees != 0xffffffffu) {
#pragma unroll
                for (int y = 0; y < 32; ++y)
                  if (!(sees >> y & 1)) sr[c][y] = __float_as_uint(-INFINITY);
              }
            }
#pragma unroll
            for (int y = 0; y < 32; y += 2)
              mx8[(y >> 1) & 7] = max3(mx8[(y >> 1) & 7], __uint_as_float(sr[c][y]), __uint_as_float(sr[c][y + 1]));
          }
        }
        if (key + kKeys > it.n_kv && it.n_kv < p.s_kv) {
          // the buffer goes on behind the sequence's end: clear those rows of V
          if (!wait_all(&v_full[g & 1], (g >> 1) & 1, abort, tp, kErrTimeoutSoftmax)) {
            ok = false;
            break;
          }
          if ((sink_half && row >= kKeys / 2 ? row - kKeys / 2 : key + row) >= it.n_kv) {
            uint8_t *v_row = kv_s + (g & 1) * 2 * kTile + kTile + row * 128;
            for (int c = 0; c < DP / 64; ++c)
              for (int y = 0; y < 8; ++y) *reinterpret_cast<uint4 *>(v_row + c * kChunkBytes + y * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_async_shared();
        }
        const float mx = max3(max3(mx8[0], mx8[1], mx8[2]), max3(mx8[3], mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7])) * p.scale_log2;
        const float m_new = fmaxf(m, mx - kLift<T>);
        const bool need = m_new > m + kRescale;
        if (__any_sync(0xffffffffu, need)) {
          const float alpha = need ? ex2(m - m_new) : 1.0f;
          if (need) {
            l *= alpha;
            m = m_new;
          }
          if (x > 0) {
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
              for (int y = 0; y < 16; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * alpha);
              tmem_st16(o_at + c * 16, o);
            }
            tmem_wait_st();
          }
        }
        // All exponentials on the MUFU unit: one pair in sixteen on the FMA pipe, as in sdpa.cu,
        // measured the same, one in eight 3% slower.
        uint64_t part2[4] = {0ull, 0ull, 0ull, 0ull};
        const uint64_t scale2 = pack2(p.scale_log2, p.scale_log2);
        const float base = m == -INFINITY ? 0.f : -m;  // nothing seen so far: all weights are 2^-inf
        const uint64_t base2 = pack2(base, base);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t packed[16];
#pragma unroll
          for (int y = 0; y < 16; ++y) {
            const uint64_t x2 = ffma2(pack2(__uint_as_float(sr[c][2 * y]), __uint_as_float(sr[c][2 * y + 1])), scale2, base2);
            const float2 xx = unpack2(x2);
            const uint64_t p2 = pack2(ex2(xx.x), ex2(xx.y));
            part2[y & 3] = fadd2(part2[y & 3], p2);
            const float2 pp = unpack2(p2);
            packed[y] = pack16<T>(pp.x, pp.y);
          }
          if (c == 2) {  // the first half of P was stored some time ago: its products may begin
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_half[t]);
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
      // the output warps have read the piece before's
      if (local > 0 && !wait_all(&o_empty[t], (local - 1) & 1, abort, tp, kErrTimeoutSoftmax)) break;
      stat[t][row] = make_float2(m, l);
      __syncwarp();
      if (lane == 0) mbar_arrive(&stat_full[t]);
      ++local;
      g0 += n;
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegs));
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const bool in_tile = row < tp.group * tp.tokens;
    const int token = row / tp.group, head = row - token * tp.group;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    int g0 = 0, local = 0;
    bool ok = true;
    // items that see nothing: zeros
    for (int index = blockIdx.x; index < tp.items; index += gridDim.x) {
      const Item it = item_of(p, tp, lens, index);
      if (it.n > 0 || !in_tile) continue;
      for (int t = 0; t < kTiles; ++t) {
        const int i = it.i0 + t * tp.tokens + token, h = it.hk * tp.group + head;
        if (i >= p.s_q) continue;
        T *out = static_cast<T *>(p.o) + it.b * p.os[0] + i * p.os[1] + h * p.os[2];
        for (int c = 0; c < p.d; c += 8) *reinterpret_cast<uint4 *>(out + c) = make_uint4(0, 0, 0, 0);
        if (p.lse) p.lse[((int64_t)it.b * p.q_heads + h) * p.s_q + i] = -INFINITY;
      }
    }
    __syncwarp();
    while (ok) {
      if (!wait_all(&piece_full[local % kRing], local / kRing & 1, abort, tp, kErrTimeoutEpilogue)) break;
      const Piece piece = ring[local % kRing];
      const Item &it = piece.it;
      const int n = piece.j1 - piece.j0;
      __syncwarp();
      if (lane == 0) mbar_arrive(&piece_empty[local % kRing]);
      if (n == 0) break;
      for (int t = 0; t < kTiles; ++t) {
        const uint32_t o_at = tmem + lane_base + kOCol + t * DP;
        const int i = it.i0 + t * tp.tokens + token, h = it.hk * tp.group + head;
        if (!wait_all(&stat_full[t], local & 1, abort, tp, kErrTimeoutEpilogue)) {
          ok = false;
          break;
        }
        const float m = stat[t][row].x, l = stat[t][row].y;
        const bool stored = in_tile && i < p.s_q;
        // sees something (a row of NaN scores has no maximum)
        const bool some = stored && i < it.n_q && it.base + i >= 0 && (m != -INFINITY || isnan(l));
        const float inv = some ? 1.0f / l : 0.f;
        const uint64_t inv2 = pack2(inv, inv);
        T *out = static_cast<T *>(p.o) + it.b * p.os[0] + i * p.os[1] + h * p.os[2];
        if (p.lse && stored && n == it.n)
          p.lse[((int64_t)it.b * p.q_heads + h) * p.s_q + i] = some ? lse_of<(int)kLift<T>>(m, l) : -INFINITY;
        if (!wait_all(&o_done[t], (g0 + n - 1) & 1, abort, tp, kErrTimeoutEpilogue)) {
          ok = false;
          break;
        }
        tc_fence_after();
        auto release = [&]() {  // O and the tile's m and l are read
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&o_empty[t]);
        };
        if (n < it.n) {  // a share of the item: unnormalised, for join_kernel
          const int64_t at = (((int64_t)blockIdx.x * 2 + (piece.j0 == 0)) * kTiles + t) * kRows + row;
          tp.stats[at] = make_float2(m, l);
          if (piece.j0 == 0 && t == 0 && row == 0) {  // the run's last piece: it goes on in the next CTA's
            const int64_t last_unit = run_end - (piece.j1 + kItemUnits) + units_of(it.n);
            tp.spans[blockIdx.x] = make_int2(piece.index, (int)((last_unit * run_ctas - 1) / run_total));
          }
#pragma unroll 1
          for (int c = 0; c < DP / 32; ++c) {
            uint32_t o[32];
            tmem_ld32(o_at + c * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int y = 0; y < 4; ++y) st_global_v8_b32(tp.sums + (at - row) * DP + ((c * 4 + y) * kRows + row) * 8, o + y * 8);
            __syncwarp();
          }
          release();
        } else {
          // 16 columns at a time, the next ones' load under this ones' division and store
          uint64_t zero[2] = {0ull, 0ull};  // NaN once a value is infinite or NaN
          uint32_t o[2][16];
          tmem_ld16(o_at, o[0]);
#pragma unroll
          for (int c = 0; c < DP / 16; ++c) {
            tmem_wait_ld();
            if (c + 1 < DP / 16) {
              tmem_ld16(o_at + (c + 1) * 16, o[(c + 1) & 1]);
            } else {
              release();
            }
            if (stored) {
              uint32_t packed[8];
#pragma unroll
              for (int x = 0; x < 8; ++x) {
                const uint64_t two = ffma2(pack2(__uint_as_float(o[c & 1][2 * x]), __uint_as_float(o[c & 1][2 * x + 1])), inv2, 0ull);
                zero[x & 1] = ffma2(two, 0ull, zero[x & 1]);
                const float2 ab = unpack2(two);
                packed[x] = some ? pack16<T>(ab.x, ab.y) : 0u;
              }
              T *to = out + c * 16;
              if (tp.o_vec == 2) {
                if (c * 16 < p.d) st_global_v8_b32(to, packed);
              } else {
#pragma unroll
                for (int x = 0; x < 2; ++x)
                  if (c * 16 + x * 8 < p.d)
                    reinterpret_cast<uint4 *>(to)[x] = make_uint4(packed[4 * x], packed[4 * x + 1], packed[4 * x + 2], packed[4 * x + 3]);
              }
            }
          }
          const float2 z = unpack2(fadd2(zero[0], zero[1]));
          if (some && !(z.x + z.y == 0.f)) any_odd = 1;
        }
      }
      ++local;
      g0 += n;
    }
  }

  __syncthreads();
  if (abort_flag) drain_delay();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
  if (any_odd && !abort_flag) {
    // Some row of some whole item holds an infinite or NaN output (a rare case: it is not
    // kept which): look at all of them.
    if (warp >= 4 && warp < 12)
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLaunchRegs));
    else
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kLaunchRegs));
    Pieces pieces = run;
    Piece piece;
    while (pieces.next(p, tp, lens, piece)) {
      if (piece.j1 - piece.j0 < piece.it.n) continue;
      for (int first = warp * 32; first < kTiles * kRows; first += kThreads)
        mend_piece<T, DP / 32>(p, tp, piece.it, first + lane);
    }
  }
}

// Adds up the items that several CTAs share.  A warp takes 8 rows, four lanes each, so
// that a load instruction reads 256 bytes together and a part's 16 of them are in
// flight at once.  DEEP (few items, many parts of each): the CTA's warps share 8 rows
// and deal the parts among themselves; blockIdx.x counts the shared items.  Else each
// warp has rows of its own, and blockIdx.x is the CTA that an item began in; most find
// nothing and leave.  19 parts of 8 items: 5 us against 16 us with rows of its own.
template <class T, int DP, bool DEEP>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ WindowParams p, const __grid_constant__ TensorParams tp) {
  constexpr int kSums = DEEP ? 8 : 1;
  __shared__ float warp_m[kSums][32], warp_l[kSums][32];
  __shared__ float2 warp_o[kSums][DP / 8][32];
  __shared__ int found;
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int first = blockIdx.x;
  if (DEEP) {  // the CTA in which the blockIdx.x-th shared item began
    if (threadIdx.x == 0) found = -1;
    __syncthreads();
    if (warp == 0) {
      int left = blockIdx.x;
      for (int base = 0; base < tp.ctas; base += 32) {
        const unsigned some = __ballot_sync(0xffffffffu, base + lane < tp.ctas && tp.spans[base + lane].x >= 0);
        const int here = __popc(some);
        if (left < here) {
          if ((some >> lane & 1) && __popc(some & ((1u << lane) - 1)) == left) found = base + lane;
          break;
        }
        left -= here;
      }
    }
    __syncthreads();
    first = found;
    if (first < 0) return;
  }
  const int2 span = tp.spans[first];
  if (span.x < 0) return;
  const Item it = item_of(p, tp, {p.q_lens, p.kv_lens}, span.x);
  const int tile_row = (DEEP ? blockIdx.y : blockIdx.y * 8 + warp) * 8 + (lane >> 2), t = tile_row / kRows, row = tile_row % kRows;
  const int token = row / tp.group, h = it.hk * tp.group + row - token * tp.group;
  const int i = it.i0 + t * tp.tokens + token, pos = it.base + i;
  const bool stored = row < tp.group * tp.tokens && i < p.s_q;
  if (!__any_sync(0xffffffffu, stored)) return;  // (the same rows in every warp where DEEP)
  // CTA c's share: the item began in CTA `first`, before every other
  auto share = [&](int c) { return ((int64_t)c * 2 + (c == first)) * kTiles + t; };
  const int begin = first + (DEEP ? warp : 0), step = DEEP ? 8 : 1;
  float m = -INFINITY, l = 0.f;
#pragma unroll 4
  for (int c = begin; c <= span.y; c += step) m = fmaxf(m, __ldcg(tp.stats + share(c) * kRows + row).x);
  const float base = m == -INFINITY ? 0.f : m;
  float2 o[DP / 8];  // columns 8 y + 2 (lane % 4) on
#pragma unroll
  for (int y = 0; y < DP / 8; ++y) o[y] = make_float2(0.f, 0.f);
#pragma unroll 2
  for (int c = begin; c <= span.y; c += step) {
    const float2 st = __ldcg(tp.stats + share(c) * kRows + row);
    const float weight = exp2f(st.x - base);
    // a share that saw nothing of the row counts nothing, whatever its sums hold
    const bool none = st.x == -INFINITY && !isnan(st.y);
    l = none ? l : fmaf(st.y, weight, l);
    const float *from = tp.sums + (share(c) * DP * kRows + row * 8) + (lane & 3) * 2;
#pragma unroll
    for (int y = 0; y < DP / 8; ++y) {
      const float2 two = __ldcg(reinterpret_cast<const float2 *>(from + y * kRows * 8));
      o[y].x = none ? o[y].x : fmaf(two.x, weight, o[y].x);
      o[y].y = none ? o[y].y : fmaf(two.y, weight, o[y].y);
    }
  }
  constexpr int kMine = DP / 8 / kSums;  // columns' groups that this warp writes
  if (DEEP) {
    warp_m[warp][lane] = m;
    warp_l[warp][lane] = l;
#pragma unroll
    for (int y = 0; y < DP / 8; ++y) warp_o[warp][y][lane] = o[y];
    __syncthreads();
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int w = 0; w < kSums; ++w) m = fmaxf(m, warp_m[w][lane]);
    const float all = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int y = 0; y < kMine; ++y) o[y] = make_float2(0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kSums; ++w) {
      const float weight = exp2f(warp_m[w][lane] - all);
      l = fmaf(warp_l[w][lane], weight, l);  // (a warp without parts has sums of zero)
#pragma unroll
      for (int y = 0; y < kMine; ++y) {
        const float2 two = warp_o[w][warp * kMine + y][lane];
        o[y].x = fmaf(two.x, weight, o[y].x);
        o[y].y = fmaf(two.y, weight, o[y].y);
      }
    }
  }
  const int col = (DEEP ? warp * kMine : 0) * 8 + (lane & 3) * 2;
  const bool some = stored && i < it.n_q && pos >= 0 && (m != -INFINITY || isnan(l));
  const float inv = some ? 1.0f / l : 0.f;
  T *out = static_cast<T *>(p.o) + it.b * p.os[0] + i * p.os[1] + h * p.os[2];
  bool odd = false;
#pragma unroll
  for (int y = 0; y < kMine; ++y) {
    const float a = some ? o[y].x * inv : 0.f, b = some ? o[y].y * inv : 0.f;
    if (stored && col + y * 8 < p.d) {
      odd |= !isfinite(a) || !isfinite(b);
      *reinterpret_cast<uint32_t *>(out + col + y * 8) = pack16<T>(a, b);
    }
  }
  if (p.lse && stored && (lane & 3) == 0 && (!DEEP || warp == 0))
    p.lse[((int64_t)it.b * p.q_heads + h) * p.s_q + i] = some ? lse_of<(int)kLift<T>>(m, l) : -INFINITY;
  if (DEEP) __syncthreads();  // the other warps' columns are there: mended once or more, but alike
  const unsigned odd_lanes = __ballot_sync(0xffffffffu, odd);
  if (odd_lanes) mend_rows<T, DP / 32>(p, (lane & 3) == 0 && (odd_lanes >> lane & 0xf) != 0, it.b, it.hk, pos, i, h);
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
// a group that fits a tile, 16-byte alignment, strides that a tensor map holds (below
// 2^40 bytes; a broadcast batch or head of K and V becomes an axis of one).
bool window_tensor(const WindowParams &p) {
  constexpr int64_t kMostStride = 1ll << 38;
  const int group = p.q_heads / p.kv_heads;
  bool ok = p.d <= 128 && p.d % 8 == 0 && group <= kRows && (group == 1 || p.qs[2] < kMostStride / group) && p.s_kv > 0 && aligned(p.q, 16) && aligned(p.k, 16) &&
            aligned(p.v, 16) && aligned(p.o, 16);
  const int sizes[4][3] = {{p.batch, p.s_q, p.q_heads}, {p.batch, p.s_kv, p.kv_heads}, {p.batch, p.s_kv, p.kv_heads}, {p.batch, p.s_q, p.q_heads}};
  const int64_t *strides[4] = {p.qs, p.ks, p.vs, p.os};
  for (int x = 0; x < 4; ++x)
    for (int a = 0; a < 3; ++a) {
      const bool repeats = (x == 1 || x == 2) && a != 1;  // may have a stride of zero
      const int64_t s = strides[x][a];
      ok = ok && (sizes[x][a] == 1 || (s % 8 == 0 && (s > 0 || (s == 0 && repeats)) && s < kMostStride));
    }
  return ok;
}

template <class T, int DP>
int launch_window(const WindowParams &p, cudaStream_t s) {
  using L = WindowLayout<DP>;
  constexpr bool kBf16 = !std::is_same<T, __half>::value;
  auto *kernel = window_kernel<T, DP>;
  TensorParams t = {};
  t.group = p.q_heads / p.kv_heads;
  t.tokens = kRows / t.group;
  CUtensorMap tq, tk, tv;
  const int64_t q_sizes[5] = {p.d, t.group, p.s_q, p.kv_heads, p.batch};
  const int64_t q_strides[5] = {1, p.qs[2], p.qs[1], p.qs[2] * t.group, p.qs[0]};
  const int q_box[5] = {64, t.group, t.tokens, 1, 1};
  if (int rc = make_map(&tq, kBf16, p.q, 5, q_sizes, q_strides, q_box)) return rc;
  const int kv_box[4] = {64, kKeys / 2, 1, 1};  // a block's halves may come from two places
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
  // Whole items, or runs of blocks: where the most loaded CTA (the first one: items come longest
  // first) has more units beyond a run's than cutting and joining cost.  With lengths on the
  // device the items may be short or empty: several items a CTA are then left to the kernel,
  // which cuts them only where whole ones would not be even.
  const int sms = std::min(sm_count(), kMostCtas);
  t.cut = 0;
  t.deep = items * 4 <= sms;  // an item spans four CTAs or more, if it is cut
  if (items <= kMaxCutItems) {
    const int heads = p.batch * p.kv_heads;
    auto units = [&](int qb) {
      const int64_t keys = (int64_t)p.s_kv - p.s_q + (int64_t)(qb + 1) * kTiles * t.tokens;
      const int64_t reach = p.window ? (int64_t)p.window + kTiles * t.tokens + p.sinks : p.s_kv;
      const int64_t seen = std::min(std::min(keys, reach), (int64_t)p.s_kv);
      return seen <= 0 ? 0 : units_of((int)((seen + kKeys - 1) / kKeys));
    };
    int64_t total = 0, most = 0;
    for (int qb = 0; qb < t.q_blocks; ++qb) total += (int64_t)units(qb) * heads;
    for (int64_t i = 0; i < items; i += sms) most += units(t.q_blocks - 1 - (int)(i / heads));
    const bool ragged = p.q_lens || p.kv_lens;
    t.cut = total < (1 << 30) && (ragged && items > sms ? units(t.q_blocks - 1) > kMinRun
                                                        : most - std::max<int64_t>(total / sms, kMinRun) > (t.deep ? kDeepCut : kWideCut));
  }
  int grid = t.items < sms ? t.items : sms;
  if (t.cut) {
    grid = t.ctas = sms;
    void *mem = nullptr;
    const size_t rows = (size_t)sms * 2 * kTiles * kRows;
    if (int rc = scratch_buffer(s, kSpansSlot, sms * sizeof(int2), &mem)) return rc;
    t.spans = static_cast<int2 *>(mem);
    if (int rc = scratch_buffer(s, kSumsSlot, rows * 128 * sizeof(float), &mem)) return rc;
    t.sums = static_cast<float *>(mem);
    if (int rc = scratch_buffer(s, kStatsSlot, rows * sizeof(float2), &mem)) return rc;
    t.stats = static_cast<float2 *>(mem);
  }
  if (int rc = check_cuda(launch_pdl(kernel, dim3(grid), dim3(kThreads), L::kBytes, s, tq, tk, tv, p, t), "lc_window_attention")) return rc;
  if (!t.cut) return LC_OK;
  const cudaError_t err = t.deep ? launch_pdl(join_kernel<T, DP, true>, dim3(t.items, kTiles * kRows / 8), dim3(256), 0, s, p, t)
                               : launch_pdl(join_kernel<T, DP, false>, dim3(sms, kTiles * kRows / 64), dim3(256), 0, s, p, t);
  return check_cuda(err, "lc_window_attention (join)");
}

template <class T>
int window_sized(const WindowParams &p, cudaStream_t s) {
  return p.d <= 64 ? launch_window<T, 64>(p, s) : launch_window<T, 128>(p, s);
}

// Few rows of few keys: a CTA per row is done before the tensor-core form has set up its
// barriers, tensor memory and copies (19 rows x 8 heads of 19 keys: 2.7 against 6.7 us,
// 16 x 32 of 64: 6.0 against 7.7; 64 x 32 of 64: 12.2 against 8.9, 1 x 8 of 256: 10.8
// against 8.0).
bool few_keys(const WindowParams &p) {
  const int64_t reach = p.window ? std::min<int64_t>((int64_t)p.window + p.sinks, p.s_kv) : p.s_kv;
  return reach <= 128 && (int64_t)p.batch * p.s_q * p.q_heads * reach <= 32768;
}

template <class T>
int launch_rows(const WindowParams &p, cudaStream_t s) {
  const dim3 grid((unsigned)p.s_q, (unsigned)p.q_heads, (unsigned)p.batch), block(kRowWarps * 32);
  return check_cuda(p.d <= 64    ? launch_pdl(window_row_kernel<T, 2>, grid, block, 0, s, p)
                    : p.d <= 128 ? launch_pdl(window_row_kernel<T, 4>, grid, block, 0, s, p)
                                 : launch_pdl(window_row_kernel<T, 8>, grid, block, 0, s, p),
                    "lc_window_attention (rows)");
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
  if (!(scale > 0.f) || scale > 2e38f) return fail(LC_ERR_INVALID, "%s: scale must be positive and finite", me);
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
  if (!few_keys(p) && window_tensor(p)) return dtype == LC_F16 ? window_sized<__half>(p, s) : window_sized<__nv_bfloat16>(p, s);
  return dtype == LC_F16 ? launch_rows<__half>(p, s) : launch_rows<__nv_bfloat16>(p, s);
}
