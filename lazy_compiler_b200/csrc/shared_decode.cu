// Attention of one new token of every sequence where sequences begin alike: samples
// of a prompt, questions to a document.  Slots with the same leader hold the same pages
// over the first `shared` tokens; that prefix is read once for all of them, what comes
// behind it by each slot alone (paged_decode.cu's kernels, over the suffix), and the two
// are joined:
//   o = (sum_x 2^(m_x - m) O_x) / (sum_x 2^(m_x - m) l_x)   over the parts x of a row,
// each an unnormalised sum of values O_x and of weights l_x relative to its reference m_x.
//
// Over the prefix the rows of a group, slots x query heads of a key-value head, are
// one operand: R = 32 rows for eight samples of groups of four heads, 256 for 64.  So
// this is a matrix product again, 4 R d flops for 4 d bytes of a key: bound by HBM up to
// some 200 rows, by the tensor pipe and the softmax beyond.  Hence tcgen05, the
// schedule of window_attention.cu with two tiles of 128 rows a CTA, S = Q K^T and
// O += P V, P over S in tensor memory, a softmax thread per row.  Where a group has more
// than 128 rows, the tiles are 256 of them and share every block of 128 keys; else both
// are the same rows, and take every other block, so that two blocks are in work at any time.
//
// Work is cut by length: all (group, key-value head, 256 rows) segments are laid end to
// end, block by block, and every CTA takes an equal run.  What a run holds of a segment
// goes to the workspace in f32; merge_kernel adds up a row's parts in CTA order.
// Pages come by cp.async, 16 bytes a lane, so any page size, stride and page that is not
// there (zero-filled, masked) is alike; four warps of copies: keys and values of even and
// of odd blocks, each the only writer of its buffer.
//
// P is rounded to the storage type before the second product, as in window_attention.cu (1.35 times the
// error of an output rounded once); all else is f32.
//
// Measured, 32/8 heads of 128, with the suffixes and the join: 8 prompts of 8000 tokens with 8 samples of
// 600 more 77 us where the bytes take 42 (the prefixes by themselves 52 us: 20 blocks a CTA, then ends and
// beginnings of segments, two or three a CTA); 64 questions to 100003 tokens 137 us in a graph, bytes 70, products
// 64 (two tiles' block takes 3660 cycles, 2080 of them products: as in window_attention.cu a tile's scores, softmax
// and products are a chain).
#include <algorithm>
#include <type_traits>

#include "paged.cuh"
#include "sm100.cuh"
#include "softmax.cuh"

namespace lc {

using namespace attend;

namespace {

using namespace sm100;
using namespace softmax;

constexpr int kRows = 128;   // of a tile
constexpr int kTiles = 2;    // per CTA
constexpr int kKeys = 128;   // of a block
constexpr int kStages = 2;
constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMostCtas = 256;
constexpr int kMostSlots = 8192;
constexpr int kLensHeld = 1024;  // slots whose lengths are kept in shared memory
constexpr int kEndUnits = 1;  // what a segment's end costs, in blocks: its sums' way to memory
constexpr int kMinRun = 4;    // units of a run: a run's beginning and its parts' join cost about as many
constexpr int kRing = 4;      // pieces of work known ahead
constexpr int kReaders = 1 + 8 + 4;  // of a piece: the warps of products, softmax and copies
constexpr int kFewRegs = 72, kManyRegs = 184;  // of 128 at launch, as in window_attention.cu
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kOCol = 256;  // S of tile t at t * 128, P over it, O of tile t at kOCol + t * DP
constexpr float kRescale = 8.0f;
template <class T>
constexpr float kLift = kLiftBf16;
template <>
constexpr float kLift<__half> = 7.f;  // with the lag of kRescale, weights reach 2^15
constexpr int kChunkBytes = kRows * 64 * 2;
constexpr int kSumsSlot = 47, kStatsSlot = 48, kWhereSlot = 49, kOwnSumsSlot = 50, kOwnStatsSlot = 51;  // scratch_buffer slots

template <int DP>
struct SharedLayout {
  static constexpr int kTileBytes = DP / 64 * kChunkBytes;
  static constexpr int kQBytes = kTiles * kTileBytes;
  static constexpr int kBuffers = kQBytes + kStages * 2 * kTileBytes;
  // the buffers, and of every slot its leader, its place in the order, and its length if there are few
  static int bytes(int slots) { return kBuffers + 1024 + slots * 4 + (slots <= kLensHeld ? slots * 4 : 0); }
};

struct SharedParams {
  DecodeParams p;
  Sharing sharing;
  // Parts of rows: [CTA][of a segment that began before the run, of one that began in it][tile][row],
  // behind them [slot][query head][tile], of segments that one CTA holds: DP sums, and (m, l).
  float *sums;
  float2 *stats;
  int4 *where;  // of every row of a prefix: first and last CTA, row of its tiles, how (kSplitKeys, kWhole)
  int *err;
  int ctas;
  int q_pieces;  // the queries are aligned to 16 bytes
  int runs;  // 16 tokens of a head, from a multiple of 16 on, are one run of memory in k and in v
};
constexpr int kSplitKeys = 1, kWhole = 2;

__host__ __device__ __forceinline__ int64_t cut_rows(int ctas) { return (int64_t)ctas * 2 * kTiles * kRows; }

// The leaders in the order of the slots; the mark says that a group with a prefix begins here.
constexpr uint16_t kBegins = 0x8000;

// The slots order[at ... at + count) and the blocks of keys that some of them see of the prefix: those of the
// sinks, then from key `start` on.
struct Group {
  int at, count, slot, keys, n_sink, start, blocks;
};
// By a whole warp.
__device__ __forceinline__ Group group_of(const SharedParams &sp, const uint16_t *leaders, const uint16_t *order, int at) {
  const DecodeParams &p = sp.p;
  const int lane = threadIdx.x & 31;
  Group g;
  g.at = at;
  g.slot = leaders[at] & ~kBegins;
  // the group's end: among the next 32 places, or by bisection behind them
  const unsigned others = __ballot_sync(0xffffffffu, at + 1 + lane >= p.slots || leaders[at + 1 + lane] != (uint16_t)g.slot);
  int lo = at + 1 + (others ? __ffs(others) - 1 : 32), hi = others ? lo : p.slots;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (leaders[mid] == (uint16_t)g.slot)
      lo = mid + 1;
    else
      hi = mid;
  }
  g.count = lo - at;
  g.keys = prefix_tokens(p, sp.sharing, g.slot);
  int first = 0, sinks = 0;
  if (p.window) {
    first = INT32_MAX;
    for (int i = lane; i < g.count; i += 32) {
      const int slot = order[at + i];
      const int n = slot < p.slots ? cached_tokens(p, slot) : 0;
      if (n <= 0) continue;
      const Visible see = visible(n - 1, p.window, p.sinks);
      first = min(first, see.lo);
      sinks = max(sinks, see.sink_end);
    }
    first = __reduce_min_sync(0xffffffffu, first);
    sinks = __reduce_max_sync(0xffffffffu, sinks);
  }
  g.n_sink = (min(sinks, g.keys) + kKeys - 1) / kKeys;
  g.start = max(min(first, g.keys), g.n_sink * kKeys);
  g.blocks = g.n_sink + max(0, g.keys - g.start + kKeys - 1) / kKeys;
  return g;
}
__device__ __forceinline__ int block_key(const Group &g, int j) { return j < g.n_sink ? j * kKeys : g.start + (j - g.n_sink) * kKeys; }

// Blocks [j0, j1) of a segment: a group's key-value head and 256 of its rows.
struct Piece {
  Group g;
  int head, row0, rows, j0, j1;
  int first, last;  // the CTAs that the segment's blocks are in
};
// a * b / c for units and CTAs; units times CTAs are below 2^32 (worth_sharing).
__device__ __forceinline__ int share_of(int a, int b, int c, bool below = false) {  // below: of one less
  return (int)(((unsigned)a * (unsigned)b - below) / (unsigned)c);
}
// A CTA's run, in units, and the segment that a reader of it is at.
struct Run {
  int begin, end, total, seg_begin;
  int ctas, seg;  // seg: (head, 256 rows) of the group
  Group g;        // at: the group's first place in the order, or behind the last
};
__device__ __forceinline__ int row_parts(int count, int group) { return (int)(((int64_t)count * group + kTiles * kRows - 1) / (kTiles * kRows)); }
struct Pieces {
  Run run;
  __device__ __forceinline__ explicit Pieces(const Run &r) : run(r) {}
  // By a whole warp.
  __device__ __forceinline__ bool next(const SharedParams &sp, const uint16_t *leaders, const uint16_t *order, Piece &out) {
    const DecodeParams &p = sp.p;
    const int lane = threadIdx.x & 31, group = p.q_heads / p.kv_heads;
    while (run.seg_begin < run.end && run.g.at < p.slots) {
      const int parts = row_parts(run.g.count, group);
      const bool some = run.g.blocks > 0;
      if (some) {
        out.g = run.g;
        out.head = run.seg / parts;
        out.row0 = (run.seg - out.head * parts) * (kTiles * kRows);
        out.rows = (int)min((int64_t)kTiles * kRows, (int64_t)run.g.count * group - out.row0);
        out.j0 = max(0, run.begin - run.seg_begin);
        out.j1 = min(run.g.blocks, run.end - run.seg_begin);
        // the CTA of a unit x: the last whose run begins at x or before, ((x + 1) ctas - 1) / total
        const bool begins = out.j0 == 0, ends = out.j1 == run.g.blocks;
        out.first = begins ? (int)blockIdx.x : share_of(run.seg_begin + 1, run.ctas, run.total, true);
        out.last = ends ? (int)blockIdx.x : share_of(run.seg_begin + run.g.blocks, run.ctas, run.total, true);
        run.seg_begin += run.g.blocks + kEndUnits;
        if (++run.seg == parts * p.kv_heads) run.seg = 0;
      }
      if (!some || run.seg == 0) {  // the next group that begins
        run.seg = 0;
        int at = run.g.at + run.g.count;
        while (at < p.slots) {
          const unsigned begins = __ballot_sync(0xffffffffu, at + lane < p.slots && (leaders[at + lane] & kBegins) != 0);
          if (begins) {
            at += __ffs(begins) - 1;
            break;
          }
          at += 32;
        }
        run.g.at = at;
        if (at < p.slots && run.seg_begin < run.end) run.g = group_of(sp, leaders, order, at);
      }
      if (some && out.j1 > out.j0) return true;
    }
    return false;
  }
};

__device__ __forceinline__ void give_up(const SharedParams &sp, volatile int *abort, int code) {
  *abort = 1;
  atomicCAS(sp.err, 0, code);
}
// Every lane waits, and the warp agrees on the outcome.
__device__ __forceinline__ bool wait_all(uint64_t *bar, uint32_t parity, volatile int *abort, const SharedParams &sp, int code) {
  const int ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, abort) ? 1 : 0);
  if (!ok && (threadIdx.x & 31) == 0) give_up(sp, abort, code);
  return ok != 0;
}

// The pieces as the planning warp leaves them, for the others to take one after the other.
struct Ring {
  Piece piece[kRing];
  uint64_t full[kRing], empty[kRing];
};
// The k-th; false: there is none (or the wait for it was given up).
__device__ __forceinline__ bool take(Ring &ring, int k, Piece &out, volatile int *abort, const SharedParams &sp, int code) {
  if (!wait_all(&ring.full[k % kRing], k / kRing & 1, abort, sp, code)) return false;
  out = ring.piece[k % kRing];
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(&ring.empty[k % kRing]);
  return out.j1 > 0;
}

// What is read once leaves L2 first, so that code, maps, queries and parts stay there.
__device__ __forceinline__ uint64_t first_to_leave() {
  uint64_t policy;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
  return policy;
}
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, int bytes, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint.L2::128B [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src), "r"(bytes), "l"(policy) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(policy) : "memory");
}
__device__ __forceinline__ void copies_done() {
  asm volatile("cp.async.commit_group;" ::: "memory");
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

template <class T, int DP>
__global__ void __launch_bounds__(kThreads, 1) shared_kernel(const __grid_constant__ SharedParams sp) {
  using L = SharedLayout<DP>;
  constexpr int kTile = L::kTileBytes;
  constexpr bool kBf16 = !std::is_same<T, __half>::value;
  const DecodeParams &p = sp.p;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t *q_s = smem, *kv_s = smem + L::kQBytes;
  uint16_t *leaders = reinterpret_cast<uint16_t *>(smem + L::kBuffers), *order = leaders + p.slots;
  int *lens = reinterpret_cast<int *>(order + p.slots);  // by place in the order
  __shared__ __align__(8) uint64_t q_full, q_empty;
  __shared__ __align__(8) uint64_t k_full[kStages], v_full[kStages], k_empty[kStages], v_empty[kStages];
  __shared__ __align__(8) uint64_t s_full[kTiles], p_full[kTiles], o_done[kTiles];
  __shared__ __align__(16) uint32_t key_bits[4][kKeys / 32];  // of a block, its number modulo 4: the keys that are there
  __shared__ uint32_t tmem_base;
  __shared__ int abort_flag;
  __shared__ int warp_units[kWarps];
  __shared__ Run run_shared;
  __shared__ __align__(16) Ring ring;
  volatile int *abort = &abort_flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int group = p.q_heads / p.kv_heads;

  if (tid == 0) {
    for (int x = 0; x < kRing; ++x) {
      mbar_init(&ring.full[x], 1);
      mbar_init(&ring.empty[x], kReaders);
    }
    mbar_init(&q_full, 8);
    mbar_init(&q_empty, 1);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int t = 0; t < kTiles; ++t) {
      mbar_init(&s_full[t], 2);
      mbar_init(&p_full[t], 4);
      mbar_init(&o_done[t], 1);
    }
    abort_flag = 0;
    fence_barrier_init();
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
  pdl_trigger();  // the suffixes' kernel: it waits at its end

  // ---- this CTA's run
  for (int i = tid; i < p.slots; i += kThreads) {
    const int slot = sp.sharing.order[i];
    uint16_t mark = 0x7fff;  // no group
    if ((unsigned)slot < (unsigned)p.slots) {
      const int leader = sp.sharing.leader[slot], keys = prefix_tokens(p, sp.sharing, slot);
      if ((unsigned)leader < (unsigned)p.slots) mark = (uint16_t)(leader | (leader == slot && keys > 0 ? kBegins : 0));
      if (p.slots <= kLensHeld) lens[i] = cached_tokens(p, slot);
    }
    leaders[i] = mark;
    order[i] = (unsigned)slot < (unsigned)p.slots ? (uint16_t)slot : 0xffff;
  }
  if (tid == 0) run_shared = {};
  if (tid == 0) run_shared.g.at = p.slots;
  __syncthreads();
  int *units = reinterpret_cast<int *>(smem);  // of the group that begins at a position
  Group *groups = reinterpret_cast<Group *>(smem + kMostSlots * sizeof(int));  // and that group, if there are few slots
  const bool held = p.slots * (int)sizeof(Group) <= L::kBuffers - kMostSlots * (int)sizeof(int);
  for (int i = warp; i < p.slots; i += kWarps) {
    int n = 0;
    if (leaders[i] & kBegins) {
      const Group g = group_of(sp, leaders, order, i);
      if (g.blocks > 0) n = (g.blocks + kEndUnits) * row_parts(g.count, group) * p.kv_heads;
      if (held && lane == 0) groups[i] = g;
    }
    if (lane == 0) units[i] = n;
  }
  __syncthreads();
  {
    const int per = (p.slots + kThreads - 1) / kThreads;
    const int i0 = min(p.slots, tid * per), i1 = min(p.slots, i0 + per);
    int own = 0;
    for (int i = i0; i < i1; ++i) own += units[i];
    int inc = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    if (lane == 31) warp_units[warp] = inc;
    __syncthreads();
    const int of_warp = lane < kWarps ? warp_units[lane] : 0;
    const int total = __reduce_add_sync(0xffffffffu, of_warp);
    int before = inc - own + __reduce_add_sync(0xffffffffu, lane < warp ? of_warp : 0);
    const int ctas = min(sp.ctas, (total + kMinRun - 1) / kMinRun);
    if ((int)blockIdx.x < ctas) {
      const int begin = share_of(blockIdx.x, total, ctas), end = share_of(blockIdx.x + 1, total, ctas);
      if (begin >= before && begin < before + own) {
        for (int i = i0; i < i1; ++i) {
          if (begin < before + units[i]) {
            run_shared.begin = begin, run_shared.end = end, run_shared.total = total;
            run_shared.seg_begin = before, run_shared.ctas = ctas, run_shared.g.at = i;
            if (held) run_shared.g = groups[i];
            break;
          }
          before += units[i];
        }
      }
    }
  }
  __syncthreads();
  // (the units have been read: the buffers are free)
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegs));
    if (warp == 0) {
      Run run = run_shared;
      if (run.ctas > 0) {
        if (!held) run.g = group_of(sp, leaders, order, run.g.at);
        run.seg = (run.begin - run.seg_begin) / (run.g.blocks + kEndUnits);
        run.seg_begin += run.seg * (run.g.blocks + kEndUnits);
      }
      Pieces pieces(run);
      Piece piece = {};
      for (int k = 0;; ++k) {
        const bool more = pieces.next(sp, leaders, order, piece);
        if (!more) piece.j1 = 0;
        if (k >= kRing && !wait_all(&ring.empty[k % kRing], (k / kRing - 1) & 1, abort, sp, kErrTimeoutProducer)) break;
        if (lane == 0) {
          ring.piece[k % kRing] = piece;
          mbar_arrive(&ring.full[k % kRing]);
        }
        __syncwarp();
        if (!more) break;
      }
    } else if (warp == 1) {
      const uint32_t leader = elect_one();
      constexpr uint32_t idesc_s = idesc_f16(kBf16, false, false, kRows, kKeys);
      constexpr uint32_t idesc_o = idesc_f16(kBf16, false, true, kRows, DP);
      const uint64_t q_desc = smem_desc_sw128(smem_u32(q_s), 16, 1024);
      const uint64_t k_desc = smem_desc_sw128(smem_u32(kv_s), 16, 1024);
      const uint64_t v_desc = smem_desc_sw128(smem_u32(kv_s) + kTile, kChunkBytes, 1024);
      constexpr uint32_t kStageStep = 2 * kTile / 16;
      Piece piece;
      int g0 = 0, local = 0, done[kTiles] = {0, 0};  // blocks and pieces so far, steps of a tile
      bool ok = true;
      while (ok && take(ring, local, piece, abort, sp, kErrTimeoutMma)) {
        // Step x is tile x & 1; of both tiles' rows one block (more than 128), else of the same rows the next.
        const bool wide = piece.rows > kRows;
        const int blocks = piece.j1 - piece.j0, steps = wide ? 2 * blocks : blocks;
        auto block_of = [&](int x) { return g0 + (wide ? x >> 1 : x); };
        auto products_s = [&](int x) {  // S_t = Q_t K^T
          const int t = x & 1, g = block_of(x);
          if ((!wide || t == 0) && !mbar_wait(&k_full[g & 1], (g >> 1) & 1, abort)) return false;
          tc_fence_after();
          const uint64_t qd = q_desc + (uint64_t)(wide ? t * kTile / 16 : 0);
          const uint64_t kd = k_desc + (uint64_t)((g & 1) * kStageStep);
#pragma unroll
          for (int k = 0; k < DP / 16; ++k) {
            const uint32_t off = ((k >> 2) * kChunkBytes + (k & 3) * 32) / 16;
            warp_mma(leader, tmem + t * kKeys, qd + off, kd + off, idesc_s, k > 0);
          }
          warp_commit(leader, &s_full[t]);
          if (leader) mbar_arrive(&s_full[t]);  // and what this warp has seen of the block (key_bits)
          if (!wide || t == 1) warp_commit(leader, &k_empty[g & 1]);
          if (x + 1 == steps) warp_commit(leader, &q_empty);
          return true;
        };
        ok = mbar_wait(&q_full, local & 1, abort);
        for (int x = 0; ok && x < min(2, steps); ++x) ok = products_s(x);
        for (int x = 0; ok && x < steps; ++x) {  // O_t (+)= P_t V
          const int t = x & 1, g = block_of(x);
          if ((!wide || t == 0) && !mbar_wait(&v_full[g & 1], (g >> 1) & 1, abort)) {
            ok = false;
            break;
          }
          if (!mbar_wait(&p_full[t], done[t] & 1, abort)) {
            ok = false;
            break;
          }
          ++done[t];
          tc_fence_after();
          const uint64_t vd = v_desc + (uint64_t)((g & 1) * kStageStep);
#pragma unroll
          for (int k = 0; k < kKeys / 16; ++k)
            warp_mma_tmem_a(leader, tmem + kOCol + t * DP, tmem + t * kKeys + k * 8, vd + (uint64_t)(k * 2048 / 16), idesc_o, !(x < 2 && k == 0));
          warp_commit(leader, &o_done[t]);
          if (!wide || t == 1) warp_commit(leader, &v_empty[g & 1]);
          if (x + 2 < steps) ok = products_s(x + 2);
        }
        g0 += blocks;
        ++local;
      }
      if (!ok && lane == 0) give_up(sp, abort, kErrTimeoutMma);
    }
  } else if (warp < 12) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManyRegs));
    const int t = (warp - 4) >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_at = tmem + lane_base + t * kKeys, o_at = tmem + lane_base + kOCol + t * DP;
    Piece piece;
    int g0 = 0, local = 0, step = 0;
    bool ok = true;
    while (ok && take(ring, local, piece, abort, sp, kErrTimeoutSoftmax)) {
      const bool wide = piece.rows > kRows;
      const int blocks = piece.j1 - piece.j0, steps = wide ? blocks : (blocks + 1 - t) / 2;
      // this thread's row: a slot of the group and one of its query heads
      const int tile_row = wide ? t * kRows + row : row;
      const bool real = tile_row < piece.rows;
      const int in_group = real ? piece.row0 + tile_row : 0, member = in_group / group;
      const int place = piece.g.at + (real ? member : 0), listed = order[place];
      const bool sound = listed < p.slots;  // (a place in the order may say anything)
      const int slot = sound ? listed : piece.g.slot;
      const int h = piece.head * group + in_group - member * group;
      const int n = p.slots <= kLensHeld && sound ? lens[place] : cached_tokens(p, slot);
      const int upto = real ? min(n, piece.g.keys) : INT32_MAX;
      const Visible see = visible(n - 1, p.window, p.sinks);
      const int lo = real ? see.lo : 0, sink_end = see.sink_end;
      if (local > 0 && !wait_all(&q_empty, (local - 1) & 1, abort, sp, kErrTimeoutSoftmax)) break;
      if (wide || t == 0) {
        // The warp's rows of Q, piece c of 16 bytes at c ^ (row & 7).  A thread a row took 7 us; every address is
        // readable, so the loads need no condition, and are on their way together.
        const int64_t at = slot * p.qs[0] + h * p.qs[1];
        const unsigned reals = __ballot_sync(0xffffffffu, real);
        uint8_t *to = q_s + (wide ? t * kTile : 0) + quarter * 32 * 128;
        if (sp.q_pieces) {
          constexpr int kPieces = DP / 8, kLoads = kPieces;  // 16 bytes a lane: 32 / kPieces rows a load
          const int c = lane % kPieces, row_in = lane / kPieces;
          const T *from = static_cast<const T *>(p.q) + (c * 8 < p.d ? c * 8 : 0);
          uint4 v[kLoads];
#pragma unroll
          for (int i = 0; i < kLoads; ++i) v[i] = __ldg(reinterpret_cast<const uint4 *>(from + __shfl_sync(0xffffffffu, at, i * (32 / kPieces) + row_in)));
#pragma unroll
          for (int i = 0; i < kLoads; ++i) {
            const int r = i * (32 / kPieces) + row_in;
            *reinterpret_cast<uint4 *>(to + (c >> 3) * kChunkBytes + r * 128 + (((c & 7) ^ (r & 7)) << 4)) =
                (reals >> r & 1) && c * 8 < p.d ? v[i] : make_uint4(0, 0, 0, 0);
          }
        } else {
          constexpr int kHalves = DP / 64, kAtOnce = 8;
          const T *column[kHalves];
#pragma unroll
          for (int x = 0; x < kHalves; ++x) column[x] = static_cast<const T *>(p.q) + (x * 64 + lane * 2 < p.d ? x * 64 + lane * 2 : 0);
#pragma unroll 1
          for (int r0 = 0; r0 < 32; r0 += kAtOnce) {
            uint32_t v[kAtOnce][kHalves];
#pragma unroll
            for (int r = 0; r < kAtOnce; ++r) {
              const int64_t from = __shfl_sync(0xffffffffu, at, r0 + r);
#pragma unroll
              for (int x = 0; x < kHalves; ++x) v[r][x] = __ldg(reinterpret_cast<const uint32_t *>(column[x] + from));
            }
#pragma unroll
            for (int r = 0; r < kAtOnce; ++r)
#pragma unroll
              for (int x = 0; x < kHalves; ++x)
                *reinterpret_cast<uint32_t *>(to + x * kChunkBytes + (r0 + r) * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4) =
                    (reals >> (r0 + r) & 1) && x * 64 + lane * 2 < p.d ? v[r][x] : 0u;
          }
        }
        fence_async_shared();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full);

      float m = -INFINITY, l = 0.f;
      for (int x = 0; x < steps; ++x, ++step) {
        const int j = wide ? x : 2 * x + t, key = block_key(piece.g, piece.j0 + j), g = g0 + j;
        if (!wait_all(&s_full[t], step & 1, abort, sp, kErrTimeoutSoftmax)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint4 there = *reinterpret_cast<const uint4 *>(key_bits[g & 3]);
        const bool whole = key + kKeys <= upto && (key >= lo || key + kKeys <= sink_end) && (there.x & there.y & there.z & there.w) == 0xffffffffu;
        const bool all_whole = __all_sync(0xffffffffu, whole);
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
            if (!all_whole) {
              const int at = key + c * 32;
              uint32_t sees = bits_between(0, upto - at) & (bits_between(lo - at, 32) | bits_between(0, sink_end - at));
              sees = real ? sees & (c == 0 ? there.x : c == 1 ? there.y : c == 2 ? there.z : there.w) : 0xffffffffu;
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
        const float mx = max3(max3(mx8[0], mx8[1], mx8[2]), max3(mx8[3], mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7])) * p.scale_log2;
        const float m_new = fmaxf(m, mx - kLift<T>);
        const bool need = m_new > m + kRescale;
        if (__any_sync(0xffffffffu, need)) {
          const float alpha = need ? ex2(m - m_new) : 1.0f;
          if (need) {
            l *= alpha;
            m = m_new;
          }
          if (x > 0) {  // S of this step came behind the product before it
            if (!wait_all(&o_done[t], (step - 1) & 1, abort, sp, kErrTimeoutCorrection)) {
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
        uint64_t part2[4] = {0ull, 0ull, 0ull, 0ull};
        const uint64_t scale2 = pack2(p.scale_log2, p.scale_log2);
        const float base = m == -INFINITY ? 0.f : -m;
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
      // the row's part
      const bool whole_segment = piece.first == piece.last;
      const int64_t at = whole_segment ? cut_rows(sp.ctas) + ((int64_t)slot * p.q_heads + h) * kTiles + (wide ? 0 : t)
                                       : (((int64_t)blockIdx.x * 2 + (piece.j0 == 0)) * kTiles + t) * kRows + row;
      // (`where` not before: an arrival on a barrier waits for the stores ahead of it, 6 us at the first)
      if (real && piece.j0 == 0 && (wide || t == 0))
        sp.where[(int64_t)slot * p.q_heads + h] = make_int4(piece.first, piece.last, tile_row, (wide ? 0 : kSplitKeys) | (whole_segment ? kWhole : 0));
      if (real) sp.stats[at] = make_float2(m, l);
      if (steps > 0) {
        if (!wait_all(&o_done[t], (step - 1) & 1, abort, sp, kErrTimeoutEpilogue)) break;
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < DP / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(o_at + c * 32, o);
          tmem_wait_ld();
          if (real) {
#pragma unroll
            for (int y = 0; y < 4; ++y) st_global_v8_b32(sp.sums + at * DP + c * 32 + y * 8, o + y * 8);
          }
        }
        tc_fence_before();
      }
      g0 += blocks;
      ++local;
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegs));
    const int stage = warp & 1;
    const bool values = warp >= 14;
    constexpr int kPieces = DP / 8, kRowsPerCopy = 32 / kPieces;  // 16-byte pieces of a row; rows of a copy
    const int c = lane % kPieces, row_in = lane / kPieces;
    const bool c_real = c * 8 < p.d;
    const T *base = static_cast<const T *>(values ? p.v : p.k);
    const int64_t *strides = values ? p.vs : p.ks;
    uint64_t *full = values ? &v_full[stage] : &k_full[stage], *empty = values ? &v_empty[stage] : &k_empty[stage];
    const uint32_t buffer = smem_u32(kv_s) + stage * 2 * kTile + (values ? kTile : 0) + (c >> 3) * kChunkBytes;
    Piece piece;
    int g = 0;
    bool ok = true;
    for (int local = 0; ok && take(ring, local, piece, abort, sp, kErrTimeoutProducer); ++local) {
      // The first queries come first: behind the copies of all CTAs they took 10 us.
      if (local == 0 && !wait_all(&q_full, 0, abort, sp, kErrTimeoutProducer)) break;
      const int *table = p.table + piece.g.slot * p.ts;
      const uint64_t policy = (int64_t)piece.g.count * group > kTiles * kRows ? l2_policy_evict_normal() : first_to_leave();
      for (int j = piece.j0; j < piece.j1; ++j, ++g) {
        if ((g & 1) != stage) continue;
        const int key = block_key(piece.g, j);
        int64_t off[4];  // of keys lane, lane + 32, ...; -1: not there
        uint32_t bits[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int k = key + x * 32 + lane;
          off[x] = -1;
          if (k < piece.g.keys) {
            const int entry = page_index(p, k), page = table[entry];
            if ((unsigned)page < (unsigned)p.pages)
              off[x] = page * strides[0] + piece.head * strides[1] + (k - entry * p.page_size) * strides[2];
          }
          bits[x] = __ballot_sync(0xffffffffu, off[x] >= 0);
        }
        if (!wait_all(empty, ((g >> 1) & 1) ^ 1, abort, sp, kErrTimeoutProducer)) {
          ok = false;
          break;
        }
        if (!values && lane == 0) *reinterpret_cast<uint4 *>(key_bits[g & 3]) = make_uint4(bits[0], bits[1], bits[2], bits[3]);
        // Where 16 keys lie in one page one behind the other, without padding, they are one run of memory: one
        // place for 16 rows, and the addresses differ by constants (issuing a block: 4400 cycles without).
        const bool whole = sp.runs && (bits[0] & bits[1] & bits[2] & bits[3]) == 0xffffffffu && (key & 15) == 0;
        if (whole) {
          const uint32_t to = buffer + row_in * 128 + (((c & 7) ^ (row_in & 7)) << 4);
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const T *from = base + __shfl_sync(0xffffffffu, off[x >> 1], (x & 1) * 16) + lane * 8;
#pragma unroll
            for (int i = 0; i < 16; i += kRowsPerCopy)  // row i + row_in: bits apart, as piece ^ row wants it
              copy16((to ^ ((i & 7) << 4)) + (x * 16 + i) * 128, from + i * DP, policy);
          }
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          if (whole) break;
#pragma unroll 8
          for (int i = 0; i < 32; i += kRowsPerCopy) {
            const int r = x * 32 + i + row_in;
            const int64_t o = __shfl_sync(0xffffffffu, off[x], i + row_in);
            const bool copied = o >= 0 && c_real;
            copy16(buffer + r * 128 + (((c & 7) ^ (r & 7)) << 4), base + (copied ? o + c * 8 : 0), copied ? 16 : 0, policy);
          }
        }
        copies_done();
        fence_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(full);
      }
    }
  }

  __syncthreads();
  if (abort_flag) drain_delay();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// Adds up a row's parts, the prefix's in CTA order, then the suffix: a CTA a row, the parts dealt to its warps.
constexpr int kMergeWarps = 4;

template <class T, int DP>
__global__ void __launch_bounds__(kMergeWarps * 32) merge_kernel(const __grid_constant__ SharedParams sp, const float *own_sums, const float2 *own_stats) {
  constexpr int kCols = DP / 32, kAtOnce = 8;
  __shared__ float sums[kMergeWarps][DP];
  __shared__ float warp_m[kMergeWarps], warp_l[kMergeWarps];
  pdl_wait();
  pdl_trigger();
  const DecodeParams &p = sp.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = blockIdx.x;
  const int slot = (int)(row / p.q_heads), h = (int)(row - (int64_t)slot * p.q_heads);
  const int4 w = __ldcg(sp.where + row);
  const float2 own = __ldcg(own_stats + row);
  int parts = 0, first = 0, tile_row = 0;
  bool split = false, whole = false;
  if (slot_prefix(p, sp.sharing, slot) > 0 && w.x >= 0 && w.x <= w.y && w.y < sp.ctas && (unsigned)w.z < kTiles * kRows) {
    first = w.x, tile_row = w.z, split = w.w & kSplitKeys, whole = w.w & kWhole;
    parts = (split ? 2 : 1) * (whole ? 1 : w.y - w.x + 1);
  }
  auto part = [&](int x) -> int64_t {
    const int cta = first + (split ? x >> 1 : x), t = split ? x & 1 : tile_row / kRows;
    if (whole) return cut_rows(sp.ctas) + row * kTiles + (split ? x : 0);
    return (((int64_t)cta * 2 + (cta == first)) * kTiles + t) * kRows + tile_row % kRows;
  };
  auto counts = [](const float2 &st) { return st.x != -INFINITY || isnan(st.y); };  // else its sums hold anything
  // this warp's parts, of which the suffix is the last: a lane a part's statistics, then the sums, kAtOnce in flight
  float m = -INFINITY, l = 0.f, o[kCols];
#pragma unroll
  for (int y = 0; y < kCols; ++y) o[y] = 0.f;
  for (int x0 = warp; x0 <= parts; x0 += 32 * kMergeWarps) {
    const int x = x0 + lane * kMergeWarps;
    float2 st = make_float2(-INFINITY, 0.f);
    const float *from = own_sums + row * DP;
    if (x < parts) {
      const int64_t at = part(x);
      st = __ldcg(sp.stats + at);
      from = sp.sums + at * DP;
    } else if (x == parts) {
      st = own;
    }
    const unsigned some = __ballot_sync(0xffffffffu, counts(st));
    const float top = fmaxf(m, warp_max(st.x)), base = top == -INFINITY ? 0.f : top, alpha = ex2(m - base);
    const float weight = ex2(st.x - base);
    m = top;
    l = l * alpha + warp_sum(counts(st) ? st.y * weight : 0.f);
#pragma unroll
    for (int y = 0; y < kCols; ++y) o[y] *= alpha;
    for (unsigned left = some; left;) {
      float2 two[kAtOnce][kCols / 2];
      float ws[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const int i = left ? __ffs(left) - 1 : 0;
        const float *src = reinterpret_cast<const float *>(__shfl_sync(0xffffffffu, (unsigned long long)from, i));
        ws[u] = __shfl_sync(0xffffffffu, weight, i);
#pragma unroll
        for (int y = 0; y < kCols / 2; ++y)
          two[u][y] = left ? __ldcg(reinterpret_cast<const float2 *>(src + lane * kCols + 2 * y)) : make_float2(0.f, 0.f);
        left &= left - 1;
      }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
        for (int y = 0; y < kCols / 2; ++y) {
          o[2 * y] = fmaf(two[u][y].x, ws[u], o[2 * y]);
          o[2 * y + 1] = fmaf(two[u][y].y, ws[u], o[2 * y + 1]);
        }
    }
  }
#pragma unroll
  for (int y = 0; y < kCols; ++y) sums[warp][lane * kCols + y] = o[y];
  if (lane == 0) warp_m[warp] = m, warp_l[warp] = l;
  __syncthreads();
  float top = -INFINITY, sum = 0.f, weights[kMergeWarps];
#pragma unroll
  for (int x = 0; x < kMergeWarps; ++x) top = fmaxf(top, warp_m[x]);
#pragma unroll
  for (int x = 0; x < kMergeWarps; ++x) {
    weights[x] = ex2(warp_m[x] - (top == -INFINITY ? 0.f : top));
    sum = fmaf(warp_l[x], weights[x], sum);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  T *out = static_cast<T *>(p.o) + slot * p.os[0] + h * p.os[1];
  const int col = threadIdx.x;
  bool odd = false;
  if (col < p.d) {
    float v = 0.f;
#pragma unroll
    for (int x = 0; x < kMergeWarps; ++x) v = fmaf(sums[x][col], weights[x], v);
    v *= inv;
    odd = !isfinite(v);
    out[col] = Elem<T>::from_float(v);
  }
  if (p.lse && threadIdx.x == 0) p.lse[row] = sum == 0.f ? -INFINITY : lse_of<(int)kLift<T>>(top, sum);
  if (__syncthreads_or(odd) && warp == 0) {  // what came out infinite or NaN again, key by key
    RowState<kCols> st;
    plain_part<T>(p, slot, h, h / (p.q_heads / p.kv_heads), st, 0, 1);
    mend_row(st, out, p.d, lane);
  }
}

template <class T, int DP>
int launch_shared(int dtype, SharedParams &sp, cudaStream_t s) {
  using L = SharedLayout<DP>;
  const DecodeParams &p = sp.p;
  auto *kernel = shared_kernel<T, DP>;
  static bool configured[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    if (int rc = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::bytes(kMostSlots)), "shared prefix memory"))
      return rc;
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  sp.ctas = std::min(sm_count(), kMostCtas);
  sp.runs = p.dense && p.page_size % 16 == 0;
  sp.q_pieces = aligned(p.q, 16) && p.qs[0] % 8 == 0 && p.qs[1] % 8 == 0;
  const int64_t rows = (int64_t)p.slots * p.q_heads, parts = cut_rows(sp.ctas) + rows * kTiles;
  void *mem = nullptr;
  Suffix suffix = {sp.sharing, nullptr, nullptr};
  if (int rc = device_error_word(&sp.err)) return rc;
  if (int rc = scratch_buffer(s, kSumsSlot, (size_t)parts * DP * 4, &mem)) return rc;
  sp.sums = static_cast<float *>(mem);
  if (int rc = scratch_buffer(s, kStatsSlot, (size_t)parts * 8, &mem)) return rc;
  sp.stats = static_cast<float2 *>(mem);
  if (int rc = scratch_buffer(s, kWhereSlot, (size_t)rows * 16, &mem)) return rc;
  sp.where = static_cast<int4 *>(mem);
  if (int rc = scratch_buffer(s, kOwnSumsSlot, (size_t)rows * DP * 4, &mem)) return rc;
  suffix.sums = static_cast<float *>(mem);
  if (int rc = scratch_buffer(s, kOwnStatsSlot, (size_t)rows * 8, &mem)) return rc;
  suffix.stats = static_cast<float2 *>(mem);
  if (int rc = check_cuda(launch_pdl(kernel, dim3(sp.ctas), dim3(kThreads), L::bytes(p.slots), s, sp), "lc_shared_decode")) return rc;
  if (int rc = decode_suffix(dtype, p, suffix, s)) return rc;
  return check_cuda(launch_pdl(merge_kernel<T, DP>, dim3((unsigned)rows), dim3(kMergeWarps * 32), 0, s, sp,
                               suffix.sums, suffix.stats),
                    "lc_shared_decode (merge)");
}

// Whether reading the prefixes once can pay, by what all slots' keys and values may come to: below, lc_paged_decode,
// which finds what another slot has read in L2, is done before three kernels are (64 samples of 300 tokens, 8 heads of
// 128, 100 MB: 25 us against 37; 8 prompts of 8 samples, 2.1 GB: 174 against 75; 4 of 16, heads of 64, 1 GB: 110, 42).
constexpr int64_t kWorthBytes = 192 << 20;
// (The units of all segments together, times the CTAs, are counted in 32 bits.)
bool worth_sharing(const DecodeParams &p) {
  const int64_t rows = (int64_t)p.slots * p.q_heads, blocks = (int64_t)p.width * p.page_size / kKeys + 3;
  if ((rows / (kTiles * kRows) + (int64_t)p.slots * p.kv_heads) * blocks >= INT32_MAX / kMostCtas) return false;
  return (int64_t)p.slots * p.width * p.page_size * p.kv_heads * p.d * 4 >= kWorthBytes;
}

}  // namespace
}  // namespace lc

extern "C" int lc_shared_decode(int dtype, const void *q, const void *k, const void *v, void *o, float *lse, const int32_t *table,
                                const int32_t *lens, const int32_t *leader, const int32_t *shared, const int32_t *order, int64_t slots,
                                int64_t width, int64_t pages, int64_t page_size, int64_t q_heads, int64_t kv_heads, int64_t d,
                                const int64_t *strides, int64_t window, int64_t sinks, float scale, void *stream) {
  using namespace lc;
  const char *me = "lc_shared_decode";
  SharedParams sp = {};
  if (int rc = decode_params(me, sp.p, dtype, q, k, v, o, lse, table, lens, slots, width, pages, page_size, q_heads, kv_heads, d, strides,
                             window, sinks, scale))
    return rc;
  if (slots > kMostSlots) return fail(LC_ERR_UNSUPPORTED, "%s: %lld slots, at most %d", me, (long long)slots, kMostSlots);
  if (slots == 0) return LC_OK;
  if (!leader || !shared || !order) return fail(LC_ERR_INVALID, "%s: null buffer", me);
  sp.sharing = {leader, shared, order};
  cudaStream_t s = as_stream(stream);
  if (d > 128 || decode_few_keys(sp.p) || !decode_tensor(sp.p) || !worth_sharing(sp.p)) return decode_all(dtype, sp.p, s);
  if (dtype == LC_F16) return d <= 64 ? launch_shared<__half, 64>(dtype, sp, s) : launch_shared<__half, 128>(dtype, sp, s);
  return d <= 64 ? launch_shared<__nv_bfloat16, 64>(dtype, sp, s) : launch_shared<__nv_bfloat16, 128>(dtype, sp, s);
}
