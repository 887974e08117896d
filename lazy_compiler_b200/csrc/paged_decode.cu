// Attention of one new token of every sequence over its paged key-value cache
// (the single-token form of window_attention.cu): slot s has lens[s] cached
// tokens, its query is the last of them, and token j is row j % page_size of
// page table[s][j / page_size].  The same kernels, instantiated with a Suffix, take
// the tokens behind the prefixes that slots share, for shared_decode.cu, and leave the
// rows unnormalised.
#include <algorithm>

#include "paged.cuh"
#include "softmax.cuh"

namespace lc {

using namespace attend;

namespace {

constexpr int kPartialsSlot = 41, kArrivedSlot = 42, kSpansSlot = 46;  // scratch_buffer slots

// ---------------------------------------------------------------- plain form
// One CTA of eight warps per (slot, query head): few keys, and what the tensor-core form
// below does not take (odd head sizes and alignments).
constexpr int kRowWarps = 8;

template <class T, int NC>
__global__ void __launch_bounds__(kRowWarps * 32) decode_row_kernel(DecodeParams p) {
  __shared__ float scratch[kRowWarps * (32 * NC + 2)];
  pdl_wait();
  pdl_trigger();
  const int slot = blockIdx.x, h = blockIdx.y;
  RowState<NC> st;
  plain_row<T, kRowWarps>(p, slot, h, h / (p.q_heads / p.kv_heads), st, scratch);
  if (threadIdx.x < 32)
    store_row(st, static_cast<T *>(p.o) + slot * p.os[0] + h * p.os[1],
              p.lse ? p.lse + (int64_t)slot * p.q_heads + h : nullptr, p.d, threadIdx.x);
}

// ---------------------------------------------------------------- tensor-core form
// Reading the cache is all the work (4 flops per element and query head), so the
// kernel is built around keeping loads in flight.
//
// Work is cut by length, not by sequence: all (slot, key-value head, group of 8 NT
// query heads) segments are laid end to end as tiles of 64 keys, and each CTA takes
// an equal contiguous run of them (kEndUnits says how equal), so a batch of unequal lengths and a single long
// sequence both fill the GPU.  A segment that spans CTAs leaves an unnormalised
// (O, m, l) per CTA in the workspace; the CTA that arrives last joins them in CTA
// order (the run boundaries depend on the lengths alone, so results repeat), or,
// where a segment may span kDeepParts of them or more, a second kernel with a CTA per row (one
// sequence of 131072 with one key-value head, 444 parts: 21 us, 167 with the last CTA, which
// reads 1.9 MB alone; 4 of 1 to 8192 tokens, 8 heads: 20.3 us, 24.7 with it from 16 parts on; one
// of 512: 9.2, 11.1).  The host chooses, by the table's width and an even share of the CTAs: it does
// not know the lengths.  So one long sequence among many short ones is joined by the last CTAs (64
// slots, 8 heads, one of 131072 tokens, the others 100: 97 us where its bytes take 87; of 32768: 40, 25).
//
// In a CTA each warp takes 16 keys of every tile and is on its own until the
// segment ends: it copies its keys' rows (cp.async, 16 bytes per lane, zeros where
// a key is not visible, so what an unused row holds never enters a product) through
// a private ring of STAGES tiles, and computes
//   S^T[16 keys, 8 heads] = K Q^T          (mma.sync m16n8k16, Q in registers)
//   O^T[D, 8 heads] += V^T P^T             (P^T by movmatrix from S^T's registers)
// with the heads along N: 8 query heads of a group fill the instruction, and a
// thread holds the same two heads in S^T and O^T, so rescaling needs no exchange.
// tcgen05 has no use here: its 128-row tiles would be 1/16 full, and the tensor
// pipe is idle most of the time as it is.
// P is split into two 16-bit parts (value and remainder) and multiplied twice: the
// extra products hide behind the loads and keep P to 16 bits or more.  An f16 part ends at
// 2^-25, where a bf16 one has f32's range, so f16 weights are taken 2^kLift larger (the row's
// reference is its maximum less kLift): a weight is off by 2^-39 of the row's largest one at most,
// and a long tail below a sink that outweighs it is not lost.
// Bound by HBM.  Measured, 32/8 heads of 128, bf16: 64 sequences of 1 to 8192 tokens
// in pages of 16: 167 us, 6440 GB/s, the rate of a copy; 64/8, f16, 100003 and 131072
// tokens: 147 us, 6430 GB/s.  Three CTAs per SM of two stages against two of three:
// the warps' own latency (a tile is a chain of some 500 instructions) needs 12 of them
// (177 us with 8).  Heads of 64, half the bytes a tile and nearly its instructions: four CTAs of
// three stages (1 to 8192 tokens, before kEndUnits: 98 us; 105 with three of four, 98 with five of two, 111 with six of two;
// groups of 16: 127, 161 with two of six).
constexpr int kDecodeWarps = 4;
constexpr int kTileKeys = 16;
constexpr int kDeepParts = 5;
constexpr int kMinTiles = 2;  // CTA tiles below which a segment is not cut further
// Runs are cut into equal numbers of units, a tile's time each: a segment's end (the warps' sums
// joined and written) counts as one too, or a CTA of nine segments of a tile each is done long after
// the one beside it (64 sequences of 1 to 1000 tokens: 44.0 us without, 33.3 with one, 32.8 with
// two, 33.0 with three; of 1 to 250: 18.7, 17.0, 17.7, 17.9; of 1 to 8192: 169, 168, 168, 170).
constexpr int kEndUnits = 1;
// A cut this many tiles or fewer from an end of a segment moves there: one tile more or less is
// cheaper than a segment that two CTAs have to join (64 sequences of 1 to 250 tokens: 16.7 -> 13.9 us,
// 8 of 1 to 512: 15.3 -> 13.3, but 64 of 1 to 500: 23.3 -> 25.2; two tiles make short caches of few
// heads worse, 2000 tokens of 2 heads: 9.0 -> 10.7).
constexpr int kSnap = 1;

// The largest weight of a row is 2^kLift: f16's far from its largest number, with sums in f32.
template <class T>
constexpr float kLift = kLiftBf16;
template <>
constexpr float kLift<__half> = 14.f;

template <class T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ void copy_async16(uint32_t dst, const void *src) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// 16 bytes to shared memory; zeros, and no read, where `bytes` is 0.
__device__ __forceinline__ void copy_async16(uint32_t dst, const void *src, int bytes) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
template <class T>
__device__ __forceinline__ uint32_t pack(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
template <class T>
__device__ __forceinline__ float round_to(float v) {
  return Elem<T>::to_float(Elem<T>::from_float(v));
}

// One slot's tiles of 16 keys: those of the sinks, then those from the window's
// start on (a tile both reach counts once).
struct SlotTiles {
  int n, sink_end, lo;       // keys, and the visible ones: j < sink_end or j >= lo
  int sink_tiles, first, tiles;  // tile x is keys 16 (x < sink_tiles ? x : x - sink_tiles + first)
  int from = 0, sink_first = 0;  // with a Suffix: its first key; the first of the sinks' tiles
};
__device__ __forceinline__ SlotTiles slot_tiles(const DecodeParams &p, int slot) {
  SlotTiles t;
  t.n = cached_tokens(p, slot);
  const Visible see = visible(t.n - 1, p.window, p.sinks);
  t.sink_end = see.sink_end;
  t.lo = see.lo;
  t.sink_tiles = (t.sink_end + kTileKeys - 1) / kTileKeys;
  t.first = max(t.lo / kTileKeys, t.sink_tiles);
  t.tiles = t.n <= 0 ? 0 : t.sink_tiles + (t.n + kTileKeys - 1) / kTileKeys - t.first;
  return t;
}
// The tiles that hold a key of the suffix.
__device__ __forceinline__ SlotTiles slot_tiles(const DecodeParams &p, int slot, const Suffix &suffix) {
  SlotTiles t;
  t.n = cached_tokens(p, slot);
  const Visible see = visible(t.n - 1, p.window, p.sinks);
  t.from = min(group_prefix(p, suffix.sharing, slot), t.n);
  t.lo = max(see.lo, t.from);
  t.sink_end = see.sink_end > t.from ? see.sink_end : 0;
  t.sink_first = t.sink_end ? t.from / kTileKeys : 0;
  t.sink_tiles = (t.sink_end + kTileKeys - 1) / kTileKeys - t.sink_first;
  t.first = max(t.lo / kTileKeys, t.sink_first + t.sink_tiles);
  t.tiles = t.n <= t.from ? 0 : t.sink_tiles + max(0, (t.n + kTileKeys - 1) / kTileKeys - t.first);
  return t;
}
__device__ __forceinline__ int cta_tiles(const SlotTiles &t) { return (t.tiles + kDecodeWarps - 1) / kDecodeWarps; }

// A place in the sequence of all tiles.
struct Cursor {
  SlotTiles tiles;
  int slot, part, t, count;  // part: (head, group) of the slot; t of count CTA tiles
};
template <class... WithSuffix>
__device__ __forceinline__ void advance(Cursor &c, const DecodeParams &p, int parts, const WithSuffix &...suffix) {
  if (++c.t < c.count) return;
  c.t = 0;
  if (++c.part < parts) return;
  c.part = 0;
  do {
    if (++c.slot >= p.slots) return;
    c.tiles = slot_tiles(p, c.slot, suffix...);
    c.count = cta_tiles(c.tiles);
  } while (c.count == 0);
}

// a / b for counts: 32 bits where a has no more, which is a fifth of the instructions.
__device__ __forceinline__ long long quotient(long long a, long long b) {
  return (a >> 32) == 0 ? (long long)((unsigned)a / (unsigned)b) : a / b;
}

struct DecodeWork {
  float *partials;    // [CTA][2][rows][DP + 4]: of a segment that began before the CTA, of one that began in it
  unsigned *arrived;  // [slots * parts], zero between launches
  // deep: segments span so many CTAs that decode_join_kernel joins them; the segment
  // (slot * parts + part) that began in a CTA and goes on after it, or -1, and its last CTA
  int deep, ctas;
  int2 *spans;
};

template <class T, int DP, int NT, int STAGES>
struct DecodeLayout {
  static constexpr int kRows = 8 * NT;
  static constexpr int kRowBytes = DP * 2;
  static constexpr int kStageBytes = 2 * kTileKeys * kRowBytes;  // K and V of 16 keys
  static constexpr int kBytes = kDecodeWarps * STAGES * kStageBytes;
  static_assert(kRows * DP * 4 <= kStageBytes, "a warp's sums are joined in its last stage");
};

// What a kernel that takes a Suffix writes of its rows.
template <class... WithSuffix>
struct SuffixRows {};
template <>
struct SuffixRows<Suffix> {
  const Suffix &suffix;
  template <int DP>
  __device__ __forceinline__ float *sums(int64_t row) const {
    return suffix.sums + row * DP;
  }
  __device__ __forceinline__ void stats(int64_t row, float m, float l) const { suffix.stats[row] = make_float2(m, l); }
};

// PAGED16: a tile of 16 keys lies in one page (page_size is a multiple of 16).
// WithSuffix: Suffix, or nothing.
template <class T, int DP, int NT, int STAGES, int CTAS, bool PAGED16, class... WithSuffix>
__device__ __forceinline__ void decode_run(const DecodeParams &p, const DecodeWork &work, const WithSuffix &...suffix) {
  constexpr bool kSuffix = sizeof...(WithSuffix) > 0;
  const SuffixRows<WithSuffix...> rows_to{suffix...};
  using L = DecodeLayout<T, DP, NT, STAGES>;
  constexpr int kRows = L::kRows;
  constexpr int kChunks = DP / 8;                   // 16-byte pieces of a row
  constexpr int kRowsPerCopy = 32 / (kChunks < 32 ? kChunks : 32);
  constexpr int kCopies = kTileKeys / kRowsPerCopy;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ unsigned masks[kDecodeWarps][STAGES];  // the visible keys of each warp's staged tiles
  __shared__ float scratch[kDecodeWarps * (DP + 2)];  // the plain form's joins
  __shared__ float merge_m[kDecodeWarps][kRows], merge_l[kDecodeWarps][kRows], merge_w[kDecodeWarps][kRows];
  __shared__ float row_m[kRows], row_l[kRows];
  __shared__ long long sums[kDecodeWarps], tile_sums[kDecodeWarps];
  __shared__ int start_slot, start_part, start_t;
  __shared__ long long unit_at[2], tile_at[2];
  __shared__ unsigned ticket;

  // Before a join the next kernel is not let in early: the join's CTAs, and the next call's behind
  // them, on SMs that are still reading cost more than their launch (5 x 32687 tokens, heads of 64,
  // call after call: 60 us, 82 let in).
  if (!work.deep) pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int group = p.q_heads / p.kv_heads;
  const int chunks = (group + kRows - 1) / kRows;
  const int parts = p.kv_heads * chunks;

  // ---- this CTA's run of tiles
  const int per = (p.slots + kDecodeWarps * 32 - 1) / (kDecodeWarps * 32);
  const int s0 = min(p.slots, tid * per), s1 = min(p.slots, s0 + per);
  // units: a segment's tiles and kEndUnits for its end
  long long own = 0, own_tiles = 0;
  auto units_of = [&](int count) { return (long long)(count ? count + kEndUnits : 0) * parts; };
  for (int s = s0; s < s1; ++s) {
    const int count = cta_tiles(slot_tiles(p, s, suffix...));
    own += units_of(count);
    own_tiles += (long long)count * parts;
  }
  long long inc = own, inc_tiles = own_tiles;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, inc, o), up_tiles = __shfl_up_sync(0xffffffffu, inc_tiles, o);
    if (lane >= o) inc += up, inc_tiles += up_tiles;
  }
  if (lane == 31) sums[warp] = inc, tile_sums[warp] = inc_tiles;
  __syncthreads();
  long long before = inc - own, total = 0, before_tiles = inc_tiles - own_tiles, total_tiles = 0;
#pragma unroll
  for (int w = 0; w < kDecodeWarps; ++w) {
    if (w < warp) before += sums[w], before_tiles += tile_sums[w];
    total += sums[w];
    total_tiles += tile_sums[w];
  }
  // a CTA for every kMinTiles tiles, or for every segment, if those are more (4 sequences of 1 to 128
  // tokens, 8 heads: 8.9 us; 10.8 with two segments a CTA)
  const long long useful = max((total_tiles + kMinTiles - 1) / kMinTiles, (total - total_tiles) / kEndUnits);
  const long long ctas = useful < (long long)gridDim.x ? useful : (long long)gridDim.x;
  const bool works = blockIdx.x < ctas;
  const long long even_begin = works ? quotient(blockIdx.x * total, ctas) : 0, even_end = works ? quotient((blockIdx.x + 1) * total, ctas) : 0;
  // where the run begins, and the numbers of its first tile and of the one behind it
  if (works) {
#pragma unroll 1
    for (int x = 0; x < 2; ++x) {
      const long long unit = x ? even_end : even_begin;
      if (unit < before || unit >= before + own) continue;
      long long at = before, at_tile = before_tiles;
      int s = s0, count;
      for (;; ++s) {
        count = cta_tiles(slot_tiles(p, s, suffix...));
        if (unit < at + units_of(count)) break;
        at += units_of(count);
        at_tile += (long long)count * parts;
      }
      const long long in = unit - at, seg = quotient(in, count + kEndUnits), t = in - seg * (count + kEndUnits);
      const int to = 2 * t < count ? (t <= kSnap ? 0 : (int)t) : (t >= count - kSnap ? count : (int)t);
      unit_at[x] = unit - t + to;
      tile_at[x] = at_tile + seg * count + to;
      if (x == 0) {
        start_slot = s;
        start_part = (int)seg;
        start_t = to;
      }
    }
    if (even_end == total && tid == 0) {
      unit_at[1] = total;
      tile_at[1] = total_tiles;
    }
  }
  // slots with nothing to see
  for (int s = blockIdx.x; s < p.slots; s += gridDim.x) {
    if (slot_tiles(p, s, suffix...).tiles != 0) continue;
    if constexpr (kSuffix) {
      for (int h = tid; h < p.q_heads; h += blockDim.x) rows_to.stats((int64_t)s * p.q_heads + h, -INFINITY, 0.f);
    } else {
      for (int i = tid; i < p.q_heads * p.d; i += blockDim.x) {
        const int h = i / p.d;
        static_cast<T *>(p.o)[s * p.os[0] + h * p.os[1] + (i - h * p.d)] = Elem<T>::from_float(0.f);
      }
      if (p.lse)
        for (int h = tid; h < p.q_heads; h += blockDim.x) p.lse[(int64_t)s * p.q_heads + h] = -INFINITY;
    }
  }
  if (work.deep && tid == 0) work.spans[blockIdx.x] = make_int2(-1, -1);
  __syncthreads();
  if (!works) return;
  const long long begin = unit_at[0], end = unit_at[1];
  const int steps = (int)(tile_at[1] - tile_at[0]);
  if (steps == 0) return;  // its cuts have moved together, or only a segment's end lies between

  Cursor load;
  load.slot = start_slot;
  load.tiles = slot_tiles(p, load.slot, suffix...);
  load.count = cta_tiles(load.tiles);
  load.part = start_part;
  load.t = start_t;
  int64_t seg_begin = begin - load.t;  // unit of the current segment's first tile in the sequence of all
  if (load.t >= load.count) {          // behind a segment's last tile: the next one
    seg_begin += load.count + kEndUnits;
    load.t = load.count - 1;
    advance(load, p, parts, suffix...);
  }
  Cursor use = load;

  // ---- loading: lane l copies piece l % kChunks of rows l / kChunks, ...
  const int piece = lane % kChunks, piece_row = lane / kChunks;
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * STAGES * L::kStageBytes;
  const bool piece_real = piece * 8 < p.d;
  int page = -1;  // of the tile the load cursor is at (PAGED16), or of its key `lane`
  auto key_of_tile = [&](const Cursor &c) {
    const int x = c.t * kDecodeWarps + warp;
    const int sink = kSuffix ? c.tiles.sink_first : 0;
    return x < c.tiles.tiles ? kTileKeys * (x < c.tiles.sink_tiles ? x + sink : x - c.tiles.sink_tiles + c.tiles.first) : -1;
  };
  auto find_page = [&]() {
    const int key = key_of_tile(load);
    page = -1;
    if (key < 0) return;
    if (PAGED16) {
      page = p.table[load.slot * p.ts + page_index(p, key)];
    } else {
      const int j = key + (lane & 15);
      if (j < load.tiles.n) page = p.table[load.slot * p.ts + page_index(p, j)];
    }
  };
  auto issue = [&](int stage) {
    const int key = key_of_tile(load);
    const int j = key + (lane & 15);
    const bool sees = key >= 0 && (unsigned)page < (unsigned)p.pages && j < load.tiles.n &&
                      (j >= load.tiles.lo || (j < load.tiles.sink_end && (!kSuffix || j >= load.tiles.from)));
    const unsigned mask = __ballot_sync(0xffffffffu, sees) & 0xffffu;
    if (lane == 0) masks[warp][stage] = mask;
    // Piece x of row r lies at x ^ (r & 7).  A lane's rows are i * kRowsPerCopy + piece_row, whose
    // two parts share no bit, so the i-th address differs from the first by constants.
    const uint32_t dst = ring + stage * L::kStageBytes + piece_row * L::kRowBytes + ((piece ^ (piece_row & 7)) << 4);
    auto dst_of = [&](int i) { return (dst ^ ((i * kRowsPerCopy & 7) << 4)) + i * kRowsPerCopy * L::kRowBytes; };
    constexpr uint32_t kV = kTileKeys * L::kRowBytes;  // V behind K
    if (PAGED16 && mask == 0xffffu && p.dense) {  // one run of memory each
      const int head = load.part / chunks, r = key - page_index(p, key) * p.page_size;
      const T *k = static_cast<const T *>(p.k) + page * p.ks[0] + head * p.ks[1] + r * DP + lane * 8;
      const T *v = static_cast<const T *>(p.v) + page * p.vs[0] + head * p.vs[1] + r * DP + lane * 8;
#pragma unroll
      for (int i = 0; i < kCopies; ++i) copy_async16(dst_of(i), k + i * 256);
#pragma unroll
      for (int i = 0; i < kCopies; ++i) copy_async16(dst_of(i) + kV, v + i * 256);
    } else if (mask) {
      const int head = load.part / chunks;
      int64_t k_off, v_off;
      if (PAGED16) {
        const int r = key - page_index(p, key) * p.page_size;
        k_off = page * p.ks[0] + head * p.ks[1] + (r + piece_row) * p.ks[2] + piece * 8;
        v_off = page * p.vs[0] + head * p.vs[1] + (r + piece_row) * p.vs[2] + piece * 8;
      } else {
        const int r = j - page_index(p, j) * p.page_size;
        k_off = page * p.ks[0] + head * p.ks[1] + r * p.ks[2];
        v_off = page * p.vs[0] + head * p.vs[1] + r * p.vs[2];
      }
#pragma unroll
      for (int i = 0; i < kCopies; ++i) {
        const int row = i * kRowsPerCopy + piece_row;
        const int bytes = (mask >> row & 1) && piece_real ? 16 : 0;
        int64_t ko, vo;
        if (PAGED16) {
          ko = k_off + (int64_t)(i * kRowsPerCopy) * p.ks[2];
          vo = v_off + (int64_t)(i * kRowsPerCopy) * p.vs[2];
        } else {
          ko = __shfl_sync(0xffffffffu, k_off, row) + piece * 8;
          vo = __shfl_sync(0xffffffffu, v_off, row) + piece * 8;
        }
        copy_async16(dst_of(i), static_cast<const T *>(p.k) + (bytes ? ko : 0), bytes);
        copy_async16(dst_of(i) + kV, static_cast<const T *>(p.v) + (bytes ? vo : 0), bytes);
      }
    }
  };

  // ---- computing
  uint32_t q[NT][DP / 16][2];
  float o[NT][DP / 16][4];
  float m[NT][2], l[NT][2];
  const int g = lane >> 2, c2 = (lane & 3) * 2;
  auto start_segment = [&]() {
    const int head = use.part / chunks, first = head * group + use.part % chunks * kRows;
    const int live = min(kRows, (head + 1) * group - first);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const T *row = static_cast<const T *>(p.q) + use.slot * p.qs[0] + (first + nt * 8 + g) * p.qs[1];
      const bool real = nt * 8 + g < live;
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int c = k * 16 + x * 8 + c2;
          q[nt][k][x] = real && c < p.d ? *reinterpret_cast<const uint32_t *>(row + c) : 0u;
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) o[nt][k][x] = 0.f;
      }
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
    }
  };
  auto compute = [&](int stage) {
    const unsigned mask = masks[warp][stage];
    if (!mask) return;
    const uint32_t k_src = ring + stage * L::kStageBytes, v_src = k_src + kTileKeys * L::kRowBytes;
    float s[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
    // K: rows 0-7, 8-15 of pieces 2k, then 2k + 1
    const int k_row = lane & 15;
    const uint32_t k_at = k_src + k_row * L::kRowBytes + (((lane >> 4) ^ (k_row & 7)) << 4);
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) {
      uint32_t a[4];
      ldmatrix4(a, (k_at ^ ((2 * k & 7) << 4)) + (2 * k >> 3) * 128);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mma16816<T>(s[nt], a, q[nt][k][0], q[nt][k][1]);
    }
    uint32_t hi[NT][2], lo[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      // s: (key g, heads c2, c2 + 1), (key g + 8, the same heads)
#pragma unroll
      for (int x = 0; x < 4; ++x) s[nt][x] *= p.scale_log2;
      if (mask != 0xffffu) {
#pragma unroll
        for (int x = 0; x < 4; ++x)
          if (!(mask >> (g + (x >> 1) * 8) & 1)) s[nt][x] = -INFINITY;
      }
      float top[2] = {fmaxf(s[nt][0], s[nt][2]), fmaxf(s[nt][1], s[nt][3])};
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 4));
        top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 8));
        top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 16)) - kLift<T>;
      }
      const bool grew = top[0] > m[nt][0] || top[1] > m[nt][1];
      if (__any_sync(0xffffffffu, grew)) {
        float alpha[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float m_new = fmaxf(m[nt][x], top[x]);
          alpha[x] = softmax::ex2(m[nt][x] - (m_new == -INFINITY ? 0.f : m_new));
          m[nt][x] = m_new;
          l[nt][x] *= alpha[x];
        }
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
          o[nt][k][0] *= alpha[0];
          o[nt][k][1] *= alpha[1];
          o[nt][k][2] *= alpha[0];
          o[nt][k][3] *= alpha[1];
        }
      }
      const float base[2] = {m[nt][0] == -INFINITY ? 0.f : m[nt][0], m[nt][1] == -INFINITY ? 0.f : m[nt][1]};
      float e[4], r[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        e[x] = softmax::ex2(s[nt][x] - base[x & 1]);
        l[nt][x & 1] += e[x];
        r[x] = round_to<T>(e[x]);
      }
      hi[nt][0] = movmatrix_trans(pack<T>(r[0], r[1]));
      hi[nt][1] = movmatrix_trans(pack<T>(r[2], r[3]));
      lo[nt][0] = movmatrix_trans(pack<T>(e[0] - r[0], e[1] - r[1]));
      lo[nt][1] = movmatrix_trans(pack<T>(e[2] - r[2], e[3] - r[3]));
    }
    // V^T: (keys 0-7, pieces 2k, 2k + 1), then keys 8-15
    const int v_row = (lane & 7) + (lane >> 4) * 8;
    const uint32_t v_at = v_src + v_row * L::kRowBytes + (((lane >> 3 & 1) ^ (v_row & 7)) << 4);
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) {
      uint32_t a[4];
      ldmatrix4_trans(a, (v_at ^ ((2 * k & 7) << 4)) + (2 * k >> 3) * 128);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        mma16816<T>(o[nt][k], a, hi[nt][0], hi[nt][1]);
        mma16816<T>(o[nt][k], a, lo[nt][0], lo[nt][1]);
      }
    }
  };

  // ---- ending a segment: the warps' states joined, and the CTAs' where there are several
  constexpr int kPartial = kRows * (DP + 4);  // floats; m and l at DP, DP + 1 of a row
  // a thread's share of the rows x DP sums: columns col + 128 y of rows first_row + kSplit x
  constexpr int kCols = DP < 128 ? DP : 128, kSplit = kDecodeWarps * 32 / kCols, kRpt = kRows / kSplit, kCpt = DP / kCols;
  const int col = tid % kCols, first_row = tid / kCols;
  auto write_rows = [&](const float (&values)[kRpt][kCpt]) {  // O / l and the log-sum-exp; whether all is finite
    const int head = use.part / chunks, first = head * group + use.part % chunks * kRows;
    const int live = min(kRows, (head + 1) * group - first);
    bool odd = false;
    if constexpr (kSuffix) {
#pragma unroll
      for (int x = 0; x < kRpt; ++x) {
        const int row = first_row + kSplit * x;
        if (row >= live) continue;
        float *to = rows_to.template sums<DP>((int64_t)use.slot * p.q_heads + first + row);
#pragma unroll
        for (int y = 0; y < kCpt; ++y) to[col + kCols * y] = values[x][y];
      }
      if (tid < live) rows_to.stats((int64_t)use.slot * p.q_heads + first + tid, row_m[tid], row_l[tid]);
    } else {
#pragma unroll
      for (int x = 0; x < kRpt; ++x) {
        const int row = first_row + kSplit * x;
        if (row >= live) continue;
        const float sum = row_l[row], inv = sum == 0.f ? 0.f : 1.f / sum;
        T *out = static_cast<T *>(p.o) + use.slot * p.os[0] + (first + row) * p.os[1];
#pragma unroll
        for (int y = 0; y < kCpt; ++y) {
          const float v = values[x][y] * inv;
          if (col + kCols * y < p.d) {
            odd |= !isfinite(v);
            out[col + kCols * y] = Elem<T>::from_float(v);
          }
        }
      }
      if (p.lse && tid < live)
        p.lse[(int64_t)use.slot * p.q_heads + first + tid] = row_l[tid] == 0.f ? -INFINITY : lse_of<(int)kLift<T>>(row_m[tid], row_l[tid]);
    }
    return odd;
  };
  // What came out infinite or NaN is computed again one key at a time: the
  // remainder's products can turn an infinite value into NaN.
  auto plain_rows = [&]() {
    const int head = use.part / chunks, first = head * group + use.part % chunks * kRows;
    const int live = min(kRows, (head + 1) * group - first);
    for (int x = 0; x < live; ++x) {
      RowState<DP / 32> st;
      __syncthreads();
      plain_row<T, kDecodeWarps>(p, use.slot, first + x, head, st, scratch);
      if (warp == 0) mend_row(st, static_cast<T *>(p.o) + use.slot * p.os[0] + (first + x) * p.os[1], p.d, lane);
    }
  };
  auto end_segment = [&](long long seg_end, int stage) {
    // The stage just used is free until the next copies: each warp leaves its sums
    // there, column c of heads 2 t, 2 t + 1 at c ^ 8 t, off each other's banks.
    auto sums_of = [&](int w) { return reinterpret_cast<float *>(smem + (w * STAGES + stage) * L::kStageBytes); };
    float *mine = sums_of(warp);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float sum = l[nt][x];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        if (g == 0) {
          merge_m[warp][nt * 8 + c2 + x] = m[nt][x];
          merge_l[warp][nt * 8 + c2 + x] = sum;
        }
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
          float *row = mine + (nt * 8 + c2 + x) * DP;
          row[(k * 16 + g) ^ (c2 << 2)] = o[nt][k][x];
          row[(k * 16 + g + 8) ^ (c2 << 2)] = o[nt][k][2 + x];
        }
      }
    }
    __syncthreads();
    if (tid < kRows) {
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < kDecodeWarps; ++w) top = fmaxf(top, merge_m[w][tid]);
#pragma unroll
      for (int w = 0; w < kDecodeWarps; ++w) {
        const float weight = exp2f(merge_m[w][tid] - (top == -INFINITY ? 0.f : top));
        merge_w[w][tid] = weight;
        sum = fmaf(merge_l[w][tid], weight, sum);
      }
      row_m[tid] = top;
      row_l[tid] = sum;
    }
    __syncthreads();
    float values[kRpt][kCpt];
#pragma unroll
    for (int x = 0; x < kRpt; ++x) {
      const int row = first_row + kSplit * x;
#pragma unroll
      for (int y = 0; y < kCpt; ++y) {
        values[x][y] = 0.f;
#pragma unroll
        for (int w = 0; w < kDecodeWarps; ++w)
          values[x][y] = fmaf(sums_of(w)[row * DP + ((col + kCols * y) ^ ((row & 6) << 2))], merge_w[w][row], values[x][y]);
      }
    }
    bool odd = false;
    if (seg_begin >= begin && seg_end <= end) {
      odd = write_rows(values);
    } else {
      float *partial = work.partials + ((int64_t)blockIdx.x * 2 + (seg_begin >= begin)) * kPartial;
#pragma unroll
      for (int x = 0; x < kRpt; ++x)
#pragma unroll
        for (int y = 0; y < kCpt; ++y) partial[(first_row + kSplit * x) * (DP + 4) + col + kCols * y] = values[x][y];
      if (tid < kRows) {
        partial[tid * (DP + 4) + DP] = row_m[tid];
        partial[tid * (DP + 4) + DP + 1] = row_l[tid];
      }
      // The CTAs whose runs hold the segment's first and last tile: as many run boundaries as there
      // are up to its first kSnap tiles lie before it, those in its last kSnap behind it.
      const int first = (int)quotient((seg_begin + kSnap + 1) * ctas - 1, total), last = (int)quotient((seg_end - kSnap) * ctas - 1, total);
      if (work.deep) {
        if (seg_begin >= begin && tid == 0) work.spans[blockIdx.x] = make_int2(use.slot * parts + use.part, last);
        __syncthreads();  // the sums have been read
        return;
      }
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        unsigned *count = work.arrived + (int64_t)use.slot * parts + use.part;
        ticket = atomicAdd(count, 1u);
        if (ticket == (unsigned)(last - first)) *count = 0;  // for the next launch
      }
      __syncthreads();
      if (ticket != (unsigned)(last - first)) return;
      __threadfence();
      // CTA c's share: the segment began in CTA `first` and before every other
      auto share = [&](int c) { return work.partials + ((int64_t)c * 2 + (c == first)) * kPartial; };
      // Weights first, 64 parts at a time into the free stage of warp 0; then the sums, 16 bytes
      // a thread and eight parts in flight: an SM reads them at the rate its loads arrive.
      constexpr int kThreads = kDecodeWarps * 32, kGroups = kThreads / kRows, kChunk = 64;
      float *weights = sums_of(0), *joined = sums_of(1);
      const int wrow = tid % kRows, wgroup = tid / kRows;
      float top = -INFINITY;
#pragma unroll 4
      for (int c = first + wgroup; c <= last; c += kGroups) top = fmaxf(top, __ldcg(share(c) + wrow * (DP + 4) + DP));
      weights[wgroup * kRows + wrow] = top;
      __syncthreads();
      for (int x = 0; x < kGroups; ++x) top = fmaxf(top, weights[x * kRows + wrow]);
      const float base = top == -INFINITY ? 0.f : top;
      constexpr int kVecs = kRows * DP / 4 / kThreads;  // 16-byte pieces of the rows that a thread adds up
      float4 sum4[kVecs];
#pragma unroll
      for (int x = 0; x < kVecs; ++x) sum4[x] = make_float4(0.f, 0.f, 0.f, 0.f);
      float sum = 0.f;
      for (int from = first; from <= last; from += kChunk) {
        const int parts_here = min(kChunk, last + 1 - from);
        __syncthreads();
        for (int c = wgroup; c < parts_here; c += kGroups) {
          const float2 ml = __ldcg(reinterpret_cast<const float2 *>(share(from + c) + wrow * (DP + 4) + DP));
          const float weight = softmax::ex2(ml.x - base);
          sum = fmaf(ml.y, weight, sum);
          weights[c * kRows + wrow] = weight;
        }
        __syncthreads();
#pragma unroll 8
        for (int c = 0; c < parts_here; ++c) {
          const float *part = share(from + c);
#pragma unroll
          for (int x = 0; x < kVecs; ++x) {
            const int vec = tid + x * kThreads, row = vec / (DP / 4);
            const float4 v = __ldcg(reinterpret_cast<const float4 *>(part + row * (DP + 4) + vec % (DP / 4) * 4));
            const float weight = weights[c * kRows + row];
            sum4[x].x = fmaf(v.x, weight, sum4[x].x);
            sum4[x].y = fmaf(v.y, weight, sum4[x].y);
            sum4[x].z = fmaf(v.z, weight, sum4[x].z);
            sum4[x].w = fmaf(v.w, weight, sum4[x].w);
          }
        }
      }
      __syncthreads();
      weights[wgroup * kRows + wrow] = sum;
#pragma unroll
      for (int x = 0; x < kVecs; ++x) reinterpret_cast<float4 *>(joined)[tid + x * kThreads] = sum4[x];
      __syncthreads();
      if (wgroup == 0) {
        sum = 0.f;
        for (int x = 0; x < kGroups; ++x) sum += weights[x * kRows + wrow];
        row_m[wrow] = top;
        row_l[wrow] = sum;
      }
#pragma unroll
      for (int x = 0; x < kRpt; ++x)
#pragma unroll
        for (int y = 0; y < kCpt; ++y) values[x][y] = joined[(first_row + kSplit * x) * DP + col + kCols * y];
      __syncthreads();
      odd = write_rows(values);
    }
    if (__syncthreads_or(odd)) plain_rows();  // (the sums have been read, too)
  };

  find_page();
#pragma unroll 1
  for (int i = 0; i < STAGES - 1; ++i) {
    if (i < steps) {
      issue(i);
      advance(load, p, parts, suffix...);
      if (i + 1 < steps) find_page();
    }
    copy_commit();
  }
  start_segment();
  int stage = 0;
#pragma unroll 1
  for (int i = 0; i < steps; ++i) {
    copy_wait<STAGES - 2>();
    __syncwarp();  // this stage has landed, and the one before has been read, in every lane
    if (i + STAGES - 1 < steps) {
      issue(stage == 0 ? STAGES - 1 : stage - 1);
      advance(load, p, parts, suffix...);
      if (i + STAGES < steps) find_page();
    }
    copy_commit();
    compute(stage);
    if (use.t + 1 == use.count || i + 1 == steps) {
      end_segment(seg_begin + use.count, stage);
      seg_begin += use.count + kEndUnits;
      if (i + 1 < steps) {
        use.t = use.count - 1;
        advance(use, p, parts, suffix...);
        start_segment();
      }
    } else {
      ++use.t;
    }
    stage = stage + 1 == STAGES ? 0 : stage + 1;
  }
}

template <class T, int DP, int NT, int STAGES, int CTAS, bool PAGED16>
__global__ void __launch_bounds__(kDecodeWarps * 32, CTAS) decode_kernel(DecodeParams p, DecodeWork work) {
  pdl_wait();
  decode_run<T, DP, NT, STAGES, CTAS, PAGED16>(p, work);
}
// The kernel before it, which takes the prefixes, let this one in when all before that was done, and neither
// reads what the other writes: so it waits at its end, for what comes after both.
template <class T, int DP, int NT, int STAGES, int CTAS, bool PAGED16>
__global__ void __launch_bounds__(kDecodeWarps * 32, CTAS) suffix_kernel(DecodeParams p, DecodeWork work, Suffix suffix) {
  decode_run<T, DP, NT, STAGES, CTAS, PAGED16>(p, work, suffix);
  pdl_wait();
}

// Joins the segments that span CTAs: blockIdx.x counts them, blockIdx.y is a row; the
// parts are dealt to eight warps, each with a running maximum.  A chain of three reads: the
// spans, the parts, all of a warp's first kAtOnce together, and the eight warps' sums.
constexpr int kJoinWarps = 8;
constexpr int kMostSpans = 4;  // of a thread: up to 1024 CTAs

template <class T, int DP, int NT, class... WithSuffix>
__global__ void __launch_bounds__(kJoinWarps * 32) decode_join_kernel(DecodeParams p, DecodeWork work, WithSuffix... suffix) {
  constexpr bool kSuffix = sizeof...(WithSuffix) > 0;
  constexpr int kRows = 8 * NT, kCols = DP / 32, kAtOnce = 8;
  __shared__ float scratch[kJoinWarps * (DP + 2)];
  __shared__ int counts[kMostSpans * kJoinWarps];
  __shared__ int2 found;  // the first and the last CTA's span
  __shared__ int found_at;
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int2 mine[kMostSpans];
#pragma unroll
  for (int x = 0; x < kMostSpans; ++x) {
    const int c = x * kJoinWarps * 32 + tid;
    mine[x] = c < work.ctas ? work.spans[c] : make_int2(-1, -1);
  }
#pragma unroll
  for (int x = 0; x < kMostSpans; ++x) {
    const unsigned some = __ballot_sync(0xffffffffu, mine[x].x >= 0);
    if (lane == 0) counts[x * kJoinWarps + warp] = __popc(some);
    if (mine[x].x >= 0) mine[x].y |= __popc(some & ((1u << lane) - 1)) << 16;  // its rank in the warp beside the CTA
  }
  if (tid == 0) found_at = -1;
  __syncthreads();
  const int upto = counts[lane];  // kMostSpans * kJoinWarps is a warp's lanes
  int before = upto;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += up;
  }
  before -= upto;
#pragma unroll
  for (int x = 0; x < kMostSpans; ++x) {
    const int rank = __shfl_sync(0xffffffffu, before, x * kJoinWarps + warp) + (mine[x].y >> 16);
    if (mine[x].x >= 0 && rank == (int)blockIdx.x) {
      found_at = x * kJoinWarps * 32 + tid;
      found = make_int2(mine[x].x, mine[x].y & 0xffff);
    }
  }
  __syncthreads();
  const int first = found_at, row = blockIdx.y;
  if (first < 0) return;
  const int2 span = found;
  const int group = p.q_heads / p.kv_heads, chunks = (group + kRows - 1) / kRows, parts = p.kv_heads * chunks;
  const int slot = span.x / parts, part = span.x % parts, head = part / chunks, h = head * group + part % chunks * kRows + row;
  if (h >= (head + 1) * group) return;
  // CTA c's share of the row: the segment began in CTA `first` and before every other
  auto share = [&](int c) { return work.partials + ((int64_t)c * 2 + (c == first)) * kRows * (DP + 4) + row * (DP + 4); };
  float top = -INFINITY, sum = 0.f, o[kCols];
#pragma unroll
  for (int x = 0; x < kCols; ++x) o[x] = 0.f;
#pragma unroll 1
  for (int c0 = first + warp; c0 <= span.y; c0 += kAtOnce * kJoinWarps) {
    float2 ml[kAtOnce], two[kAtOnce][kCols / 2];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int c = c0 + u * kJoinWarps;
      ml[u] = make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int x = 0; x < kCols / 2; ++x) two[u][x] = make_float2(0.f, 0.f);
      if (c <= span.y) {
        const float *from = share(c);
        ml[u] = __ldcg(reinterpret_cast<const float2 *>(from + DP));
#pragma unroll
        for (int x = 0; x < kCols / 2; ++x) two[u][x] = __ldcg(reinterpret_cast<const float2 *>(from + lane * kCols + x * 2));
      }
    }
    float top_new = top;
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) top_new = fmaxf(top_new, ml[u].x);
    const float base = top_new == -INFINITY ? 0.f : top_new, alpha = softmax::ex2(top - base);
    top = top_new;
    sum *= alpha;
#pragma unroll
    for (int x = 0; x < kCols; ++x) o[x] *= alpha;
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const float weight = softmax::ex2(ml[u].x - base);
      sum = fmaf(ml[u].y, weight, sum);
#pragma unroll
      for (int x = 0; x < kCols / 2; ++x) {
        o[x * 2] = fmaf(two[u][x].x, weight, o[x * 2]);
        o[x * 2 + 1] = fmaf(two[u][x].y, weight, o[x * 2 + 1]);
      }
    }
  }
#pragma unroll
  for (int x = 0; x < kCols; ++x) scratch[warp * (DP + 2) + lane * kCols + x] = o[x];
  if (lane == 0) {
    scratch[warp * (DP + 2) + DP] = sum;
    scratch[warp * (DP + 2) + DP + 1] = top;
  }
  __syncthreads();
  float weights[kJoinWarps];
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) top = fmaxf(top, scratch[w * (DP + 2) + DP + 1]);
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) {
    weights[w] = softmax::ex2(scratch[w * (DP + 2) + DP + 1] - (top == -INFINITY ? 0.f : top));
    sum = fmaf(scratch[w * (DP + 2) + DP], weights[w], sum);
  }
  if constexpr (kSuffix) {
    const SuffixRows<WithSuffix...> rows_to{suffix...};
    const int64_t row_at = (int64_t)slot * p.q_heads + h;
    if (tid < DP) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < kJoinWarps; ++w) v = fmaf(scratch[w * (DP + 2) + tid], weights[w], v);
      rows_to.template sums<DP>(row_at)[tid] = v;
    }
    if (tid == 0) rows_to.stats(row_at, top, sum);
    return;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  T *out = static_cast<T *>(p.o) + slot * p.os[0] + h * p.os[1];
  bool odd = false;
  if (tid < p.d) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) v = fmaf(scratch[w * (DP + 2) + tid], weights[w], v);
    v *= inv;
    odd = !isfinite(v);
    out[tid] = Elem<T>::from_float(v);
  }
  if (p.lse && tid == 0) p.lse[(int64_t)slot * p.q_heads + h] = sum == 0.f ? -INFINITY : lse_of<(int)kLift<T>>(top, sum);
  if (__syncthreads_or(odd)) {  // as in decode_kernel
    RowState<DP / 32> st;
    plain_row<T, kJoinWarps>(p, slot, h, head, st, scratch);
    if (warp == 0) mend_row(st, out, p.d, lane);
  }
}

template <class T, int DP, int NT, int STAGES, int CTAS, bool PAGED16, class... WithSuffix>
int launch_decode(const DecodeParams &p, cudaStream_t s, const WithSuffix &...suffix) {
  using L = DecodeLayout<T, DP, NT, STAGES>;
  auto *kernel = [] {
    if constexpr (sizeof...(WithSuffix) > 0)
      return suffix_kernel<T, DP, NT, STAGES, CTAS, PAGED16>;
    else
      return decode_kernel<T, DP, NT, STAGES, CTAS, PAGED16>;
  }();
  static int configured[64] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    if (int rc = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes), "decode shared memory"))
      return rc;
    if (dev >= 0 && dev < 64) configured[dev] = 1;
  }
  const int ctas = std::min(sm_count(), kMostSpans * kJoinWarps * 32 / CTAS) * CTAS;
  const int group = p.q_heads / p.kv_heads;
  const int64_t parts = (int64_t)p.kv_heads * ((group + L::kRows - 1) / L::kRows);
  DecodeWork w = {};
  void *mem = nullptr;
  if (int rc = scratch_buffer(s, kPartialsSlot, (size_t)ctas * 2 * L::kRows * (DP + 4) * 4, &mem)) return rc;
  w.partials = static_cast<float *>(mem);
  if (int rc = zeroed_buffer(s, kArrivedSlot, (size_t)(p.slots * parts * 4), &mem)) return rc;
  w.arrived = static_cast<unsigned *>(mem);
  w.ctas = ctas;
  // the CTAs that a segment may span, if every slot's cache is as long as it can be
  const int64_t most = (int64_t)p.width * p.page_size, reach = p.window ? (int64_t)p.window + p.sinks : most;
  const int64_t cuts = (std::min(most, reach) / (kTileKeys * kDecodeWarps) + kMinTiles) / kMinTiles;
  w.deep = std::min<int64_t>(cuts, ctas / (p.slots * parts)) >= kDeepParts;
  if (w.deep) {
    if (int rc = scratch_buffer(s, kSpansSlot, ctas * sizeof(int2), &mem)) return rc;
    w.spans = static_cast<int2 *>(mem);
  }
  if (int rc = check_cuda(launch_pdl(kernel, dim3(ctas), dim3(kDecodeWarps * 32), L::kBytes, s, p, w, suffix...), "lc_paged_decode")) return rc;
  if (!w.deep) return LC_OK;
  return check_cuda(launch_pdl(decode_join_kernel<T, DP, NT, WithSuffix...>, dim3((unsigned)(p.slots * parts), L::kRows), dim3(kJoinWarps * 32), 0, s,
                               p, w, suffix...),
                    "lc_paged_decode (join)");
}

template <class T, bool PAGED16, class... WithSuffix>
int launch_sized(const DecodeParams &p, cudaStream_t s, const WithSuffix &...suffix) {
  // NT: 8 or 16 query heads of a group in one pass over its keys (a group of 9 to 16
  // read twice, 8 heads at a time, would take the loads twice; larger groups are cut in sixteens)
  const bool wide = p.q_heads / p.kv_heads > 8;
  if (p.d <= 64) return wide ? launch_decode<T, 64, 2, 3, 4, PAGED16>(p, s, suffix...) : launch_decode<T, 64, 1, 3, 4, PAGED16>(p, s, suffix...);
  if (p.d <= 128) return wide ? launch_decode<T, 128, 2, 3, 2, PAGED16>(p, s, suffix...) : launch_decode<T, 128, 1, 2, 3, PAGED16>(p, s, suffix...);
  if constexpr (sizeof...(WithSuffix) == 0)
    return wide ? launch_decode<T, 256, 2, 3, 1, PAGED16>(p, s) : launch_decode<T, 256, 1, 3, 1, PAGED16>(p, s);
  else
    return fail(LC_ERR_UNSUPPORTED, "lc_paged_decode: head size %d behind a prefix", p.d);
}

template <class T>
int launch_rows(const DecodeParams &p, cudaStream_t s) {
  const dim3 grid((unsigned)p.slots, (unsigned)p.q_heads), block(kRowWarps * 32);
  return check_cuda(p.d <= 64    ? launch_pdl(decode_row_kernel<T, 2>, grid, block, 0, s, p)
                    : p.d <= 128 ? launch_pdl(decode_row_kernel<T, 4>, grid, block, 0, s, p)
                                 : launch_pdl(decode_row_kernel<T, 8>, grid, block, 0, s, p),
                    "lc_paged_decode (rows)");
}

}  // namespace

// The tensor-core form takes 16-byte pieces of keys and values and pairs of the query.
bool decode_tensor(const DecodeParams &p) {
  bool ok = p.d % 8 == 0 && aligned(p.k, 16) && aligned(p.v, 16) && aligned(p.q, 4) && p.pages > 0 && p.width > 0;
  for (int i = 0; i < 3; ++i) ok = ok && p.ks[i] % 8 == 0 && p.vs[i] % 8 == 0;
  for (int i = 0; i < 2; ++i) ok = ok && p.qs[i] % 2 == 0;
  return ok;
}

// Few rows of few keys, by what any slot can see: as in window_attention.cu (1 x 8 rows
// of 68 keys: 4.7 against 5.5 us, 16 x 8: 5.1 against 6.4; 64 x 8 of 68: 9.4 against 6.6, 1 x 8 of 128: 6.2 against 5.5).
bool decode_few_keys(const DecodeParams &p) {
  const int64_t most = (int64_t)p.width * p.page_size;
  const int64_t reach = p.window ? std::min<int64_t>((int64_t)p.window + p.sinks, most) : most;
  return reach <= 96 && (int64_t)p.slots * p.q_heads * reach <= 16384;
}

int decode_params(const char *me, DecodeParams &p, int dtype, const void *q, const void *k, const void *v, void *o, float *lse,
                  const int32_t *table, const int32_t *lens, int64_t slots, int64_t width, int64_t pages, int64_t page_size,
                  int64_t q_heads, int64_t kv_heads, int64_t d, const int64_t *strides, int64_t window, int64_t sinks, float scale) {
  if (dtype != LC_F16 && dtype != LC_BF16) return fail(LC_ERR_INVALID, "%s: dtype %d is not f16 or bf16", me, dtype);
  if (slots < 0 || width < 0 || pages < 0 || page_size < 1 || q_heads < 1 || kv_heads < 1 || d < 1 || window < 0 || sinks < 0)
    return fail(LC_ERR_INVALID, "%s: negative or zero size", me);
  if (q_heads % kv_heads) return fail(LC_ERR_INVALID, "%s: %lld query heads over %lld key-value heads", me, (long long)q_heads, (long long)kv_heads);
  if (!strides) return fail(LC_ERR_INVALID, "%s: null strides", me);
  if (!(scale > 0.f) || scale > 2e38f) return fail(LC_ERR_INVALID, "%s: scale must be positive and finite", me);
  if (d > attend::kMaxHead) return fail(LC_ERR_UNSUPPORTED, "%s: head size %lld is over 256", me, (long long)d);
  if (slots > (1 << 20) || q_heads > 65535 || pages > INT32_MAX || page_size > (1 << 20) || width * page_size > (1ll << 30))
    return fail(LC_ERR_UNSUPPORTED, "%s: shape too large", me);
  if (slots == 0) return LC_OK;
  if (!q || !o || !lens || (width > 0 && !table) || (pages > 0 && (!k || !v))) return fail(LC_ERR_INVALID, "%s: null buffer", me);
  if (!aligned(q, 2) || !aligned(k, 2) || !aligned(v, 2) || !aligned(o, 2)) return fail(LC_ERR_ALIGN, "%s: elements are two bytes", me);
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
  p.page_shift = -1;
  for (int x = 0; x < 21; ++x)
    if (page_size == 1ll << x) p.page_shift = x;
  const int padded = d <= 64 ? 64 : d <= 128 ? 128 : 256;
  p.dense = d == padded && p.ks[2] == d && p.vs[2] == d;
  return LC_OK;
}

int decode_all(int dtype, const DecodeParams &p, cudaStream_t s) {
  if (!decode_few_keys(p) && decode_tensor(p)) {
    if (dtype == LC_F16) return p.page_size % 16 == 0 ? launch_sized<__half, true>(p, s) : launch_sized<__half, false>(p, s);
    return p.page_size % 16 == 0 ? launch_sized<__nv_bfloat16, true>(p, s) : launch_sized<__nv_bfloat16, false>(p, s);
  }
  return dtype == LC_F16 ? launch_rows<__half>(p, s) : launch_rows<__nv_bfloat16>(p, s);
}

int decode_suffix(int dtype, const DecodeParams &p, const Suffix &suffix, cudaStream_t s) {
  if (dtype == LC_F16) return p.page_size % 16 == 0 ? launch_sized<__half, true>(p, s, suffix) : launch_sized<__half, false>(p, s, suffix);
  return p.page_size % 16 == 0 ? launch_sized<__nv_bfloat16, true>(p, s, suffix) : launch_sized<__nv_bfloat16, false>(p, s, suffix);
}

}  // namespace lc

extern "C" int lc_paged_decode(int dtype, const void *q, const void *k, const void *v, void *o, float *lse,
                               const int32_t *table, const int32_t *lens, int64_t slots, int64_t width, int64_t pages,
                               int64_t page_size, int64_t q_heads, int64_t kv_heads, int64_t d, const int64_t *strides,
                               int64_t window, int64_t sinks, float scale, void *stream) {
  using namespace lc;
  attend::DecodeParams p;
  if (int rc = decode_params("lc_paged_decode", p, dtype, q, k, v, o, lse, table, lens, slots, width, pages, page_size, q_heads, kv_heads,
                             d, strides, window, sinks, scale))
    return rc;
  return slots == 0 ? LC_OK : decode_all(dtype, p, as_stream(stream));
}
