// Page operations of a paged key-value cache, all on the device: what is free,
// whose pages are whose and how long each sequence is lives in three int32
// arrays (`refs[pages]`: how many sequences hold the page; `table[slots, width]`:
// a sequence's pages in order; `lens[slots]`: its tokens), so a serving loop
// needs no host round trip and can be captured in a CUDA graph.
//
//   extend   takes the lowest-numbered free pages for new tokens, in slot order
//   write    puts new tokens' keys and values into their pages
//   fork     slot i goes on as a copy of slot parent[i]: full pages are shared,
//            a last page that is not full belongs to one sequence, so all but the
//            lowest slot of a parent get a page of their own with its tokens
//   release  drops whole sequences, or the pages a sliding window has left behind
//   compact  moves the pages in use onto the lowest numbers
//   copy     copies listed pages
//   prefixes tells which slots begin with the same pages, and how far (it changes nothing)
//
// A map kernel is one cluster, whose barrier separates the phases where a grid would
// need another launch.  It is a chain of some six dependent reads, each as long as an
// L2 access takes, so its size goes by the table's and refs' entries: one CTA of 256
// threads up to 2048 of them, 8 of 512 up to 65536, 8 of 1024 beyond (compact, 312
// entries: 6.6, 9.2 us; extend, 12662: 12.1, 9.1, 9.6 us; 200652: 55, 19.5, 14.3 us).
// Every result is independent of scheduling: ranks come from scans in index order, and
// atomics only count.
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"

namespace lc {
namespace {

namespace cg = cooperative_groups;

constexpr int kMostCtas = 8;
constexpr int kMostThreads = 1024;
constexpr int kMostWarps = kMostThreads / 32;
constexpr int kItems = 4;  // consecutive items of a thread in the scans, independent ones elsewhere
constexpr int kScratchSlot = 40;  // scratch_buffer slot of the page operations

// Exclusive prefix of v over the CTA's threads, and the CTA's total.
struct BlockScan {
  int warp_sums[kMostWarps + 1];
  __device__ __forceinline__ int exclusive(int v, int &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    int inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    __syncthreads();  // the previous scan has been read
    if (lane == 31) warp_sums[warp] = inc;
    __syncthreads();
    if (warp == 0) {
      const int own = lane < warps ? warp_sums[lane] : 0;
      int sum = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
      }
      __syncwarp();
      if (lane < warps) warp_sums[lane] = sum - own;
      if (lane == 31) warp_sums[kMostWarps] = sum;
    }
    __syncthreads();
    total = warp_sums[kMostWarps];
    return warp_sums[warp] + inc - v;
  }
};

__device__ __forceinline__ int pages_of(int tokens, int page_size) {
  return tokens <= 0 ? 0 : (tokens - 1) / page_size + 1;
}

// This CTA's contiguous share of n items.
struct Share {
  int begin, end;
};
__device__ __forceinline__ Share share_of(int n, int rank, int ctas) {
  const int per = (n + ctas - 1) / ctas;
  const int begin = min(n, rank * per);
  return {begin, min(n, begin + per)};
}

// How many of share [begin, end) of refs are free.
__device__ __forceinline__ int count_free(const int *refs, const Share &share) {
  int n = 0;
  for (int i = share.begin + threadIdx.x; i < share.end; i += kItems * blockDim.x) {
    int r[kItems];
#pragma unroll
    for (int x = 0; x < kItems; ++x) r[x] = i + x * (int)blockDim.x < share.end ? refs[i + x * blockDim.x] : 1;
#pragma unroll
    for (int x = 0; x < kItems; ++x) n += r[x] == 0;
  }
  return n;
}

// Adds v over the CTA and leaves the sum for the cluster in *mine; after the
// cluster barrier, before_and_total gives the sums of the lower CTAs and of all.
__device__ __forceinline__ void publish(int v, BlockScan &scan, int *mine) {
  int total;
  scan.exclusive(v, total);
  if (threadIdx.x == 0) *mine = total;
}
__device__ __forceinline__ void before_and_total(cg::cluster_group &cluster, int *mine, int &before, int &total) {
  before = total = 0;
  const int rank = (int)cluster.block_rank();
  for (int r = 0; r < (int)cluster.num_blocks(); ++r) {
    const int x = *cluster.map_shared_rank(mine, r);
    if (r < rank) before += x;
    total += x;
  }
}

// ---------------------------------------------------------------- extend

struct ExtendParams {
  const int *table_in, *lens_in, *refs_in, *add;
  int *table_out, *lens_out, *refs_out, *status;
  int *refusals;  // null, or the first refusal and the last call's
  int *offsets;   // scratch: each slot's first new page in `list`, which lies behind them: the pages taken
  int slots, width, pages, page_size;
};
// The host's part of a launch takes 0.4 us longer with eight bytes more.
static_assert(sizeof(ExtendParams) <= 96, "parameters of a map kernel");

__global__ void __launch_bounds__(kMostThreads, 1) extend_kernel(ExtendParams p) {
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ BlockScan scan;
  __shared__ int free_here;
  pdl_wait();
  pdl_trigger();
  const int rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks(), threads = blockDim.x, warps = threads >> 5, tid = threadIdx.x;
  int *list = p.offsets + p.slots;
  // every CTA adds up the demand of all slots; CTA 0 keeps each slot's offset
  int need = 0, wide = 0;
  for (int base = 0; base < p.slots; base += threads) {
    const int i = base + tid;
    int n = 0;
    if (i < p.slots) {
      const int len = max(p.lens_in[i], 0), more = p.add[i];
      const int64_t end = (int64_t)len + max(more, 0);
      const int64_t want = (end + p.page_size - 1) / p.page_size;
      const int held = pages_of(len, p.page_size);
      if (more < 0 || want > p.width)
        wide = 1;
      else
        n = (int)want - held;
    }
    int total;
    const int at = scan.exclusive(n, total);
    if (rank == 0 && i < p.slots) p.offsets[i] = need + at;
    need += total;
  }
  wide = __syncthreads_or(wide);
  // count the free pages of this CTA's share
  const Share mine = share_of(p.pages, rank, ctas);
  publish(count_free(p.refs_in, mine), scan, &free_here);
  cluster.sync();
  int before, total_free;
  before_and_total(cluster, &free_here, before, total_free);
  const bool fits = !wide && need <= total_free;
  const int take = fits ? need : 0;
  // take the lowest `take` free pages
  for (int base = mine.begin; base < mine.end; base += kItems * threads) {
    const int i = base + tid * kItems;
    int refs[kItems], n = 0, total = 0, at = 0;
#pragma unroll
    for (int x = 0; x < kItems; ++x) {
      refs[x] = i + x < mine.end ? p.refs_in[i + x] : 1;
      n += refs[x] == 0;
    }
    if (before < take) at = before + scan.exclusive(n, total);  // uniform: all lower pages are accounted for
#pragma unroll
    for (int x = 0; x < kItems; ++x) {
      const bool taken = before < take && refs[x] == 0 && at < take;
      if (i + x < mine.end) p.refs_out[i + x] = taken ? 1 : refs[x];
      if (taken) list[at] = i + x;
      at += refs[x] == 0;
    }
    before += total;
  }
  cluster.sync();  // the list and the offsets are complete, and no CTA reads another's shared memory any more
  for (int i = rank * warps + (tid >> 5); i < p.slots; i += ctas * warps) {
    const int lane = tid & 31;
    const int len = max(p.lens_in[i], 0), more = fits ? p.add[i] : 0;
    const int held = pages_of(len, p.page_size), want = pages_of(len + more, p.page_size);
    const int *in = p.table_in + (int64_t)i * p.width;
    int *out = p.table_out + (int64_t)i * p.width;
    if (in != out)
      for (int j = lane; j < p.width; j += 32)
        if (j < held || j >= want) out[j] = in[j];
    for (int j = held + lane; j < want; j += 32) out[j] = list[p.offsets[i] + j - held];
    __syncwarp();
    if (lane == 0) p.lens_out[i] = fits ? len + more : p.lens_in[i];
  }
  if (rank == 0 && tid == 0) {
    const int code = wide ? -1 : fits ? 0 : need - total_free;
    p.status[0] = code;
    p.status[1] = total_free - take;
    if (p.refusals) {
      if (code != 0 && p.refusals[0] == 0) p.refusals[0] = code;
      p.refusals[1] = code;
    }
  }
}

// ---------------------------------------------------------------- fork

struct CopyList {  // pages to copy, written by a map kernel and read by copy_kernel
  int *count;      // one int
  int *src, *dst, *tokens;
};

constexpr int kMostForkSlots = 8192;

struct ForkParams {
  const int *table_in, *lens_in, *refs_in, *parent;
  int *table_out, *lens_out, *refs_out, *status;
  int *refusals;    // null, or the first refusal
  CopyList copies;  // scratch; the pages taken lie behind the count
  int slots, width, pages, page_size;
};

__global__ void __launch_bounds__(kMostThreads, 1) fork_kernel(ForkParams p) {
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ BlockScan scan;
  __shared__ int free_here, lowest[kMostForkSlots];  // the lowest slot of each parent
  pdl_wait();
  pdl_trigger();  // copy_kernel may be scheduled; it waits for this kernel's end
  const int rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks(), threads = blockDim.x, warps = threads >> 5, tid = threadIdx.x, lane = tid & 31;
  const Share mine = share_of(p.pages, rank, ctas);
  int *list = p.copies.count + 1;
  const Share own = share_of(p.slots, rank, ctas);
  for (int i = mine.begin + tid; i < mine.end; i += threads) p.refs_out[i] = 0;
  for (int i = tid; i < p.slots; i += threads) lowest[i] = 0x7fffffff;
  __syncthreads();
  for (int i = tid; i < p.slots; i += threads) {
    const int from = p.parent[i];
    if (from >= 0 && from < p.slots) atomicMin(lowest + from, i);
  }
  __syncthreads();
  // demand: every CTA counts all slots' copies (the same result in each)
  int need = 0, bad = 0;
  for (int base = 0; base < p.slots; base += threads) {
    const int i = base + tid;
    int n = 0;
    if (i < p.slots) {
      const int from = p.parent[i];
      if (from < -1 || from >= p.slots)
        bad = 1;
      else if (from >= 0) {
        const int len = max(p.lens_in[from], 0);
        n = len % p.page_size != 0 && lowest[from] != i && len / p.page_size < p.width;
      }
    }
    int total;
    const int at = scan.exclusive(n, total);
    if (rank == 0 && n) {
      const int from = p.parent[i], len = p.lens_in[from];
      p.copies.src[need + at] = p.table_in[(int64_t)from * p.width + len / p.page_size];
      p.copies.dst[need + at] = i;  // the slot; the page follows once it is known
      p.copies.tokens[need + at] = len % p.page_size;
    }
    need += total;
  }
  bad = __syncthreads_or(bad);
  cluster.sync();  // refs_out is zero
  // the new rows, and how often each page is held
  for (int i = rank * warps + (tid >> 5); i < p.slots; i += ctas * warps) {
    const int from = bad ? -1 : p.parent[i];
    const int len = from >= 0 ? max(p.lens_in[from], 0) : 0;
    const int own_page = from >= 0 && len % p.page_size != 0 && lowest[from] != i ? len / p.page_size : -1;
    const int *in = p.table_in + (int64_t)(from >= 0 ? from : 0) * p.width;
    int *out = p.table_out + (int64_t)i * p.width;
    for (int j = lane; j < p.width; j += 32) {
      const int page = from >= 0 ? in[j] : -1;
      out[j] = page;
      if (j != own_page && page >= 0 && page < p.pages) atomicAdd(p.refs_out + page, 1);
    }
    if (lane == 0) p.lens_out[i] = from >= 0 ? p.lens_in[from] : 0;
  }
  cluster.sync();
  publish(count_free(p.refs_out, mine), scan, &free_here);
  cluster.sync();
  int before, total_free;
  before_and_total(cluster, &free_here, before, total_free);
  const bool fits = !bad && need <= total_free;
  const int short_by = need - total_free;
  if (fits) {
    for (int base = mine.begin; base < mine.end && before < need; base += kItems * threads) {
      const int i = base + tid * kItems;
      bool is_free[kItems];
      int n = 0, total;
#pragma unroll
      for (int x = 0; x < kItems; ++x) {
        is_free[x] = i + x < mine.end && p.refs_out[i + x] == 0;
        n += is_free[x];
      }
      int at = before + scan.exclusive(n, total);
#pragma unroll
      for (int x = 0; x < kItems; ++x) {
        if (is_free[x] && at < need) {
          p.refs_out[i + x] = 1;
          list[at] = i + x;
        }
        at += is_free[x];
      }
      before += total;
    }
    cluster.sync();
    for (int i = rank * threads + tid; i < need; i += ctas * threads) {
      const int slot = p.copies.dst[i], page = list[i];
      const int from = p.parent[slot];
      p.table_out[(int64_t)slot * p.width + p.lens_in[from] / p.page_size] = page;
      p.copies.dst[i] = page;
    }
  } else {  // nothing changes
    int count = 0;
    for (int i = mine.begin + tid; i < mine.end; i += threads) {
      const int refs = p.refs_in[i];
      p.refs_out[i] = refs;
      count += refs == 0;
    }
    for (int i = own.begin + tid; i < own.end; i += threads) p.lens_out[i] = p.lens_in[i];
    const int64_t cells = (int64_t)p.slots * p.width;
    for (int64_t i = rank * threads + tid; i < cells; i += ctas * threads) p.table_out[i] = p.table_in[i];
    cluster.sync();  // every CTA has read free_here
    publish(count, scan, &free_here);
    cluster.sync();
    before_and_total(cluster, &free_here, before, total_free);
  }
  if (rank == 0 && tid == 0) {
    const int code = bad ? -1 : fits ? 0 : short_by;
    p.status[0] = code;
    p.status[1] = fits ? total_free - need : total_free;
    if (p.refusals && code != 0 && p.refusals[0] == 0) p.refusals[0] = code;
    *p.copies.count = fits ? need : 0;
  }
  cluster.sync();  // no CTA leaves while its shared memory is read
}

// ---------------------------------------------------------------- release

struct ReleaseParams {
  int *table, *lens, *refs, *status;
  const int *gone;    // drop the slots where this is not zero; null: trim
  int window, sinks;  // trim: pages that no position from lens[i] on sees
  int slots, width, pages, page_size;
};

__global__ void __launch_bounds__(kMostThreads, 1) release_kernel(ReleaseParams p) {
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ BlockScan scan;
  __shared__ int free_here;
  pdl_wait();
  pdl_trigger();
  const int rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks(), threads = blockDim.x, warps = threads >> 5, tid = threadIdx.x, lane = tid & 31;
  for (int i = rank * warps + (tid >> 5); i < p.slots; i += ctas * warps) {
    const int len = max(p.lens[i], 0);
    int begin = 0, end = min(pages_of(len, p.page_size), p.width);
    if (p.gone) {
      if (p.gone[i] == 0) continue;
    } else {
      // the next token's position is len: it sees j > len - window and j < sinks
      begin = pages_of(p.sinks, p.page_size);
      end = min(end, max(len - p.window + 1, 0) / p.page_size);
    }
    int *row = p.table + (int64_t)i * p.width;
    for (int j = begin + lane; j < end; j += 32) {
      const int page = row[j];
      if (page >= 0 && page < p.pages) atomicSub(p.refs + page, 1);
      row[j] = -1;
    }
    __syncwarp();
    if (p.gone && lane == 0) p.lens[i] = 0;
  }
  cluster.sync();
  const Share mine = share_of(p.pages, rank, ctas);
  publish(count_free(p.refs, mine), scan, &free_here);
  cluster.sync();
  int before, total;
  before_and_total(cluster, &free_here, before, total);
  if (rank == 0 && tid == 0) {
    p.status[0] = 0;
    p.status[1] = total;
  }
  cluster.sync();  // no CTA leaves while its shared memory is read
}

// ---------------------------------------------------------------- compact

struct CompactParams {
  const int *table_in, *lens_in, *refs_in;
  int *table_out, *lens_out, *refs_out, *status;
  int *rank_of;  // scratch: a page's rank among the pages in use
  CopyList copies;
  int slots, width, pages;
};

// With U pages in use, L(p) of them below page p: a free page p < U is hole
// p - L(p), and the pages in use from U on have the ranks L = U - holes .. U - 1;
// the r-th of them moves into hole r.  No source is a destination.
__global__ void __launch_bounds__(kMostThreads, 1) compact_kernel(CompactParams p) {
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ BlockScan scan;
  __shared__ int used_here, holes_here;
  pdl_wait();
  pdl_trigger();  // copy_kernel may be scheduled; it waits for this kernel's end
  const int rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks(), threads = blockDim.x, tid = threadIdx.x;
  const Share mine = share_of(p.pages, rank, ctas);
  publish((tid == 0 ? mine.end - mine.begin : 0) - count_free(p.refs_in, mine), scan, &used_here);
  cluster.sync();
  int below, used;
  before_and_total(cluster, &used_here, below, used);
  int holes = 0;
  for (int base = mine.begin; base < mine.end; base += kItems * threads) {
    const int i = base + tid * kItems;
    bool live[kItems];
    int n = 0, total;
#pragma unroll
    for (int x = 0; x < kItems; ++x) {
      live[x] = i + x < mine.end && p.refs_in[i + x] != 0;
      n += live[x];
    }
    int at = below + scan.exclusive(n, total);
#pragma unroll
    for (int x = 0; x < kItems; ++x) {
      const int page = i + x;
      if (page < mine.end) {
        if (page >= used) p.rank_of[page] = live[x] ? at : -1;
        if (!live[x] && page < used) {
          p.copies.dst[page - at] = page;
          ++holes;
        }
      }
      at += live[x];
    }
    below += total;
  }
  publish(holes, scan, &holes_here);
  cluster.sync();
  int before, total_holes;
  before_and_total(cluster, &holes_here, before, total_holes);
  const int first = used - total_holes;  // the lowest rank that moves
  for (int i = mine.begin + tid; i < mine.end; i += threads) {
    const int refs = p.refs_in[i];
    if (i >= used) {
      if (refs != 0) {
        const int r = p.rank_of[i] - first;
        p.copies.src[r] = i;
        p.refs_out[p.copies.dst[r]] = refs;
      }
      p.refs_out[i] = 0;
    } else if (refs != 0 && p.refs_in != p.refs_out) {
      p.refs_out[i] = refs;
    }
  }
  const int64_t cells = (int64_t)p.slots * p.width;
  const int64_t stride = (int64_t)ctas * threads;
  for (int64_t i = rank * threads + tid; i < cells; i += kItems * stride) {
    int page[kItems], r[kItems];
#pragma unroll
    for (int x = 0; x < kItems; ++x) page[x] = i + x * stride < cells ? p.table_in[i + x * stride] : -1;
#pragma unroll
    for (int x = 0; x < kItems; ++x) r[x] = page[x] >= used && page[x] < p.pages ? p.rank_of[page[x]] : -1;
#pragma unroll
    for (int x = 0; x < kItems; ++x)
      if (r[x] >= first) page[x] = p.copies.dst[r[x] - first];
#pragma unroll
    for (int x = 0; x < kItems; ++x)
      if (i + x * stride < cells) p.table_out[i + x * stride] = page[x];
  }
  const Share own = share_of(p.slots, rank, ctas);
  if (p.lens_in != p.lens_out)
    for (int i = own.begin + tid; i < own.end; i += threads) p.lens_out[i] = p.lens_in[i];
  if (rank == 0 && tid == 0) {
    p.status[0] = 0;
    p.status[1] = p.pages - used;
    *p.copies.count = total_holes;
  }
  cluster.sync();  // no CTA leaves while its shared memory is read
}

// ---------------------------------------------------------------- copy

struct PoolParams {
  char *pool;
  int planes, pages, heads, page_size;
  int64_t token_bytes, plane, page, head;  // strides in bytes
};

struct CopyParams {
  PoolParams pool;
  const int *src, *dst, *tokens, *count;  // tokens: null = whole pages; count: null = n
  int n;
};

__device__ __forceinline__ uint4 load_once(const uint4 *p) { return ld_stream_u4(p); }
__device__ __forceinline__ uint8_t load_once(const uint8_t *p) { return *p; }
__device__ __forceinline__ void store_once(uint4 *p, uint4 v) { st_stream_u4(p, v); }
__device__ __forceinline__ void store_once(uint8_t *p, uint8_t v) { *p = v; }

// A warp moves up to 8 x 32 vectors (4 KB) of one run at a time: a head's tokens of one
// page of one plane, or the whole page where its heads lie together.  Eight loads are in
// flight before the first store, whatever the pages' size (1.1 GB of 32 KB pages: 168 us,
// 6500 GB/s; of 4 KB pages 64 us against 114 with a CTA per page).
template <class Vec>
__global__ void __launch_bounds__(256) copy_kernel(CopyParams p) {
  pdl_wait();
  pdl_trigger();
  constexpr int V = sizeof(Vec), U = 8;
  const int n = p.count ? *p.count : p.n, lane = threadIdx.x & 31;
  const bool together = !p.tokens && p.pool.head == p.pool.page_size * p.pool.token_bytes;
  const unsigned runs = together ? 1 : p.pool.heads;
  const int64_t most = p.pool.page_size * p.pool.token_bytes * (together ? p.pool.heads : 1);
  const unsigned pieces = (unsigned)((most + U * 32 * V - 1) / (U * 32 * V));
  const unsigned per_plane = runs * pieces;
  const int64_t units = (int64_t)n * p.pool.planes * per_plane;
  for (int64_t unit = blockIdx.x * 8 + (threadIdx.x >> 5); unit < units; unit += gridDim.x * 8) {
    const int64_t page = unit / per_plane;  // (pair, plane)
    const unsigned in_plane = (unsigned)(unit - page * per_plane), head = in_plane / pieces, piece = in_plane - head * pieces;
    const int pair = (int)(page / p.pool.planes), plane = (int)(page - (int64_t)pair * p.pool.planes);
    const int src = p.src[pair], dst = p.dst[pair];
    if (src < 0 || src >= p.pool.pages || dst < 0 || dst >= p.pool.pages || src == dst) continue;
    const int64_t bytes = p.tokens ? p.tokens[pair] * p.pool.token_bytes : most;
    const int64_t at = plane * p.pool.plane + head * p.pool.head + ((int64_t)piece * U * 32 + lane) * V;
    const int left = (int)((bytes - ((int64_t)piece * U * 32 + lane) * V + V - 1) / V);  // of this lane's vectors on
    const Vec *from = reinterpret_cast<const Vec *>(p.pool.pool + at + src * p.pool.page);
    Vec *to = reinterpret_cast<Vec *>(p.pool.pool + at + dst * p.pool.page);
    Vec v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (u * 32 < left) v[u] = load_once(from + u * 32);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (u * 32 < left) store_once(to + u * 32, v[u]);
  }
}

// ---------------------------------------------------------------- write

struct WriteParams {
  const char *k, *v;
  char *k_pages, *v_pages;
  const int *table, *lens, *add, *refused;  // refused: null, or a word; nothing is written where it is not 0
  int slots, most, width, pages, page_size, heads;
  int64_t row_bytes;              // head_dim elements
  int64_t ks[3], vs[3];           // byte strides of the new tokens: slot, token, head
  int64_t kp[3], vp[3];           // byte strides of the pages: page, head, token
};

// New token t of slot i goes to position lens[i] - add[i] + t.  A CTA takes
// tokens of one slot, its threads the 16-byte pieces of their heads.  Pure traffic:
// 82000 tokens of 8 heads of 128: 100 us, 6700 GB/s.
constexpr int kWriteTokens = 8;

template <class Vec>
__global__ void __launch_bounds__(256) write_kernel(WriteParams p) {
  pdl_wait();
  pdl_trigger();
  const int slot = blockIdx.y;
  const int refused = p.refused ? *p.refused : 0;
  const int add = min(max(p.add[slot], 0), p.most);
  const int first = blockIdx.x * kWriteTokens;
  if (first >= add || refused) return;
  const int64_t start = (int64_t)p.lens[slot] - p.add[slot];
  if (start < 0) return;
  constexpr int V = sizeof(Vec);
  const int row = (int)(p.row_bytes / V), token = row * p.heads;
  const int tokens = min(kWriteTokens, add - first);
  for (int i = threadIdx.x; i < tokens * token; i += 256) {
    const int t = i / token, in_token = i - t * token;
    const int head = in_token / row, c = in_token - head * row;
    const int64_t pos = start + first + t;
    const int64_t entry = pos / p.page_size;
    if (entry >= p.width) continue;
    const int page = p.table[(int64_t)slot * p.width + entry];
    if (page < 0 || page >= p.pages) continue;
    const int r = (int)(pos - entry * p.page_size);
    const int64_t in_k = slot * p.ks[0] + (first + t) * p.ks[1] + head * p.ks[2] + (int64_t)c * V;
    const int64_t in_v = slot * p.vs[0] + (first + t) * p.vs[1] + head * p.vs[2] + (int64_t)c * V;
    const Vec k = *reinterpret_cast<const Vec *>(p.k + in_k), v = *reinterpret_cast<const Vec *>(p.v + in_v);
    *reinterpret_cast<Vec *>(p.k_pages + page * p.kp[0] + head * p.kp[1] + r * p.kp[2] + (int64_t)c * V) = k;
    *reinterpret_cast<Vec *>(p.v_pages + page * p.vp[0] + head * p.vp[1] + r * p.vp[2] + (int64_t)c * V) = v;
  }
}

// ---------------------------------------------------------------- prefixes

struct PrefixParams {
  const int *table, *lens;
  int *leader, *shared, *order;
  int *least;  // scratch: of each leader, the pages that its group has in common so far
  int slots, width, pages, page_size;
};
constexpr int kCompare = 16;  // table entries of a lane at a time

// A group is the slots whose first page, a full one, is the same; its lowest slot leads. What they share is the
// least number of full pages at which every slot's row is the leader's. Rows are compared in pieces of 512
// entries, dealt to all warps, none behind a difference that is known. Ranks by counting: slots^2 / 8192 steps a
// thread at most, and slots are few.
__global__ void __launch_bounds__(kMostThreads, 1) prefixes_kernel(PrefixParams p) {
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ int keys[kMostForkSlots];  // first pages, then leaders
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, lane = tid & 31, warps = cluster.num_blocks() * (blockDim.x >> 5);
  const int warp = cluster.block_rank() * (blockDim.x >> 5) + (tid >> 5);
  auto full_pages = [&](int s) {
    const int64_t most = (int64_t)p.width * p.page_size;
    return (int)min((int64_t)max(p.lens[s], 0), most) / p.page_size;
  };
  for (int s = tid; s < p.slots; s += blockDim.x) {
    const int page = full_pages(s) > 0 ? p.table[(int64_t)s * p.width] : -1;
    keys[s] = (unsigned)page < (unsigned)p.pages ? page : -1;
  }
  __syncthreads();
  for (int s = warp; s < p.slots; s += warps) {
    int lowest = s;
    if (keys[s] >= 0)
      for (int j = lane; j < s; j += 32)
        if (keys[j] == keys[s]) {
          lowest = j;
          break;
        }
    lowest = __reduce_min_sync(0xffffffffu, lowest);
    if (lane == 0) {
      p.leader[s] = lowest;
      p.least[s] = full_pages(s);
    }
  }
  cluster.sync();
  for (int s = tid; s < p.slots; s += blockDim.x) keys[s] = __ldcg(p.leader + s);
  __syncthreads();
  constexpr int kPiece = 32 * kCompare;
  const int pieces = (p.width + kPiece - 1) / kPiece;
  for (int64_t x = warp; x < (int64_t)p.slots * pieces; x += warps) {
    const int s = (int)(x / pieces), begin = (int)(x - (int64_t)s * pieces) * kPiece;
    const int leader = keys[s];
    if (leader == s) continue;
    const int end = min(min(full_pages(s), full_pages(leader)), begin + kPiece);
    if (begin == 0 && lane == 0) atomicMin(p.least + leader, full_pages(s));
    if (begin >= end || begin >= __ldcg(p.least + leader)) continue;
    const int *a = p.table + (int64_t)s * p.width + begin, *b = p.table + (int64_t)leader * p.width + begin;
    int other = end;
#pragma unroll
    for (int i = kCompare - 1; i >= 0; --i) {
      const int j = lane + 32 * i;
      if (begin + j < end && a[j] != b[j]) other = begin + j;
    }
    other = __reduce_min_sync(0xffffffffu, other);
    if (other < end && lane == 0) atomicMin(p.least + leader, other);
  }
  cluster.sync();
  for (int s = warp; s < p.slots; s += warps) {
    int before = 0, members = 0;
    for (int j = lane; j < p.slots; j += 32) {
      const int same = keys[j] == keys[s];
      before += keys[j] < keys[s] || (same && j < s);
      members += same;
    }
    before = __reduce_add_sync(0xffffffffu, before);
    members = __reduce_add_sync(0xffffffffu, members);
    if (lane == 0) {
      p.shared[s] = members > 1 ? __ldcg(p.least + keys[s]) * p.page_size : 0;
      p.order[before] = s;
    }
  }
}

// ---------------------------------------------------------------- host side

template <class Params>
int launch_maps(const char *me, void (*kernel)(Params), int64_t cells, cudaStream_t s, const Params &p) {
  const unsigned ctas = cells <= 2048 ? 1 : kMostCtas, threads = cells <= 2048 ? 256 : cells <= 65536 ? 512 : kMostThreads;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(threads);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {ctas, 1, 1};
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return check_cuda(cudaLaunchKernelEx(&cfg, kernel, p), me);
}

int check_maps(const char *me, int64_t slots, int64_t width, int64_t pages, int64_t page_size) {
  if (slots < 0 || width < 0 || pages < 0 || page_size < 1) return fail(LC_ERR_INVALID, "%s: negative or zero size", me);
  if (slots > (1 << 20) || pages > (1 << 30) || page_size > (1 << 20) || width > (1 << 24) || width * page_size > (1ll << 30) ||
      slots * width > INT32_MAX)  // the demand of all slots is an int, too
    return fail(LC_ERR_UNSUPPORTED, "%s: shape too large", me);
  return LC_OK;
}

int make_pool(const char *me, PoolParams *out, void *pool, int64_t planes, int64_t pages, int64_t heads,
              int64_t page_size, int64_t token_bytes, const int64_t *strides) {
  if (planes < 0 || heads < 1 || token_bytes < 1) return fail(LC_ERR_INVALID, "%s: negative or zero pool size", me);
  if (!strides) return fail(LC_ERR_INVALID, "%s: null strides", me);
  if (planes > (1 << 20) || heads > (1 << 16) || token_bytes > (1 << 16) || heads * page_size * token_bytes > (1ll << 30))
    return fail(LC_ERR_UNSUPPORTED, "%s: pool too large", me);
  if (planes > 0 && pages > 0 && !pool) return fail(LC_ERR_INVALID, "%s: null pool", me);
  *out = {static_cast<char *>(pool), (int)planes, (int)pages, (int)heads, (int)page_size, token_bytes, strides[0], strides[1], strides[2]};
  return LC_OK;
}

bool all_multiple(const int64_t *v, int n, int64_t of) {
  for (int i = 0; i < n; ++i)
    if (v[i] % of) return false;
  return true;
}

int launch_copy(const char *me, const CopyParams &p, int64_t most_pairs, cudaStream_t s) {
  const int64_t sizes[4] = {p.pool.token_bytes, p.pool.plane, p.pool.page, p.pool.head};
  const bool wide = aligned(p.pool.pool, 16) && all_multiple(sizes, 4, 16);
  // as many CTAs as there can be units of 4 KB for, up to 32 per SM (whole pages,
  // 1.1 GB: 195 us with 8, 182 with 32, 180 with 64; where fewer move than could, the rest leave at once)
  const int64_t page_bytes = p.pool.heads * p.pool.page_size * p.pool.token_bytes;
  const int64_t units = most_pairs * p.pool.planes * std::max<int64_t>(p.pool.heads, (page_bytes + 4095) / 4096);
  const unsigned grid = (unsigned)std::min<int64_t>(sm_count() * 32, (units + 7) / 8);
  const cudaError_t err = wide ? launch_pdl(copy_kernel<uint4>, dim3(grid), dim3(256), 0, s, p)
                               : launch_pdl(copy_kernel<uint8_t>, dim3(grid), dim3(256), 0, s, p);
  return check_cuda(err, me);
}

}  // namespace
}  // namespace lc

extern "C" int lc_cache_extend_recorded(const int32_t *table_in, int32_t *table_out, const int32_t *lens_in, int32_t *lens_out,
                                        const int32_t *refs_in, int32_t *refs_out, const int32_t *add, int32_t *status,
                                        int32_t *refusals, int64_t slots, int64_t width, int64_t pages, int64_t page_size,
                                        void *stream) {
  using namespace lc;
  const char *me = "lc_cache_extend";
  if (int rc = check_maps(me, slots, width, pages, page_size)) return rc;
  if (!status || (slots > 0 && (!lens_in || !lens_out || !add || (width > 0 && (!table_in || !table_out)))) ||
      (pages > 0 && (!refs_in || !refs_out)))
    return fail(LC_ERR_INVALID, "%s: null buffer", me);
  cudaStream_t s = as_stream(stream);
  void *scratch = nullptr;
  if (int rc = scratch_buffer(s, kScratchSlot, (size_t)(slots + pages + 1) * 4, &scratch)) return rc;
  int *ints = static_cast<int *>(scratch);
  const ExtendParams p = {table_in, lens_in, refs_in, add, table_out, lens_out, refs_out, status, refusals, ints,
                          (int)slots, (int)width, (int)pages, (int)page_size};
  return launch_maps(me, extend_kernel, slots * width + pages, s, p);
}

extern "C" int lc_cache_extend(const int32_t *table_in, int32_t *table_out, const int32_t *lens_in, int32_t *lens_out,
                               const int32_t *refs_in, int32_t *refs_out, const int32_t *add, int32_t *status,
                               int64_t slots, int64_t width, int64_t pages, int64_t page_size, void *stream) {
  return lc_cache_extend_recorded(table_in, table_out, lens_in, lens_out, refs_in, refs_out, add, status, nullptr, slots, width, pages,
                                  page_size, stream);
}

extern "C" int lc_cache_write_unless(const void *k, const void *v, void *k_pages, void *v_pages, const int32_t *table,
                                     const int32_t *lens, const int32_t *add, int64_t slots, int64_t most, int64_t width,
                                     int64_t pages, int64_t page_size, int64_t kv_heads, int64_t row_bytes,
                                     const int64_t *strides, const int32_t *refused, void *stream) {
  using namespace lc;
  const char *me = "lc_cache_write";
  if (int rc = check_maps(me, slots, width, pages, page_size)) return rc;
  if (most < 0 || kv_heads < 1 || row_bytes < 1) return fail(LC_ERR_INVALID, "%s: negative or zero size", me);
  if (!strides) return fail(LC_ERR_INVALID, "%s: null strides", me);
  if (most > (1 << 30) || kv_heads > (1 << 16) || row_bytes > (1 << 12) || slots > 65535 ||
      kWriteTokens * kv_heads * row_bytes > INT32_MAX - 256)  // a CTA counts its tokens' pieces in an int
    return fail(LC_ERR_UNSUPPORTED, "%s: shape too large", me);
  if (slots == 0 || most == 0 || width == 0 || pages == 0) return LC_OK;
  if (!k || !v || !k_pages || !v_pages || !table || !lens || !add) return fail(LC_ERR_INVALID, "%s: null buffer", me);
  WriteParams p = {static_cast<const char *>(k), static_cast<const char *>(v), static_cast<char *>(k_pages), static_cast<char *>(v_pages),
                   table, lens, add, refused, (int)slots, (int)most, (int)width, (int)pages, (int)page_size, (int)kv_heads, row_bytes, {}, {}, {}, {}};
  for (int i = 0; i < 3; ++i) p.ks[i] = strides[i], p.vs[i] = strides[3 + i], p.kp[i] = strides[6 + i], p.vp[i] = strides[9 + i];
  const bool wide = aligned(k, 16) && aligned(v, 16) && aligned(k_pages, 16) && aligned(v_pages, 16) &&
                    row_bytes % 16 == 0 && all_multiple(strides, 12, 16);
  const dim3 grid((unsigned)((most + kWriteTokens - 1) / kWriteTokens), (unsigned)slots);
  cudaStream_t s = as_stream(stream);
  return check_cuda(wide ? launch_pdl(write_kernel<uint4>, grid, dim3(256), 0, s, p) : launch_pdl(write_kernel<uint8_t>, grid, dim3(256), 0, s, p), me);
}

extern "C" int lc_cache_write(const void *k, const void *v, void *k_pages, void *v_pages, const int32_t *table,
                              const int32_t *lens, const int32_t *add, int64_t slots, int64_t most, int64_t width,
                              int64_t pages, int64_t page_size, int64_t kv_heads, int64_t row_bytes,
                              const int64_t *strides, void *stream) {
  return lc_cache_write_unless(k, v, k_pages, v_pages, table, lens, add, slots, most, width, pages, page_size, kv_heads, row_bytes,
                               strides, nullptr, stream);
}

extern "C" int lc_cache_fork_recorded(void *pool, int64_t planes, int64_t kv_heads, int64_t token_bytes, const int64_t *strides,
                                      const int32_t *table_in, int32_t *table_out, const int32_t *lens_in, int32_t *lens_out,
                                      const int32_t *refs_in, int32_t *refs_out, const int32_t *parent, int32_t *status,
                                      int32_t *refusals, int64_t slots, int64_t width, int64_t pages, int64_t page_size,
                                      void *stream) {
  using namespace lc;
  const char *me = "lc_cache_fork";
  if (int rc = check_maps(me, slots, width, pages, page_size)) return rc;
  CopyParams c = {};
  if (int rc = make_pool(me, &c.pool, pool, planes, pages, kv_heads, page_size, token_bytes, strides)) return rc;
  if (!status || (slots > 0 && (!lens_in || !lens_out || !parent || (width > 0 && (!table_in || !table_out)))) ||
      (pages > 0 && (!refs_in || !refs_out)))
    return fail(LC_ERR_INVALID, "%s: null buffer", me);
  if (slots > kMostForkSlots) return fail(LC_ERR_UNSUPPORTED, "%s: %lld slots, at most %d", me, (long long)slots, kMostForkSlots);
  if ((slots > 0 && (lens_in == lens_out || (width > 0 && table_in == table_out))) || (pages > 0 && refs_in == refs_out))
    return fail(LC_ERR_INVALID, "%s: the new maps may not overwrite the old ones", me);
  cudaStream_t s = as_stream(stream);
  void *scratch = nullptr;
  if (int rc = scratch_buffer(s, kScratchSlot, (size_t)(4 * slots + 1) * 4, &scratch)) return rc;
  int *ints = static_cast<int *>(scratch);
  ForkParams p = {table_in, lens_in, refs_in, parent, table_out, lens_out, refs_out, status, refusals,
                  {ints, ints + 1 + slots, ints + 1 + 2 * slots, ints + 1 + 3 * slots},
                  (int)slots, (int)width, (int)pages, (int)page_size};
  if (int rc = launch_maps(me, fork_kernel, slots * width + pages, s, p)) return rc;
  if (planes == 0 || pages == 0 || slots == 0) return LC_OK;
  c.src = p.copies.src, c.dst = p.copies.dst, c.tokens = p.copies.tokens, c.count = p.copies.count;
  return launch_copy(me, c, slots, s);
}

extern "C" int lc_cache_fork(void *pool, int64_t planes, int64_t kv_heads, int64_t token_bytes, const int64_t *strides,
                             const int32_t *table_in, int32_t *table_out, const int32_t *lens_in, int32_t *lens_out,
                             const int32_t *refs_in, int32_t *refs_out, const int32_t *parent, int32_t *status,
                             int64_t slots, int64_t width, int64_t pages, int64_t page_size, void *stream) {
  return lc_cache_fork_recorded(pool, planes, kv_heads, token_bytes, strides, table_in, table_out, lens_in, lens_out, refs_in, refs_out,
                                parent, status, nullptr, slots, width, pages, page_size, stream);
}

extern "C" int lc_cache_release(int32_t *table, int32_t *lens, int32_t *refs, const int32_t *gone, int64_t window,
                                int64_t sinks, int32_t *status, int64_t slots, int64_t width, int64_t pages,
                                int64_t page_size, void *stream) {
  using namespace lc;
  const char *me = "lc_cache_release";
  if (int rc = check_maps(me, slots, width, pages, page_size)) return rc;
  if (!gone && (window < 1 || sinks < 0)) return fail(LC_ERR_INVALID, "%s: trimming needs a window and sinks >= 0", me);
  if (!status || (slots > 0 && (!lens || (width > 0 && !table))) || (pages > 0 && !refs))
    return fail(LC_ERR_INVALID, "%s: null buffer", me);
  const int64_t most = 1ll << 30;
  const ReleaseParams p = {table, lens, refs, status, gone, (int)(window < most ? window : most), (int)(sinks < most ? sinks : most),
                           (int)slots, (int)width, (int)pages, (int)page_size};
  return launch_maps(me, release_kernel, slots * width + pages, as_stream(stream), p);
}

extern "C" int lc_cache_compact(void *pool, int64_t planes, int64_t kv_heads, int64_t token_bytes,
                                const int64_t *strides, const int32_t *table_in, int32_t *table_out,
                                const int32_t *lens_in, int32_t *lens_out, const int32_t *refs_in, int32_t *refs_out,
                                int32_t *status, int64_t slots, int64_t width, int64_t pages, int64_t page_size,
                                void *stream) {
  using namespace lc;
  const char *me = "lc_cache_compact";
  if (int rc = check_maps(me, slots, width, pages, page_size)) return rc;
  CopyParams c = {};
  if (int rc = make_pool(me, &c.pool, pool, planes, pages, kv_heads, page_size, token_bytes, strides)) return rc;
  if (!status || (slots > 0 && (!lens_in || !lens_out || (width > 0 && (!table_in || !table_out)))) ||
      (pages > 0 && (!refs_in || !refs_out)))
    return fail(LC_ERR_INVALID, "%s: null buffer", me);
  cudaStream_t s = as_stream(stream);
  void *scratch = nullptr;
  if (int rc = scratch_buffer(s, kScratchSlot, (size_t)(3 * pages + 1) * 4, &scratch)) return rc;
  int *ints = static_cast<int *>(scratch);
  const CompactParams p = {table_in, lens_in, refs_in, table_out, lens_out, refs_out, status, ints + 1,
                           {ints, ints + 1 + pages, ints + 1 + 2 * pages, nullptr}, (int)slots, (int)width, (int)pages};
  if (int rc = launch_maps(me, compact_kernel, slots * width + pages, s, p)) return rc;
  if (planes == 0 || pages == 0) return LC_OK;
  c.src = p.copies.src, c.dst = p.copies.dst, c.count = p.copies.count;
  return launch_copy(me, c, (pages + 1) / 2, s);
}

extern "C" int lc_cache_copy(void *pool, int64_t planes, int64_t kv_heads, int64_t token_bytes, const int64_t *strides,
                             const int32_t *src, const int32_t *dst, int64_t n, int64_t pages, int64_t page_size,
                             void *stream) {
  using namespace lc;
  const char *me = "lc_cache_copy";
  if (int rc = check_maps(me, 0, 0, pages, page_size)) return rc;
  CopyParams c = {};
  if (int rc = make_pool(me, &c.pool, pool, planes, pages, kv_heads, page_size, token_bytes, strides)) return rc;
  if (n < 0) return fail(LC_ERR_INVALID, "%s: negative count", me);
  if (n > (1 << 30)) return fail(LC_ERR_UNSUPPORTED, "%s: too many pages", me);
  if (n == 0 || planes == 0 || pages == 0) return LC_OK;
  if (!src || !dst) return fail(LC_ERR_INVALID, "%s: null buffer", me);
  c.src = src, c.dst = dst, c.n = (int)n;
  return launch_copy(me, c, n, as_stream(stream));
}

extern "C" int lc_cache_prefixes(const int32_t *table, const int32_t *lens, int32_t *leader, int32_t *shared, int32_t *order,
                                 int64_t slots, int64_t width, int64_t pages, int64_t page_size, void *stream) {
  using namespace lc;
  const char *me = "lc_cache_prefixes";
  if (int rc = check_maps(me, slots, width, pages, page_size)) return rc;
  if (slots > kMostForkSlots) return fail(LC_ERR_UNSUPPORTED, "%s: %lld slots, at most %d", me, (long long)slots, kMostForkSlots);
  if (slots == 0) return LC_OK;
  if (!lens || !leader || !shared || !order || (width > 0 && !table)) return fail(LC_ERR_INVALID, "%s: null buffer", me);
  cudaStream_t s = as_stream(stream);
  void *scratch = nullptr;
  if (int rc = scratch_buffer(s, kScratchSlot, (size_t)slots * 4, &scratch)) return rc;
  const PrefixParams p = {table, lens, leader, shared, order, static_cast<int *>(scratch), (int)slots, (int)width, (int)pages, (int)page_size};
  return launch_maps(me, prefixes_kernel, slots * width, s, p);
}
