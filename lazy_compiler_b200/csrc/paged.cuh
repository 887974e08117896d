// What the kernels of single-token attention share (paged_decode.cu, shared_decode.cu): a call's
// parameters, a slot's tokens, its row key by key, and what of a slot is a shared prefix.
#pragma once

#include "attend.cuh"

namespace lc {
namespace attend {

struct DecodeParams {
  const void *q, *k, *v;
  void *o;
  float *lse;
  const int *table, *lens;
  int slots, width, pages, page_size, q_heads, kv_heads, d;
  int64_t qs[2], ks[3], vs[3], os[2], ts;  // element strides: q, o slot and head; k, v page, head, token; table slot
  int window, sinks;
  float scale_log2;
  int page_shift;  // page_size is 1 << page_shift, or -1
  int dense;       // a head's tokens follow each other in k and v, without padding
};

__device__ __forceinline__ int page_index(const DecodeParams &p, int key) {
  return p.page_shift >= 0 ? key >> p.page_shift : key / p.page_size;
}

__device__ __forceinline__ int cached_tokens(const DecodeParams &p, int slot) {
  const int64_t most = (int64_t)p.width * p.page_size;
  const int n = max(p.lens[slot], 0);
  return n < most ? n : (int)most;
}

// What a slot's group shares: of each slot its group's lowest slot, and the tokens that all of the group have in
// common; `order` lists the slots by group (shared_decode.cu).
struct Sharing {
  const int *leader, *shared, *order;
};
// Prefixes below this many tokens are read by each slot alone.
constexpr int kLeastPrefix = 128;
__device__ __forceinline__ int prefix_tokens(const DecodeParams &p, const Sharing &g, int leader) {
  const int64_t most = (int64_t)p.width * p.page_size;
  const int n = g.shared[leader];
  return n < kLeastPrefix ? 0 : n < most ? n : (int)most;
}
__device__ __forceinline__ int group_prefix(const DecodeParams &p, const Sharing &g, int slot) {
  const int leader = g.leader[slot];
  return (unsigned)leader < (unsigned)p.slots ? prefix_tokens(p, g, leader) : 0;
}
// The tokens of a slot that belong to the prefix.
__device__ __forceinline__ int slot_prefix(const DecodeParams &p, const Sharing &g, int slot) {
  return min(group_prefix(p, g, slot), cached_tokens(p, slot));
}

// ---------------------------------------------------------------- plain form
// What warp `warp` of `warps` takes of a row, key by key.
template <class T, int NC>
__device__ __forceinline__ void plain_part(const DecodeParams &p, int slot, int h, int head, RowState<NC> &st, int warp, int warps) {
  const int lane = threadIdx.x & 31;
  const int n = cached_tokens(p, slot);
  float q[NC];
  load_row(q, static_cast<const T *>(p.q) + slot * p.qs[0] + h * p.qs[1], p.d, lane, p.scale_log2);
  const int *row = p.table + slot * p.ts;
  auto at = [&](int j, const T *&k, const T *&v) {
    const int entry = row[page_index(p, j)], r = j - page_index(p, j) * p.page_size;
    const bool held = (unsigned)entry < (unsigned)p.pages;
    const int64_t page = held ? entry : 0;
    k = static_cast<const T *>(p.k) + page * p.ks[0] + head * p.ks[1] + r * p.ks[2];
    v = static_cast<const T *>(p.v) + page * p.vs[0] + head * p.vs[1] + r * p.vs[2];
    return held;
  };
  if (n > 0 && p.pages > 0) {
    const Visible see = visible(n - 1, p.window, p.sinks);
    attend_keys<T>(st, q, p.d, lane, warp, see.sink_end, warps, at);
    attend_keys<T>(st, q, p.d, lane, see.lo + warp, n, warps, at);
  }
}
// A row by the WARPS warps of a CTA; warp 0 receives it.
template <class T, int WARPS, int NC>
__device__ __forceinline__ void plain_row(const DecodeParams &p, int slot, int h, int head, RowState<NC> &st, float *scratch) {
  plain_part<T>(p, slot, h, head, st, threadIdx.x >> 5, WARPS);
  join_warps<WARPS>(st, scratch);
}

}  // namespace attend

// Attention over the tokens behind every slot's prefix, unnormalised: sums[slots * q_heads][padded head size]
// and (reference, sum of weights) of every row.  The caller has checked the arguments and that
// decode_tensor() holds.
struct Suffix {
  attend::Sharing sharing;
  float *sums;
  float2 *stats;
};
int decode_suffix(int dtype, const attend::DecodeParams &p, const Suffix &suffix, cudaStream_t s);
// Whether the tensor-core form takes a call, and whether it pays (few keys go row by row).
bool decode_tensor(const attend::DecodeParams &p);
bool decode_few_keys(const attend::DecodeParams &p);
// The arguments of a call as the kernels take them, checked.
int decode_params(const char *me, attend::DecodeParams &p, int dtype, const void *q, const void *k, const void *v, void *o, float *lse,
                  const int32_t *table, const int32_t *lens, int64_t slots, int64_t width, int64_t pages, int64_t page_size,
                  int64_t q_heads, int64_t kv_heads, int64_t d, const int64_t *strides, int64_t window, int64_t sinks, float scale);
// lc_paged_decode behind its checks.
int decode_all(int dtype, const attend::DecodeParams &p, cudaStream_t s);

}  // namespace lc
