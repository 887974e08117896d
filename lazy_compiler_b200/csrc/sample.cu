// One token of every row of logits: temperature, the k likeliest, of them the shortest run
// of the likeliest that holds p of their sum, of them those of at least min_p times the
// likeliest's weight, and of what is left the one at which the sum in index order passes u
// times its total (u is given).
//
// Weights are whole numbers: W = round(2^s 2^((x - max) log2(e) / T)), s = 62 - log2(vocab)
// rounded up, 50 at most, from an exponential in f64 (2^-42 or so off).  So every sum is exact
// and the same in any order, for any split of the row and whatever atomics do; and since a cut
// is off by the weights' rounding alone, some 1e-11 of the total, the token is that of the
// definition in 64 bits but for one draw in a million even where the whole vocabulary is kept.
//
// A row is a cluster's: up to eight CTAs of 16 warps, a run of consecutive elements each.
//   1  the largest element (the pass that reads HBM; the others find the row in L2)
//   2  a threshold that at least J elements reach: the J-th largest of the threads' own maxima;
//      what reaches it goes to a list, and where top-p needs it the total is added up
//   3  where the list holds all that can be kept (the rule), one CTA has its entries in
//      registers and finds the k-th, the end of the run and the token by bisection, each a
//      sum over the CTA: of the keys' bits, of the indices' bits
//   or, where it does not: histograms over the range of keys that the cut may be in, 2048
//      bins of counts and weights each, until a bin is one key; then the sums of the warps'
//      runs, and the run that holds the token again, element by element
// Equal logits are taken in index order throughout.
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"

namespace lc {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kMostCtas = 8;
constexpr int kListed = 4, kList = kListed * kThreads;  // entries of a thread, of the list
constexpr int kBinBits = 11, kBins = 1 << kBinBits;
constexpr uint32_t kNone = 0x007fffffu;  // the key of -infinity

struct SampleParams {
  const void *logits;
  int64_t stride;
  const float *uniform;
  const float *temperature, *top_p, *min_p;  // null: the value beside it
  const int *top_k;
  float temperature_all, top_p_all, min_p_all;
  int top_k_all;
  int *token;
  float *logprob;
  int vocab, scale;  // s
};

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }

// Whole numbers in the order of the floats; -0 is 0.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ ((int32_t)b < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key ^ (key >> 31 ? 0x80000000u : 0xffffffffu));
}

// 2^(y / 256) for y <= 0 as a whole number of 2^-s: a table of 2^(i / 256), and 1 + r a1 + ... + r^3 a3 for
// the rest, |r| <= 1/2 (off by 1.4e-13).
struct Weights {
  const double *table;
  double max, factor;  // y = (x - max) factor, factor = 256 log2(e) / T
  int scale;
  __device__ __forceinline__ double place(float x) const { return x == (float)max ? 0.0 : ((double)x - max) * factor; }
  __device__ __forceinline__ uint64_t at(double y) const {
    if (!(y > -256.0 * (scale + 1))) return 0;  // rounds to nothing; NaN
    constexpr double kMagic = 6755399441055744.0, kStep = 0.6931471805599453 / 256;  // 1.5 * 2^52
    const double z = y + kMagic, r = y - (z - kMagic);
    const int j = __double2loint(z);
    double f = fma(r, kStep * kStep * kStep / 6, kStep * kStep / 2);
    f = fma(r, f, kStep);
    f = fma(r, f, 1.0) * table[j & 255];
    // times 2^(s + j / 256), then the whole number in the low bits
    f = __hiloint2double(__double2hiint(f) + ((scale + (j >> 8)) << 20), __double2loint(f)) + 4503599627370496.0;
    return (uint64_t)(__double_as_longlong(f) & 0xfffffffffffffll);
  }
  __device__ __forceinline__ uint64_t of(float x) const { return at(place(x)); }
};

struct SampleShared {
  double table[256];
  union {
    struct {
      uint32_t key[kList];
      int index[kList];
    } list;
    struct {
      uint32_t count[kBins], low[kBins], high[kBins];
    } bins;
    struct {
      uint64_t sum[kMostCtas * kWarps];
      int ties[kMostCtas * kWarps];
    } runs;
  };
  uint64_t parts[2][kWarps];
  // what the cluster's other CTAs read
  float max, threshold;
  int listed;
  uint64_t total, listed_sum;
  uint64_t run_sum[kWarps];
  int run_ties[kWarps];
  // a histogram's crossing
  uint32_t found;
  uint64_t found_sum;
  uint64_t found_count;
};

__device__ __forceinline__ uint64_t warp_total(uint64_t v) {
  // in pieces of 26 bits, whose sums over a warp fit 32
  const uint64_t a = __reduce_add_sync(0xffffffffu, (uint32_t)(v & 0x3ffffff)), b = __reduce_add_sync(0xffffffffu, (uint32_t)(v >> 26 & 0x3ffffff));
  const uint64_t c = __reduce_add_sync(0xffffffffu, (uint32_t)(v >> 52));
  return a + (b << 26) + (c << 52);
}

// Sum over the CTA, the same for every thread; one barrier a call, `turn` alternates.
__device__ __forceinline__ uint64_t block_total(uint64_t v, SampleShared &s, int &turn) {
  v = warp_total(v);
  turn ^= 1;
  if ((threadIdx.x & 31) == 0) s.parts[turn][threadIdx.x >> 5] = v;
  __syncthreads();
  uint64_t sum = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) sum += s.parts[turn][w];
  return sum;
}

// The largest key in [lo, hi] whose sum over entries of at least it reaches `want` (lo does).
template <class F>
__device__ __forceinline__ uint32_t bisect_down(uint32_t lo, uint32_t hi, uint64_t want, SampleShared &s, int &turn, const F &sum_from) {
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo + 1) / 2;
    if (block_total(sum_from(mid), s, turn) >= want)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}
// The smallest index in [0, hi] whose sum over entries up to it reaches `want` (hi does).
template <class F>
__device__ __forceinline__ int bisect_up(int hi, uint64_t want, SampleShared &s, int &turn, const F &sum_to) {
  int lo = 0;
  while (lo < hi) {
    const int mid = lo + (hi - lo) / 2;
    if (block_total(sum_to(mid), s, turn) >= want)
      hi = mid;
    else
      lo = mid + 1;
  }
  return lo;
}

// u times a total, as the whole number that a sum has to pass; p of a total, as the one it has to reach.
__device__ __forceinline__ uint64_t passed(float u, uint64_t total) {
  if (!(u > 0.f)) return 0;
  const double t = (double)u * (double)total;
  return u < 1.f && t < (double)(total - 1) ? (uint64_t)t : total - 1;
}
__device__ __forceinline__ uint64_t reached(float p, uint64_t total) {
  const double t = ceil((double)p * (double)total);
  return t < 1.0 ? 1 : t < (double)total ? (uint64_t)t : total;
}

template <class T>
struct Row {
  static constexpr int E = 16 / sizeof(T);  // elements of a vector
  const T *at;       // element 0
  int vocab, skew;   // of vector 0, the elements before element 0
  int begin, end;    // this warp's vectors
  __device__ __forceinline__ int index(int v, int e) const { return v * E + e - skew; }
  // A vector's elements; NaN where it reaches over the row's ends.
  __device__ __forceinline__ void load(int v, float (&x)[E]) const {
    const int first = index(v, 0);
    if (first >= 0 && first + E <= vocab) {
      union {
        uint4 raw;
        T t[E];
      } u;
      u.raw = __ldg(reinterpret_cast<const uint4 *>(at + first));
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = widen(u.t[e]);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = first + e >= 0 && first + e < vocab ? widen(at[first + e]) : NAN;
    }
  }
  // f(vector, elements) for the vectors of this lane, U in flight.
  template <int U, class F>
  __device__ __forceinline__ void each(const F &f) const {
    for (int v = begin + (threadIdx.x & 31); v < end; v += 32 * U) {
      float x[U][E];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (v + 32 * u < end) load(v + 32 * u, x[u]);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (v + 32 * u < end) f(v + 32 * u, x[u]);
    }
  }
};

template <class T>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const __grid_constant__ SampleParams p) {
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ SampleShared s;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), r = blockIdx.x / ctas;
  if (tid < 256) s.table[tid] = exp2(tid / 256.0);
  if (tid == 0) s.listed = 0, s.total = s.listed_sum = 0;
  pdl_wait();
  pdl_trigger();
  Row<T> row;
  row.at = static_cast<const T *>(p.logits) + r * p.stride;
  row.vocab = p.vocab;
  row.skew = (int)((reinterpret_cast<uintptr_t>(row.at) & 15) / sizeof(T));
  const int vectors = (row.skew + p.vocab + Row<T>::E - 1) / Row<T>::E;
  const int per = (vectors + ctas * kWarps - 1) / (ctas * kWarps);
  row.begin = min(vectors, (rank * kWarps + warp) * per);
  row.end = min(vectors, row.begin + per);

  const float temperature = p.temperature ? p.temperature[r] : p.temperature_all;
  const bool greedy = !(temperature > 0.f);
  int top_k = p.top_k ? p.top_k[r] : p.top_k_all;
  const float top_p = p.top_p ? p.top_p[r] : p.top_p_all, min_p = p.min_p ? p.min_p[r] : p.min_p_all;
  if (top_k <= 0 || top_k >= p.vocab) top_k = 0;
  const bool nucleus = top_p < 1.f;
  const float uniform = p.uniform[r];

  // ---- 1: the largest, and a threshold
  float largest = -INFINITY;
  row.template each<4>([&](int, const float (&x)[Row<T>::E]) {
#pragma unroll
    for (int e = 0; e < Row<T>::E; ++e) largest = fmaxf(largest, x[e]);
  });
  int turn = 0;
  const bool lists = !greedy && (top_k || nucleus);
  const uint32_t own = key_of(largest);
  {
    const uint32_t top = __reduce_max_sync(0xffffffffu, own);
    if (lane == 0) s.parts[0][warp] = top;
    __syncthreads();
    uint32_t most = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) most = max(most, (uint32_t)s.parts[0][w]);
    // at least `wanted` elements of the CTA reach it: the maxima of so many threads do
    uint32_t reach = kNone;
    const int wanted = top_k ? (top_k + ctas - 1) / ctas : 128;
    if (lists && p.vocab > kList && wanted <= kThreads / 2) {
      uint32_t lo = kNone, hi = most;
      while (lo < hi) {
        const uint32_t mid = lo + (hi - lo + 1) / 2;
        if (__syncthreads_count(own >= mid) >= wanted)
          lo = mid;
        else
          hi = mid - 1;
      }
      reach = lo;
    }
    if (tid == 0) {
      s.max = value_of(most);
      s.threshold = value_of(reach);
    }
  }
  cluster.sync();
  float threshold = INFINITY;
  for (int c = 0; c < ctas; ++c) {
    const SampleShared &other = *cluster.map_shared_rank(&s, c);
    largest = fmaxf(c ? largest : -INFINITY, other.max);
    threshold = fminf(threshold, other.threshold);
  }
  if (largest == -INFINITY) {  // nothing to take
    if (rank == 0 && tid == 0) {
      p.token[r] = -1;
      if (p.logprob) p.logprob[r] = -INFINITY;
    }
    cluster.sync();  // no CTA leaves while its shared memory is read
    return;
  }

  if (greedy) {
    int first = INT32_MAX;
    row.template each<4>([&](int v, const float (&x)[Row<T>::E]) {
#pragma unroll
      for (int e = Row<T>::E - 1; e >= 0; --e)
        if (x[e] == largest) first = min(first, row.index(v, e));
    });
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0) s.run_ties[warp] = first;
    cluster.sync();
    if (rank == 0 && warp == 0) {
      for (int x = lane; x < ctas * kWarps; x += 32) first = min(first, cluster.map_shared_rank(&s, x / kWarps)->run_ties[x % kWarps]);
      first = __reduce_min_sync(0xffffffffu, first);
      if (lane == 0) {
        p.token[r] = first;
        if (p.logprob) p.logprob[r] = 0.f;
      }
    }
    cluster.sync();
    return;
  }

  const Weights weights = {s.table, largest, 256.0 * 1.4426950408889634 / (double)temperature, p.scale};
  const double least = min_p > 0.f ? 256.0 * log2((double)fminf(min_p, 1.f)) : -INFINITY;  // of y
  // the token and the logarithm of its share
  auto answer = [&](int index, float x, uint64_t total) {
    p.token[r] = index;
    if (p.logprob) p.logprob[r] = (float)(weights.place(x) * (0.6931471805599453 / 256) + (p.scale * 0.6931471805599453 - log((double)total)));
  };
  // what is kept: keys over `cut`, and the first `ties` elements of that key
  uint32_t cut = kNone;
  int64_t ties = 0;

  if (lists) {
    // ---- 2: what reaches the threshold, and the total
    const bool sums = nucleus && !top_k;
    uint64_t total = 0;
    row.template each<2>([&](int v, const float (&x)[Row<T>::E]) {
      bool some = false;
#pragma unroll
      for (int e = 0; e < Row<T>::E; ++e) some |= x[e] >= threshold;
      if (some && *(volatile int *)&s.listed <= kList) {  // (not all of a flat row)
#pragma unroll
        for (int e = 0; e < Row<T>::E; ++e)
          if (x[e] >= threshold && x[e] > -INFINITY) {
            const int at = atomicAdd(&s.listed, 1);
            if (at < kList) s.list.key[at] = key_of(x[e]), s.list.index[at] = row.index(v, e);
          }
      }
      if (sums) {
#pragma unroll
        for (int e = 0; e < Row<T>::E; ++e) total += weights.of(x[e]);
      }
    });
    total = block_total(total, s, turn);  // (its barrier: the list is complete)
    int listed = s.listed;
    uint64_t inside = 0;
    if (sums && listed <= kList)
      for (int x = tid; x < listed; x += kThreads) inside += weights.of(value_of(s.list.key[x]));
    inside = block_total(inside, s, turn);
    if (tid == 0) s.total = total, s.listed_sum = inside;
    cluster.sync();
    total = inside = 0;
    int before = 0, all = 0;
    for (int c = 0; c < ctas; ++c) {
      const SampleShared &other = *cluster.map_shared_rank(&s, c);
      if (c == rank) before = all;
      all = (int)min((int64_t)all + other.listed, (int64_t)kList + 1);
      total += other.total;
      inside += other.listed_sum;
    }
    if (all <= kList && (!sums || inside >= reached(top_p, total))) {
      // ---- 3: all entries to the first CTA
      if (rank != 0) {
        SampleShared &to = *cluster.map_shared_rank(&s, 0);
        for (int x = tid; x < listed; x += kThreads) to.list.key[before + x] = s.list.key[x], to.list.index[before + x] = s.list.index[x];
      }
      cluster.sync();
      if (rank != 0) return;
      uint32_t key[kListed];
      int index[kListed];
      uint64_t w[kListed];
      bool kept[kListed];
#pragma unroll
      for (int x = 0; x < kListed; ++x) {
        const int at = x * kThreads + tid;
        kept[x] = at < all;
        key[x] = kept[x] ? s.list.key[at] : 0;
        index[x] = kept[x] ? s.list.index[at] : INT32_MAX;
        w[x] = kept[x] ? weights.of(value_of(key[x])) : 0;
      }
      const uint32_t lowest = key_of(threshold), highest = key_of(largest);
      // cuts the kept entries behind the `want`-th unit of `amount`, in the order of keys, then of indices
      auto cut_at = [&](uint64_t want, const uint64_t (&amount)[kListed]) {
        const uint32_t last = bisect_down(lowest, highest, want, s, turn, [&](uint32_t from) {
          uint64_t sum = 0;
#pragma unroll
          for (int x = 0; x < kListed; ++x) sum += kept[x] && key[x] >= from ? amount[x] : 0;
          return sum;
        });
        uint64_t over = 0;
#pragma unroll
        for (int x = 0; x < kListed; ++x) over += kept[x] && key[x] > last ? amount[x] : 0;
        over = block_total(over, s, turn);
        const int end = bisect_up(p.vocab - 1, want - over, s, turn, [&](int to) {
          uint64_t sum = 0;
#pragma unroll
          for (int x = 0; x < kListed; ++x) sum += kept[x] && key[x] == last && index[x] <= to ? amount[x] : 0;
          return sum;
        });
#pragma unroll
        for (int x = 0; x < kListed; ++x) kept[x] = kept[x] && (key[x] > last || (key[x] == last && index[x] <= end));
      };
      if (top_k && top_k < all) {
        const uint64_t one[kListed] = {1, 1, 1, 1};
        cut_at(top_k, one);
      }
      if (nucleus) {
        if (top_k) {
          total = 0;
#pragma unroll
          for (int x = 0; x < kListed; ++x) total += kept[x] ? w[x] : 0;
          total = block_total(total, s, turn);
        }
        cut_at(reached(top_p, total), w);
      }
      total = 0;
#pragma unroll
      for (int x = 0; x < kListed; ++x) {
        kept[x] = kept[x] && weights.place(value_of(key[x])) >= least;
        total += kept[x] ? w[x] : 0;
      }
      total = block_total(total, s, turn);
      const int token = bisect_up(p.vocab - 1, passed(uniform, total) + 1, s, turn, [&](int to) {
        uint64_t sum = 0;
#pragma unroll
        for (int x = 0; x < kListed; ++x) sum += kept[x] && index[x] <= to ? w[x] : 0;
        return sum;
      });
#pragma unroll
      for (int x = 0; x < kListed; ++x)
        if (kept[x] && index[x] == token) answer(token, value_of(key[x]), total);
      return;
    }
    // ---- or histograms.  First the k-th key by counts, then the run's end by weights.
    for (int by = top_k ? 0 : 1; by < (nucleus ? 2 : 1); ++by) {
      const uint64_t want = by == 0 ? (uint64_t)top_k : reached(top_p, total);
      uint32_t lo = kNone + 1, hi = key_of(largest);
      uint64_t over = 0, over_count = 0;  // of keys over hi: weights, elements
      for (;;) {
        const int shift = max(0, 32 - __clz(hi - lo) - kBinBits);
        cluster.sync();  // the histograms before, and the list, have been read
        for (int b = tid; b < kBins; b += kThreads) s.bins.count[b] = s.bins.low[b] = s.bins.high[b] = 0;
        if (tid == 0) s.found = UINT32_MAX;
        __syncthreads();
        row.template each<2>([&](int, const float (&x)[Row<T>::E]) {
#pragma unroll
          for (int e = 0; e < Row<T>::E; ++e) {
            const uint32_t key = key_of(x[e]);
            if (!(x[e] > -INFINITY) || key < lo || key > hi) continue;
            const uint32_t b = (hi - key) >> shift;
            const uint64_t w = weights.of(x[e]);
            atomicAdd(&s.bins.count[b], 1u);
            if (w == 0) continue;
            const uint32_t add = (uint32_t)w, old = atomicAdd(&s.bins.low[b], add);
            const uint32_t up = (uint32_t)(w >> 32) + (old + add < old);
            if (up) atomicAdd(&s.bins.high[b], up);
          }
        });
        cluster.sync();
        // a thread's consecutive bins, of all CTAs
        constexpr int kOwn = kBins / kThreads;
        uint64_t count[kOwn] = {0}, sum[kOwn] = {0}, amount = 0;
        for (int c = 0; c < ctas; ++c) {
          const SampleShared &other = *cluster.map_shared_rank(&s, c);
#pragma unroll
          for (int x = 0; x < kOwn; ++x) {
            const int b = tid * kOwn + x;
            count[x] += other.bins.count[b];
            sum[x] += ((uint64_t)other.bins.high[b] << 32) + other.bins.low[b];
          }
        }
        uint64_t counts = 0, sums_here = 0;
#pragma unroll
        for (int x = 0; x < kOwn; ++x) counts += count[x], sums_here += sum[x];
        // exclusive prefixes over the threads
        uint64_t run[2] = {counts, sums_here};
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const uint64_t mine = run[q];
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const uint64_t up = __shfl_up_sync(0xffffffffu, run[q], o);
            if (lane >= o) run[q] += up;
          }
          __syncthreads();
          if (lane == 31) s.parts[q][warp] = run[q];
          run[q] -= mine;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWarps; ++w)
          if (w < warp) run[0] += s.parts[0][w], run[1] += s.parts[1][w];
        run[0] += over_count, run[1] += over;
        amount = run[by];
#pragma unroll
        for (int x = 0; x < kOwn; ++x) {
          const uint64_t next = amount + (by ? sum[x] : count[x]);
          if (amount < want && next >= want) {
            s.found = tid * kOwn + x;
            s.found_count = run[0];
            s.found_sum = run[1];
          }
          amount = next;
          run[0] += count[x], run[1] += sum[x];
        }
        __syncthreads();
        if (s.found == UINT32_MAX) {  // fewer elements than k: all are kept
          cut = kNone, ties = 0;
          if (by == 0) {
            total = over;
            for (int w = 0; w < kWarps; ++w) total += s.parts[1][w];
          }
          break;
        }
        over_count = s.found_count, over = s.found_sum;
        hi -= s.found << shift;
        if (shift == 0) {
          const uint64_t w = weights.of(value_of(hi));
          const int64_t last = by == 0 ? (int64_t)(want - over_count) : (int64_t)((want - over + w - 1) / w);
          if (by == 0) total = over + last * w;
          // a run that ends at the k-th key keeps no more of it than the k
          ties = by == 1 && top_k && hi == cut ? min(ties, last) : last;
          cut = hi;
          break;
        }
        lo = max(lo, hi - ((1u << shift) - 1));
      }
    }
    cluster.sync();  // the histograms have been read
  }

  // ---- what is kept of every warp's run
  uint64_t sum = 0;
  int tied = 0;
  row.template each<2>([&](int, const float (&x)[Row<T>::E]) {
#pragma unroll
    for (int e = 0; e < Row<T>::E; ++e) {
      const uint32_t key = key_of(x[e]);
      if (!(x[e] > -INFINITY) || key < cut) continue;
      const double y = weights.place(x[e]);
      if (!(y >= least)) continue;
      if (key == cut)
        ++tied;
      else
        sum += weights.at(y);
    }
  });
  sum = warp_total(sum);
  tied = __reduce_add_sync(0xffffffffu, tied);
  if (lane == 0) s.run_sum[warp] = sum, s.run_ties[warp] = tied;
  cluster.sync();
  const uint64_t tie = ties ? weights.of(value_of(cut)) : 0;
  const int runs = ctas * kWarps;
  for (int x = tid; x < runs; x += kThreads) {
    const SampleShared &other = *cluster.map_shared_rank(&s, x / kWarps);
    s.runs.sum[x] = other.run_sum[x % kWarps];
    s.runs.ties[x] = other.run_ties[x % kWarps];
  }
  cluster.sync();
  // every thread the same: the total, then this warp's share of it
  uint64_t total = 0, begin = 0, end = 0;
  int64_t left = ties, left_here = 0;
  for (int x = 0; x < runs; ++x) {
    const int64_t some = min(left, (int64_t)s.runs.ties[x]);
    if (x == rank * kWarps + warp) begin = total, left_here = left;
    total += s.runs.sum[x] + some * tie;
    if (x == rank * kWarps + warp) end = total;
    left -= some;
  }
  const uint64_t target = passed(uniform, total);
  if (target < begin || target >= end) return;
  // the warp with the token: its run again
  uint64_t seen = begin;
  for (int base = row.begin; base < row.end; base += 32) {
    float x[Row<T>::E];
    const int v = base + lane;
    if (v < row.end) {
      row.load(v, x);
    } else {
#pragma unroll
      for (int e = 0; e < Row<T>::E; ++e) x[e] = NAN;
    }
    int mine = 0;  // elements of the cut's key
#pragma unroll
    for (int e = 0; e < Row<T>::E; ++e) mine += x[e] > -INFINITY && key_of(x[e]) == cut && weights.place(x[e]) >= least;
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += up;
    }
    const int64_t mine_left = left_here - (upto - mine);
    left_here -= __shfl_sync(0xffffffffu, upto, 31);
    auto weight = [&](int e, int64_t &quota) -> uint64_t {
      const uint32_t key = key_of(x[e]);
      if (!(x[e] > -INFINITY) || key < cut) return 0;
      const double y = weights.place(x[e]);
      if (!(y >= least)) return 0;
      return key != cut || quota-- > 0 ? weights.at(y) : 0;
    };
    uint64_t here = 0;
    int64_t quota = mine_left;
#pragma unroll
    for (int e = 0; e < Row<T>::E; ++e) here += weight(e, quota);
    uint64_t run = here;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t up = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += up;
    }
    const uint64_t stop = seen + run;  // behind this lane's elements
    if (target >= stop - here && target < stop) {
      uint64_t at = stop - here;
      quota = mine_left;
      bool done = false;
#pragma unroll
      for (int e = 0; e < Row<T>::E; ++e) {
        at += weight(e, quota);
        if (!done && at > target) {
          answer(row.index(v, e), x[e], total);
          done = true;
        }
      }
    }
    seen = __shfl_sync(0xffffffffu, stop, 31);
    if (seen > target) return;
  }
}

template <class T>
int launch_sample(const SampleParams &p, int64_t rows, cudaStream_t s) {
  // CTAs of a row: for few rows as many as have a vector or two a thread, for many what fills the GPU.
  const int64_t vectors = p.vocab / Row<T>::E;
  int ctas = 1;
  while (ctas < kMostCtas && vectors / ctas > kThreads && rows * ctas < 8 * sm_count()) ctas *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {(unsigned)ctas, 1, 1};
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return check_cuda(cudaLaunchKernelEx(&cfg, sample_kernel<T>, p), "lc_sample");
}

}  // namespace
}  // namespace lc

extern "C" int lc_sample(int dtype, const void *logits, const float *uniform, const float *temperature, const int32_t *top_k,
                         const float *top_p, const float *min_p, float temperature_all, int64_t top_k_all, float top_p_all,
                         float min_p_all, int32_t *token, float *logprob, int64_t rows, int64_t vocab, int64_t stride,
                         void *stream) {
  using namespace lc;
  const char *me = "lc_sample";
  if (dtype != LC_F32 && dtype != LC_F16 && dtype != LC_BF16) return fail(LC_ERR_INVALID, "%s: dtype %d is not f32, f16 or bf16", me, dtype);
  if (rows < 0 || vocab < 1) return fail(LC_ERR_INVALID, "%s: negative or zero size", me);
  if (rows > (1 << 24) || vocab > (1 << 24)) return fail(LC_ERR_UNSUPPORTED, "%s: shape too large", me);
  if (rows == 0) return LC_OK;
  if (!logits || !uniform || !token) return fail(LC_ERR_INVALID, "%s: null buffer", me);
  if (!aligned(logits, dtype == LC_F32 ? 4 : 2)) return fail(LC_ERR_ALIGN, "%s: an element's address", me);
  SampleParams p = {logits, stride, uniform, temperature, top_p, min_p, top_k, temperature_all, top_p_all, min_p_all,
                    (int)std::min<int64_t>(std::max<int64_t>(top_k_all, 0), INT32_MAX), token, logprob, (int)vocab, 0};
  int bits = 0;
  while ((1ll << bits) < vocab) ++bits;
  p.scale = std::min(50, 62 - bits);
  cudaStream_t s = as_stream(stream);
  return dtype == LC_F32 ? launch_sample<float>(p, rows, s) : dtype == LC_F16 ? launch_sample<__half>(p, rows, s) : launch_sample<__nv_bfloat16>(p, rows, s);
}
