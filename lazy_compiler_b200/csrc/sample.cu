// One token of every row of logits: temperature, the k likeliest, of them the shortest run
// of the likeliest that holds p of their sum, of them those of at least min_p times the
// likeliest's weight, and of what is left the one at which the sum in index order passes u
// times its total (u is given).
//
// Weights are whole numbers: W = round(2^s 2^((x - max) log2(e) / T)), s = 62 - log2(vocab)
// rounded up, 50 at most, from an exponential in f64 (1e-12 or so off).  So every sum is exact
// and the same in any order, for any split of the row and whatever atomics do; and since a cut
// is off by the weights' rounding alone, some 1e-11 of the total, the token is that of the
// definition in 64 bits but for one draw in a million even where the whole vocabulary is kept.
//
// A row is a cluster's: up to eight CTAs of 16 warps, a run of consecutive elements each.
//   1  the largest element, from HBM (the passes after it find the row in L2), and a threshold
//      that some hundred elements reach, from the lanes' own largest
//   2  what reaches the threshold goes to a list; where top-p asks for it, the total
//   3  one CTA has the list in registers and finds the k-th, the end of the run and the token
//      by bisection of (logit, index) and of the index, each step a sum over the threads; of a
//      short list by looking through all of it
// Where the list does not hold what may be kept, the cut is looked for first: a histogram of
// counts over 4096 equal steps of the logits, the steps that the cut may lie in (a step's weights
// are nearly one), and the list is of those, with the exact sums of what lies above them; where even
// they hold too many (equal logits), histograms of counts and weights over the keys, down to one. (Top-k with
// top-p lists the k and the rest of the last of their steps, and takes 3: 256 rows of 151643, 591 -> 195 us.)
// Then, and where nothing is cut: the sums of the warps' runs, and the run that holds the token
// again, element by element.  Equal logits are taken in index order throughout.
//
// Bound by instructions: the pass for the total takes some 10 operations in f64 and 20 others an
// element (measured by itself, 4 elements a clock and SM, 34 us of 256 rows of 151643), the list
// chains of sums over the CTA; by latencies for few rows. Measured: one row of 32000, f16, top-k and
// top-p 9 us a call; in a graph, 64 rows of 50257, bf16: top-k 17, top-p 24; 256 rows of 151643,
// f32: largest only 31 (5 TB/s), top-k 69, top-p of 0.9 107, of 0.99 249, nothing cut 99.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"

namespace lc {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kMostCtas = 8;
constexpr int kListed = 4, kList = kListed * kThreads;  // entries of a thread, of the list
constexpr int kWanted = 256;                             // entries of a list for top-p alone, at least
constexpr int kFew = 128;                                // threads that a short list is dealt to
constexpr int kOwnFew = 2;                               // entries of each of them, at which looking through all pays
constexpr int kBinBits = 11, kBins = 1 << kBinBits;     // of keys
constexpr int kSteps = 4096;                             // of logits
constexpr uint32_t kNone = 0x007fffffu;                  // the key of -infinity
constexpr float kLowest = -3.402823466e38f;              // the lowest f32
constexpr double kLn2 = 0.6931471805599453, kLog2e = 1.4426950408889634;

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
// 2^(i / 32).
__constant__ double kPowers[32] = {
    1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237, 1.0905077326652577, 1.1143867425958924,
    1.1387886347566916, 1.1637248587775775, 1.189207115002721, 1.215247359980469, 1.241857812073484,
    1.2690509571917332, 1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832,
    1.4142135623730951, 1.4451808069770467, 1.4768261459394993, 1.5091644275934228, 1.5422108254079407,
    1.5759808451078865, 1.6104903319492543, 1.645755478153965, 1.681792830507429, 1.718619298122478,
    1.7562521603732995, 1.7947090750031072, 1.8340080864093424, 1.8741676341103, 1.9152065613971474,
    1.9571441241754002};

// The next f32 below.
__device__ __forceinline__ float below(float x) {
  const uint32_t b = __float_as_uint(x);
  return __uint_as_float(x > 0.f ? b - 1 : x < 0.f ? b + 1 : 0x80000001u);
}

// 2^(y / 32), y = (x - max) factor, as a whole number of 2^-s: 2^(i / 32) from lane i, times a polynomial of
// degree 4 for the rest, |r| <= 1/2 (off by 1.2e-12 at the ends, and with r's sign).  By whole warps.  f32
// only where it is exact: the larger of x and `floor`, which weighs nothing (so does NaN, then).
struct Weights {
  double max, factor;
  float floor;
  double power;  // 2^(s + lane / 32)
  // N at a time, step by step: one after the other, the chain of ten f64 operations would be waited for.
  template <int N>
  __device__ __forceinline__ void of(const float (&x)[N], uint64_t (&w)[N]) const {
    constexpr double kMagic = 6755399441055744.0, kStep = kLn2 / 32;  // 1.5 * 2^52
    double f[N], r[N];
    int j[N], lo[N], hi[N];
#pragma unroll
    for (int e = 0; e < N; ++e) r[e] = ((double)fmaxf(x[e], floor) - max) * factor;  // (x factor - max factor would cancel where T is small)
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = r[e] + kMagic;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      j[e] = __double2loint(f[e]);
      lo[e] = __shfl_sync(0xffffffffu, __double2loint(power), j[e]);
      hi[e] = __shfl_sync(0xffffffffu, __double2hiint(power), j[e]) + ((j[e] & ~31) << 15);
      r[e] -= f[e] - kMagic;
    }
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = fma(r[e], kStep * kStep * kStep * kStep / 24, kStep * kStep * kStep / 6);
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = fma(r[e], f[e], kStep * kStep / 2);
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = fma(r[e], f[e], kStep);
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = fma(r[e], f[e], 1.0);
#pragma unroll
    for (int e = 0; e < N; ++e)  // plus 2^52: the whole number in the low bits
      w[e] = (uint64_t)__double_as_longlong(fma(f[e], __hiloint2double(hi[e], lo[e]), 4503599627370496.0)) - 0x4330000000000000ull;
  }
  __device__ __forceinline__ uint64_t of(float x) const {
    const float one[1] = {x};
    uint64_t w[1];
    of(one, w);
    return w[0];
  }
  // Temperatures that f32's logits cannot tell from none, or from infinite, are brought to where the numbers above
  // keep their range: one step of f32 below the largest weighs nothing already; 1e29.
  __device__ __forceinline__ void set(float temperature, int scale) {
    factor = 32.0 * kLog2e / fmin((double)temperature, 1e29);
    power = kPowers[threadIdx.x & 31];
    power = __hiloint2double(__double2hiint(power) + (scale << 20), __double2loint(power));
  }
  __device__ __forceinline__ void set_largest(float largest, int scale) {  // above the lowest f32
    const float next = below(largest);
    max = largest;
    factor = fmin(factor, (double)__fdiv_rd(16384.f, largest - next));
    floor = fmaxf(fminf(__fsub_rd(largest, __fdiv_ru(33.f * (scale + 2), (float)factor)), next), kLowest);
  }
};

struct alignas(16) SampleShared {
  union {
    struct {
      uint32_t key[kList];
      int index[kList];
      union {
        uint32_t count[kSteps];
        struct {  // in the first CTA: the lists, each in its part
          uint32_t in_key[kList];
          int in_index[kList];
        };
      };
    } list;
    struct {
      uint32_t count[kBins], low[kBins], high[kBins];  // (high follows low: add_word)
    } bins;
  };
  struct Part {
    uint64_t sum;
    uint32_t count, pad;
  } parts[2][kWarps];
  double scan[2][kWarps];
  float scan_steps[2][kWarps];
  // what the cluster's CTAs have left here, each in its place
  struct {
    float max, threshold, min;
    int listed;
    uint64_t total, inside, count;
  } from[2][kMostCtas];
  int first[kMostCtas * kWarps];
  uint64_t run_sum[kMostCtas * kWarps];
  int listed;
  uint64_t count;
  // what the first CTA has found
  uint32_t cut;
  int cut_index, run;
  uint64_t run_begin, kept;
  uint64_t runs[kMostCtas * kWarps];
  // a histogram's crossing
  uint32_t found, found_end;
  uint64_t found_sum, found_count;
};

struct Sum {
  uint64_t sum;
  uint32_t count;
};
// Over a warp; the counts are below 2^16 in all.
__device__ __forceinline__ Sum warp_total(uint64_t v, uint32_t count) {
  // in pieces of 26 bits, whose sums over a warp fit 32; the counts with the last, which is short
  const uint32_t a = __reduce_add_sync(0xffffffffu, (uint32_t)v & 0x3ffffff), b = __reduce_add_sync(0xffffffffu, (uint32_t)(v >> 26) & 0x3ffffff);
  const uint32_t c = __reduce_add_sync(0xffffffffu, (uint32_t)(v >> 52) | count << 16);
  return {a + ((uint64_t)b << 26) + ((uint64_t)(c & 0xffff) << 52), c >> 16};
}

// Sums over the first `threads` threads of the CTA, the same for each; one barrier a call, `turn` alternates.
struct Totals {
  SampleShared &s;
  int threads, turn;
  __device__ __forceinline__ Sum operator()(uint64_t v, uint32_t count = 0) {
    const Sum w = warp_total(v, count);
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) s.parts[turn][threadIdx.x >> 5] = {w.sum, w.count, 0};
    asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory");
    // a lane a part: sixteen warps reading sixteen parts each take a thousand cycles
    const int lane = threadIdx.x & 31;
    const bool part = lane < threads / 32;
    return warp_total(part ? s.parts[turn][lane].sum : 0, part ? s.parts[turn][lane].count : 0);
  }
};

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

// Adds a thread's N words of shared memory, maybe another CTA's, by 16 bytes: word by word, the lanes' strides make
// many accesses of one (a histogram of eight CTAs: 57000 cycles).
template <int N, class Word>
__device__ __forceinline__ void add_words(Word (&to)[N], const uint32_t *from) {
  static_assert(N % 4 == 0, "whole vectors");
#pragma unroll
  for (int x = 0; x < N; x += 4) {
    const uint4 v = *reinterpret_cast<const uint4 *>(from + x);
    to[x] += v.x, to[x + 1] += v.y, to[x + 2] += v.z, to[x + 3] += v.w;
  }
}

// Adds to 64 bits in shared memory, the upper half `high` words behind the lower: by halves, since a 64-bit addition
// there is a loop that tries until no other thread comes between.
__device__ __forceinline__ void add_word(uint32_t *low, int high, uint64_t w) {
  const uint32_t add = (uint32_t)w, old = atomicAdd(low, add);
  const uint32_t up = (uint32_t)(w >> 32) + (old + add < old);
  if (up) atomicAdd(low + high, up);
}

template <class T>
struct Row {
  static constexpr int E = 16 / sizeof(T);  // elements of a vector
  const T *at;       // element 0
  int vocab, skew;   // of vector 0, the elements before element 0
  int begin, end;    // this warp's vectors
  bool single;       // only elements that are `only` weigh anything: they are 0, the others nothing
  float only;
  __device__ __forceinline__ int index(int v, int e) const { return v * E + e - skew; }
  // A vector as it lies there; NaN where it reaches over the ends of the row or of the run.
  union Raw {
    uint4 all;
    T t[E];
  };
  __device__ __forceinline__ Raw fetch(int v) const {
    Raw raw;
    const int first = index(v, 0);
    if (v < end && first >= 0 && first + E <= vocab) {
      raw.all = __ldg(reinterpret_cast<const uint4 *>(at + first));
    } else {
      raw.all = make_uint4(UINT32_MAX, UINT32_MAX, UINT32_MAX, UINT32_MAX);  // NaN in any type
      if (v < end) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (first + e >= 0 && first + e < vocab) raw.t[e] = at[first + e];
      }
    }
    return raw;
  }
  __device__ __forceinline__ void open(const Raw &raw, float (&x)[E]) const {
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = widen(raw.t[e]);
    if (single) {
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = x[e] == only ? 0.f : -INFINITY;
    }
  }
  // A vector's elements, of a lane of this warp's.
  __device__ __forceinline__ void load(int v, float (&x)[E]) const { open(fetch(v), x); }
  // f(vector, elements) by whole warps for all vectors of this lane, U in flight while U are worked on; behind
  // the end they are NaN.
  template <int U, class F>
  __device__ __forceinline__ void each(const F &f) const {
    const int first = begin + (threadIdx.x & 31);
    Raw next[U];
#pragma unroll
    for (int u = 0; u < U; ++u) next[u] = fetch(first + 32 * u);
    for (int base = begin; base < end; base += 32 * U) {
      Raw now[U];
#pragma unroll
      for (int u = 0; u < U; ++u) now[u] = next[u];
      const int v = base + (threadIdx.x & 31);
#pragma unroll
      for (int u = 0; u < U; ++u) next[u] = fetch(v + 32 * (U + u));
      __syncwarp();
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float x[E];
        open(now[u], x);
        f(v + 32 * u, x);
      }
    }
  }
};

template <class T>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const __grid_constant__ SampleParams p) {
  constexpr int E = Row<T>::E, U = 8 / E;
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ SampleShared s;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), r = blockIdx.x / ctas;
  auto other = [&](int c) -> SampleShared & { return *cluster.map_shared_rank(&s, c); };
  if (tid == 0) s.listed = 0;
  pdl_wait();
  pdl_trigger();
  Row<T> row;
  row.at = static_cast<const T *>(p.logits) + r * p.stride;
  row.vocab = p.vocab;
  row.skew = (int)((reinterpret_cast<uintptr_t>(row.at) & 15) / sizeof(T));
  row.single = false;
  const int vectors = (row.skew + p.vocab + E - 1) / E;
  const int per = (vectors + ctas * kWarps - 1) / (ctas * kWarps);  // of a warp's run
  row.begin = min(vectors, (rank * kWarps + warp) * per);
  row.end = min(vectors, row.begin + per);

  const float temperature = p.temperature ? p.temperature[r] : p.temperature_all;
  const bool greedy = !(temperature > 0.f);
  int top_k = p.top_k ? p.top_k[r] : p.top_k_all;
  const float top_p = p.top_p ? p.top_p[r] : p.top_p_all, min_p = p.min_p ? p.min_p[r] : p.min_p_all;
  if (top_k <= 0 || top_k >= p.vocab) top_k = 0;
  const bool nucleus = top_p < 1.f, lists = !greedy && (top_k || nucleus);
  const float uniform = p.uniform[r];

  Weights weights;
  weights.set(temperature, p.scale);

  // ---- 1: the largest, where it is first, and a threshold
  float largest = -INFINITY, lowest = INFINITY;
  int place = -1;  // its vector
  row.template each<4>([&](int v, const float (&x)[E]) {
    float most = x[0];
#pragma unroll
    for (int e = 1; e < E; ++e) most = fmaxf(most, x[e]);
#pragma unroll
    for (int e = 0; e < E; ++e) lowest = fminf(lowest, x[e]);
    if (most > largest) largest = most, place = v;
  });
  {
    const uint32_t own = key_of(largest), most = __reduce_max_sync(0xffffffffu, own);
    if (lane == 0) s.parts[0][warp].sum = most;
    __syncthreads();
    const uint32_t block_most = __reduce_max_sync(0xffffffffu, lane < kWarps ? (uint32_t)s.parts[0][lane].sum : 0);
    // A key that the largest of `wanted` threads reach, and not many more: as many elements do.
    uint32_t reach = kNone;
    const int wanted = top_k ? (top_k + ctas - 1) / ctas : kWanted / ctas;
    if (lists && p.vocab > kList && wanted <= kThreads / 2) {
      uint32_t hi = block_most;
      while (reach < hi) {
        const uint32_t mid = reach + (hi - reach + 1) / 2;
        const int n = __syncthreads_count(own >= mid);
        if (n >= wanted)
          reach = mid;
        else
          hi = mid - 1;
        if (n >= wanted && n <= wanted + wanted / 16 + 2) break;  // (of half the threads: some 1600 elements, of 2048 there is room for)
      }
    }
    if (tid < ctas) {
      auto &to = other(tid).from[0][rank];
      to.max = value_of(block_most), to.threshold = value_of(reach);
    }
  }
  cluster.sync();
  const float own_largest = largest;
  const bool reads = lane < ctas;  // a lane a CTA
  largest = value_of(__reduce_max_sync(0xffffffffu, reads ? key_of(s.from[0][lane].max) : 0));
  float threshold = value_of(__reduce_min_sync(0xffffffffu, reads ? key_of(s.from[0][lane].threshold) : UINT32_MAX));
  if (greedy || largest == -INFINITY) {
    int first = INT32_MAX;
    if (own_largest == largest && place >= 0) {
      float x[E];
      row.load(place, x);
#pragma unroll
      for (int e = E - 1; e >= 0; --e)
        if (x[e] == largest) first = row.index(place, e);
    }
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0) other(0).first[rank * kWarps + warp] = first;
    cluster.sync();
    if (rank == 0 && warp == 0) {
      for (int x = lane; x < ctas * kWarps; x += 32) first = min(first, s.first[x]);
      first = __reduce_min_sync(0xffffffffu, first);
      if (lane == 0) {
        p.token[r] = largest == -INFINITY ? -1 : first;
        if (p.logprob) p.logprob[r] = largest == -INFINITY ? -INFINITY : 0.f;
      }
    }
    return;
  }
  if (largest == INFINITY || largest == kLowest) {
    row.single = true;
    row.only = largest;
    threshold = threshold == largest ? 0.f : -INFINITY;
    largest = lowest = 0.f;
  }
  weights.set_largest(largest, p.scale);
  // the least logit of weight min_p: the next f32 from the bound on
  float least = -INFINITY;
  if (min_p > 0.f) least = min_p < 1.f ? __double2float_ru((double)largest + (double)temperature * log((double)min_p)) : largest;
  // the sum of a vector's weights
  auto weigh = [&](const float (&x)[E]) {
    uint64_t sum = 0;  // four at a time: eight leave the 64 registers
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      const float four[4] = {x[e], x[e + 1], x[e + 2], x[e + 3]};
      uint64_t w[4];
      weights.of(four, w);
      sum += w[0] + w[1] + w[2] + w[3];
    }
    return sum;
  };
  // the token and the logarithm of its share
  auto answer = [&](int index, float x, uint64_t total) {
    p.token[r] = index;
    const double of_largest = x == largest ? 0.0 : ((double)x - (double)largest) / (double)temperature;
    if (p.logprob) p.logprob[r] = (float)(of_largest + (p.scale * kLn2 - log((double)total)));
  };
  Totals totals = {s, kThreads, 0};
  // What is kept: keys over `cut`, and of that key the indices up to `cut_index`.
  uint32_t cut = kNone;
  int cut_index = -1;
  bool have_runs = false;

  if (lists) {
    // ---- 2: what reaches the threshold, and the total
    const bool sums = nucleus && !top_k;
    auto list = [&](int v, const float (&x)[E], float from, float to) {  // logits from .. to
      bool some = false;
#pragma unroll
      for (int e = 0; e < E; ++e) some |= x[e] >= from && x[e] <= to;
      if (some && *(volatile int *)&s.listed <= kList) {  // (not all of a flat row)
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (x[e] >= from && x[e] <= to && x[e] > -INFINITY) {
            const int at = atomicAdd(&s.listed, 1);
            if (at < kList) s.list.key[at] = key_of(x[e]), s.list.index[at] = row.index(v, e);
          }
      }
      __syncwarp();
    };
    float list_lo = threshold, list_hi = largest;
    uint64_t total = 0, inside = 0;  // of weights: of all (or above a list), in the list
    uint64_t count = 0;              // above the list
    int all = 0;                     // entries of all
    // Sums up `total`, `count` and the list over the cluster, and takes the lists to the first CTA, if each fits its part.
    const int part = kList / ctas;
    int exchanges = 0;
    auto exchange = [&](bool weighs, bool counts) {
      exchanges ^= 1;
      if (weighs)
        total = totals(total).sum;  // (its barrier: the list is complete)
      else
        __syncthreads();
      if (counts) count = totals(count).sum;
      const int listed = s.listed;
      inside = 0;
      if (sums && listed <= part) {
        for (int x = 0; x < listed; x += kThreads) inside += weights.of(x + tid < listed ? value_of(s.list.key[x + tid]) : NAN);
        inside = totals(inside).sum;
      }
      if (tid < ctas) {
        auto &to = other(tid).from[exchanges][rank];
        to.listed = listed <= part ? listed : kList + 1;
        to.total = total, to.inside = inside, to.count = count;
      }
      if (listed <= part) {
        SampleShared &to = other(0);
        for (int x = tid; x < listed; x += kThreads) to.list.in_key[rank * part + x] = s.list.key[x], to.list.in_index[rank * part + x] = s.list.index[x];
      }
      cluster.sync();
      const auto &have = s.from[exchanges][lane & (kMostCtas - 1)];
      total = warp_total(reads ? have.total : 0, 0).sum;
      if (sums) inside = warp_total(reads ? have.inside : 0, 0).sum;
      if (counts) count = warp_total(reads ? have.count : 0, 0).sum;
      all = min((int)__reduce_add_sync(0xffffffffu, reads ? have.listed : 0), kList + 1);
    };
    row.template each<1>([&](int v, const float (&x)[E]) {
      list(v, x, threshold, INFINITY);
      if (sums) total += weigh(x);
    });
    lowest = value_of(__reduce_min_sync(0xffffffffu, key_of(lowest)));
    if (lane < ctas) other(lane).first[rank * kWarps + warp] = (int)(key_of(lowest) ^ 0x80000000u);  // in the order of ints
    exchange(sums, false);
    const uint64_t row_total = total, want_sum = sums ? reached(top_p, total) : 0;

    // In the first CTA: the lists' entries into the registers of its first threads.
    uint32_t key[kListed];
    int index[kListed];
    uint64_t w[kListed];
    bool kept[kListed];
    int threads = 0;
    auto gather = [&] {
      threads = all <= kListed * kFew ? kFew : kThreads;
      totals.threads = threads;
      if (tid >= threads) return;
#pragma unroll
      for (int x = 0; x < kListed; ++x) {
        int at = x * threads + tid, c = 0;
        kept[x] = at < all;
        if (kept[x])
          for (int n; at >= (n = s.from[exchanges][c].listed); ++c) at -= n;
        key[x] = kept[x] ? s.list.in_key[c * part + at] : 0;
        index[x] = kept[x] ? s.list.in_index[c * part + at] : 0;
      }
      __syncwarp();
#pragma unroll
      for (int x = 0; x < kListed; ++x) w[x] = weights.of(kept[x] ? value_of(key[x]) : NAN);
    };
    // Keys, then indices from the lowest, as one number in the order of what is kept first: of as few bits as tell the
    // type's keys and the row's indices apart, each of which may be a step (64 rows of 50257, bf16, top-k of 50: 25 -> 17 us).
    constexpr int kSame = sizeof(T) == 4 ? 0 : std::is_same<T, __half>::value ? 13 : 16;  // a widened number's last bits
    const int index_bits = 32 - __clz(p.vocab - 1 | 1);
    auto place_of = [&](uint32_t key, int index) { return (uint64_t)(key >> kSame) << index_bits | (unsigned)(p.vocab - 1 - index); };
    auto order_of = [&](int x) { return place_of(key[x], index[x]); };
    // The entry that holds the `want`-th unit of `amount` of the kept entries: those up to it stay.
    auto cut_list = [&](uint64_t want, auto amount) {
      uint64_t lo = place_of(key_of(list_lo), p.vocab - 1), hi = place_of(key_of(list_hi), 0);
      uint32_t n = 0;
#pragma unroll
      for (int x = 0; x < kListed; ++x) n += kept[x];
      for (n = totals(0, n).count; n > 1;) {  // the entry is one of the n in lo .. hi
        const uint64_t mid = lo + (hi - lo) / 2 + 1;
        uint64_t sum = 0;
        uint32_t upper = 0;
#pragma unroll
        for (int x = 0; x < kListed; ++x)
          if (kept[x] && order_of(x) >= mid) sum += amount(x), upper += order_of(x) <= hi;
        const Sum t = totals(sum, upper);
        if (t.sum >= want)
          lo = mid, n = t.count;
        else
          hi = mid - 1, n -= t.count;
      }
#pragma unroll
      for (int x = 0; x < kListed; ++x) kept[x] = kept[x] && order_of(x) >= lo;
    };
    auto one = [](int) -> uint64_t { return 1; };
    auto weight = [&](int x) -> uint64_t { return w[x]; };

    bool found = false;
    for (bool again = false;;) {  // once, or once more with another list
      if (all <= kList && (!sums || inside >= want_sum) && (!again || all >= top_k)) {
        // ---- 3
        if (rank != 0) return;
        gather();
        if (tid >= threads) return;
        if (all <= kOwnFew * kFew) {
          // So few that each thread looks through all of them for what lies before its own: twice, where bisection
          // takes some twenty sums a cut (in a graph, with this and without; top-k of 50 with top-p of 0.9: 64 rows of
          // 50257, bf16, 17.0 and 20.1 us, one of 32000 13.3 and 14.4; top-k alone: 16.8 and 17.8, 13.0 and 12.5).
          struct Entry {
            uint64_t place, weight;
          };
          Entry *entries = reinterpret_cast<Entry *>(s.list.key);  // (the first CTA's own list has gone to in_key)
          uint64_t place[kOwnFew], before[kOwnFew], sum = 0;
          int above[kOwnFew];
          auto look = [&] {
#pragma unroll
            for (int x = 0; x < kOwnFew; ++x) {
              if (x * kFew + tid < all) entries[x * kFew + tid] = {place[x], kept[x] ? w[x] : 0};
              before[x] = 0, above[x] = 0;
            }
            asm volatile("bar.sync 1, %0;" ::"n"(kFew) : "memory");
#pragma unroll 4
            for (int i = 0; i < all; ++i) {
              const Entry e = entries[i];
#pragma unroll
              for (int x = 0; x < kOwnFew; ++x)
                if (e.place > place[x]) before[x] += e.weight, ++above[x];
            }
          };
#pragma unroll
          for (int x = 0; x < kOwnFew; ++x) place[x] = order_of(x);
          look();
          if (top_k) {
#pragma unroll
            for (int x = 0; x < kOwnFew; ++x) kept[x] = kept[x] && above[x] < top_k;
          }
          if (nucleus) {
            if (top_k) {
#pragma unroll
              for (int x = 0; x < kOwnFew; ++x) sum += kept[x] ? w[x] : 0;
              sum = totals(sum).sum;
            }
            const uint64_t want = reached(top_p, sums ? row_total : sum);
#pragma unroll
            for (int x = 0; x < kOwnFew; ++x) kept[x] = kept[x] && before[x] < want;
          }
          sum = 0;
#pragma unroll
          for (int x = 0; x < kOwnFew; ++x) {
            kept[x] = kept[x] && value_of(key[x]) >= least;
            sum += kept[x] ? w[x] : 0;
            place[x] = (unsigned)(p.vocab - 1 - index[x]);  // now by the index alone
          }
          const uint64_t left = totals(sum).sum, target = passed(uniform, left);
          look();
#pragma unroll
          for (int x = 0; x < kOwnFew; ++x)
            if (kept[x] && before[x] <= target && target - before[x] < w[x]) answer(index[x], value_of(key[x]), left);
          return;
        }
        if (top_k && top_k < all) cut_list(top_k, one);
        uint64_t sum = 0;
        if (nucleus) {
          if (top_k) {
#pragma unroll
            for (int x = 0; x < kListed; ++x) sum += kept[x] ? w[x] : 0;
            sum = totals(sum).sum;
          }
          cut_list(reached(top_p, sums ? row_total : sum), weight);
        }
        sum = 0;
        uint32_t n = 0;
#pragma unroll
        for (int x = 0; x < kListed; ++x) {
          kept[x] = kept[x] && value_of(key[x]) >= least;
          sum += kept[x] ? w[x] : 0;
          n += kept[x];
        }
        const Sum left = totals(sum, n);
        const uint64_t target = passed(uniform, left.sum);
        n = left.count;
        int lo = 0, hi = p.vocab - 1;
        while (n > 1) {  // the token is one of the n in lo .. hi
          const int mid = lo + (hi - lo) / 2;
          sum = 0;
          uint32_t lower = 0;
#pragma unroll
          for (int x = 0; x < kListed; ++x)
            if (kept[x] && index[x] <= mid) sum += w[x], lower += index[x] >= lo;
          const Sum t = totals(sum, lower);
          if (t.sum > target)
            hi = mid, n = t.count;
          else
            lo = mid + 1, n -= t.count;
        }
#pragma unroll
        for (int x = 0; x < kListed; ++x)
          if (kept[x] && index[x] >= lo && index[x] <= hi) answer(index[x], value_of(key[x]), left.sum);
        return;
      }

      if (again) break;
      {
        // ---- the steps of the logits that the cut may lie in: by weights below the list, if there is one, down to
        // where weights are nothing
        const bool under = sums && all <= kList;
        for (int x = lane; x < ctas * kWarps; x += 32) lowest = fminf(lowest, value_of((uint32_t)s.first[x] ^ 0x80000000u));
        lowest = value_of(__reduce_min_sync(0xffffffffu, key_of(lowest)));
        const float range_hi = under ? threshold : largest;
        const float range_lo = fmaxf(lowest, largest - (float)((p.scale + 2) * kLn2 * (double)temperature));
        const float step = (range_hi - range_lo) / kSteps, per_step = kSteps / (range_hi - range_lo);
        const float range_to = under ? range_hi : INFINITY;  // the largest is at range_hi, and counts
        float lo = range_lo, hi = range_hi;
        if (step > 0.f && step < 1e30f && per_step < 1e30f) {
          cluster.sync();  // the list has been read
          for (int b = tid; b < kSteps; b += kThreads) s.list.count[b] = 0;
          if (tid == 0) s.found = s.found_end = UINT32_MAX, s.listed = 0;
          __syncthreads();
          row.template each<U>([&](int, const float (&x)[E]) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
              const int b = min(kSteps - 1, (int)((range_hi - x[e]) * per_step));
              if (x[e] >= range_lo && x[e] < range_to) atomicAdd(&s.list.count[b], 1u);
            }
          });
          if (ctas > 1) {
            // A CTA adds up its part of the steps, for all of them (each reading all of eight took 21000 cycles).
            cluster.sync();
            for (int x = tid; x < kSteps / 4 / ctas; x += kThreads) {
              const int at = rank * (kSteps / ctas) + 4 * x;
              uint32_t n[4] = {0};
#pragma unroll
              for (int c = 0; c < kMostCtas; ++c)
                if (c < ctas) add_words(n, other(c).list.count + at);
#pragma unroll
              for (int c = 0; c < kMostCtas; ++c)
                if (c < ctas) *reinterpret_cast<uint4 *>(other(c).list.count + at) = make_uint4(n[0], n[1], n[2], n[3]);
            }
          }
          cluster.sync();
          // A thread's consecutive steps: their elements, and the least and the most that their weights (of the
          // largest's) may come to: of the steps' edges, a little wider for the rounding of a step's number, of
          // the exponential and of the weights.
          constexpr int kOwn = kSteps / kThreads;
          uint32_t n[kOwn] = {0};
          add_words(n, s.list.count + tid * kOwn);
          const float unit = exp2f(-(float)p.scale), octaves = (float)(weights.factor / 32);
          const float wider = exp2f(0.01f * step * octaves) * (1 + 1e-4f);
          float amounts[2][kOwn];
          float edge = exp2f(fminf(0.f, (range_hi - (float)(tid * kOwn) * step - largest) * octaves));
#pragma unroll
          for (int x = 0; x < kOwn; ++x) {
            const float next = exp2f(fminf(0.f, (range_hi - (float)(tid * kOwn + x + 1) * step - largest) * octaves));
            amounts[0][x] = sums ? n[x] * fmaxf(0.f, next / wider - unit) : n[x];
            amounts[1][x] = sums ? n[x] * (edge * wider + unit) : n[x];
            edge = next;
          }
          float run[2];
#pragma unroll
          for (int side = 0; side < 2; ++side) {
            float mine = 0.f;
#pragma unroll
            for (int x = 0; x < kOwn; ++x) mine += amounts[side][x];
            run[side] = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const float up = __shfl_up_sync(0xffffffffu, run[side], o);
              if (lane >= o) run[side] += up;
            }
            if (lane == 31) s.scan_steps[side][warp] = run[side];
            run[side] -= mine;
          }
          __syncthreads();
#pragma unroll
          for (int x = 0; x < kWarps; ++x) {
            run[0] += x < warp ? s.scan_steps[0][x] : 0.f;
            run[1] += x < warp ? s.scan_steps[1][x] : 0.f;
          }
          // the first step that may hold the cut, and the first by which it is surely reached: f32's sums of weights are
          // off by 4e-6 or less (40 additions one after the other, and a difference), its counts are exact
          const float need = sums ? (float)((double)(under ? want_sum - inside : want_sum) * (double)unit) : (float)top_k, off = sums ? 1e-5f : 0.f;
          uint32_t from = UINT32_MAX, to = UINT32_MAX;
#pragma unroll
          for (int x = 0; x < kOwn; ++x) {
            run[0] += amounts[0][x];
            run[1] += amounts[1][x];
            if (n[x] && run[1] * (1 + off) >= need) from = min(from, tid * kOwn + x);
            if (n[x] && run[0] * (1 - off) >= need) to = min(to, tid * kOwn + x);
          }
          from = __reduce_min_sync(0xffffffffu, from);
          to = __reduce_min_sync(0xffffffffu, to);
          if (lane == 0 && from != UINT32_MAX) atomicMin(&s.found, from);
          if (lane == 0 && to != UINT32_MAX) atomicMin(&s.found_end, to);
          __syncthreads();
          const uint32_t step_from = s.found, step_to = s.found_end;
          if (step_from == UINT32_MAX && !nucleus) {
            found = true;  // fewer than k elements weigh anything: no cut
          } else if (step_from != UINT32_MAX) {
            if (step_from > 0) hi = range_hi - ((float)step_from - 0.01f) * step;
            if (step_to < kSteps - 1) lo = range_hi - ((float)step_to + 1.01f) * step;
            // the list of lo .. hi, and the sums of what lies above it
            list_lo = lo, list_hi = hi;
            cluster.sync();  // the histogram has been read, in whose place lists may arrive
            if (nucleus && !sums) {  // the k and what else the last step holds, as a list of another threshold
              list_hi = largest;
              row.template each<1>([&](int v, const float (&x)[E]) { list(v, x, lo, INFINITY); });
              exchange(false, false);
              again = true;
              continue;
            }
            uint64_t mine = 0;  // of this warp's run, of those that min_p leaves
            total = count = 0;
            row.template each<1>([&](int v, const float (&x)[E]) {
              list(v, x, lo, hi);
              float over[E];
              bool some = false;
#pragma unroll
              for (int e = 0; e < E; ++e) {
                const bool is = x[e] > hi;
                some |= is;
                count += is;
                over[e] = is ? x[e] : -INFINITY;
              }
              if (!__any_sync(0xffffffffu, some)) return;
              total += weigh(over);
              if (least > hi) {
#pragma unroll
                for (int e = 0; e < E; ++e) over[e] = over[e] >= least ? over[e] : -INFINITY;
                mine += weigh(over);
              }
            });
            if (!(least > hi)) mine = total;
            mine = warp_total(mine, 0).sum;
            if (lane == 0) other(0).run_sum[rank * kWarps + warp] = mine;
            exchange(true, true);
            if (all <= kList && (sums ? total < want_sum && total + inside >= want_sum : count < (uint64_t)top_k && count + all >= (uint64_t)top_k)) {
              found = have_runs = true;
              if (rank == 0) {
                for (int x = tid; x < ctas * kWarps; x += kThreads) s.runs[x] = s.run_sum[x];
                gather();
              }
              if (rank == 0 && tid < threads) {
                if (sums)
                  cut_list(want_sum - total, weight);
                else
                  cut_list(top_k - count, one);
                // the kept entries join their runs
#pragma unroll
                for (int x = 0; x < kListed; ++x)
                  if (kept[x] && value_of(key[x]) >= least) add_word(reinterpret_cast<uint32_t *>(&s.runs[(index[x] + row.skew) / E / per]), 1, w[x]);
                // the last of them is the cut
                uint32_t last = UINT32_MAX;
#pragma unroll
                for (int x = 0; x < kListed; ++x)
                  if (kept[x]) last = min(last, key[x]);
                if (tid == 0) s.found = UINT32_MAX, s.cut_index = -1;
                totals(0);
                last = __reduce_min_sync(0xffffffffu, last);
                if (lane == 0) atomicMin(&s.found, last);
                totals(0);
#pragma unroll
                for (int x = 0; x < kListed; ++x)
                  if (kept[x] && key[x] == s.found) atomicMax(&s.cut_index, index[x]);
                totals(0);
                if (tid == 0) s.cut = s.found;
              }
              totals.threads = kThreads;
              totals.turn = 0;  // the others have not taken part
              cluster.sync();
              cut = other(0).cut;
              cut_index = other(0).cut_index;
            }
          }
        }
      }
      break;
    }
    if (!found) {
      // ---- histograms of the keys.  First the k-th key by counts, then the run's end by weights.
      total = row_total;
      uint32_t k_cut = kNone;
      int64_t ties = 0, all_ties = 0;  // of the cut's key: those kept, those there are
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
          row.template each<U>([&](int, const float (&x)[E]) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
              const uint32_t key = key_of(x[e]);
              const bool in = x[e] > -INFINITY && key >= lo && key <= hi;
              if (!__any_sync(0xffffffffu, in)) continue;
              const uint64_t w = weights.of(x[e]);
              if (!in) continue;
              const uint32_t b = (hi - key) >> shift;
              atomicAdd(&s.bins.count[b], 1u);
              if (w != 0) add_word(&s.bins.low[b], kBins, w);
            }
            __syncwarp();
          });
          cluster.sync();
          // a thread's consecutive bins, of all CTAs
          constexpr int kOwn = kBins / kThreads;
          uint64_t counts[kOwn] = {0}, weighs[kOwn] = {0};
          for (int c = 0; c < ctas; ++c) {
            add_words(counts, other(c).bins.count + tid * kOwn);
            add_words(weighs, other(c).bins.low + tid * kOwn);
            uint64_t high[kOwn] = {0};
            add_words(high, other(c).bins.high + tid * kOwn);
#pragma unroll
            for (int x = 0; x < kOwn; ++x) weighs[x] += high[x] << 32;
          }
          uint64_t run[2] = {0, 0};
#pragma unroll
          for (int x = 0; x < kOwn; ++x) run[0] += counts[x], run[1] += weighs[x];
          // exclusive prefixes over the threads
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const uint64_t mine = run[q];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const uint64_t up = __shfl_up_sync(0xffffffffu, run[q], o);
              if (lane >= o) run[q] += up;
            }
            if (lane == 31) s.scan[q][warp] = __longlong_as_double((long long)run[q]);
            run[q] -= mine;
          }
          __syncthreads();
          uint64_t whole = over;
          for (int x = 0; x < kWarps; ++x) {
            const uint64_t a = __double_as_longlong(s.scan[0][x]), b = __double_as_longlong(s.scan[1][x]);
            if (x < warp) run[0] += a, run[1] += b;
            whole += b;
          }
          run[0] += over_count, run[1] += over;
#pragma unroll
          for (int x = 0; x < kOwn; ++x) {
            const uint64_t next[2] = {run[0] + counts[x], run[1] + weighs[x]};
            if (run[by] < want && next[by] >= want) {
              s.found = tid * kOwn + x;
              s.found_count = run[0];
              s.found_sum = run[1];
              s.count = counts[x];
            }
            run[0] = next[0], run[1] = next[1];
          }
          __syncthreads();
          if (s.found == UINT32_MAX) {  // fewer elements than k: all are kept
            total = whole;
            break;
          }
          over_count = s.found_count, over = s.found_sum;
          hi -= s.found << shift;
          if (shift == 0) {
            const uint64_t w = weights.of(value_of(hi));
            int64_t last = by == 0 ? (int64_t)(want - over_count) : (int64_t)((want - over + w - 1) / w);
            if (by == 0) total = over + last * w, k_cut = hi;
            // a run that ends at the k-th key keeps no more of it than the k
            if (by == 1 && top_k && hi == k_cut) last = min(ties, last);
            ties = last;
            all_ties = (int64_t)s.count;
            cut = hi;
            break;
          }
          lo = max(lo, hi - ((1u << shift) - 1));
        }
      }
      cut_index = INT32_MAX;
      if (ties < all_ties) {
        // the index of the last of them: the warps' runs count theirs, and the one that has it looks again
        int64_t mine = 0;
        row.template each<U>([&](int, const float (&x)[E]) {
#pragma unroll
          for (int e = 0; e < E; ++e) mine += x[e] > -INFINITY && key_of(x[e]) == cut;
        });
        mine = (int64_t)warp_total((uint64_t)mine, 0).sum;
        if (lane < ctas) other(lane).run_sum[rank * kWarps + warp] = (uint64_t)mine;
        cluster.sync();
        int64_t before_me = 0;
        for (int x = lane; x < rank * kWarps + warp; x += 32) before_me += (int64_t)s.run_sum[x];
        before_me = (int64_t)warp_total((uint64_t)before_me, 0).sum;
        if (before_me < ties && before_me + mine >= ties) {
          int left = (int)(ties - before_me);
          for (int base = row.begin; base < row.end && left > 0; base += 32) {
            float x[E];
            row.load(base + lane, x);
            __syncwarp();
            int here = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) here += x[e] > -INFINITY && key_of(x[e]) == cut;
            int upto = here;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const int up = __shfl_up_sync(0xffffffffu, upto, o);
              if (lane >= o) upto += up;
            }
            int at = upto - here;
#pragma unroll
            for (int e = 0; e < E; ++e)
              if (x[e] > -INFINITY && key_of(x[e]) == cut && ++at == left) other(0).cut_index = row.index(base + lane, e);
            left -= __shfl_sync(0xffffffffu, upto, 31);
          }
        }
        cluster.sync();
        cut_index = other(0).cut_index;
      }
    }
  }

  // A logit that is kept, or nothing in its place: those over `bound`, and of it the indices up to `bound_index`.
  float bound = value_of(cut);
  int bound_index = cut_index;
  if (least > bound) {
    bound = below(least);
    bound_index = -1;
  }
  auto kept_of = [&](float x, int index) { return x > bound || (bound_index >= 0 && x == bound && index <= bound_index) ? x : -INFINITY; };
  if (!have_runs) {
    // ---- what is kept of every warp's run
    uint64_t sum = 0;
    row.template each<1>([&](int v, const float (&x)[E]) {
      float kept[E];
#pragma unroll
      for (int e = 0; e < E; ++e) kept[e] = kept_of(x[e], row.index(v, e));
      sum += weigh(kept);
    });
    sum = warp_total(sum, 0).sum;
    if (lane == 0) other(0).runs[rank * kWarps + warp] = sum;
    cluster.sync();
  }
  if (rank == 0) {
    __syncthreads();
    if (warp == 0) {  // the run with the token, and the sum of those before it
      constexpr int kOwn = kMostCtas * kWarps / 32;
      uint64_t sums[kOwn], upto = 0;
#pragma unroll
      for (int x = 0; x < kOwn; ++x) {
        sums[x] = lane * kOwn + x < ctas * kWarps ? s.runs[lane * kOwn + x] : 0;
        upto += sums[x];
      }
      uint64_t at = upto;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint64_t up = __shfl_up_sync(0xffffffffu, at, o);
        if (lane >= o) at += up;
      }
      const uint64_t kept = __shfl_sync(0xffffffffu, at, 31), target = passed(uniform, kept);
      at -= upto;
#pragma unroll
      for (int x = 0; x < kOwn; ++x) {
        if (target >= at && target < at + sums[x]) s.run = lane * kOwn + x, s.run_begin = at;
        at += sums[x];
      }
      if (lane == 0) s.kept = kept;
    }
  }
  cluster.sync();
  const int run = other(0).run;
  const uint64_t total = other(0).kept, target = passed(uniform, total);
  uint64_t seen = other(0).run_begin;
  cluster.sync();
  if (run / kWarps != rank) return;
  // ---- that run again, a sixteenth a warp, and the sixteenth that holds the token once more
  const int run_end = min(vectors, (run + 1) * per), share = (per + kWarps - 1) / kWarps;
  row.begin = min(run_end, run * per + warp * share);
  row.end = min(run_end, row.begin + share);
  uint64_t mine = 0;
  row.template each<1>([&](int v, const float (&x)[E]) {
    float kept[E];
#pragma unroll
    for (int e = 0; e < E; ++e) kept[e] = kept_of(x[e], row.index(v, e));
    mine += weigh(kept);
  });
  mine = warp_total(mine, 0).sum;
  if (lane == 0) s.run_sum[warp] = mine;
  __syncthreads();
  for (int x = 0; x < warp; ++x) seen += s.run_sum[x];
  if (target < seen || target >= seen + mine) return;
  for (int base = row.begin; base < row.end; base += 32) {
    float x[E];
    const int v = base + lane;
    row.load(v, x);
    __syncwarp();
    uint64_t w[E], here = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = kept_of(x[e], row.index(v, e));
    weights.of(x, w);
#pragma unroll
    for (int e = 0; e < E; ++e) here += w[e];
    uint64_t upto = here;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t up = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += up;
    }
    uint64_t at = seen + upto - here;
    seen += __shfl_sync(0xffffffffu, upto, 31);
    if (seen <= target) continue;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (target >= at && target < at + w[e]) answer(row.index(v, e), x[e], total);
      at += w[e];
    }
    return;
  }
}

template <class T>
int launch_sample(const SampleParams &p, int64_t rows, cudaStream_t s) {
  // CTAs of a row: for few rows as many as have a vector a thread, for many so that all rows are in work at once;
  // but two where there are vectors for them, since a row whose cut lies deep holds its CTAs twice as long (256
  // rows of 151643, f32, every fourth of them: 169 us with two, 213 with one, 218 with four).
  const int64_t vectors = p.vocab / Row<T>::E;
  int ctas = 1;
  while (ctas < kMostCtas && vectors / ctas > kThreads && (ctas == 1 || rows * ctas * 2 <= 2 * sm_count())) ctas *= 2;
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
