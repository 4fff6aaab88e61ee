// The k largest scores of each row, in descending order, equal ones by ascending class, and the row's
// log-sum-exp.
//
// Every score gets a key that no other of its row has: its value as an ordered integer, then the
// complement of its class.  NaN is above everything, -0 equals +0.
//
// Rows above kWarpCols are taken by a block, whose threads see one group of elements each.  A bound tau that at
// least k, and hardly more, of the groups' best keys reach is found bit by bit (one warp counts, until few
// too many are left); at least k elements reach it, and all that do lie in those groups: only these are read
// again, from L1 or L2, dealt out anew to all threads.  Random rows leave little more than k candidates whatever
// the row's length; each finds its place by counting the larger ones.  Where there are more than the list
// holds, the k-th key itself is found bit by bit.  Shorter rows stay in the registers of a warp, which
// finds its bound by votes on all of them, and many rows of up to 16 KB are a
// warp's that reads them twice.  Rows of a few classes are taken by one thread each, from a tile in
// shared memory, which keeps its best sorted in registers.
//
// Bound by memory: one pass over the scores, which also takes the running maximum and sum of the
// log-sum-exp.  Of a thread's best score that pass keeps the value and the 16 bytes that hold it; the keys of
// their first and last element stand for its own above and below.
// Where rows are few, several blocks share one: up to eight as a cluster, whose first block joins the lists over
// distributed shared memory; of longer rows a second kernel does.
//
// The same kernels give a row's scores (score_common.cuh) with its best classes, of which the log probabilities are then
// written: kScored.  (With a pass of its own for the scores 4096 x 32,768 bf16, k 8, took
// 138 us, now 74; 1 x 50,001 fp32, k 20, 23.5 and 10.3; 1,000,003 x 10 fp32, k 3, 467 and 33.)
#include <cooperative_groups.h>

#include <algorithm>

#include "score_common.cuh"

namespace b2fil {
namespace distill {
namespace {

constexpr int kThreads  = 256;   // groups of a block: at least the largest k
constexpr int kList     = 2048;  // candidates of a block
constexpr int kWarpList = 320;   // candidates of a warp: at least the largest k
constexpr int kWarpCols = 2048;  // longest rows of a warp (fp64: 1024)
constexpr int kWarpTop  = 24;    // k up to which a warp finds its bound by its lanes' best alone, and the largest of
                                 // rows above 1024 (30,000 x 2000: fp32, k 10 70 us, by blocks 258; bf16, k 100
                                 // 414 and 367)
// Rows of a warp that its registers do not hold: bytes, and rows per SM from which on.  (By blocks and this way, us:
// 30,000 x 3000 bf16, k 10, 268 and 104; 20,000 x 8192 bf16 189 and 107, fp32 equal; 20,000 x 2048 fp64 456 and 136;
// 1184 x 4096 bf16 14.8 and 12.8, x 8192 14.7 and 16.8.)
constexpr int kLongBytes = 16384;
constexpr int kLongLeast = 8;
// Bytes of scored rows that a warp takes by groups where there are kLongLeast rows per SM, as many times that as there are more of them, and at
// most kGroupMost.  (us of a call, k 8, by blocks and this way: 20,000 x 3000 bf16 204 and 53, 4096 x 4096 fp32 44 and 23, 4096 x 16,384 bf16 57
// and 43, x 20,001 72 and 55, x 32,768 82 and 85 (one after the other 74 and 68; k 24 88 and 98), 8192 x 32,768 156 and 147, x 50,001 217 and
// 213, k 24 242 and 257, 8192 x 12,000 fp32 145 and 100, 20,000 x 40,000 bf16 465 and 377, 1300 x 16,384 22 and 26, x 8192 17 and 16, 2600 x
// 32,768 59 and 66.)
constexpr int64_t kGroupBytes = 16384;
constexpr int64_t kGroupMost  = 6 * kGroupBytes;
constexpr int kCount    = 160;   // candidates of a block that are placed by counting; more are sorted
constexpr int kCluster  = 8;     // blocks that share a row of up to kJoinCols and join their lists themselves
constexpr int64_t kJoinCols = 1 << 17;  // (1 x 50,001, k 20: 13.8 us by two kernels, 10.7 this way, 14.2 by 16 blocks)
constexpr int kMore     = 8;     // groups more than k that end the search of the bound
constexpr int kInFlight = 4;
// Rows for one thread each: tiles of kTileRows.  A thread takes some 5 k instructions per score, a warp with a row
// 20 per score and lane and 300 more: many short rows are a thread's (200,000 x 64 fp32, k 4: 155 us by
// warps), few or long ones a warp's, since a thread's steps follow one another.
constexpr int kTileBytes = 512;  // of a row
constexpr int kTileTop   = 32;   // largest k, and most classes where k is above 8
constexpr int kTileSteps = 160;  // classes x (k + 1) that a thread takes however few rows there are
constexpr int kTileLeast = 32;   // rows per SM from which on threads take the others
static_assert(kThreads >= kMostTop, "a group per entry");

// ---- keys ----------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t ordered(float x)
{
  x += 0.f;
  const uint32_t b = __float_as_uint(x);
  return x != x ? ~0u : b ^ ((b >> 31) ? ~0u : 0x80000000u);
}
__device__ __forceinline__ uint64_t ordered(double x)
{
  x += 0.0;
  const uint64_t b = __double_as_longlong(x);
  return x != x ? ~0ull : b ^ ((b >> 63) ? ~0ull : 0x8000000000000000ull);
}
__device__ __forceinline__ float from_ordered(uint32_t k)
{
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : ~0u));
}
__device__ __forceinline__ double from_ordered(uint64_t k)
{
  return __longlong_as_double(k ^ ((k >> 63) ? 0x8000000000000000ull : ~0ull));
}

// 32-bit values: one word holds both parts
struct Key32 {
  uint64_t w;
  static __device__ __forceinline__ Key32 none() { return {0}; }
  static __device__ __forceinline__ Key32 of(float x, uint32_t i)
  {
    return {static_cast<uint64_t>(ordered(x)) << 32 | static_cast<uint32_t>(~i)};
  }
  __device__ __forceinline__ bool above(const Key32& o) const { return w > o.w; }
  __device__ __forceinline__ float value() const { return from_ordered(static_cast<uint32_t>(w >> 32)); }
  __device__ __forceinline__ uint32_t index() const { return ~static_cast<uint32_t>(w); }
  static constexpr int kBits = 64;
  __device__ __forceinline__ Key32 with(int bit) const { return {w | 1ull << bit}; }
};
struct Key64 {
  uint64_t v;
  uint32_t i;
  static __device__ __forceinline__ Key64 none() { return {0, 0}; }
  static __device__ __forceinline__ Key64 of(double x, uint32_t i) { return {ordered(x), ~i}; }
  __device__ __forceinline__ bool above(const Key64& o) const { return v > o.v || (v == o.v && i > o.i); }
  __device__ __forceinline__ double value() const { return from_ordered(v); }
  __device__ __forceinline__ uint32_t index() const { return ~i; }
  static constexpr int kBits = 96;
  __device__ __forceinline__ Key64 with(int bit) const
  {
    return bit >= 32 ? Key64{v | 1ull << (bit - 32), i} : Key64{v, i | 1u << bit};
  }
};
template <class T>
struct KeyOf {
  using type = Key32;
};
template <>
struct KeyOf<double> {
  using type = Key64;
};

// Bitonic sort, descending: `n` keys (a power of two) of shared memory.
template <class K>
__device__ void sort_list(K* list, int n)
{
  for (int size = 2; size <= n; size <<= 1) {
    for (int d = size >> 1; d; d >>= 1) {
      for (int i = threadIdx.x; i < n / 2; i += kThreads) {
        const int a = 2 * i - (i & (d - 1)), b = a + d;
        const K x = list[a], y = list[b];
        if (((a & size) == 0) == y.above(x)) {
          list[a] = y;
          list[b] = x;
        }
      }
      __syncthreads();
    }
  }
}

template <class V>
__device__ __forceinline__ V log_of(V x);
template <>
__device__ __forceinline__ float log_of(float x) { return logf(x); }
template <>
__device__ __forceinline__ double log_of(double x) { return log(x); }

enum { kScores = 0, kProbabilities = 1, kScored = 2 };  // what a kernel is given, and whether it scores

// Best classes with a row's scores: values and logsumexp are not used.
struct ScoredTopArgs : TopArgs {
  Target target;
  Temperature temperature;
  Scores out;
  float* top;
};
template <int MODE>
using ArgsOf = std::conditional_t<MODE == kScored, ScoredTopArgs, TopArgs>;

// Exponents' factor log2(e) / T, as the gradient takes it.
template <class V, class A>
__device__ __forceinline__ V factor_of(const A& a)
{
  if constexpr (std::is_same_v<A, ScoredTopArgs>)
    return a.temperature.c;
  else
    return static_cast<V>(1.4426950408889634 * a.inv_temperature);
}

// Entry j of a scored row: m and log s, as in finish_score.
template <class K>
__device__ __forceinline__ void write_scored(const ScoredTopArgs& a, int64_t row, int j, const K& key, float m, const RowScore& score)
{
  const double x = (static_cast<double>(key.value()) - m) * a.temperature.inverse - score.log_s;
  a.top[row * a.k + j]   = !score.counts ? 0.f : static_cast<float>(x > 0 ? 0 : x);
  a.index[row * a.k + j] = score.counts ? static_cast<int32_t>(key.index()) : -1;
}
// A row that does not count, by `threads` threads.
__device__ __forceinline__ void write_uncounted_top(const ScoredTopArgs& a, int64_t row, int tid, int threads)
{
  for (int j = tid; j < a.k; j += threads) {
    a.top[row * a.k + j]   = 0.f;
    a.index[row * a.k + j] = -1;
  }
}
__device__ __forceinline__ void write_uncounted(const ScoredTopArgs& a, int64_t row, int tid, int threads)
{
  if (tid == 0) finish_score(a.out, row, Scored(), a.temperature.inverse, -2, 0.f);
  write_uncounted_top(a, row, tid, threads);
}
// Scores of a row: written by one thread, known to all that call.
template <class T>
__device__ __forceinline__ RowScore score_row(const ScoredTopArgs& a, int64_t row, const T* x, const Scored& r, int at, bool writes)
{
  if (writes) return finish_score(a.out, row, r, a.temperature.inverse, at, at >= 0 ? widen(x[at]) : 0.f);
  return {log_sum(r.s), at != -2 && !(r.s == 0.f)};
}

// Writes entry j of a row.
template <class T, class K>
__device__ __forceinline__ void write_top(const TopArgs& a, int64_t row, int j, const K& key)
{
  using V = typename ValueOf<T>::type;
  V v     = key.value();
  if (a.probabilities) v = log_of(v);
  static_cast<T*>(a.values)[row * a.k + j] = narrow<T>(v);
  a.index[row * a.k + j]                   = static_cast<int32_t>(key.index());
}

// Scores over T of this size and above are more than 31, the logarithm of the longest row, apart or equal: the
// log-sum-exp is the largest, to half a step (2^30: 64).
template <class V>
constexpr double kHuge = sizeof(V) == 4 ? 0x1p30 : 0x1p59;

// The sum over a row: of 2^(x c - r), c = log2(e) / T, x the score or the probability's logarithm.  r is m c of an m that
// no x exceeds by more than kSlack powers of two, or -2 kHuge, below which terms are 0: the difference keeps what m c is
// rounded by, which has to be an exponent of a number.  Probabilities add up to nearly 1, whose
// logarithm is a difference: at T = 1 (`plain`) the sum is their own and keeps what each addition drops.
template <class V, bool PROB>
struct Sum {
  V r = V(0), s = V(0), limit = lowest<V>(), dropped = V(0);
  bool first = true;
  __device__ __forceinline__ void reach(V most, V c, bool plain)  // most, limit: scores or probabilities themselves
  {
    if (plain || !(most > limit)) return;
    const V to = larger((PROB ? log_of(most) : most) * c, V(-2 * kHuge<V>));
    s          = first ? s : s * power(r - to);
    r          = to;
    first      = false;
    limit      = PROB ? most * smaller(power(V(kSlack * 1.4426950408889634) / c), V(1e30)) : most + V(kSlack) / c;
  }
  __device__ __forceinline__ void add(V x, V c, bool plain)
  {
    if (plain) {
      const V t = s + x, b = t - s;
      dropped += (s - (t - b)) + (x - b);
      s = t;
    } else {
      s += power(fma(PROB ? log_of(x) : x, c, -r));
    }
  }
};

// The same with what scores need.
// (of rows in registers, whose maximum is known)
struct ScoredSum : ScoredStream {
  float slack;
  __device__ __forceinline__ explicit ScoredSum(float c) : slack(kSlack / c) {}
  __device__ __forceinline__ void reach(float most, float c, bool) { ScoredStream::reach(most, c, slack); }
  __device__ __forceinline__ void add(float x, float c, bool) { Scored::add(x, base, c); }
};
template <class V, int MODE>
__device__ __forceinline__ auto new_sum(V c)
{
  if constexpr (MODE == kScored)
    return ScoredSum(c);
  else
    return Sum<V, MODE == kProbabilities>();
}
// ... and of a row that is read once.
template <class T, int MODE>
struct StreamOf {
  using type = Sum<typename ValueOf<T>::type, MODE == kProbabilities>;
};
template <class T>
struct StreamOf<T, kScored> {
  using type = PairedStream<T>;
};
template <class V, bool PROB>
__device__ __forceinline__ bool is_nan(const Sum<V, PROB>& sum) { return sum.s != sum.s; }
template <class T>
__device__ __forceinline__ bool is_nan(const PairedStream<T>& sum)
{
  float lo, hi;
  split_pair(sum.s, lo, hi);
  return lo != lo || hi != hi;
}
// The logarithm of s + dropped, which may be nearly 1: of its 32-bit part, and what that leaves.
__device__ __forceinline__ float log_of_sum(float s, double dropped)
{
  const double all = s + dropped;
  const float high = static_cast<float>(all);
  return high > 0.f && high < INFINITY ? logf(high) + static_cast<float>(all - high) / high : logf(high);
}
__device__ __forceinline__ double log_of_sum(double s, double dropped) { return log(s + dropped); }

__device__ __forceinline__ double log_of_terms(float s) { return log_sum(s); }
__device__ __forceinline__ double log_of_terms(double s) { return log(s); }

// log-sum-exp of a row from its sum; best: the row's largest key.
// m: the terms are relative to 2^m.
template <class V, class K>
__device__ __forceinline__ void write_lse(const TopArgs& a, int64_t row, V m, V s, double dropped, const K& best)
{
  if (!a.logsumexp) return;
  const bool plain = a.probabilities && a.inv_temperature == 1.0;
  V top = best.value(), r;  // (infinite, or NaN, of a score that is)
  if (plain) {
    r = top < V(INFINITY) ? log_of_sum(s, dropped) : top;
  } else {
    if (a.probabilities) top = log_of(top);
    r = top != top || top == lowest<V>() || top == -lowest<V>() ? top
        : fabs(top * a.inv_temperature) >= kHuge<V>             ? static_cast<V>(top * a.inv_temperature)
                                                                : static_cast<V>(m * 0.69314718055994530942 + log_of_terms(s));
  }
  static_cast<V*>(a.logsumexp)[row] = r;
}

// Places `got` keys of `list` in descending order: put(place, key).  By a block; at most kList.
template <class K, class F>
__device__ __forceinline__ void arrange(K* list, int got, int k, F put)
{
  const int tid = threadIdx.x;
  if (got <= kCount) {  // a key's place is the number of larger ones
    if (tid < got) {
      const K key = list[tid];
      int place   = 0;
#pragma unroll 4
      for (int j = 0; j < got; ++j) place += list[j].above(key);
      if (place < k) put(place, key);
    }
  } else {
    int size = 256;
    while (size < got) size <<= 1;
    for (int i = got + tid; i < size; i += kThreads) list[i] = K::none();
    __syncthreads();
    sort_list(list, size);
    if (tid < k) put(tid, list[tid]);
  }
}

// The first NaN among a thread's elements of a row, or ~0.
template <class T>
__device__ __forceinline__ uint32_t first_nan(const T* x, int64_t n, int tid, int threads)
{
  uint32_t first = ~0u;
  visit_row<1>(
    x, n, tid, threads,
    [&](int64_t i, T e) {
      if (widen(e) != widen(e)) first = min(first, static_cast<uint32_t>(i));
    },
    [&](int64_t i, const Piece<T>& p) {
#pragma unroll
      for (int e = 0; e < Piece<T>::N; ++e)
        if (widen(p.v[e]) != widen(p.v[e])) first = min(first, static_cast<uint32_t>(i + e));
    });
  return first;
}

// A segment of a row per block.  segs == 1: the row's answer; else its k best keys and its sum, which the first
// block of a cluster of segs blocks joins, or top_join does.
template <class T, int MODE>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 8 ? 3 : 5) top_segments(ArgsOf<MODE> a, int segs, int64_t seg_cols,
                                                                                 bool clustered,
                                                                                 typename KeyOf<T>::type* keys, double* sums)
{
  using V = typename ValueOf<T>::type;
  using K = typename KeyOf<T>::type;
  constexpr int N     = Piece<T>::N;
  constexpr bool PROB = MODE == kProbabilities;
  __shared__ K list[kList], best[kMostTop], shared_tau;
  __shared__ double best_sum[3];
  __shared__ float joined_m;
  __shared__ RowScore joined_score;
  __shared__ int16_t groups[kThreads];
  __shared__ int found, chosen;
  __shared__ double room[64];
  const int tid       = threadIdx.x;
  const int seg       = blockIdx.x % segs;
  const int64_t begin = seg * seg_cols;
  const int64_t n     = min(seg_cols, a.n_cols - begin);
  const int k         = static_cast<int>(min(static_cast<int64_t>(a.k), n));
  const V c           = factor_of<V>(a);
  const bool plain    = PROB && a.inv_temperature == 1.0;
  for (int64_t row = blockIdx.x / segs; row < a.n_rows; row += gridDim.x / segs) {
    const T* x       = static_cast<const T*>(a.scores) + row * a.row_stride + begin;
    const int lead   = lead_of(x, n);
    const int pieces = static_cast<int>((n - lead) / N);
    const T* body    = x + lead;
    int given        = -1;
    if constexpr (MODE == kScored) {
      given = target_of(a.target, row, a.n_cols);
      if (given == -2) {  // (for all blocks of a cluster)
        if (seg == 0) write_uncounted(a, row, tid, kThreads);
        continue;
      }
    }
    // the thread's best score, the first element of the piece that holds it, and the sum
    typename StreamOf<T, MODE>::type sum;
    const V slack = static_cast<V>(kSlack) / c;
    V top       = lowest<V>();
    uint32_t at = ~0u;  // none yet
    visit_row<kInFlight>(
      x, n, tid, kThreads,
      [&](int64_t i, T e) {
        const V v = widen(e);
        if (v > top || at == ~0u) at = static_cast<uint32_t>(i);
        top = larger(top, v);
        if constexpr (MODE == kScored) {
          sum.take(v, c, slack);
        } else {
          sum.reach(v, c, plain);
          sum.add(v, c, plain);
        }
      },
      [&](int64_t i, const Piece<T>& p) {
        if constexpr (MODE == kScored) {
          const V most = largest_of(p);
          if (most > top || at == ~0u) at = static_cast<uint32_t>(i);
          top = larger(top, most);
          sum.take(p, most, c, slack);
          return;
        }
        V v[N], most;
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = widen(p.v[e]);
        most = v[0];
#pragma unroll
        for (int e = 1; e < N; ++e) most = larger(most, v[e]);
        if (most > top || at == ~0u) at = static_cast<uint32_t>(i);
        top = larger(top, most);
        if constexpr (MODE != kScored) {
          sum.reach(most, c, plain);
#pragma unroll
          for (int e = 0; e < N; ++e) sum.add(v[e], c, plain);
        }
      });
    if (is_nan(sum)) {  // a NaN, or infinities: the first NaN of the group is its best
      const uint32_t first = first_nan(x, n, tid, kThreads);
      if (first != ~0u) {
        top = static_cast<V>(NAN);
        at  = first;
      }
    }
    // bounds of the best element's key
    const bool any = at != ~0u;
    const K below  = any ? K::of(top, static_cast<uint32_t>(begin) + at + N - 1) : K::none();
    const K above  = any ? K::of(top, static_cast<uint32_t>(begin) + at) : K::none();
    double dropped = 0;
    Running<V> all;
    all.m = V(0);
    Scored scored;
    if constexpr (MODE == kScored) {
      scored = sum.scored(c);
      join_scored<kThreads>(scored, c, reinterpret_cast<float*>(room));
      if (!sum.usable(scored.m, c)) scored = visit_any<T, kThreads, kInFlight>(x, n, tid, c, reinterpret_cast<float*>(room));
    } else if (plain) {
      // (in 64 bits: see Sum)
      dropped = sum_row<kThreads>(static_cast<double>(sum.s) + sum.dropped, room);
    } else {
      all.m = sum.first ? lowest<V>() : sum.r;
      all.s = sum.s;
      join_row<kThreads>(all, V(1), reinterpret_cast<V*>(room));
    }
    // tau: a bound that k groups reach, and at most kMore more unless its last bit is reached; the first warp
    // counts for all
    K tau = K::none();
    list[tid] = below;
    __syncthreads();
    if (tid < 32) {
      constexpr int G = kThreads / 32;
      K group[G];
#pragma unroll
      for (int g = 0; g < G; ++g) group[g] = list[tid + 32 * g];
      auto reached = [&](const K& by) {
        int some = 0;
#pragma unroll
        for (int g = 0; g < G; ++g) some += !by.above(group[g]);
        return static_cast<int>(__reduce_add_sync(~0u, some));
      };
      const int seen = reached(K::none().with(0));  // (a group without elements has no key)
      if (seen > k + kMore || (seen >= k && n > kList)) {
        for (int bit = K::kBits - 1; bit >= 0; --bit) {
          const K next  = tau.with(bit);
          const int got = reached(next);
          if (got < k) continue;
          tau = next;
          if (got <= k + kMore) break;
        }
      }
      if (tid == 0) shared_tau = tau;
    }
    if (tid == 0) found = chosen = 0;
    __syncthreads();
    tau                = shared_tau;
    const bool reaches = any && !tau.above(above);
    if (reaches) groups[atomicAdd(&chosen, 1)] = static_cast<int16_t>(tid);
    __syncthreads();
    const int reached_by = chosen;
    // A group's pieces, to the next power of two: those behind the last are left out below.
    const int per   = (pieces + kThreads - 1) / kThreads;
    const int shift = per <= 1 ? 0 : 32 - __clz(per - 1);
    auto collect    = [&](const K& bound) {
      auto take = [&](int64_t i) {
        const K key = K::of(widen(x[i]), static_cast<uint32_t>(begin + i));
        if (bound.above(key)) return;
        const int to = atomicAdd(&found, 1);
        if (to < kList) list[to] = key;
      };
      // (values below the bound's are left out at once; NaN is not below)
      const V least = bound.value();
#pragma unroll 4
      for (int i = tid; i < reached_by << shift; i += kThreads) {
        const int p = groups[i >> shift] + (i & ((1 << shift) - 1)) * kThreads;
        if (p >= pieces) continue;
        const Piece<T> v = load_piece(body + static_cast<int64_t>(p) * N);
        uint32_t some = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) some |= !(widen(v.v[e]) < least) ? 1u << e : 0u;
        for (; some; some &= some - 1) take(lead + static_cast<int64_t>(p) * N + (__ffs(some) - 1));
      }
      // the elements before the first and behind the last boundary
      if (tid < lead) take(tid);
      const int64_t end = lead + static_cast<int64_t>(pieces) * N + tid;
      if (end < n) take(end);
      __syncthreads();
      const int got = found;
      __syncthreads();
      if (tid == 0) found = 0;
      __syncthreads();
      return got;
    };
    // Where the list is too short, the largest bound that k keys reach is found bit by bit: keys differ, so
    // exactly k do.
    int got = 0;
    K bound = K::none(), next = tau;
    for (int bit = -1;;) {
      got = collect(next);
      if (bit < 0) {
        if (got <= kList) break;
        bit = K::kBits;
      } else if (got >= k) {
        bound = next;
      }
      next = --bit < 0 ? bound : bound.with(bit);
    }
    const int64_t part = row * segs + seg;
    if (segs == 1) {
      arrange(list, got, k, [&](int place, const K& key) {
        if constexpr (MODE == kScored) {
          write_scored(a, row, place, key, scored.m, score_row(a, row, x, scored, given, place == 0));
        } else {
          write_top<T>(a, row, place, key);
          if (place == 0) write_lse(a, row, all.m, all.s, dropped, key);
        }
      });
      __syncthreads();
      continue;
    }
    K* to = clustered ? best : keys + part * a.k;
    arrange(list, got, k, [&](int place, const K& key) { to[place] = key; });
    for (int j = k + tid; j < a.k; j += kThreads) to[j] = K::none();
    if (tid == 0) {
      double* sum_to = clustered ? best_sum : sums + 3 * part;
      if constexpr (MODE == kScored) {
        sum_to[0] = scored.s;
        sum_to[1] = scored.m;
        sum_to[2] = scored.u;
      } else {
        sum_to[0] = plain ? dropped : static_cast<double>(all.s);
        sum_to[1] = all.m;
      }
    }
    if (clustered) {
      // With r = k / segs rounded up, at least k keys reach the least of the lists' r-th keys.
      namespace cg = cooperative_groups;
      cg::cluster_group cluster = cg::this_cluster();
      cluster.sync();
      if (seg == 0) {
        const int r_th = (a.k + segs - 1) / segs - 1;
        K least        = K::of(static_cast<V>(NAN), 0u);  // nothing is above
        for (int i = 0; i < segs; ++i) {
          const K key = *cluster.map_shared_rank(best + r_th, i);
          if (least.above(key)) least = key;
        }
        for (int i = tid; i < segs * a.k; i += kThreads) {
          const K key = *cluster.map_shared_rank(best + i % a.k, i / a.k);
          if (!least.above(key)) list[atomicAdd(&found, 1)] = key;
        }
        if constexpr (MODE == kScored) {
          if (tid < 32) {
            Scored r;
            if (tid < segs) {
              const double* from = cluster.map_shared_rank(best_sum, tid);
              r.s = static_cast<float>(from[0]);
              r.m = static_cast<float>(from[1]);
              r.u = static_cast<float>(from[2]);
            }
            r.join_lanes(c);
            if (tid == 0) {
              joined_m     = r.m;
              joined_score = score_row(a, row, x, r, given, true);  // (the first block's part begins with the row)
            }
          }
        }
        __syncthreads();
        arrange(list, found, a.k, [&](int place, const K& key) {
          if constexpr (MODE == kScored) {
            write_scored(a, row, place, key, joined_m, joined_score);
            return;
          } else {
            write_top<T>(a, row, place, key);
            if (place > 0) return;
            Running<double> r;
            for (int i = 0; i < segs; ++i) {
              const double* from = cluster.map_shared_rank(best_sum, i);
              if (plain)
                r.s += from[0];
              else
                r.join(from[1], from[0], 1.0);
            }
            write_lse(a, row, static_cast<V>(r.m), static_cast<V>(plain ? 0.0 : r.s), plain ? r.s : 0.0, key);
          }
        });
      }
      cluster.sync();  // the others' lists have been read
    }
    __syncthreads();
  }
}

// Joins the segments' sorted lists of a row.  With r = k / segs rounded up, at least k keys reach the least of the
// lists' r-th keys: these alone are sorted, where they fit; else as many as fit with the best so far.
template <class T, int MODE>
__global__ void __launch_bounds__(kThreads) top_join(ArgsOf<MODE> a, int segs, const typename KeyOf<T>::type* keys,
                                                     const double* sums)
{
  using V = typename ValueOf<T>::type;
  using K = typename KeyOf<T>::type;
  __shared__ K list[kList];
  __shared__ double room[64];
  __shared__ int found;
  const bool plain = a.probabilities && a.inv_temperature == 1.0;
  for (int64_t row = blockIdx.x; row < a.n_rows; row += gridDim.x) {
    int given = -1;
    if constexpr (MODE == kScored) {
      given = target_of(a.target, row, a.n_cols);
      if (given == -2) continue;  // (written already)
    }
    const K* from = keys + row * segs * a.k;
    const int all = segs * a.k, r_th = (a.k + segs - 1) / segs - 1;
    if (threadIdx.x == 0) found = 0;
    __syncthreads();
    K bound = K::of(static_cast<V>(NAN), 0u);  // nothing is above
    for (int i = 0; i < segs; ++i) {
      const K key = from[i * a.k + r_th];
      if (bound.above(key)) bound = key;
    }
    for (int i = threadIdx.x; i < all; i += kThreads) {
      const K key = from[i];
      if (bound.above(key)) continue;
      const int to = atomicAdd(&found, 1);
      if (to < kList) list[to] = key;
    }
    __syncthreads();
    const int got = found;
    if (got <= kList) {
      int size = 1;
      while (size < got) size <<= 1;
      for (int i = got + threadIdx.x; i < size; i += kThreads) list[i] = K::none();
      __syncthreads();
      sort_list(list, size);
    } else {
      int have = 0;
      for (int i = 0; i < all;) {
        const int more = min(all - i, kList - have);
        int size       = 1;
        while (size < have + more) size <<= 1;
        for (int j = threadIdx.x; j < size - have; j += kThreads) list[have + j] = j < more ? from[i + j] : K::none();
        __syncthreads();
        sort_list(list, size);
        i += more;
        have = min(a.k, have + more);
      }
    }
    if constexpr (MODE == kScored) {
      const float c = factor_of<V>(a);
      Scored r;
      for (int i = threadIdx.x; i < segs; i += kThreads) {
        const double* part = sums + 3 * (row * segs + i);
        r.join(static_cast<float>(part[1]), static_cast<float>(part[0]), static_cast<float>(part[2]), c);
      }
      join_scored<kThreads>(r, c, reinterpret_cast<float*>(room));
      const T* x           = static_cast<const T*>(a.scores) + row * a.row_stride;
      const RowScore score = score_row(a, row, x, r, given, threadIdx.x == 0);
      for (int j = threadIdx.x; j < a.k; j += kThreads) write_scored(a, row, j, list[j], r.m, score);
      __syncthreads();
    } else {
      for (int j = threadIdx.x; j < a.k; j += kThreads) write_top<T>(a, row, j, list[j]);
      Running<double> r;
      for (int i = threadIdx.x; i < segs; i += kThreads) {
        const double s = sums[3 * (row * segs + i)], m = sums[3 * (row * segs + i) + 1];
        if (plain)
          r.s += s;
        else
          r.join(m, s, 1.0);
      }
      if (plain)
        r.s = sum_row<kThreads>(r.s, room);
      else
        join_row<kThreads>(r, 1.0, room);
      if (threadIdx.x == 0) write_lse(a, row, static_cast<V>(r.m), static_cast<V>(plain ? 0.0 : r.s), plain ? r.s : 0.0, list[0]);
      __syncthreads();
    }
  }
}

// Ordered integers of one thread's best scores.
template <class V>
struct Ordered {
  using type = uint32_t;
};
template <>
struct Ordered<double> {
  using type = uint64_t;
};

__device__ __forceinline__ uint32_t max_of(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint64_t max_of(uint64_t a, uint64_t b) { return a > b ? a : b; }

// Blocks of an SM whose lanes hold `bytes` of elements each.
__host__ __device__ constexpr int warps_fit(size_t bytes) { return bytes <= 128 ? 4 : 2; }

// A row per warp, in registers.  Short rows: every 32nd element is a lane's, S of them.  Longer ones: U pieces of
// 16 bytes and at most one element from before the first or behind the last boundary per lane, and S is 0.
template <class T, int U, int S, int MODE>
__global__ void __launch_bounds__(kThreads, warps_fit(U * 16 / sizeof(T) * sizeof(typename ValueOf<T>::type))) top_warps(ArgsOf<MODE> a)
{
  using V = typename ValueOf<T>::type;
  using K = typename KeyOf<T>::type;
  using O = typename Ordered<V>::type;
  constexpr int N = Piece<T>::N, E = S ? S : U * N + 1, ROWS = kThreads / 32, kBits = sizeof(O) * 8;
  constexpr bool PROB = MODE == kProbabilities;
  __shared__ K lists[ROWS][kWarpList];
  const int lane = threadIdx.x % 32, n = static_cast<int>(a.n_cols), k = a.k;
  K* list          = lists[threadIdx.x / 32];
  const V c        = factor_of<V>(a);
  const bool plain = PROB && a.inv_temperature == 1.0;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x / 32; row < a.n_rows;
       row += static_cast<int64_t>(gridDim.x) * ROWS) {
    const T* x       = static_cast<const T*>(a.scores) + row * a.row_stride;
    int given        = -1;
    if constexpr (MODE == kScored) {
      given = target_of(a.target, row, a.n_cols);
      if (given == -2) {
        write_uncounted(a, row, lane, 32);
        continue;
      }
    }
    const int lead   = S ? 0 : lead_of(x, n), pieces = S ? 0 : (n - lead) / N;
    // the odd element: the first lanes' before, the last lanes' behind the pieces
    const int behind = lead + pieces * N + 31 - lane;
    const int odd    = lane < lead ? lane : behind < n ? behind : -1;
    auto place_of    = [&](int e) { return S ? lane + 32 * e : e == E - 1 ? odd : lead + (lane + 32 * (e / N)) * N + e % N; };
    auto is_there    = [&](int e) { return S ? lane + 32 * e < n : e == E - 1 ? odd >= 0 : lane + 32 * (e / N) < pieces; };
    V v[E], top = lowest<V>();
    if constexpr (S > 0) {
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = lane + 32 * e < n ? widen(x[lane + 32 * e]) : lowest<V>();
    } else {
      const T* body = x + lead;
      Piece<T> w[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (lane + 32 * u < pieces) w[u] = load_piece(body + (lane + 32 * u) * N);
      v[E - 1] = odd >= 0 ? widen(x[odd]) : lowest<V>();
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < N; ++e) v[u * N + e] = lane + 32 * u < pieces ? widen(w[u].v[e]) : lowest<V>();
    }
#pragma unroll
    for (int e = 0; e < E; ++e) top = larger(top, v[e]);
    const V most = top;
#pragma unroll
    for (int d = 16; d; d >>= 1) top = larger(top, __shfl_xor_sync(~0u, top, d));
    // the sum (what is not there is -inf and adds nothing to a sum of powers)
    auto sum = new_sum<V, MODE>(c);
    sum.reach(top, c, plain);
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (!PROB || is_there(e)) sum.add(v[e], c, plain);
    V s            = sum.s;
    double dropped = 0;
    if constexpr (MODE == kScored) {
      s = sum.s = sum_lanes(sum.s);
      sum.u     = sum_lanes(sum.u);
    } else if (plain) {
      dropped = sum_lanes(static_cast<double>(sum.s) + sum.dropped);
      s       = V(0);
    } else {
      s = sum_lanes(s);
    }
    int got = 0;
    const bool nan = plain ? dropped != dropped : s != s;
    // Few of many: a bound that at least k lanes' best reach, a ballot per bit.
    bool done = false;
    if (k <= kWarpTop && (S ? E > 2 : pieces >= 32) && !nan) {
      const O best = ordered(most);
      O tau        = 0;
      for (int bit = kBits - 1; bit >= 0; --bit) {
        const O next   = tau | O(1) << bit;
        const int some = __popc(__ballot_sync(~0u, best >= next));
        if (some < k) continue;
        tau = next;
        if (some <= k + 2) break;
      }
      const V least = tau > ordered(lowest<V>()) ? from_ordered(tau) : lowest<V>();
      // the lane's hits, then its part of the list
      constexpr int H = E < 64 ? E : 64;  // (a 65th is the odd one)
      uint64_t hits   = 0;
      bool last_hit   = false;
      if (least > lowest<V>()) {
#pragma unroll
        for (int e = 0; e < H; ++e) hits |= v[e] >= least ? 1ull << e : 0ull;
        if (E > H) last_hit = v[E - 1] >= least;
      } else {
#pragma unroll
        for (int e = 0; e < H; ++e) hits |= is_there(e) ? 1ull << e : 0ull;
        if (E > H) last_hit = is_there(E - 1);
      }
      const int mine = __popcll(hits) + last_hit;
      int to         = mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(~0u, to, d);
        if (lane >= d) to += o;
      }
      got  = __shfl_sync(~0u, to, 31);
      done = got <= kWarpList;
      if (done) {
        to -= mine;
        for (; hits; hits &= hits - 1) {
          const int at = place_of(__ffsll(hits) - 1);
          list[to++]   = K::of(widen(x[at]), static_cast<uint32_t>(at));
        }
        if (last_hit) list[to] = K::of(v[E - 1], static_cast<uint32_t>(odd));
      }
    }
    if (!done) {
      // All elements as ordered integers (0: not there); tau: a value that k of them reach and, unless equal ones are
      // among them, hardly more.
      O o[E], tau = 1;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = is_there(e) ? ordered(v[e]) : O(0);
      auto reached = [&](O by) {
        int some = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) some += o[e] >= by;
        return static_cast<int>(__reduce_add_sync(~0u, some));
      };
      int some = n;
      if (n > k + kMore) {
        O t = 0;
        for (int bit = kBits - 1; bit >= 0; --bit) {
          const O next = t | O(1) << bit;
          const int up = reached(next);
          if (up < k) continue;
          t    = next;
          some = up;
          if (some <= k + kMore) break;
        }
        tau = max_of(t, O(1));
      }
      // equal ones at the bound beyond what the list holds: the first of them only
      int last = n;
      if (some > kWarpList) {
        const int over = tau == ~O(0) ? 0 : reached(tau + 1);
        int low = 0, high = n - 1;  // the least place up to which k - over of them lie
        while (low < high) {
          const int mid = (low + high) / 2;
          int up        = 0;
#pragma unroll
          for (int e = 0; e < E; ++e) up += o[e] == tau && place_of(e) <= mid;
          if (static_cast<int>(__reduce_add_sync(~0u, up)) >= k - over)
            high = mid;
          else
            low = mid + 1;
        }
        last = low;
      }
      got = 0;
      // puts an element of each lane that has one into the list
      auto push = [&](bool is, int e) {
        const unsigned all = __ballot_sync(~0u, is);
        if (all == 0) return;
        if (is) list[got + __popc(all & ((1u << lane) - 1))] = K::of(from_ordered(o[e]), static_cast<uint32_t>(place_of(e)));
        got += __popc(all);
      };
#pragma unroll
      for (int e = 0; e < E; ++e) push(o[e] > tau || (o[e] == tau && place_of(e) <= last), e);
    }
    __syncwarp();
    for (int i = lane; i < got; i += 32) {
      const K key = list[i];
      int place   = 0;
#pragma unroll 4
      for (int j = 0; j < got; ++j) place += list[j].above(key);
      if (place >= k) continue;
      if constexpr (MODE == kScored) {
        write_scored(a, row, place, key, sum.m, score_row(a, row, x, sum, given, place == 0));
      } else {
        write_top<T>(a, row, place, key);
        if (place == 0) write_lse(a, row, sum.r, s, dropped, key);
      }
    }
    __syncwarp();
  }
}

// A row per warp that its registers do not hold, of more than 32 x 32 elements; k <= kWarpTop.  Its lanes' best give the
// bound, as above, and what reaches it is read again; where that is more than the list holds the k-th key is found
// bit by bit as in top_segments.  (A bound by values alone took 5.7 ms where all but five of 4096 scores of 8192 rows
// were -inf.)
template <class T, bool PROB>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 8 ? 3 : 4) top_long(TopArgs a)
{
  using V = typename ValueOf<T>::type;
  using K = typename KeyOf<T>::type;
  constexpr int N = Piece<T>::N, ROWS = kThreads / 32;
  __shared__ K lists[ROWS][kWarpList];
  __shared__ int counts[ROWS];
  const int lane = threadIdx.x % 32, k = a.k;
  K* list          = lists[threadIdx.x / 32];
  int* found       = &counts[threadIdx.x / 32];
  const V c        = factor_of<V>(a);
  const bool plain = PROB && a.inv_temperature == 1.0;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x / 32; row < a.n_rows;
       row += static_cast<int64_t>(gridDim.x) * ROWS) {
    const T* x = static_cast<const T*>(a.scores) + row * a.row_stride;
    // the lane's best score, the first element of the piece that holds it, and the sum
    V best      = lowest<V>();
    uint32_t at = ~0u;
    Sum<V, PROB> sum;
    visit_row<2 * kInFlight>(
      x, a.n_cols, lane, 32,
      [&](int64_t i, T e) {
        const V v = widen(e);
        if (v > best || at == ~0u) at = static_cast<uint32_t>(i);
        best      = larger(best, v);
        sum.reach(v, c, plain);
        sum.add(v, c, plain);
      },
      [&](int64_t i, const Piece<T>& p) {
        V v[N], most;
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = widen(p.v[e]);
        most = v[0];
#pragma unroll
        for (int e = 1; e < N; ++e) most = larger(most, v[e]);
        if (most > best || at == ~0u) at = static_cast<uint32_t>(i);
        best = larger(best, most);
        sum.reach(most, c, plain);
#pragma unroll
        for (int e = 0; e < N; ++e) sum.add(v[e], c, plain);
      });
    double dropped = 0;
    Running<V> all;
    all.m = V(0);
    if (plain) {
      dropped = sum_lanes(static_cast<double>(sum.s) + sum.dropped);
    } else {
      all.m = sum.first ? lowest<V>() : sum.r;
      all.s = sum.s;
      all.join_lanes(V(1));
    }
    if (sum.s != sum.s) {  // a NaN, or infinities
      const uint32_t first = first_nan(x, a.n_cols, lane, 32);
      if (first != ~0u) {
        best = static_cast<V>(NAN);
        at   = first;
      }
    }
    // Puts what is above or equal into the list, as far as that goes; how many there are.
    auto collect = [&](const K& bound, V least) {
      __syncwarp();
      if (lane == 0) *found = 0;
      __syncwarp();
      auto take = [&](int64_t i, T e) {
        const K key = K::of(widen(e), static_cast<uint32_t>(i));
        if (bound.above(key)) return;
        const int to = atomicAdd(found, 1);
        if (to < kWarpList) list[to] = key;
      };
      visit_row<kInFlight>(x, a.n_cols, lane, 32, take, [&](int64_t i, const Piece<T>& p) {
        uint32_t some = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) some |= !(widen(p.v[e]) < least) ? 1u << e : 0u;
        if (some == 0) return;
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (some >> e & 1) take(i + e, p.v[e]);
      });
      __syncwarp();
      return *static_cast<volatile int*>(found);
    };
    // tau: a key that k lanes' best reach; the last element of its piece stands for a lane's best
    const K mine = K::of(best, at + N - 1);
    K tau        = K::none();
    for (int bit = K::kBits - 1; bit >= 0; --bit) {
      const K next   = tau.with(bit);
      const int some = __popc(__ballot_sync(~0u, !next.above(mine)));
      if (some < k) continue;
      tau = next;
      if (some <= k + 2) break;
    }
    int got = collect(tau, tau.value());
    if (got > kWarpList) {
      K bound = K::none();
      for (int bit = K::kBits - 1; bit >= 0 && got > kWarpList; --bit) {
        const K next   = bound.with(bit);
        const int some = collect(next, next.value());
        if (some < k) continue;
        bound = next;
        got   = some;
      }
    }
    for (int i = lane; i < got; i += 32) {
      const K key = list[i];
      int place   = 0;
#pragma unroll 4
      for (int j = 0; j < got; ++j) place += list[j].above(key);
      if (place >= k) continue;
      write_top<T>(a, row, place, key);
      if (place == 0) write_lse(a, row, all.m, all.s, dropped, key);
    }
    __syncwarp();
  }
}

// The best classes of a scored row from the largest of kBestGroups groups of its pieces, kGroups of a lane: group g of lane l is
// l + 32 g.  By a warp; k <= kWarpTop.  A value tau that k of them reach is found by votes, and only the groups that reach it
// are read again.  Where that is more than the list holds, what is above tau is taken, and of its equals (a mask, for
// instance) the first of the row.
constexpr int kBestGroups = 256, kGroups = kBestGroups / 32;
struct GroupRoom {
  Key32 list[kWarpList];
  uint8_t chosen[kBestGroups];
  int count;
};
template <class T, class F>
__device__ __forceinline__ void best_of_groups(const T* x, int n, int k, const float (&best)[kGroups], bool nan, GroupRoom& room, F put)
{
  constexpr int N = Piece<T>::N, R = kBestGroups;
  using K = Key32;
  const int lane       = threadIdx.x % 32;
  const unsigned below = (1u << lane) - 1;
  const int lead = lead_of(x, n), pieces = (n - lead) / N, behind = lead + pieces * N + lane;
  // the elements before the first and behind the last boundary are looked at whatever they are
  const float before = lane < lead ? widen(x[lane]) : 0.f, after = behind < n ? widen(x[behind]) : 0.f;
  uint32_t o[kGroups], tau = 0;
#pragma unroll
  for (int g = 0; g < kGroups; ++g) o[g] = ordered(best[g]);
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t next = tau | 1u << bit;
    int some            = 0;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) some += o[g] >= next;
    some = __reduce_add_sync(~0u, some);
    if (some < k) continue;
    tau = next;
    if (some <= k + kMore) break;
  }
  int reached_by = 0;
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    const unsigned all = __ballot_sync(~0u, o[g] >= tau);
    if (o[g] >= tau) room.chosen[reached_by + __popc(all & below)] = static_cast<uint8_t>(g * 32 + lane);
    reached_by += __popc(all);
  }
  __syncwarp();
  // Puts those of the reached groups, or of the whole row, whose keys are `bound` or above into the list; how many there are, or
  // that there are more than it holds.
  auto collect = [&](const K& bound, bool whole) {
    volatile int* count = &room.count;
    __syncwarp();
    if (lane == 0) *count = 0;
    __syncwarp();
    auto take = [&](int i, float v) {
      const K key = K::of(v, static_cast<uint32_t>(i));
      if (bound.above(key)) return;
      const int to = atomicAdd(&room.count, 1);
      if (to < kWarpList) room.list[to] = key;
    };
    const float least = bound.value();  // (NaN is not below)
    const int rounds = (pieces + R - 1) / R, all = whole ? pieces : reached_by * rounds;
    for (int i = lane; i - lane < all; i += 32) {
      if (__any_sync(~0u, *count > kWarpList)) break;
      const int p = i >= all ? pieces : whole ? i : room.chosen[i / rounds] + i % rounds * R;
      if (p >= pieces) continue;
      float v[N];
      numbers_of(piece_of<T>(__ldg(reinterpret_cast<const uint4*>(x + lead + static_cast<int64_t>(p) * N))), v);
      uint32_t some = 0;
#pragma unroll
      for (int e = 0; e < N; ++e) some |= !(v[e] < least) ? 1u << e : 0u;
      for (; some; some &= some - 1) {
        const int e = lead + p * N + __ffs(some) - 1;
        take(e, widen(x[e]));
      }
    }
    if (lane < lead) take(lane, before);
    if (behind < n) take(behind, after);
    __syncwarp();
    return *count;
  };
  int got = nan ? kWarpList + 1 : collect(K{static_cast<uint64_t>(tau) << 32}, false);
  if (got > kWarpList && !nan) {
    got = tau == ~0u ? 0 : collect(K{static_cast<uint64_t>(tau + 1) << 32}, false);
    // equals of tau, in the order of their classes
    for (int first = 0; first < n && got < k; first += 32) {
      const int i        = first + lane;
      const bool is      = i < n && ordered(widen(x[i])) == tau;
      const unsigned all = __ballot_sync(~0u, is);
      if (is) room.list[got + __popc(all & below)] = K::of(widen(x[i]), static_cast<uint32_t>(i));
      got += __popc(all);
    }
    __syncwarp();
  }
  if (got > kWarpList) {  // NaN, or many above tau in few groups: the k-th key bit by bit
    K bound = K::none();
    for (int bit = K::kBits - 1; bit >= 0 && got > kWarpList; --bit) {
      const K next   = bound.with(bit);
      const int some = collect(next, true);
      if (some < k) continue;
      bound = next;
      got   = some;
    }
  }
  for (int i = lane; i < got; i += 32) {
    const K key = room.list[i];
    int place   = 0;
#pragma unroll 4
    for (int j = 0; j < got; ++j) place += room.list[j].above(key);
    if (place < k) put(place, key);
  }
  __syncwarp();
}

// A scored row per warp, of more than kWarpCols elements.
constexpr int kGroupThreads = 128;  // (small blocks: few rows are spread evenly over the SMs)
constexpr int kGroupBlocks  = 8;    // of an SM, all there at once
template <class T>
__global__ void __launch_bounds__(kGroupThreads, kGroupBlocks) top_groups(ScoredTopArgs a)
{
  constexpr int N = Piece<T>::N, ROWS = kGroupThreads / 32, U = kInFlight, R = kBestGroups;
  __shared__ GroupRoom rooms[ROWS];
  const int lane = threadIdx.x % 32, n = static_cast<int>(a.n_cols);
  const float c  = a.temperature.c, slack = kSlack / c;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x / 32; row < a.n_rows;
       row += static_cast<int64_t>(gridDim.x) * ROWS) {
    const T* x      = static_cast<const T*>(a.scores) + row * a.row_stride;
    const int given = target_of(a.target, row, a.n_cols);
    if (given == -2) {
      write_uncounted(a, row, lane, 32);
      continue;
    }
    const int lead = lead_of(x, n), pieces = (n - lead) / N, behind = lead + pieces * N + lane;
    const T* body  = x + lead;
    PairedStream<T> sum;
    float best[kGroups];
#pragma unroll
    for (int g = 0; g < kGroups; ++g) best[g] = lowest<float>();
    for (int first = lane; first - lane < pieces; first += R) {
      const bool full = first - lane + R <= pieces;
#pragma unroll
      for (int h = 0; h < kGroups; h += U) {
        Piece<T> r[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (full || first + (h + u) * 32 < pieces)
            r[u] = piece_of<T>(__ldg(reinterpret_cast<const uint4*>(body + static_cast<int64_t>(first + (h + u) * 32) * N)));
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (!full && first + (h + u) * 32 >= pieces) continue;
          const float most = largest_of(r[u]);
          best[h + u]      = fmaxf(best[h + u], most);
          sum.take(r[u], most, c, slack);
        }
      }
    }
    sum.take(lane < lead ? widen(x[lane]) : lowest<float>(), behind < n ? widen(x[behind]) : lowest<float>(), c, slack);
    const bool nan = __any_sync(~0u, is_nan(sum));  // (or an infinite one)
    Scored scored  = sum.scored(c);
    scored.join_lanes(c);
    if (!sum.usable(scored.m, c)) scored = visit_any<T, 32, kInFlight>(x, a.n_cols, lane, c, nullptr);
    if (scored.s == 0.f) {
      write_uncounted(a, row, lane, 32);
      continue;
    }
    best_of_groups(x, n, a.k, best, nan, rooms[threadIdx.x / 32], [&](int place, const Key32& key) {
      write_scored(a, row, place, key, scored.m, score_row(a, row, x, scored, given, place == 0));
    });
  }
}

// A row per thread: n_cols x sizeof(T) <= kTileBytes, k <= TOP.
template <class T, int TOP, int MODE>
__global__ void __launch_bounds__(kTileRows) top_tiles(ArgsOf<MODE> a)
{
  constexpr bool PROB = MODE == kProbabilities;
  using V = typename ValueOf<T>::type;
  using K = typename KeyOf<T>::type;
  using O = typename Ordered<V>::type;
  extern __shared__ __align__(16) char smem[];
  T* tile       = reinterpret_cast<T*>(smem);
  const int c_n = static_cast<int>(a.n_cols);
  const TileShape<T> shape(c_n);
  const V c        = factor_of<V>(a);
  const bool plain = PROB && a.inv_temperature == 1.0;
  const bool whole = without_gaps<T>(a.scores, a.row_stride, c_n);
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * kTileRows; first < a.n_rows;
       first += static_cast<int64_t>(gridDim.x) * kTileRows) {
    const int rows = static_cast<int>(min(static_cast<int64_t>(kTileRows), a.n_rows - first));
    __syncthreads();  // the last tile has been used
    load_tile(tile, shape, static_cast<const T*>(a.scores) + first * a.row_stride, a.row_stride, rows, whole);
    __syncthreads();
    if (threadIdx.x >= rows) continue;
    const T* x = tile + threadIdx.x * shape.pitch;
    // Sorted insertion without branches: of the entries that x exceeds the first becomes x, the others move down.
    V top[TOP], odd = V(0);
    int at[TOP];
#pragma unroll
    for (int j = 0; j < TOP; ++j) {
      top[j] = lowest<V>();
      at[j]  = j < c_n ? j : 0;  // (a row of -inf)
    }
    for (int i = 0; i < c_n; ++i) {
      const V v = widen(x[i]);
      odd       = fma(v, V(0), odd);  // NaN where one of the scores is infinite or no number
      bool up[TOP];
#pragma unroll
      for (int j = 0; j < TOP; ++j) up[j] = v > top[j];
#pragma unroll
      for (int j = TOP - 1; j > 0; --j) {
        top[j] = larger(top[j], smaller(top[j - 1], v));
        at[j]  = up[j - 1] ? at[j - 1] : up[j] ? i : at[j];
      }
      top[0] = larger(top[0], v);
      at[0]  = up[0] ? i : at[0];
    }
    if (odd != V(0)) {  // by ordered integers
      O key[TOP];
#pragma unroll
      for (int j = 0; j < TOP; ++j) {
        key[j] = 0;
        at[j]  = 0;
      }
      for (int i = 0; i < c_n; ++i) {
        O o     = ordered(widen(x[i]));
        int p   = i;
        bool up = false;  // all entries behind the new one move down (equal ones: the earlier class stays)
#pragma unroll
        for (int j = 0; j < TOP; ++j) {
          up |= o > key[j];
          const O ko   = key[j];
          const int ka = at[j];
          key[j]       = up ? o : ko;
          at[j]        = up ? p : ka;
          o            = up ? ko : o;
          p            = up ? ka : p;
        }
      }
#pragma unroll
      for (int j = 0; j < TOP; ++j) top[j] = from_ordered(key[j]);
    }
    auto sum = new_sum<V, MODE>(c);
    if (plain) {
      for (int i = 0; i < c_n; ++i) sum.add(widen(x[i]), c, true);
    } else {
      sum.reach(top[0], c, false);
      for (int i = 0; i < c_n; ++i) sum.add(widen(x[i]), c, false);
    }
    const int64_t row = first + threadIdx.x;
    if constexpr (MODE == kScored) {
      const int given      = target_of(a.target, row, a.n_cols);
      const RowScore score = score_row(a, row, x, sum, given, true);
#pragma unroll
      for (int j = 0; j < TOP; ++j)
        if (j < a.k) write_scored(a, row, j, K::of(top[j], static_cast<uint32_t>(at[j])), sum.m, score);
    } else {
      T* values         = static_cast<T*>(a.values) + row * a.k;
      int32_t* index    = a.index + row * a.k;
#pragma unroll
      for (int j = 0; j < TOP; ++j) {
        if (j >= a.k) break;
        values[j] = narrow<T>(PROB ? log_of(top[j]) : top[j]);
        index[j]  = at[j];
      }
      write_lse(a, row, sum.r, sum.s, static_cast<double>(sum.dropped), K::of(top[0], 0u));
    }
  }
}

// Parts of a row: enough blocks to fill the machine, none below 2048 elements.
int segments(int64_t n_rows, int64_t n_cols, int n_sms)
{
  if (n_rows == 0) return 1;
  const int64_t fill = (4 * n_sms + n_rows - 1) / n_rows;
  const int64_t most = (n_cols + 2047) / 2048;
  const int64_t segs = fill < most ? fill : most;
  return static_cast<int>(n_rows >= 2 * n_sms || segs < 1 ? 1 : segs);
}
int64_t part_cols(int64_t n_cols, int segs)
{
  return segs == 1 ? n_cols : ((n_cols + segs - 1) / segs + 63) / 64 * 64;
}

// `a`'s kernel of the three modes.
template <class A, class K>
auto kernel_of(const A& a, K scores, K probabilities)
{
  return a.probabilities ? probabilities : scores;
}

template <class T, int TOP, class A>
cudaError_t run_tiles(const A& a, int n_sms, cudaStream_t s)
{
  const size_t bytes   = TileShape<T>(static_cast<int>(a.n_cols)).bytes();
  const int64_t blocks = (a.n_rows + kTileRows - 1) / kTileRows, most = 16ll * n_sms;
  const auto kernel    = [&] {
    if constexpr (std::is_same_v<A, ScoredTopArgs>)
      return top_tiles<T, TOP, kScored>;
    else
      return kernel_of(a, top_tiles<T, TOP, kScores>, top_tiles<T, TOP, kProbabilities>);
  }();
  if (bytes > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
    if (e != cudaSuccess) return e;
  }
  kernel<<<static_cast<unsigned>(blocks < most ? blocks : most), kTileRows, bytes, s>>>(a);
  count_launches(1);
  return cudaGetLastError();
}

template <class T, int U, int S, class A>
cudaError_t run_warps(const A& a, int n_sms, cudaStream_t s)
{
  const int64_t need = (a.n_rows + kThreads / 32 - 1) / (kThreads / 32), most = 16ll * n_sms;
  const auto kernel  = [&] {
    if constexpr (std::is_same_v<A, ScoredTopArgs>)
      return top_warps<T, U, S, kScored>;
    else
      return kernel_of(a, top_warps<T, U, S, kScores>, top_warps<T, U, S, kProbabilities>);
  }();
  kernel<<<static_cast<unsigned>(need < most ? need : most), kThreads, 0, s>>>(a);
  count_launches(1);
  return cudaGetLastError();
}

// Scored rows by a warp each.
bool by_groups(int64_t n_rows, int64_t n_cols, int k, int element, int n_sms)
{
  const int64_t per = n_rows / n_sms, most = std::min(kGroupBytes * per / kLongLeast, kGroupMost);
  return n_cols > kWarpCols && k <= kWarpTop && per >= kLongLeast && n_cols * element <= most;
}

template <class T, class A>
cudaError_t run_top(const A& a, void* workspace, int n_sms, cudaStream_t s)
{
  constexpr bool kIsScored = std::is_same_v<A, ScoredTopArgs>;
  using K = typename KeyOf<T>::type;
  const int64_t bytes = a.n_cols * static_cast<int64_t>(sizeof(T));
  if (a.n_cols <= kTileTop && a.k > 8 && a.n_rows >= kTileLeast * n_sms)
    return a.k <= 16 ? run_tiles<T, 16>(a, n_sms, s) : run_tiles<T, kTileTop>(a, n_sms, s);
  if (bytes <= kTileBytes && a.k <= 8 && (a.n_cols * (a.k + 1) <= kTileSteps || a.n_rows >= kTileLeast * n_sms)) {
    switch (a.k) {
      case 1: return run_tiles<T, 1>(a, n_sms, s);
      case 2: return run_tiles<T, 2>(a, n_sms, s);
      case 3: return run_tiles<T, 3>(a, n_sms, s);
      case 4: return run_tiles<T, 4>(a, n_sms, s);
      default: return run_tiles<T, 8>(a, n_sms, s);
    }
  }
  if (a.n_cols <= 32) return run_warps<T, 0, 1>(a, n_sms, s);
  if (a.n_cols <= 64) return run_warps<T, 0, 2>(a, n_sms, s);
  if (a.n_cols <= 128) return run_warps<T, 0, 4>(a, n_sms, s);
  if (a.n_cols <= 256) return run_warps<T, 0, 8>(a, n_sms, s);
  constexpr int kPieces = sizeof(T) == 8 ? 8 : sizeof(T);  // 512 elements
  if (a.n_cols <= 512) return run_warps<T, kPieces, 0>(a, n_sms, s);
  if (a.n_cols <= 1024) return run_warps<T, 2 * kPieces, 0>(a, n_sms, s);
  if constexpr (sizeof(T) < 8) {
    if (a.n_cols <= kWarpCols && a.k <= kWarpTop) return run_warps<T, 4 * kPieces, 0>(a, n_sms, s);
  }
  if constexpr (kIsScored) {
    const int64_t blocks = std::min<int64_t>((a.n_rows + kGroupThreads / 32 - 1) / (kGroupThreads / 32), kGroupBlocks * n_sms);
    if (by_groups(a.n_rows, a.n_cols, a.k, sizeof(T), n_sms)) {
      top_groups<T><<<static_cast<unsigned>(blocks), kGroupThreads, 0, s>>>(a);
      count_launches(1);
      return cudaGetLastError();
    }
  } else if (bytes <= kLongBytes && a.k <= kWarpTop && a.n_rows >= static_cast<int64_t>(kLongLeast) * n_sms) {
    const int64_t need = (a.n_rows + kThreads / 32 - 1) / (kThreads / 32), most = 16ll * n_sms;
    const auto kernel  = kernel_of(a, top_long<T, false>, top_long<T, true>);
    kernel<<<static_cast<unsigned>(need < most ? need : most), kThreads, 0, s>>>(a);
    count_launches(1);
    return cudaGetLastError();
  }
  int segs             = segments(a.n_rows, a.n_cols, n_sms);
  const bool clustered = segs > 1 && a.n_cols <= kJoinCols;
  if (clustered) {
    // (a part has more than the largest k: rounded up, segs is less than one for 1024 elements)
    int power = 2;
    while (power < segs && power < kCluster) power *= 2;
    segs = power;
  }
  int64_t cols = part_cols(a.n_cols, segs);
  if (!clustered) segs = static_cast<int>((a.n_cols + cols - 1) / cols);
  double* sums       = static_cast<double*>(workspace);
  K* keys            = reinterpret_cast<K*>(sums + (segs > 1 ? 3 * a.n_rows * segs : 0));
  const int64_t most = 16ll * n_sms;
  const unsigned rows = static_cast<unsigned>(a.n_rows < most ? a.n_rows : most);
  cudaLaunchConfig_t config{};
  config.gridDim  = dim3(rows * segs);
  config.blockDim = dim3(kThreads);
  config.stream   = s;
  cudaLaunchAttribute attribute{};
  attribute.id               = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim.x = segs;
  attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
  config.attrs    = &attribute;
  config.numAttrs = clustered ? 1 : 0;
  const auto kernel   = [&] {
    if constexpr (kIsScored)
      return top_segments<T, kScored>;
    else
      return kernel_of(a, top_segments<T, kScores>, top_segments<T, kProbabilities>);
  }();
  const cudaError_t e = cudaLaunchKernelEx(&config, kernel, a, segs, cols, clustered, keys, sums);
  if (e != cudaSuccess) return e;
  const bool join = segs > 1 && !clustered;
  if (join) top_join<T, kIsScored ? kScored : kScores><<<rows, kThreads, 0, s>>>(a, segs, keys, sums);
  count_launches(join ? 2 : 1);
  return cudaGetLastError();
}

}  // namespace

size_t top_workspace(int dtype, const TopArgs& a, int n_sms)
{
  const int64_t segs = segments(a.n_rows, a.n_cols, n_sms);
  if (segs <= 1 || a.n_cols <= kJoinCols) return 0;
  return a.n_rows * segs * (a.k * (dtype == kF64 ? sizeof(Key64) : sizeof(Key32)) + 3 * sizeof(double));
}

cudaError_t launch_top(int dtype, const TopArgs& a, void* workspace, int n_sms, cudaStream_t s)
{
  switch (dtype) {
    case kF32: return run_top<float>(a, workspace, n_sms, s);
    case kF64: return run_top<double>(a, workspace, n_sms, s);
    case kBF16: return run_top<__nv_bfloat16>(a, workspace, n_sms, s);
    case kF16: return run_top<__half>(a, workspace, n_sms, s);
  }
  return cudaErrorInvalidValue;
}

size_t scored_top_workspace(int dtype, const ScoreArgs& a, int n_sms)
{
  if (by_groups(a.n_rows, a.n_cols, a.k, dtype == kF32 ? 4 : 2, n_sms)) return 0;
  TopArgs t{};
  t.n_rows = a.n_rows;
  t.n_cols = a.n_cols;
  t.k      = a.k;
  return top_workspace(dtype, t, n_sms);
}

cudaError_t launch_scored_top(int dtype, const ScoreArgs& g, void* workspace, int n_sms, cudaStream_t s)
{
  ScoredTopArgs a{};
  a.scores      = g.logits;
  a.n_rows      = g.n_rows;
  a.n_cols      = g.n_cols;
  a.row_stride  = g.row_stride;
  a.k           = g.k;
  a.index       = g.top_index;
  a.target      = g.target;
  a.temperature = g.temperature;
  a.out         = g.out;
  a.top         = g.top;
  switch (dtype) {
    case kF32: return run_top<float>(a, workspace, n_sms, s);
    case kBF16: return run_top<__nv_bfloat16>(a, workspace, n_sms, s);
    case kF16: return run_top<__half>(a, workspace, n_sms, s);
  }
  return cudaErrorInvalidValue;
}

}  // namespace distill
}  // namespace b2fil
