// The k largest scores of each row, in descending order, equal ones by ascending class, and the row's
// log-sum-exp.
//
// Every score gets a key that no other of its row has: its value as an ordered integer, then the
// complement of its class.  NaN is above everything, -0 equals +0.  The thread t of a block sees the
// elements of its own group; the k-th largest of the groups' best keys is a bound tau that at least k
// elements reach, and all that reach it lie in the k groups whose best does: only these are read
// again (from L1 or L2).  Random rows leave little more than k candidates, which are sorted; where there
// are more than the list holds, the k-th key itself is found bit by bit.
//
// Bound by memory: one pass over the scores, which also takes the running maximum and sum of the
// log-sum-exp (the maximum is the thread's best score, so that both cost one comparison per 16 bytes).
// A block takes a segment of a row; the lists of several segments are joined by a second kernel.
#include "distill_common.cuh"

namespace b2fil {
namespace distill {
namespace {

constexpr int kThreads  = 256;   // groups: at least the largest k
constexpr int kSegment  = 16384; // largest part of a row that one block takes
constexpr int kList     = 2048;  // candidates that a block sorts
constexpr int kInFlight = 4;
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
  __device__ __forceinline__ Key32 lane_xor(int d) const { return {__shfl_xor_sync(~0u, w, d)}; }
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
  __device__ __forceinline__ Key64 lane_xor(int d) const { return {__shfl_xor_sync(~0u, v, d), __shfl_xor_sync(~0u, i, d)}; }
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
// One key per thread of the block, descending by thread; `room`: kThreads keys.
template <class K>
__device__ K sort_threads(K x, K* room)
{
  const int t = threadIdx.x;
  for (int size = 2; size <= kThreads; size <<= 1) {
    const bool down = (t & size) == 0;
    for (int d = size >> 1; d; d >>= 1) {
      K y;
      if (d >= 32) {
        __syncthreads();
        room[t] = x;
        __syncthreads();
        y = room[t ^ d];
      } else {
        y = x.lane_xor(d);
      }
      const bool first = (t & d) == 0;
      if ((first == down) == y.above(x)) x = y;
    }
  }
  return x;
}

template <class V>
__device__ __forceinline__ V log_of(V x);
template <>
__device__ __forceinline__ float log_of(float x) { return logf(x); }
template <>
__device__ __forceinline__ double log_of(double x) { return log(x); }

// What a score adds to the sum: exp((x - m) / T), or x^(1/T) for a probability.
template <class V>
__device__ __forceinline__ V term(V x, V m, V c, bool prob, bool plain)
{
  if (!prob) return power((x - base_of(m)) * c);
  // (the exponent of a probability is taken from its logarithm; T = 1 needs neither)
  return plain ? x : x == V(0) ? V(0) : power(log_of(x) * c);
}

// Writes the sorted keys of a row.
template <class T, class K>
__device__ __forceinline__ void write_top(const TopArgs& a, int64_t row, int j, const K& key)
{
  using V = typename ValueOf<T>::type;
  V v     = key.value();
  if (a.probabilities) v = log_of(v);
  static_cast<T*>(a.values)[row * a.k + j] = narrow<T>(v);
  a.index[row * a.k + j]                   = static_cast<int32_t>(key.index());
}
// m, s: of exp((x - m) / T), or of x^(1/T) (m unused); best: the row's largest key.
template <class V, class K>
__device__ __forceinline__ void write_lse(const TopArgs& a, int64_t row, V m, V s, const K& best)
{
  if (!a.logsumexp) return;
  const V top = best.value();
  V r;
  if (top != top)
    r = top;
  else if (a.probabilities)
    r = log_of(s);
  else
    r = top == lowest<V>() || top == -lowest<V>() ? top : static_cast<V>(top * a.inv_temperature) + log_of(s);
  static_cast<V*>(a.logsumexp)[row] = r;
}

// A segment of a row per block.  segs == 1: the row's answer; else its k best keys and its sum.
template <class T>
__global__ void __launch_bounds__(kThreads) top_segments(TopArgs a, int64_t seg_cols, typename KeyOf<T>::type* keys,
                                                         typename ValueOf<T>::type* sums)
{
  using V = typename ValueOf<T>::type;
  using K = typename KeyOf<T>::type;
  __shared__ K list[kList];
  __shared__ V room[64];
  __shared__ int found;
  const int segs      = gridDim.x;
  const int64_t begin = blockIdx.x * seg_cols;
  const int64_t n     = min(seg_cols, a.n_cols - begin);
  const int k         = static_cast<int>(min(static_cast<int64_t>(a.k), n));
  const V c           = static_cast<V>(1.4426950408889634 * a.inv_temperature);
  const bool plain    = a.inv_temperature == 1.0;
  const bool prob     = a.probabilities;
  for (int64_t row = blockIdx.y; row < a.n_rows; row += gridDim.y) {
    const T* x = static_cast<const T*>(a.scores) + row * a.row_stride + begin;
    // the thread's best score and its place, and the sum
    Running<V> r;
    uint32_t at  = ~0u;  // none yet
    bool nan     = false;
    visit_row<kInFlight>(
      x, n, threadIdx.x, kThreads,
      [&](int64_t i, T e) {
        const V v = widen(e);
        nan |= v != v;
        if (v > r.m || at == ~0u) {
          if (!prob && v > r.m) r.raise(v, c);
          r.m = larger(r.m, v);
          at  = static_cast<uint32_t>(i);
        }
        r.s += term(v, r.m, c, prob, plain);
      },
      [&](int64_t i, const Piece<T>& p) {
        constexpr int N = Piece<T>::N;
        V v[N], most;
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = widen(p.v[e]);
        most = v[0];
#pragma unroll
        for (int e = 1; e < N; ++e) most = larger(most, v[e]);
        if (most > r.m || at == ~0u) {
          if (!prob && most > r.m) r.raise(most, c);
          r.m = larger(r.m, most);
          at  = static_cast<uint32_t>(i);
#pragma unroll
          for (int e = N - 1; e >= 0; --e)
            if (v[e] == most) at = static_cast<uint32_t>(i + e);
        }
#pragma unroll
        for (int e = 0; e < N; ++e) {
          nan |= v[e] != v[e];
          r.s += term(v[e], r.m, c, prob, plain);
        }
      });
    K best = K::none();
    if (nan) {  // the first NaN of the group is its best
      uint32_t first = ~0u;
      visit_row<1>(
        x, n, threadIdx.x, kThreads,
        [&](int64_t i, T e) {
          if (widen(e) != widen(e)) first = min(first, static_cast<uint32_t>(i));
        },
        [&](int64_t i, const Piece<T>& p) {
#pragma unroll
          for (int e = 0; e < Piece<T>::N; ++e)
            if (widen(p.v[e]) != widen(p.v[e])) first = min(first, static_cast<uint32_t>(i + e));
        });
      best = K::of(static_cast<V>(NAN), static_cast<uint32_t>(begin) + first);
    } else if (at != ~0u) {
      best = K::of(r.m, static_cast<uint32_t>(begin) + at);
    }
    if (prob) {
      r.s = sum_row<kThreads>(r.s, room);
      r.m = V(0);
    } else {
      join_row<kThreads>(r, c, room);
    }
    // tau: the k-th largest of the groups' best keys (no key where there are fewer groups)
    const K mine = sort_threads(best, list);
    __syncthreads();
    if (threadIdx.x == k - 1) list[0] = mine;
    if (threadIdx.x == 0) found = 0;
    __syncthreads();
    const K tau = list[0];
    __syncthreads();
    auto collect = [&](const K& bound, bool store) {
      auto take = [&](int64_t i, T e) {
        const K key = K::of(widen(e), static_cast<uint32_t>(begin + i));
        if (!bound.above(key)) {
          const int to = atomicAdd(&found, 1);
          if (store && to < kList) list[to] = key;
        }
      };
      if (!bound.above(best))
        visit_row<1>(x, n, threadIdx.x, kThreads, take, [&](int64_t i, const Piece<T>& p) {
#pragma unroll
          for (int e = 0; e < Piece<T>::N; ++e) take(i + e, p.v[e]);
        });
      __syncthreads();
      const int got = found;
      __syncthreads();
      if (threadIdx.x == 0) found = 0;
      __syncthreads();
      return got;
    };
    int got = collect(tau, true);
    if (got > kList) {
      // the largest bound that k keys reach, bit by bit: keys differ, so exactly k do
      K bound = K::none();
      for (int bit = K::kBits - 1; bit >= 0; --bit) {
        const K next = bound.with(bit);
        if (collect(next, false) >= k) bound = next;
      }
      got = collect(bound, true);
    }
    int size = 1;
    while (size < got) size <<= 1;
    for (int i = got + threadIdx.x; i < size; i += kThreads) list[i] = K::none();
    __syncthreads();
    sort_list(list, size);
    if (segs == 1) {
      for (int j = threadIdx.x; j < a.k; j += kThreads) write_top<T>(a, row, j, list[j]);
      if (threadIdx.x == 0) write_lse(a, row, r.m, r.s, list[0]);
    } else {
      const int64_t part = row * segs + blockIdx.x;
      for (int j = threadIdx.x; j < a.k; j += kThreads) keys[part * a.k + j] = j < k ? list[j] : K::none();
      if (threadIdx.x == 0) {
        sums[2 * part]     = r.m;
        sums[2 * part + 1] = r.s;
      }
    }
    __syncthreads();
  }
}

// Joins the segments' lists of a row: as many as fit are sorted with the best so far.
template <class T>
__global__ void __launch_bounds__(kThreads) top_join(TopArgs a, int segs, const typename KeyOf<T>::type* keys,
                                                     const typename ValueOf<T>::type* sums)
{
  using V = typename ValueOf<T>::type;
  using K = typename KeyOf<T>::type;
  __shared__ K list[kList];
  __shared__ V room[64];
  const V c = static_cast<V>(1.4426950408889634 * a.inv_temperature);
  for (int64_t row = blockIdx.x; row < a.n_rows; row += gridDim.x) {
    const K* from = keys + row * segs * a.k;
    const int all = segs * a.k;
    int have      = 0;
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
    for (int j = threadIdx.x; j < a.k; j += kThreads) write_top<T>(a, row, j, list[j]);
    Running<V> r;
    for (int i = threadIdx.x; i < segs; i += kThreads) {
      const V m = sums[2 * (row * segs + i)], s = sums[2 * (row * segs + i) + 1];
      if (a.probabilities)
        r.s += s;
      else
        r.join(m, s, c);
    }
    if (a.probabilities)
      r.s = sum_row<kThreads>(r.s, room);
    else
      join_row<kThreads>(r, c, room);
    if (threadIdx.x == 0) write_lse(a, row, r.m, r.s, list[0]);
    __syncthreads();
  }
}

// Parts of a row: enough blocks to fill the machine, none below 2048 elements or above kSegment.
int segments(int64_t n_rows, int64_t n_cols, int n_sms)
{
  const int64_t least = (n_cols + kSegment - 1) / kSegment;
  const int64_t fill  = (4 * n_sms + n_rows - 1) / (n_rows ? n_rows : 1);
  const int64_t most  = (n_cols + 2047) / 2048;
  const int64_t segs  = fill < most ? fill : most;
  return static_cast<int>(segs < least ? least : segs);
}
int64_t part_cols(int64_t n_cols, int segs)
{
  return segs == 1 ? n_cols : ((n_cols + segs - 1) / segs + 63) / 64 * 64;
}

template <class T>
cudaError_t run_top(const TopArgs& a, void* workspace, int n_sms, cudaStream_t s)
{
  using K = typename KeyOf<T>::type;
  using V = typename ValueOf<T>::type;
  int segs           = segments(a.n_rows, a.n_cols, n_sms);
  const int64_t cols = part_cols(a.n_cols, segs);
  segs               = static_cast<int>((a.n_cols + cols - 1) / cols);
  K* keys            = static_cast<K*>(workspace);
  V* sums            = reinterpret_cast<V*>(keys + (segs > 1 ? a.n_rows * segs * a.k : 0));
  const unsigned rows = static_cast<unsigned>(a.n_rows < 65535 ? a.n_rows : 65535);
  top_segments<T><<<dim3(segs, rows), kThreads, 0, s>>>(a, cols, keys, sums);
  if (segs > 1) {
    const int64_t most = 16ll * n_sms;
    top_join<T><<<static_cast<unsigned>(a.n_rows < most ? a.n_rows : most), kThreads, 0, s>>>(a, segs, keys, sums);
  }
  count_launches(segs > 1 ? 2 : 1);
  return cudaGetLastError();
}

}  // namespace

size_t top_workspace(int dtype, const TopArgs& a, int n_sms)
{
  const int64_t segs = segments(a.n_rows, a.n_cols, n_sms);
  if (segs <= 1) return 0;
  const size_t key = dtype == kF64 ? sizeof(Key64) : sizeof(Key32);
  return a.n_rows * segs * (a.k * key + 2 * (dtype == kF64 ? 8 : 4)) + 16;
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

}  // namespace distill
}  // namespace b2fil
