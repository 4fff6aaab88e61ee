// T^2 KL(teacher || student) of rows of logits over the teacher's top classes, and its gradient.
//
// With q = softmax(z / T), p the teacher's probabilities of the classes that it names and, where the rest
// of its distribution is one more class, p_r and q_r what is left on either side:
//   loss  = T^2 [ sum_named p (log p - log q) + p_r (log p_r - log q_r) ]
//   dloss / dz_c = T (q_c - p_c) for named classes, T (q_r - p_r) s_c for the others, s the softmax over these:
// T q_c (1 - p_r / q_r), whose parts leave the range where q_r does, though p_r s_c does not.  Where no class is left for
// the rest, p adds up to P < 1, and q is P q in the gradient.
// Softmax cross entropy is the case of one named class of probability 1 and T = 1.
//
// Bound by memory: the forward pass reads the logits once (running maximum and sum), the backward pass
// reads them again and writes as much.  What a teacher names in a row is the work of one warp, whose chain of
// dependent loads, votes and logarithms takes as long as reading some 32 KB.  Short rows
// therefore belong to one warp altogether, and many warps hide it; longer ones to a block of eight
// warps that read, while a ninth prepares the next row and a tenth finishes the last.  Where rows are few,
// several blocks read parts of one and a warp joins their maxima and sums.  Many rows of a few classes belong to one
// thread each, from a tile in shared memory.
#include <cooperative_groups.h>

#include "distill_common.cuh"

namespace b2fil {
namespace distill {
namespace {

constexpr int kThreads  = 256;
constexpr int kWide     = kThreads + 64;  // eight warps that read, two for the teacher
constexpr int kWideRows = 3;              // blocks of an SM (four with 4 pieces: 204 against 197 us, 4096 x 131,072)
constexpr int kWarpCols = 2048;           // rows that belong to one warp
// ... and where there are kWarpLeast of them per SM: longer ones whose logits take up to kWarpBytes, and in the
// gradient, of 16 bits, which the instructions bound, up to kWarpLong.  (Loss and gradient by blocks and by warps, us:
// 20,000 x 3000 bf16 101, 94 and 50, 46; 20,000 x 6000 bf16 135, 123 and 83, 97; 20,000 x 3000 fp32 121, 86 and 73, 97.)
constexpr int kWarpLeast = 8;
constexpr int kWarpBytes = 16384;
constexpr int kWarpLong  = 8192;
constexpr int kSegment  = 8192;           // fewest elements of a row that are worth a block of their own
constexpr int kMostBits = 1 << 17;        // classes that a block marks (three rows of it: 48 KB)
constexpr int kMostSegs = 64;
constexpr int kInFlight = 8;              // pieces of a thread (the gradient of long rows: 4, as it writes as much)
constexpr int kCluster  = 8;              // blocks that add up their losses without another kernel
// Rows for one thread each: classes (the bits of one word), entries, and rows per SM from which on.  (1,000,000 x 10
// fp32, k 3, rest as a class, loss and gradient: 1646 us with a warp per row, 100 this way; 292,366 x 13 bf16: 474
// and 37.)
constexpr int kTileCols  = 64;
constexpr int kTileTop   = 16;
constexpr int kTileLeast  = 32;
constexpr int kTileBlocks = 8;  // of an SM, all there at once (292,366 x 13 bf16, rest as a class: 26.8 us, 28.8 with the seven that
                                // 72 registers allow)

// Bits of the named classes: bit 32 stands for the first element on a 16-byte boundary.
__host__ __device__ __forceinline__ size_t bit_bytes(int64_t cols) { return cols ? ((cols + 32) / 32 + 2) * 4 : 0; }

// Running maximum and sum of n elements; with REST those whose bit is set are left out.  Bit 32 stands for
// the first element on a 16-byte boundary, so that a piece's bits lie in one word.
template <class T, bool REST>
__device__ __forceinline__ Running<float> visit_logits(const T* row, int64_t n, int tid, int threads, float c,
                                                       const uint32_t* bits)
{
  constexpr int N = Piece<T>::N;
  Stream<float> r;
  const int lead    = lead_of(row, n);
  const float slack = kSlack / c;
  visit_row<kInFlight>(
    row, n, tid, threads,
    [&](int64_t i, T x) {
      if (REST) {
        const uint32_t at = static_cast<uint32_t>(i - lead + 32);
        if (bits[at >> 5] >> (at & 31) & 1) return;
      }
      r.take(widen(x), c, slack);
    },
    [&](int64_t i, const Piece<T>& v) {
      float x[N], most;
#pragma unroll
      for (int e = 0; e < N; ++e) x[e] = widen(v.v[e]);
      if (REST) {
        const uint32_t at  = static_cast<uint32_t>(i - lead + 32);
        const uint32_t set = bits[at >> 5] >> (at & 31) & ((1u << N) - 1);
        if (set) {
#pragma unroll
          for (int e = 0; e < N; ++e)
            if (set >> e & 1) x[e] = lowest<float>();
        }
      }
      most = x[0];
#pragma unroll
      for (int e = 1; e < N; ++e) most = fmaxf(most, x[e]);
      if (most > r.limit) r.raise(most, c, slack);
#pragma unroll
      for (int e = 0; e < N; ++e) r.add(x[e], c);
    });
  return r.running();
}

// Marks (or unmarks) the entries that lie in n columns from `begin` on.  By one warp.
template <bool SET>
__device__ __forceinline__ void mark(const Entries& e, int k, int64_t begin, int64_t n, int lead, uint32_t* bits)
{
  for (int j = threadIdx.x % 32; j < k; j += 32) {
    const int64_t c = e.at[j] - begin;
    if (e.at[j] < 0 || c < 0 || c >= n) continue;
    const uint32_t at = static_cast<uint32_t>(c - lead + 32);
    if (SET)
      atomicOr(&bits[at >> 5], 1u << (at & 31));
    else
      atomicAnd(&bits[at >> 5], ~(1u << (at & 31)));
  }
}

// One part of a row per block: (row, segment) -> its maximum and sum.
template <class T, bool REST>
__global__ void __launch_bounds__(kThreads) loss_parts(LossArgs a, int64_t seg_cols, float2* parts)
{
  extern __shared__ __align__(16) char smem[];
  __shared__ float room[2 * kThreads / 32];
  uint32_t* bits      = reinterpret_cast<uint32_t*>(smem);
  const int64_t begin = blockIdx.x * seg_cols;
  const int64_t n     = min(seg_cols, a.n_cols - begin);
  const float c       = a.temperature.c;
  for (int64_t row = blockIdx.y; row < a.n_rows; row += gridDim.y) {
    const T* x = static_cast<const T*>(a.logits) + row * a.row_stride + begin;
    if (REST) {
      const int lead = lead_of(x, n);
      __syncthreads();
      for (int w = threadIdx.x; w < bit_bytes(n) / 4; w += kThreads) bits[w] = 0;
      __syncthreads();
      for (int j = threadIdx.x; j < a.teacher.k; j += kThreads) {
        const int64_t at = teacher_index(a.teacher, row, j);
        if (at < begin || at >= begin + n || at == a.teacher.ignore) continue;
        const uint32_t bit = static_cast<uint32_t>(at - begin - lead + 32);
        atomicOr(&bits[bit >> 5], 1u << (bit & 31));
      }
      __syncthreads();
    }
    Running<float> r = visit_logits<T, REST>(x, n, threadIdx.x, kThreads, c, bits);
    join_row<kThreads>(r, c, room);
    if (threadIdx.x == 0) parts[row * gridDim.x + blockIdx.x] = make_float2(r.m, r.s);
  }
}

// The named and the other classes of a row together.  With d the logarithm of their sums' ratio, log q_r = -log(1 + e^d) and
// q_r - p_r = (1 - p_r) - (1 - q_r): where both rests are nearly 1 the loss is a difference of small numbers, which keep their
// relative exactness.
struct Split {
  double log_s;      // of all, relative to m
  double log_rest;   // log q_r
  float difference;  // q_r - p_r
};
__device__ __forceinline__ Split split(const Running<float>& named, const Running<float>& others, float m, double inv_t, double rest)
{
  const double a = (static_cast<double>(named.m) - m) * inv_t + log_sum(named.s);
  const double b = (static_cast<double>(others.m) - m) * inv_t + log_sum(others.s);
  const double d = a - b;
  const float e = expf(-fabsf(static_cast<float>(d))), more = log1pf(e), less = e / (1.f + e);
  const bool few = d <= 0;  // less of the student is on the named classes
  return {(few ? b : a) + more, (few ? 0.0 : -d) - more, few ? static_cast<float>(1.0 - rest) - less : less - static_cast<float>(rest)};
}
// log p_r: where p_r is small it is off by 2^-24 / p_r, and weighs with p_r.
__device__ __forceinline__ float log_of_rest(double rest) { return log1pf(-static_cast<float>(1.0 - rest)); }

// A row's loss, by one warp.  r: maximum and sum of the logits (REST: of those that are not named).
template <class T, bool REST>
__device__ __forceinline__ void finish_row(const LossArgs& a, int64_t row, const T* x, const Entries& e, const TeacherRow& t,
                                           double inv_t, float c, Running<float> r, double& sum, double& count)
{
  const int lane = threadIdx.x % 32, k = a.teacher.k;
  const Running<float> others = r;
  Split both;
  if (REST) {
    Running<float> mine;
    for (int j = lane; j < k; j += 32)
      if (e.at[j] >= 0) mine.take(widen(x[e.at[j]]), c);
    mine.join_lanes(c);
    r.join(mine.m, mine.s, c);
    both = split(mine, others, r.m, inv_t, t.rest);
  }
  const double log_s = REST ? both.log_s : log_sum(r.s);
  const bool counts  = t.counts && !(r.s == 0.f);  // (no class has a finite logit: no softmax)
  double loss        = named_loss(e, k, t, inv_t, r.m, log_s, [&](int, int at) { return widen(x[at]); });
  float4 stats       = make_float4(r.m, t.mass / r.s, r.m, t.mass / r.s);
  if (REST && t.rest != 0.0) {
    loss += t.rest * (log_of_rest(t.rest) - both.log_rest);
    stats.z = others.m;
    stats.w = both.difference / others.s;
  }
  if (!counts) loss = 0;
  loss *= a.temperature.t * a.temperature.t;
  for (int j = lane; j < k; j += 32) {
    a.named.p[row * k + j]  = e.p[j];
    a.named.at[row * k + j] = e.at[j];
  }
  if (lane == 0) {
    a.row_loss[row]  = static_cast<float>(loss);
    a.row_stats[row] = counts ? stats : make_float4(0.f, 0.f, 0.f, 0.f);
    sum += loss;
    count += counts;
  }
}

// Adds up the losses of a launch of one cluster, or leaves the block's for reduce_loss.
template <int THREADS>
__device__ __forceinline__ void finish_block(double sum, double count, bool one_cluster, const Reduced& out, double2* block_sums)
{
  __shared__ double2 room[THREADS / 32];
  __shared__ double2 mine;
  if (out.reduction == 0) return;
  const double2 all = sum_block<THREADS>(sum, count, room);
  if (!one_cluster) {
    if (threadIdx.x == 0) block_sums[blockIdx.x] = all;
    return;
  }
  namespace cg = cooperative_groups;
  if (threadIdx.x == 0) mine = all;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    double2 total = make_double2(0, 0);
    for (int i = 0; i < static_cast<int>(gridDim.x); ++i) {
      const double2 o = *cluster.map_shared_rank(&mine, i);
      total.x += o.x;
      total.y += o.y;
    }
    write_reduced(out, total);
  }
  cluster.sync();  // the others' shared memory has been read
}

// A row per warp.  segs > 0: maxima and sums come from `parts`.
template <class T, bool REST>
__global__ void __launch_bounds__(kThreads, 5) loss_narrow(LossArgs a, int segs, const float2* parts, size_t warp_room,
                                                        bool one_cluster, Reduced out, double2* block_sums)
{
  extern __shared__ __align__(16) char smem[];
  constexpr int ROWS = kThreads / 32;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, k = a.teacher.k;
  const Entries e    = entries_at(smem + warp * warp_room, k);
  uint32_t* bits     = reinterpret_cast<uint32_t*>(e.at + k);
  const float c      = a.temperature.c;
  const double inv_t = a.temperature.inverse;
  double sum = 0, count = 0;
  if (REST && segs == 0) {
    for (int w = lane; w < bit_bytes(a.n_cols) / 4; w += 32) bits[w] = 0;
    __syncwarp();
  }
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + warp; row < a.n_rows; row += static_cast<int64_t>(gridDim.x) * ROWS) {
    const T* x         = static_cast<const T*>(a.logits) + row * a.row_stride;
    const int lead     = lead_of(x, a.n_cols);
    const TeacherRow t = read_teacher<REST>(a.teacher, row, a.n_cols, inv_t, e);
    Running<float> r;
    if (segs > 0) {
      for (int i = lane; i < segs; i += 32) r.join(parts[row * segs + i].x, parts[row * segs + i].y, c);
    } else {
      if (REST) {
        mark<true>(e, k, 0, a.n_cols, lead, bits);
        __syncwarp();
      }
      r = visit_logits<T, REST>(x, a.n_cols, lane, 32, c, bits);
    }
    r.join_lanes(c);
    finish_row<T, REST>(a, row, x, e, t, inv_t, c, r, sum, count);
    if (REST && segs == 0) mark<false>(e, k, 0, a.n_cols, lead, bits);
    __syncwarp();
  }
  finish_block<kThreads>(sum, count, one_cluster, out, block_sums);
}

// A row per thread.  What is not named is what the word's bits leave.
template <class T, bool REST>
__global__ void __launch_bounds__(kTileRows, kTileBlocks) loss_tiles(LossArgs a, Reduced out, double2* block_sums)
{
  extern __shared__ __align__(16) char smem[];
  T* tile         = reinterpret_cast<T*>(smem);
  const Teacher t = a.teacher;
  const int k = t.k, cols = static_cast<int>(a.n_cols);
  const TileShape<T> shape(cols);
  const float c = a.temperature.c, ti = static_cast<float>(a.temperature.inverse);
  const double inv_t = a.temperature.inverse;
  const bool whole   = without_gaps<T>(a.logits, a.row_stride, cols);
  double sum = 0, count = 0;
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * kTileRows; first < a.n_rows;
       first += static_cast<int64_t>(gridDim.x) * kTileRows) {
    const int rows = static_cast<int>(min(static_cast<int64_t>(kTileRows), a.n_rows - first));
    __syncthreads();  // the last tile has been used
    load_tile(tile, shape, static_cast<const T*>(a.logits) + first * a.row_stride, a.row_stride, rows, whole);
    __syncthreads();
    if (threadIdx.x >= rows) continue;
    const T* x        = tile + threadIdx.x * shape.pitch;
    const int64_t row = first + threadIdx.x;
    // the teacher: classes, the largest score, classes named twice
    float* p       = a.named.p + row * k;
    int32_t* at    = a.named.at + row * k;
    const float* v = t.values ? t.values + row * t.values_stride : nullptr;
    uint64_t named = 0;
    float top      = lowest<float>();
    bool merged    = false;
    for (int j = 0; j < k; ++j) {
      const int64_t cls = teacher_index(t, row, j);
      const bool is     = cls >= 0 && cls < cols && cls != t.ignore;
      at[j]             = is ? static_cast<int>(cls) : -1;
      if (!is) continue;
      merged |= named >> cls & 1;
      named |= 1ull << cls;
      top = fmaxf(top, v ? v[j] : 0.f);
    }
    double log_norm;
    double rest = 0.0;
    float norm = 1.f, all_p = 1.f;
    bool counts;
    if (REST) {
      log_norm    = t.logsumexp[row];
      counts      = !(log_norm == -INFINITY);
      double mass = 0;
      for (int j = 0; j < k; ++j) {
        const double q = at[j] >= 0 && counts ? exp((v ? v[j] : 0.f) * inv_t - log_norm) : 0.0;
        p[j]           = static_cast<float>(q);
        mass += q;
      }
      const bool all = __popcll(named) >= cols;
      rest           = all || 1.0 - mass < least_rest(log_norm) ? 0.0 : 1.0 - mass;
      if (rest == 0.0) all_p = static_cast<float>(mass);
    } else {
      const float most = base_of(top);
      float total      = 0.f;
      for (int j = 0; j < k; ++j) {
        const float e = at[j] >= 0 ? expf(((v ? v[j] : 0.f) - most) * ti) : 0.f;
        p[j]          = e;
        total += e;
      }
      log_norm = most * inv_t + log_sum(total);
      counts   = !(total == 0.f);
      norm     = counts ? 1.f / total : 1.f;
    }
    // the student: maximum and sum, with REST of the others apart
    Running<float> r, others;
    for (int i = 0; i < cols; ++i) r.m = fmaxf(r.m, widen(x[i]));
    const float base = base_of(r.m);
    for (int i = 0; i < cols; ++i) {
      const float e = power((widen(x[i]) - base) * c);
      if (REST && !(named >> i & 1))
        others.s += e;
      else
        r.s += e;
    }
    Split both;
    if (REST) {
      const Running<float> mine = r;
      r.s += others.s;
      others.m = r.m;
      // far below the named ones (or none): relative to their own maximum, or the gradient's terms leave the range (2^-126) at more
      // than 2^-96 of the largest
      if (others.s < 0x1p-30f) {
        others = Running<float>();
        for (int i = 0; i < cols; ++i)
          if (!(named >> i & 1)) others.m = fmaxf(others.m, widen(x[i]));
        for (int i = 0; i < cols; ++i)
          if (!(named >> i & 1)) others.s += power((widen(x[i]) - base_of(others.m)) * c);
      }
      both = split(mine, others, r.m, inv_t, rest);
    }
    const double log_s = REST ? both.log_s : log_sum(r.s);
    counts             = counts && !(r.s == 0.f);
    double loss        = 0;
    for (int j = 0; j < k; ++j) {
      float q = p[j] * norm;
      if (merged && at[j] >= 0) {  // the first entry of a class has the sum, the others are none
        for (int i = j + 1; i < k; ++i)
          if (at[i] == at[j]) {
            q += p[i] * norm;
            at[i] = -1;
          }
      }
      p[j] = q;
      if (at[j] < 0 || q == 0.f) continue;
      const double log_p = merged ? log(static_cast<double>(q)) : (v ? v[j] : 0.f) * inv_t - log_norm;
      loss += q * (log_p - ((static_cast<double>(widen(x[at[j]])) - r.m) * inv_t - log_s));
    }
    float4 stats = make_float4(r.m, all_p / r.s, r.m, all_p / r.s);
    if (REST && rest != 0.0) {
      loss += rest * (log_of_rest(rest) - both.log_rest);
      stats.z = others.m;
      stats.w = both.difference / others.s;
    }
    if (!counts) loss = 0;
    loss *= a.temperature.t * a.temperature.t;
    a.row_loss[row]  = static_cast<float>(loss);
    a.row_stats[row] = counts ? stats : make_float4(0.f, 0.f, 0.f, 0.f);
    sum += loss;
    count += counts;
  }
  finish_block<kTileRows>(sum, count, false, out, block_sums);
}

// Its gradient.
template <class T>
__global__ void __launch_bounds__(kTileRows) grad_tiles(LossGradArgs g)
{
  extern __shared__ __align__(16) char smem[];
  T* tile           = reinterpret_cast<T*>(smem);
  const LossArgs& a = g.fwd;
  const int k = a.teacher.k, cols = static_cast<int>(a.n_cols);
  const TileShape<T> shape(cols);
  const float c     = a.temperature.c;
  const float scale = (g.factor ? *g.factor : 1.f) * static_cast<float>(a.temperature.t);
  const bool whole_in = without_gaps<T>(a.logits, a.row_stride, cols), whole_out = without_gaps<T>(g.grad, g.grad_stride, cols);
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * kTileRows; first < a.n_rows;
       first += static_cast<int64_t>(gridDim.x) * kTileRows) {
    const int rows = static_cast<int>(min(static_cast<int64_t>(kTileRows), a.n_rows - first));
    __syncthreads();  // the last tile has been stored
    load_tile(tile, shape, static_cast<const T*>(a.logits) + first * a.row_stride, a.row_stride, rows, whole_in);
    __syncthreads();
    if (threadIdx.x < rows) {
      T* x              = tile + threadIdx.x * shape.pitch;
      const int64_t row = first + threadIdx.x;
      const float4 s    = a.row_stats[row];
      const float up    = g.upstream[row * g.upstream_stride] * scale;
      const bool counts = s.y != 0.f;
      const float base = base_of(s.x), base_others = base_of(s.z), f = s.w * up;
      // the named classes' from their logits, which are then put over the others'
      float named[kTileTop];
#pragma unroll
      for (int j = 0; j < kTileTop; ++j) {
        const int at = j < k ? a.named.at[row * k + j] : -1;
        named[j]     = at >= 0 ? (power((widen(x[at]) - base) * c) * s.y - a.named.p[row * k + j]) * up : 0.f;
      }
      for (int i = 0; i < cols; ++i) x[i] = narrow<T>(counts ? power((widen(x[i]) - base_others) * c) * f : 0.f);
#pragma unroll
      for (int j = 0; j < kTileTop; ++j) {
        const int at = j < k && counts ? a.named.at[row * k + j] : -1;
        if (at >= 0) x[at] = narrow<T>(named[j]);
      }
    }
    __syncthreads();
    store_tile(static_cast<T*>(g.grad) + first * g.grad_stride, g.grad_stride, tile, shape, rows, whole_out);
  }
}

// A row per block: while eight warps read row i, one prepares row i + 1 and one finishes row i - 1.
template <class T, bool REST>
__global__ void __launch_bounds__(kWide, kWideRows) loss_wide(LossArgs a, size_t bits_room, bool one_cluster, Reduced out,
                                                              double2* block_sums)
{
  extern __shared__ __align__(16) char smem[];
  constexpr int W = kThreads / 32;
  __shared__ float2 parts[2][W];
  __shared__ TeacherRow teachers[3];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, k = a.teacher.k;
  const float c      = a.temperature.c;
  const double inv_t = a.temperature.inverse;
  auto entries       = [&](int i) { return entries_at(smem + 3 * bits_room + i * entry_bytes(k), k); };
  auto bits          = [&](int i) { return reinterpret_cast<uint32_t*>(smem + i * bits_room); };
  auto logits        = [&](int64_t row) { return static_cast<const T*>(a.logits) + row * a.row_stride; };
  double sum = 0, count = 0;
  if (REST)
    for (int w = threadIdx.x; w < 3 * bits_room / 4; w += kWide) reinterpret_cast<uint32_t*>(smem)[w] = 0;
  // (bits and entries of rows i - 1, i and i + 1 are in use at a time)
  auto prepare = [&](int64_t row, int at) {
    const TeacherRow t = read_teacher<REST>(a.teacher, row, a.n_cols, inv_t, entries(at));
    if (lane == 0) teachers[at] = t;
    if (REST) mark<true>(entries(at), k, 0, a.n_cols, lead_of(logits(row), a.n_cols), bits(at));
  };
  __syncthreads();
  if (warp == W && blockIdx.x < a.n_rows) prepare(blockIdx.x, 0);
  int last = 2, now = 0, next = 1, half = 0;
  for (int64_t row = blockIdx.x; row - gridDim.x < a.n_rows; row += gridDim.x) {
    __syncthreads();  // this row is marked, the last one has been read
    if (warp < W) {
      if (row < a.n_rows) {
        Running<float> r = visit_logits<T, REST>(logits(row), a.n_cols, threadIdx.x, kThreads, c, bits(now));
        r.join_lanes(c);
        if (lane == 0) parts[half][warp] = make_float2(r.m, r.s);
      }
    } else if (warp == W) {
      if (row + gridDim.x < a.n_rows) prepare(row + gridDim.x, next);
    } else if (row != blockIdx.x) {
      const int64_t done = row - gridDim.x;
      Running<float> r;
      if (lane < W) {
        r.m = parts[half ^ 1][lane].x;
        r.s = parts[half ^ 1][lane].y;
      }
      r.join_lanes(c);
      finish_row<T, REST>(a, done, logits(done), entries(last), teachers[last], inv_t, c, r, sum, count);
      if (REST) mark<false>(entries(last), k, 0, a.n_cols, lead_of(logits(done), a.n_cols), bits(last));
    }
    const int first = last;
    last = now;
    now  = next;
    next = first;
    half ^= 1;
  }
  finish_block<kWide>(sum, count, one_cluster, out, block_sums);
}

__global__ void __launch_bounds__(kThreads) reduce_loss(const double2* block_sums, int n, Reduced out)
{
  __shared__ double2 room[kThreads / 32];
  double sum = 0, count = 0;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    sum += block_sums[i].x;
    count += block_sums[i].y;
  }
  const double2 all = sum_block<kThreads>(sum, count, room);
  if (threadIdx.x == 0) write_reduced(out, all);
}

// Gradient of a part of a row by THREADS threads; blockIdx.y: the part.
template <class T, int THREADS>
__global__ void __launch_bounds__(kThreads) loss_grad(LossGradArgs g, int64_t seg_cols)
{
  constexpr int ROWS = kThreads / THREADS, N = Piece<T>::N;
  const LossArgs& a = g.fwd;
  const int slot = threadIdx.x / THREADS, tid = threadIdx.x % THREADS, k = a.teacher.k;
  const float c       = a.temperature.c;
  const int64_t begin = blockIdx.y * seg_cols;
  const int64_t n     = min(seg_cols, a.n_cols - begin);
  const float scale   = (g.factor ? *g.factor : 1.f) * static_cast<float>(a.temperature.t);
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + slot; row < a.n_rows;
       row += static_cast<int64_t>(gridDim.x) * ROWS) {
    const T* x     = static_cast<const T*>(a.logits) + row * a.row_stride + begin;
    T* d           = static_cast<T*>(g.grad) + row * g.grad_stride + begin;
    const float4 s = a.row_stats[row];
    const float up = g.upstream[row * g.upstream_stride] * scale;
    const bool counts = s.y != 0.f;
    // zero for rows that do not count, whatever their logits are
    const float base = base_of(s.x), base_others = base_of(s.z), f = s.w * up;
    auto one = [&](int64_t i, T v) { d[i] = narrow<T>(counts ? power((widen(v) - base_others) * c) * f : 0.f); };
    if (((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(d)) & 15) == 0) {
      visit_row<THREADS == 32 ? kInFlight : kInFlight / 2>(x, n, tid, THREADS, one, [&](int64_t i, const Piece<T>& v) {
        Piece<T> w;
#pragma unroll
        for (int e = 0; e < N; ++e) w.v[e] = narrow<T>(counts ? power((widen(v.v[e]) - base_others) * c) * f : 0.f);
        *reinterpret_cast<uint4*>(d + i) = *reinterpret_cast<const uint4*>(&w);
      });
    } else {
      for (int64_t i = tid; i < n; i += THREADS) one(i, x[i]);
    }
    sync_row<THREADS>();
    if (counts) {
      for (int j = tid; j < k; j += THREADS) {
        const int cls    = a.named.at[row * k + j];
        const int64_t at = cls - begin;
        if (cls < 0 || at < 0 || at >= n) continue;
        d[at] = narrow<T>((power((widen(x[at]) - base) * c) * s.y - a.named.p[row * k + j]) * up);
      }
    }
  }
}

int segments(int64_t n_rows, int64_t n_cols, int n_sms, bool rest)
{
  const int64_t least = rest ? (n_cols + kMostBits - 1) / kMostBits : 1;
  if (n_rows == 0 || n_cols <= kWarpCols || n_rows >= 2 * n_sms) return static_cast<int>(least);
  const int64_t want = (4 * n_sms + n_rows - 1) / n_rows;
  const int64_t most = (n_cols + kSegment - 1) / kSegment;
  int64_t segs       = want < most ? want : most;
  segs               = segs < 1 ? 1 : segs > kMostSegs ? kMostSegs : segs;
  return static_cast<int>(segs < least ? least : segs);
}
// length of a part: whole 128-byte lines of every type
int64_t part_cols(int64_t n_cols, int segs)
{
  return segs == 1 ? n_cols : ((n_cols + segs - 1) / segs + 63) / 64 * 64;
}

template <class K>
cudaError_t allow(K kernel, size_t bytes)
{
  return bytes <= 48 * 1024 ? cudaSuccess
                            : cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
}

// Launches a kernel whose blocks, up to kCluster of them, are one cluster and add up their losses.
template <class... P, class... A>
cudaError_t launch_rows(void (*kernel)(P...), int blocks, bool one_cluster, int threads, size_t bytes, cudaStream_t s, A... args)
{
  cudaError_t e = allow(kernel, bytes);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t config{};
  config.gridDim          = dim3(blocks);
  config.blockDim         = dim3(threads);
  config.dynamicSmemBytes = bytes;
  config.stream           = s;
  cudaLaunchAttribute attribute{};
  attribute.id               = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim.x = blocks;
  attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
  config.attrs    = &attribute;
  config.numAttrs = one_cluster ? 1 : 0;
  return cudaLaunchKernelEx(&config, kernel, static_cast<P>(args)...);
}

bool by_warps(const LossArgs& a, int n_sms, bool longer)
{
  return a.n_cols <= kWarpCols || (longer && a.n_rows >= static_cast<int64_t>(kWarpLeast) * n_sms);
}
bool by_tiles(const LossArgs& a, int n_sms)
{
  return a.n_cols <= kTileCols && a.teacher.k <= kTileTop && a.n_rows >= static_cast<int64_t>(kTileLeast) * n_sms;
}

template <class T, bool REST>
cudaError_t run_loss(const LossArgs& a, const Reduced& out, void* workspace, int n_sms, cudaStream_t s)
{
  if (by_tiles(a, n_sms)) {
    const int64_t need = (a.n_rows + kTileRows - 1) / kTileRows, most = static_cast<int64_t>(kTileBlocks) * n_sms;
    const int blocks   = static_cast<int>(need < most ? need : most);
    double2* sums      = static_cast<double2*>(workspace);
    loss_tiles<T, REST><<<blocks, kTileRows, TileShape<T>(static_cast<int>(a.n_cols)).bytes(), s>>>(a, out, sums);
    if (out.reduction != 0) reduce_loss<<<1, kThreads, 0, s>>>(sums, blocks, out);
    count_launches(out.reduction != 0 ? 2 : 1);
    return cudaGetLastError();
  }
  int segs           = segments(a.n_rows, a.n_cols, n_sms, REST);
  const int64_t cols = part_cols(a.n_cols, segs);
  segs               = segs == 1 ? 1 : static_cast<int>((a.n_cols + cols - 1) / cols);
  const bool narrow  = segs > 1 || by_warps(a, n_sms, a.n_cols * sizeof(T) <= kWarpBytes);
  const int per      = narrow ? kThreads / 32 : 1;
  const int64_t need = (a.n_rows + per - 1) / per, most = (narrow ? 8ll : kWideRows) * n_sms;
  int blocks         = static_cast<int>(need < most ? need : most);
  double2* sums      = static_cast<double2*>(workspace);
  float2* parts      = reinterpret_cast<float2*>(sums + 8 * n_sms);
  const bool cluster = out.reduction != 0 && blocks >= 1 && blocks <= kCluster;
  while (cluster && (blocks & (blocks - 1))) ++blocks;
  int launched  = 0;
  cudaError_t e = cudaSuccess;
  if (segs > 1 && a.n_rows > 0) {
    const size_t bytes = REST ? bit_bytes(cols) : 0;
    const unsigned rows = static_cast<unsigned>(a.n_rows < 65535 ? a.n_rows : 65535);
    if ((e = allow(loss_parts<T, REST>, bytes)) != cudaSuccess) return e;
    loss_parts<T, REST><<<dim3(segs, rows), kThreads, bytes, s>>>(a, cols, parts);
    ++launched;
  }
  if (blocks > 0) {
    const size_t bits = REST && segs == 1 ? (bit_bytes(a.n_cols) + 15) / 16 * 16 : 0;
    if (narrow) {
      const size_t room = (entry_bytes(a.teacher.k) + bits + 15) / 16 * 16;
      e = launch_rows(loss_narrow<T, REST>, blocks, cluster, kThreads, room * per, s, a, segs > 1 ? segs : 0, parts, room,
                      cluster, out, sums);
    } else {
      e = launch_rows(loss_wide<T, REST>, blocks, cluster, kWide, 3 * (bits + entry_bytes(a.teacher.k)), s, a, bits, cluster,
                      out, sums);
    }
    if (e != cudaSuccess) return e;
    ++launched;
  }
  if (out.reduction != 0 && !cluster) {
    reduce_loss<<<1, kThreads, 0, s>>>(sums, blocks, out);
    ++launched;
  }
  count_launches(launched);
  return cudaGetLastError();
}

template <class T>
cudaError_t run_grad(const LossGradArgs& g, int n_sms, cudaStream_t s)
{
  const LossArgs& a  = g.fwd;
  if (by_tiles(a, n_sms)) {
    const int64_t need = (a.n_rows + kTileRows - 1) / kTileRows, most = 16ll * n_sms;
    grad_tiles<T><<<static_cast<unsigned>(need < most ? need : most), kTileRows,
                    TileShape<T>(static_cast<int>(a.n_cols)).bytes(), s>>>(g);
    count_launches(1);
    return cudaGetLastError();
  }
  const bool warp    = by_warps(a, n_sms, sizeof(T) == 2 && a.n_cols <= kWarpLong);
  const int per      = warp ? kThreads / 32 : 1;
  int segs           = warp ? 1 : segments(a.n_rows, a.n_cols, n_sms, false);
  const int64_t cols = part_cols(a.n_cols, segs);
  segs               = segs == 1 ? 1 : static_cast<int>((a.n_cols + cols - 1) / cols);
  const int64_t need = (a.n_rows + per - 1) / per;
  const int blocks   = static_cast<int>(need < 8 * n_sms ? need : 8 * n_sms);
  if (warp)
    loss_grad<T, 32><<<dim3(blocks, 1), kThreads, 0, s>>>(g, cols);
  else
    loss_grad<T, kThreads><<<dim3(blocks, segs), kThreads, 0, s>>>(g, cols);
  count_launches(1);
  return cudaGetLastError();
}

}  // namespace

size_t loss_workspace(const LossArgs& a, int n_sms)
{
  const int segs = segments(a.n_rows, a.n_cols, n_sms, true);  // (as many as either kind of tail takes)
  return 8 * n_sms * sizeof(double2) + (segs > 1 ? a.n_rows * segs * sizeof(float2) : 0);
}

cudaError_t launch_loss(int dtype, const LossArgs& a, const Reduced& out, void* workspace, int n_sms, cudaStream_t s)
{
  const bool rest = a.teacher.logsumexp != nullptr;
#define B2FIL_CASE(id, T) \
  case id: return rest ? run_loss<T, true>(a, out, workspace, n_sms, s) : run_loss<T, false>(a, out, workspace, n_sms, s);
  switch (dtype) {
    B2FIL_CASE(kF32, float)
    B2FIL_CASE(kBF16, __nv_bfloat16)
    B2FIL_CASE(kF16, __half)
  }
#undef B2FIL_CASE
  return cudaErrorInvalidValue;
}

cudaError_t launch_loss_grad(int dtype, const LossGradArgs& g, int n_sms, cudaStream_t s)
{
  switch (dtype) {
    case kF32: return run_grad<float>(g, n_sms, s);
    case kBF16: return run_grad<__nv_bfloat16>(g, n_sms, s);
    case kF16: return run_grad<__half>(g, n_sms, s);
  }
  return cudaErrorInvalidValue;
}

}  // namespace distill
}  // namespace b2fil
