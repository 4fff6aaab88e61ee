// Log probability of each row's given class, the row's entropy and its best classes, from logits; and the gradient by the
// logits.  The formulas are in score_common.cuh.
//
// Bound by memory: the forward pass reads the logits once (maximum, sum and mean exponent in one pass), the backward
// pass reads them again and writes as much; rows that do not count are not read.
#include "score_common.cuh"

namespace b2fil {
namespace distill {
namespace {

constexpr int kThreads  = 256;
constexpr int kWarpCols = 2048;  // rows that belong to one warp
constexpr int kSegment  = 8192;  // fewest elements of a row that are worth a block of their own
constexpr int kMostSegs = 64;
constexpr int kInFlight = 4;     // pieces of a thread
// Rows for one thread each: classes, and rows per SM from which on.
constexpr int kTileCols   = 64;
constexpr int kTileLeast  = 32;
constexpr int kTileBlocks = 8;   // of an SM

// n elements of a row by THREADS threads, joined for all of them.
template <class T, int THREADS>
__device__ __forceinline__ Scored visit_ordinary(const T* row, int64_t n, int tid, float c, float* room)
{
  PairedStream<T> r;
  const float slack = kSlack / c;
  visit_row<kInFlight>(
    row, n, tid, THREADS, [&](int64_t, T x) { r.take(widen(x), c, slack); },
    [&](int64_t, const Piece<T>& v) { r.take(v, largest_of(v), c, slack); });
  Scored o = r.scored(c);
  join_scored<THREADS>(o, c, room);
  return o;
}
template <class T, int THREADS>
__device__ __noinline__ Scored visit_any(const T* row, int64_t n, int tid, float c, float* room)
{
  constexpr int N = Piece<T>::N;
  ScoredStream r;
  const float slack = kSlack / c;
  visit_row<kInFlight>(
    row, n, tid, THREADS,
    [&](int64_t, T x) {
      const float one[1] = {widen(x)};
      r.take(one, c, slack);
    },
    [&](int64_t, const Piece<T>& v) {
      float x[N];
#pragma unroll
      for (int e = 0; e < N; ++e) x[e] = widen(v.v[e]);
      r.take(x, c, slack);
    });
  join_scored<THREADS>(r, c, room);
  return r;
}
template <class T, int THREADS>
__device__ __forceinline__ Scored visit_scores(const T* row, int64_t n, int tid, float c, float* room)
{
  const Scored r = visit_ordinary<T, THREADS>(row, n, tid, c, room);
  return PairedStream<T>::usable(r.m, c) ? r : visit_any<T, THREADS>(row, n, tid, c, room);
}

// One part of a row per block: (row, segment) -> its m, s and u.
template <class T>
__global__ void __launch_bounds__(kThreads) score_parts(ScoreArgs a, int64_t seg_cols, float4* parts)
{
  __shared__ float room[3 * kThreads / 32];
  const int64_t begin = blockIdx.x * seg_cols;
  const int64_t n     = min(seg_cols, a.n_cols - begin);
  const float c       = a.temperature.c;
  for (int64_t row = blockIdx.y; row < a.n_rows; row += gridDim.y) {
    const T* x = static_cast<const T*>(a.logits) + row * a.row_stride + begin;
    const Scored r = visit_scores<T, kThreads>(x, n, threadIdx.x, c, room);
    if (threadIdx.x == 0) parts[row * gridDim.x + blockIdx.x] = make_float4(r.m, r.s, r.u, 0.f);
  }
}

// A row by THREADS threads.  segs > 0: its parts are joined (by a warp).
template <class T, int THREADS>
__global__ void __launch_bounds__(kThreads) score_rows(ScoreArgs a, int segs, const float4* parts)
{
  constexpr int ROWS = kThreads / THREADS;
  __shared__ float room[3 * kThreads / 32];
  const int slot = threadIdx.x / THREADS, tid = threadIdx.x % THREADS;
  const float c = a.temperature.c;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + slot; row < a.n_rows;
       row += static_cast<int64_t>(gridDim.x) * ROWS) {
    const T* x   = static_cast<const T*>(a.logits) + row * a.row_stride;
    const int at = target_of(a.target, row, a.n_cols);
    Scored r;
    if (at == -2) {  // not read
    } else if (segs > 0) {
      for (int i = tid; i < segs; i += THREADS) {
        const float4 p = parts[row * segs + i];
        r.join(p.x, p.y, p.z, c);
      }
      join_scored<THREADS>(r, c, room);
    } else {
      r = visit_scores<T, THREADS>(x, a.n_cols, tid, c, room);
    }
    if (tid == 0) finish_score(a.out, row, r, a.temperature.inverse, at, at >= 0 ? widen(x[at]) : 0.f);
  }
}

// A row per thread, from a tile in shared memory.
template <class T>
__global__ void __launch_bounds__(kTileRows, kTileBlocks) score_tiles(ScoreArgs a)
{
  extern __shared__ __align__(16) char smem[];
  T* tile        = reinterpret_cast<T*>(smem);
  const int cols = static_cast<int>(a.n_cols);
  const TileShape<T> shape(cols);
  const float c    = a.temperature.c;
  const bool whole = without_gaps<T>(a.logits, a.row_stride, cols);
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * kTileRows; first < a.n_rows;
       first += static_cast<int64_t>(gridDim.x) * kTileRows) {
    const int rows = static_cast<int>(min(static_cast<int64_t>(kTileRows), a.n_rows - first));
    __syncthreads();  // the last tile has been used
    load_tile(tile, shape, static_cast<const T*>(a.logits) + first * a.row_stride, a.row_stride, rows, whole);
    __syncthreads();
    if (threadIdx.x >= rows) continue;
    const T* x        = tile + threadIdx.x * shape.pitch;
    const int64_t row = first + threadIdx.x;
    const int at      = target_of(a.target, row, cols);
    Scored r;
    for (int i = 0; i < cols; ++i) r.m = fmaxf(r.m, widen(x[i]));
    const float base = base_of(r.m);
    for (int i = 0; i < cols; ++i) r.add(widen(x[i]), base, c);
    finish_score(a.out, row, r, a.temperature.inverse, at, at >= 0 ? widen(x[at]) : 0.f);
  }
}

// Its gradient.
template <class T>
__global__ void __launch_bounds__(kTileRows, kTileBlocks) grad_tiles(ScoreGradArgs g)
{
  extern __shared__ __align__(16) char smem[];
  T* tile            = reinterpret_cast<T*>(smem);
  const ScoreArgs& a = g.fwd;
  const int cols     = static_cast<int>(a.n_cols);
  const TileShape<T> shape(cols);
  const float c       = a.temperature.c, inv_t = static_cast<float>(a.temperature.inverse);
  const bool whole_in = without_gaps<T>(a.logits, a.row_stride, cols), whole_out = without_gaps<T>(g.grad, g.grad_stride, cols);
  const ScoreUpstream& up = g.upstream;
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * kTileRows; first < a.n_rows;
       first += static_cast<int64_t>(gridDim.x) * kTileRows) {
    const int rows = static_cast<int>(min(static_cast<int64_t>(kTileRows), a.n_rows - first));
    __syncthreads();  // the last tile has been stored
    load_tile(tile, shape, static_cast<const T*>(a.logits) + first * a.row_stride, a.row_stride, rows, whole_in);
    __syncthreads();
    if (threadIdx.x < rows) {
      T* x              = tile + threadIdx.x * shape.pitch;
      const int64_t row = first + threadIdx.x;
      const RowGrad r   = row_grad(a.out.kept[row], up.log_prob ? up.log_prob[row * up.log_prob_stride] * inv_t : 0.f,
                                   up.entropy ? up.entropy[row * up.entropy_stride] * inv_t : 0.f);
      for (int i = 0; i < cols; ++i) x[i] = narrow<T>(r.counts ? r(widen(x[i]), c) + (i == r.at ? r.add : 0.f) : 0.f);
    }
    __syncthreads();
    store_tile(static_cast<T*>(g.grad) + first * g.grad_stride, g.grad_stride, tile, shape, rows, whole_out);
  }
}

template <class T>
__device__ __forceinline__ void zero_row(T* row, int64_t n, int tid, int threads)
{
  constexpr int N   = Piece<T>::N;
  const int lead    = lead_of(row, n);
  const int64_t end = lead + (n - lead) / N * N;
  if (tid < lead) row[tid] = narrow<T>(0.f);
  for (int64_t i = lead + static_cast<int64_t>(tid) * N; i < end; i += static_cast<int64_t>(threads) * N)
    *reinterpret_cast<uint4*>(row + i) = make_uint4(0, 0, 0, 0);
  if (end + tid < n) row[end + tid] = narrow<T>(0.f);
}

// Gradient of a part of a row by THREADS threads; blockIdx.y: the part.
template <class T, int THREADS>
__global__ void __launch_bounds__(kThreads) score_grad(ScoreGradArgs g, int64_t seg_cols)
{
  constexpr int ROWS = kThreads / THREADS, N = Piece<T>::N;
  const ScoreArgs& a = g.fwd;
  const int slot = threadIdx.x / THREADS, tid = threadIdx.x % THREADS;
  const float c       = a.temperature.c, inv_t = static_cast<float>(a.temperature.inverse);
  const int64_t begin = blockIdx.y * seg_cols;
  const int64_t n     = min(seg_cols, a.n_cols - begin);
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + slot; row < a.n_rows;
       row += static_cast<int64_t>(gridDim.x) * ROWS) {
    const T* x = static_cast<const T*>(a.logits) + row * a.row_stride + begin;
    T* d       = static_cast<T*>(g.grad) + row * g.grad_stride + begin;
    const ScoreUpstream& up = g.upstream;
    const RowGrad r  = row_grad(a.out.kept[row], up.log_prob ? up.log_prob[row * up.log_prob_stride] * inv_t : 0.f,
                                up.entropy ? up.entropy[row * up.entropy_stride] * inv_t : 0.f);
    const int64_t at = r.at < 0 ? -1 : r.at - begin;
    if (!r.counts) {
      zero_row(d, n, tid, THREADS);
      continue;
    }
    auto one = [&](int64_t i, T v) { d[i] = narrow<T>(r(widen(v), c) + (i == at ? r.add : 0.f)); };
    if (((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(d)) & 15) == 0) {
      visit_row<kInFlight>(x, n, tid, THREADS, one, [&](int64_t i, const Piece<T>& v) {
        float y[N];
#pragma unroll
        for (int e = 0; e < N; ++e) y[e] = r(widen(v.v[e]), c);
        if (at >= i && at < i + N) {
#pragma unroll
          for (int e = 0; e < N; ++e) y[e] += at - i == e ? r.add : 0.f;
        }
        Piece<T> w;
#pragma unroll
        for (int e = 0; e < N; ++e) w.v[e] = narrow<T>(y[e]);
        *reinterpret_cast<uint4*>(d + i) = *reinterpret_cast<const uint4*>(&w);
      });
    } else {
      for (int64_t i = tid; i < n; i += THREADS) one(i, x[i]);
    }
  }
}

// Parts of a row where rows are few.
int segments(int64_t n_rows, int64_t n_cols, int n_sms)
{
  if (n_rows == 0 || n_cols <= kWarpCols || n_rows >= 2 * n_sms) return 1;
  const int64_t want = (4 * n_sms + n_rows - 1) / n_rows;
  const int64_t most = (n_cols + kSegment - 1) / kSegment;
  const int64_t segs = want < most ? want : most;
  return static_cast<int>(segs < 1 ? 1 : segs > kMostSegs ? kMostSegs : segs);
}
// length of a part: whole 128-byte lines of every type
int64_t part_cols(int64_t n_cols, int segs)
{
  return segs == 1 ? n_cols : ((n_cols + segs - 1) / segs + 63) / 64 * 64;
}
unsigned blocks_of(int64_t need, int64_t most) { return static_cast<unsigned>(need < most ? need : most); }

bool by_tiles(const ScoreArgs& a, int n_sms) { return a.n_cols <= kTileCols && a.n_rows >= static_cast<int64_t>(kTileLeast) * n_sms; }
template <class T, class A>
cudaError_t run_tiles(void (*kernel)(A), const A& args, const ScoreArgs& a, int n_sms, cudaStream_t s)
{
  const unsigned blocks = blocks_of((a.n_rows + kTileRows - 1) / kTileRows, static_cast<int64_t>(kTileBlocks) * n_sms);
  kernel<<<blocks, kTileRows, TileShape<T>(static_cast<int>(a.n_cols)).bytes(), s>>>(args);
  count_launches(1);
  return cudaGetLastError();
}

template <class T>
cudaError_t run_score(const ScoreArgs& a, void* workspace, int n_sms, cudaStream_t s)
{
  if (by_tiles(a, n_sms)) return run_tiles<T>(score_tiles<T>, a, a, n_sms, s);
  int segs           = segments(a.n_rows, a.n_cols, n_sms);
  const int64_t cols = part_cols(a.n_cols, segs);
  segs               = segs == 1 ? 1 : static_cast<int>((a.n_cols + cols - 1) / cols);
  float4* parts      = static_cast<float4*>(workspace);
  if (segs > 1) score_parts<T><<<dim3(segs, blocks_of(a.n_rows, 65535)), kThreads, 0, s>>>(a, cols, parts);
  const bool warp    = segs > 1 || a.n_cols <= kWarpCols;
  const int per      = warp ? kThreads / 32 : 1;
  const unsigned blocks = blocks_of((a.n_rows + per - 1) / per, 8ll * n_sms);
  if (warp)
    score_rows<T, 32><<<blocks, kThreads, 0, s>>>(a, segs > 1 ? segs : 0, parts);
  else
    score_rows<T, kThreads><<<blocks, kThreads, 0, s>>>(a, 0, parts);
  count_launches(segs > 1 ? 2 : 1);
  return cudaGetLastError();
}

template <class T>
cudaError_t run_grad(const ScoreGradArgs& g, int n_sms, cudaStream_t s)
{
  const ScoreArgs& a = g.fwd;
  if (by_tiles(a, n_sms)) return run_tiles<T>(grad_tiles<T>, g, a, n_sms, s);
  const bool warp    = a.n_cols <= kWarpCols;
  const int per      = warp ? kThreads / 32 : 1;
  int segs           = warp ? 1 : segments(a.n_rows, a.n_cols, n_sms);
  const int64_t cols = part_cols(a.n_cols, segs);
  segs               = segs == 1 ? 1 : static_cast<int>((a.n_cols + cols - 1) / cols);
  const unsigned blocks = blocks_of((a.n_rows + per - 1) / per, 8ll * n_sms);
  if (warp)
    score_grad<T, 32><<<blocks, kThreads, 0, s>>>(g, cols);
  else
    score_grad<T, kThreads><<<dim3(blocks, segs), kThreads, 0, s>>>(g, cols);
  count_launches(1);
  return cudaGetLastError();
}

}  // namespace

size_t score_workspace(int dtype, const ScoreArgs& a, int n_sms)
{
  if (a.k > 0) {
    TopArgs t{};
    t.n_rows = a.n_rows;
    t.n_cols = a.n_cols;
    t.k      = a.k;
    return top_workspace(dtype, t, n_sms);
  }
  const int segs = segments(a.n_rows, a.n_cols, n_sms);
  return segs > 1 ? a.n_rows * segs * sizeof(float4) : 0;
}

cudaError_t launch_score(int dtype, const ScoreArgs& a, void* workspace, int n_sms, cudaStream_t s)
{
  if (a.k > 0) return launch_scored_top(dtype, a, workspace, n_sms, s);
  switch (dtype) {
    case kF32: return run_score<float>(a, workspace, n_sms, s);
    case kBF16: return run_score<__nv_bfloat16>(a, workspace, n_sms, s);
    case kF16: return run_score<__half>(a, workspace, n_sms, s);
  }
  return cudaErrorInvalidValue;
}

cudaError_t launch_score_grad(int dtype, const ScoreGradArgs& g, int n_sms, cudaStream_t s)
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
