// Log probability of each row's given class, the row's entropy and its best classes, from logits; and the gradient by the
// logits.  The formulas are in score_common.cuh.
//
// Bound by memory: the forward pass reads the logits once (maximum, sum and mean exponent in one pass), the backward
// pass reads them again and writes as much.  Rows that do not count are not read, but where a thread has a row: a tile of rows is copied
// to shared memory as a whole.
#include <algorithm>

#include "score_common.cuh"

namespace b2fil {
namespace distill {
namespace {

constexpr int kThreads  = 256;
constexpr int kWarpCols = 2048;  // rows that belong to one warp
// ... or, up to kSubCols, to eight lanes of one.  (Both passes, us, by warps and by eight lanes: 200,000 x 100 fp32 59, 53 and 28, 27; 100,000 x
// 200 bf16 33, 31 and 19, 18; 60,000 x 500 bf16 31, 29 and 24, 20; x 1000 equal.)
constexpr int kSubCols    = 512;
constexpr int kSubThreads = 8;
constexpr int kSegment  = 8192;  // fewest elements of a row that are worth a block of their own
constexpr int kMostSegs = 64;
constexpr int kInFlight = 4;     // pieces of a thread
// Blocks of an SM, all there at once: of rows by blocks, rows by warps and gradients.  (4096 x 131,072 bf16, 164 us at memory's
// rate: the reading alone takes 186 us with four, 172 with five.)  Their rows lie next to one another at any time (60,000 x 1001 bf16,
// both passes: 41 and 44 us; 72 and 73 where a warp has 32 rows in a row).
constexpr int kRowBlocks  = 5;
constexpr int kWarpBlocks = 4;
constexpr int kGradBlocks = 4;
// Bytes of a row that is worth a block's start, and of one of the gradient's.  (us with a block for each row and with those that are there
// at once taking several: 4096 x 131,072 bf16 184 and 191, gradient 319 and 345; x 32,768 66 and 58, gradient 78 and 83; 4096 x 8192
// fp32 38 and 32.  Copies to shared memory ahead of the sums, the next row's among them, made the warps of a block drift apart:
// 191 and 66.)
constexpr int64_t kLongRow     = 1 << 17;
constexpr int64_t kLongGradRow = 1 << 16;
// Where there are kWarpLeast rows per SM, a warp takes longer ones, too: whose logits take up to kWarpBytes, and in the
// gradient, of 16 bits, up to kWarpLong.  (20,000 x 3000 bf16, both passes: 96 and 66 us by blocks, 34 and 43 so; the gradient of fp32: 72 and
// 77, 1200 x 3000 5.4 and 6.9, 4096 x 3000 15.1 and 13.8.)
constexpr int kWarpLeast = 8;
constexpr int kWarpBytes = 16384;
constexpr int kWarpLong  = 8192;
// Rows for one thread each: rows per SM from which on, and per SM and class, classes, bytes of a row; and of the gradient's, which writes the tile
// back, too.  A tile takes a time of its own by its classes, however few tiles there are.  (us of each pass by eight lanes and by threads:
// 1,000,000 x 10 fp32 93, 78 and 24, 25, x 48 95, 90 and 60, 85, x 64 94, 94 and 95, 147; 200,000 x 56 fp32 23, 19 and 19, 22, bf16 22, 18
// and 14, 19; 120,000 x 64 fp32 14, 12 and 17, 19; 40,000 x 33 fp32 8.6, 5.5 and 6.5, 6.8, x 64 7.7, 5.4 and 8.5, 9.4; 20,000 x 10 bf16 5.9,
// 4.5 and 4.1, 3.7, x 48 5.5, 4.1 and 5.5, 6.7; 5000 x 10 fp32 4.1, 3.1 and 4.0, 3.7, x 64 4.1, 3.0 and 7.0, 7.8.)
constexpr int kTileLeast    = 32;
constexpr int kTilePer      = 4;
constexpr int kTileCols     = 64;
constexpr int kTileBytes    = 224;
constexpr int kTileGradPer  = 12;
constexpr int kTileGradCols = 48;
constexpr int kTileBlocks = 8;   // of an SM

// n elements of a row by `threads` threads; the thread's part.
template <class T>
__device__ __forceinline__ Scored visit_ordinary(const T* row, int n, int tid, int threads, float c)
{
  PairedStream<T> r;
  const float slack = kSlack / c;
  visit_all<kInFlight>(
    row, n, tid, threads,
    [&](int i, T x, int k, T y) {
      constexpr float kFloor = Ordinary<T>::kFloor;
      r.take(i < 0 ? kFloor : widen(x), k < 0 ? kFloor : widen(y), c, slack);
    },
    [&](int, const Piece<T>& v) { r.take(v, largest_of(v), c, slack); });
  return r.scored(c);
}
// One part of a row per block: (row, segment) -> its m, s and u, nothing for rows that do not count.  (Asking for the class first costs a
// row's 0.5 us, of which the join gives back 0.3: 100 x 131,072 fp32, both kernels: 21.3 us with and 22.0 without reading such rows,
// where half of them are that 21.3 and 13.4.)
template <class T>
__global__ void __launch_bounds__(kThreads) score_parts(ScoreArgs a, int64_t seg_cols, float4* parts)
{
  __shared__ float room[3 * kThreads / 32];
  const int64_t begin = blockIdx.x * seg_cols;
  const int n         = static_cast<int>(min(seg_cols, a.n_cols - begin));
  const float c       = a.temperature.c;
  for (int64_t row = blockIdx.y; row < a.n_rows; row += gridDim.y) {
    if (target_of(a.target, row, a.n_cols) == -2) continue;  // not read
    const T* x = static_cast<const T*>(a.logits) + row * a.row_stride + begin;
    Scored r   = visit_ordinary(x, n, threadIdx.x, kThreads, c);
    join_scored<kThreads>(r, c, room);
    if (!PairedStream<T>::usable(r.m, c)) r = visit_any<T, kThreads, kInFlight>(x, n, threadIdx.x, c, room);
    if (threadIdx.x == 0) parts[row * gridDim.x + blockIdx.x] = make_float4(r.m, r.s, r.u, 0.f);
  }
}
// ... and a row's scores from them, by a warp.
template <class T>
__global__ void __launch_bounds__(kThreads) score_join(ScoreArgs a, int segs, const float4* parts)
{
  constexpr int ROWS = kThreads / 32;
  const int lane = threadIdx.x % 32;
  const float c  = a.temperature.c;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x / 32; row < a.n_rows; row += static_cast<int64_t>(gridDim.x) * ROWS) {
    const int at      = target_of(a.target, row, a.n_cols);
    const float given = at >= 0 ? widen(static_cast<const T*>(a.logits)[row * a.row_stride + at]) : 0.f;
    Scored r;
    for (int i = lane; i < segs && at != -2; i += 32) {
      const float4 p = parts[row * segs + i];
      r.join(p.x, p.y, p.z, c);
    }
    r.join_lanes(c);
    if (lane == 0) finish_score(a.out, row, r, a.temperature.inverse, at, given);
  }
}

// Rows by a block each.  What a row takes besides its logits is done for 32 of them at a time, a lane each: the given
// classes before, the scores behind.  The warps of a block go through the rows on their own.
template <class T>
__global__ void __launch_bounds__(kThreads, kRowBlocks) score_blocks(ScoreArgs a)
{
  constexpr int W = kThreads / 32;
  __shared__ float room[3 * W];
  __shared__ float parts[32 * W * 3];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const float c      = a.temperature.c;
  const int64_t step = gridDim.x;
  for (int64_t row0 = blockIdx.x; row0 < a.n_rows; row0 += 32 * step) {
    const int count = static_cast<int>(min(static_cast<int64_t>(32), (a.n_rows - row0 + step - 1) / step));
    auto logits     = [&](int j) { return static_cast<const T*>(a.logits) + (row0 + j * step) * a.row_stride; };
    const int at    = lane < count ? target_of(a.target, row0 + lane * step, a.n_cols) : -2;
    for (int j = 0; j < count; ++j) {
      if (__shfl_sync(~0u, at, j) == -2) continue;  // not read
      Scored r = visit_ordinary(logits(j), static_cast<int>(a.n_cols), threadIdx.x, kThreads, c);
      r.join_lanes(c);
      if (lane == 0) {
        float* p = parts + (j * W + warp) * 3;
        p[0]     = r.m;
        p[1]     = r.s;
        p[2]     = r.u;
      }
    }
    __syncthreads();
    Scored mine;  // of the lane's row
    if (at != -2) {
      for (int w = 0; w < W; ++w) {
        const float* p = parts + (lane * W + w) * 3;
        mine.join(p[0], p[1], p[2], c);
      }
    }
    for (unsigned again = __ballot_sync(~0u, at != -2 && !PairedStream<T>::usable(mine.m, c)); again; again &= again - 1) {
      const int j    = __ffs(again) - 1;
      const Scored r = visit_any<T, kThreads, kInFlight>(logits(j), a.n_cols, threadIdx.x, c, room);
      if (lane == j) mine = r;
    }
    if (lane < count && warp == 0)
      finish_score(a.out, row0 + lane * step, mine, a.temperature.inverse, at, at >= 0 ? widen(logits(lane)[at]) : 0.f);
    __syncthreads();  // `parts` has been read
  }
}

// The rows of a warp, which takes 32 / THREADS of them at a time, or of a block: those that are read at a time lie next to one
// another.  row(j): the j-th of 32.
template <int THREADS>
struct RowOrder {
  static constexpr int kAtOnce = THREADS < 32 ? 32 / THREADS : 1;
  static constexpr int kPer    = THREADS > 32 ? 1 : kThreads / 32;
  int64_t slot = static_cast<int64_t>(blockIdx.x) * kPer + (THREADS > 32 ? 0 : threadIdx.x / 32);
  static __device__ __forceinline__ int64_t slots() { return static_cast<int64_t>(gridDim.x) * kPer; }
  __device__ __forceinline__ int64_t row(int j) const { return (slot + j / kAtOnce * slots()) * kAtOnce + j % kAtOnce; }
  __device__ __forceinline__ void next() { slot += 32 / kAtOnce * slots(); }
};

// The same by a warp, or eight lanes, each.
template <class T, int THREADS>
__global__ void __launch_bounds__(kThreads, kWarpBlocks) score_rows(ScoreArgs a)
{
  const int tid = threadIdx.x % THREADS, lane = threadIdx.x % 32;
  const float c = a.temperature.c;
  using Order   = RowOrder<THREADS>;
  constexpr int kAtOnce = Order::kAtOnce;
  for (Order rows; rows.row(0) < a.n_rows; rows.next()) {
    auto logits  = [&](int j) { return static_cast<const T*>(a.logits) + rows.row(j) * a.row_stride; };
    const int at = rows.row(lane) < a.n_rows ? target_of(a.target, rows.row(lane), a.n_cols) : -2;
    Scored mine;  // of the lane's row
    for (int first = 0; first < 32 && rows.row(first) < a.n_rows; first += kAtOnce) {
      const int j       = first + (kAtOnce > 1 ? lane / THREADS : 0);
      const bool counts = __shfl_sync(~0u, at, j) != -2;  // (else not read)
      if (kAtOnce == 1 && !counts) continue;
      Scored r = visit_ordinary(logits(j), counts ? static_cast<int>(a.n_cols) : 0, tid, THREADS, c);
      __syncwarp();
      r.join_some<THREADS>(c);
      if (kAtOnce == 1) {
        if (lane == j) mine = r;
        continue;
      }
      // to the lanes whose rows they are
      const int from = lane % kAtOnce * THREADS;
      const float m = __shfl_sync(~0u, r.m, from), s = __shfl_sync(~0u, r.s, from), u = __shfl_sync(~0u, r.u, from);
      if (lane - lane % kAtOnce == first) {
        mine.m = m;
        mine.s = s;
        mine.u = u;
      }
    }
    for (unsigned again = __ballot_sync(~0u, at != -2 && !PairedStream<T>::usable(mine.m, c)); again; again &= again - 1) {
      const int j    = __ffs(again) - 1;
      const Scored r = visit_any<T, 32, kInFlight>(logits(j), a.n_cols, lane, c, nullptr);
      if (lane == j) mine = r;
    }
    if (rows.row(lane) < a.n_rows)
      finish_score(a.out, rows.row(lane), mine, a.temperature.inverse, at, at >= 0 ? widen(logits(lane)[at]) : 0.f);
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

// Gradient of a part (blockIdx.y) of rows by THREADS threads.  Rows' factors are made by a lane each, 32 at a time.
template <class T, int THREADS>
__global__ void __launch_bounds__(kThreads, kGradBlocks) score_grad(ScoreGradArgs g, int64_t seg_cols)
{
  constexpr int N    = Piece<T>::N;
  const ScoreArgs& a = g.fwd;
  const int tid = threadIdx.x % THREADS, lane = threadIdx.x % 32;
  using Order   = RowOrder<THREADS>;
  constexpr int kAtOnce = Order::kAtOnce;
  const float c       = a.temperature.c, inv_t = static_cast<float>(a.temperature.inverse);
  const int64_t begin = blockIdx.y * seg_cols;
  const int n         = static_cast<int>(min(seg_cols, a.n_cols - begin));
  const ScoreUpstream& up = g.upstream;
  for (Order rows; rows.row(0) < a.n_rows; rows.next()) {
    RowGrad mine{};
    if (rows.row(lane) < a.n_rows) {
      const int64_t row = rows.row(lane);
      mine = row_grad(a.out.kept[row], up.log_prob ? up.log_prob[row * up.log_prob_stride] * inv_t : 0.f,
                      up.entropy ? up.entropy[row * up.entropy_stride] * inv_t : 0.f);
      if (!mine.counts) mine.at = -2;
    }
    for (int first = 0; first < 32 && rows.row(first) < a.n_rows; first += kAtOnce) {
      const int j = first + (kAtOnce > 1 ? lane / THREADS : 0);
      RowGrad r;
      r.at   = __shfl_sync(~0u, mine.at, j);
      r.base = __shfl_sync(~0u, mine.base, j);
      r.A    = __shfl_sync(~0u, mine.A, j);
      r.B    = __shfl_sync(~0u, mine.B, j);
      r.add  = __shfl_sync(~0u, mine.add, j);
      if (kAtOnce > 1 && rows.row(j) >= a.n_rows) continue;
      const T* x = static_cast<const T*>(a.logits) + rows.row(j) * a.row_stride + begin;
      T* d       = static_cast<T*>(g.grad) + rows.row(j) * g.grad_stride + begin;
      if (r.at == -2) {
        zero_row(d, n, tid, THREADS);
        continue;
      }
      const int at = r.at >= begin && r.at - begin < n ? static_cast<int>(r.at - begin) : -1;
      auto one     = [&](int i, T v) { d[i] = narrow<T>(r(widen(v), c) + (i == at ? r.add : 0.f)); };
      if (((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(d)) & 15) == 0) {
        visit_all<kInFlight>(
          x, n, tid, THREADS,
          [&](int i, T v, int k, T w) {
            if (i >= 0) one(i, v);
            if (k >= 0) one(k, w);
          },
          [&](int i, const Piece<T>& v) {
            float y[N];
            grads_of(r, v, c, y);
            if (static_cast<unsigned>(at - i) < N) {
#pragma unroll
              for (int e = 0; e < N; ++e) y[e] += at - i == e ? r.add : 0.f;
            }
            Piece<T> w;
#pragma unroll
            for (int e = 0; e < N; ++e) w.v[e] = narrow<T>(y[e]);
            *reinterpret_cast<uint4*>(d + i) = words_of(w);
          });
      } else {
        for (int i = tid; i < n; i += THREADS) one(i, x[i]);
      }
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

bool by_warps(const ScoreArgs& a, int n_sms, bool longer)
{
  return a.n_cols <= kWarpCols || (longer && a.n_rows >= static_cast<int64_t>(kWarpLeast) * n_sms);
}
// Blocks of a launch: a block for each long row, else as many as are there at once.
unsigned row_blocks(const ScoreArgs& a, bool warp, int element, int64_t at_once, int64_t long_row)
{
  const int per = kThreads / (a.n_cols <= kSubCols ? kSubThreads : 32);
  if (warp) return blocks_of((a.n_rows + per - 1) / per, at_once);
  return blocks_of(a.n_rows, a.n_cols * element >= long_row ? 1 << 30 : at_once);
}
bool by_tiles(const ScoreArgs& a, int element, int n_sms)
{
  return a.n_cols <= kTileCols && a.n_cols * element <= kTileBytes && a.n_rows >= std::max<int64_t>(kTileLeast, kTilePer * a.n_cols) * n_sms;
}
bool grad_by_tiles(const ScoreArgs& a, int n_sms)
{
  return a.n_cols <= kTileGradCols && a.n_rows >= std::max<int64_t>(kTileLeast, kTileGradPer * a.n_cols) * n_sms;
}
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
  if (by_tiles(a, sizeof(T), n_sms)) return run_tiles<T>(score_tiles<T>, a, a, n_sms, s);
  int segs           = segments(a.n_rows, a.n_cols, n_sms);
  const int64_t cols = part_cols(a.n_cols, segs);
  segs               = segs == 1 ? 1 : static_cast<int>((a.n_cols + cols - 1) / cols);
  if (segs > 1) {
    float4* parts = static_cast<float4*>(workspace);
    score_parts<T><<<dim3(segs, blocks_of(a.n_rows, 65535)), kThreads, 0, s>>>(a, cols, parts);
    score_join<T><<<blocks_of((a.n_rows + kThreads / 32 - 1) / (kThreads / 32), 8ll * n_sms), kThreads, 0, s>>>(a, segs, parts);
    count_launches(2);
    return cudaGetLastError();
  }
  if (a.n_cols <= kSubCols)
    score_rows<T, kSubThreads><<<row_blocks(a, true, sizeof(T), kWarpBlocks * n_sms, kLongRow), kThreads, 0, s>>>(a);
  else if (by_warps(a, n_sms, a.n_cols * sizeof(T) <= kWarpBytes))
    score_rows<T, 32><<<row_blocks(a, true, sizeof(T), kWarpBlocks * n_sms, kLongRow), kThreads, 0, s>>>(a);
  else
    score_blocks<T><<<row_blocks(a, false, sizeof(T), kRowBlocks * n_sms, kLongRow), kThreads, 0, s>>>(a);
  count_launches(1);
  return cudaGetLastError();
}

template <class T>
cudaError_t run_grad(const ScoreGradArgs& g, int n_sms, cudaStream_t s)
{
  const ScoreArgs& a = g.fwd;
  if (grad_by_tiles(a, n_sms)) return run_tiles<T>(grad_tiles<T>, g, a, n_sms, s);
  const bool warp    = by_warps(a, n_sms, sizeof(T) == 2 && a.n_cols <= kWarpLong);
  const unsigned rows = row_blocks(a, warp, sizeof(T), kGradBlocks * n_sms, kLongGradRow);
  int segs           = warp ? 1 : segments(a.n_rows, a.n_cols, n_sms);
  const int64_t cols = part_cols(a.n_cols, segs);
  segs               = segs == 1 ? 1 : static_cast<int>((a.n_cols + cols - 1) / cols);
  if (a.n_cols <= kSubCols)
    score_grad<T, kSubThreads><<<rows, kThreads, 0, s>>>(g, cols);
  else if (warp)
    score_grad<T, 32><<<rows, kThreads, 0, s>>>(g, cols);
  else
    score_grad<T, kThreads><<<dim3(rows, segs), kThreads, 0, s>>>(g, cols);
  count_launches(1);
  return cudaGetLastError();
}

}  // namespace

size_t score_workspace(int dtype, const ScoreArgs& a, int n_sms)
{
  if (a.k > 0) {
    return scored_top_workspace(dtype, a, n_sms);
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
