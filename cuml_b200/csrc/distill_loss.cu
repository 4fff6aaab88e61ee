// T^2 KL(teacher || student) of rows of logits over the teacher's top classes, and its gradient.
//
// With q = softmax(z / T), p the teacher's probabilities of the classes that it names and, where the rest
// of its distribution is one more class, p_r and q_r what is left on either side:
//   loss  = T^2 [ sum_named p (log p - log q) + p_r (log p_r - log q_r) ]
//   dloss / dz_c = T (q_c - p_c) for named classes, T q_c (1 - p_r / q_r) for the others.
// Softmax cross entropy is the case of one named class of probability 1 and T = 1.
//
// Bound by memory: the forward pass reads the logits once (running maximum and sum), the backward pass
// reads them again and writes as much.  A row is visited by a warp (up to kWarpCols classes; eight rows
// per block, so that narrow rows fill the machine) or by a block; where rows are few, by several blocks
// whose maxima and sums are joined by the kernel that reads the teacher.
#include "distill_common.cuh"

namespace b2fil {
namespace distill {
namespace {

constexpr int kThreads  = 256;
constexpr int kWarpCols = 2048;   // widest rows that one warp visits
constexpr int kSegment  = 8192;   // fewest elements of a row that are worth a block of their own
constexpr int kMostSegs = 64;
constexpr int kInFlight = 4;

// Shared memory of one row: room for reductions, p, at and (REST) the bits of the named classes.
struct RowRoom {
  double* room;
  float* p;
  int* at;
  uint32_t* bits;
};
__host__ __device__ __forceinline__ size_t row_bytes(int k, int64_t bit_cols)
{
  const size_t bits = bit_cols ? ((bit_cols + 32) / 32 + 2) * 4 : 0;
  return (32 * 8 + static_cast<size_t>(k) * 8 + bits + 7) / 8 * 8;
}
__device__ __forceinline__ RowRoom room_of(char* base, int k)
{
  RowRoom r;
  r.room = reinterpret_cast<double*>(base);
  r.p    = reinterpret_cast<float*>(base + 256);
  r.at   = reinterpret_cast<int*>(r.p + k);
  r.bits = reinterpret_cast<uint32_t*>(r.at + k);
  return r;
}

// Running maximum and sum of n elements; with REST those whose bit is set are left out.  Bit 32 stands for
// the first element on a 16-byte boundary, so that a piece's bits lie in one word.
template <class T, bool REST>
__device__ __forceinline__ Running<float> visit_logits(const T* row, int64_t n, int tid, int threads, float c,
                                                       const uint32_t* bits)
{
  constexpr int N = Piece<T>::N;
  Running<float> r;
  const int lead = lead_of(row, n);
  visit_row<kInFlight>(
    row, n, tid, threads,
    [&](int64_t i, T x) {
      if (REST) {
        const uint32_t at = static_cast<uint32_t>(i - lead + 32);
        if (bits[at >> 5] >> (at & 31) & 1) return;
      }
      r.take(widen(x), c);
    },
    [&](int64_t i, const Piece<T>& v) {
      if (REST) {
        const uint32_t at  = static_cast<uint32_t>(i - lead + 32);
        const uint32_t set = bits[at >> 5] >> (at & 31) & ((1u << N) - 1);
        if (set) {
#pragma unroll
          for (int e = 0; e < N; ++e)
            if (!(set >> e & 1)) r.take(widen(v.v[e]), c);
          return;
        }
      }
      float x[N], most;
#pragma unroll
      for (int e = 0; e < N; ++e) x[e] = widen(v.v[e]);
      most = x[0];
#pragma unroll
      for (int e = 1; e < N; ++e) most = fmaxf(most, x[e]);
      if (most > r.m) r.raise(most, c);
      const float b = base_of(r.m);
#pragma unroll
      for (int e = 0; e < N; ++e) r.s += power((x[e] - b) * c);
    });
  return r;
}

template <int THREADS>
__device__ __forceinline__ void mark_named(const Teacher& t, int64_t row, int64_t n_cols, int64_t begin, int64_t n,
                                           int lead, int tid, uint32_t* bits)
{
  for (int w = tid; w < (n - lead + 32) / 32 + 1; w += THREADS) bits[w] = 0;
  sync_row<THREADS>();
  for (int j = tid; j < t.k; j += THREADS) {
    const int64_t c = teacher_index(t, row, j);
    if (c < begin || c >= begin + n || c >= n_cols || c == t.ignore) continue;
    const uint32_t at = static_cast<uint32_t>(c - begin - lead + 32);
    atomicOr(&bits[at >> 5], 1u << (at & 31));
  }
  sync_row<THREADS>();
}

// One part of a row per block: (row, segment) -> its maximum and sum.
template <class T, bool REST>
__global__ void __launch_bounds__(kThreads) loss_parts(LossArgs a, int64_t seg_cols, float2* parts)
{
  extern __shared__ __align__(16) char smem[];
  const RowRoom room  = room_of(smem, a.teacher.k);
  const int64_t begin = blockIdx.x * seg_cols;
  const int64_t n     = min(seg_cols, a.n_cols - begin);
  const float c       = 1.4426950408889634f / a.temperature;
  for (int64_t row = blockIdx.y; row < a.n_rows; row += gridDim.y) {
    const T* x = static_cast<const T*>(a.logits) + row * a.row_stride + begin;
    if (REST) {
      __syncthreads();
      mark_named<kThreads>(a.teacher, row, a.n_cols, begin, n, lead_of(x, n), threadIdx.x, room.bits);
    }
    Running<float> r = visit_logits<T, REST>(x, n, threadIdx.x, kThreads, c, room.bits);
    join_row<kThreads>(r, c, reinterpret_cast<float*>(room.room));
    if (threadIdx.x == 0) parts[row * gridDim.x + blockIdx.x] = make_float2(r.m, r.s);
  }
}

// Losses of rows; THREADS threads per row.  segs > 0: maxima and sums come from `parts`.
template <class T, int THREADS, bool REST>
__global__ void __launch_bounds__(kThreads) loss_rows(LossArgs a, int segs, const float2* parts, size_t row_room,
                                                      double2* block_sums)
{
  extern __shared__ __align__(16) char smem[];
  constexpr int ROWS = kThreads / THREADS;
  const int slot = threadIdx.x / THREADS, tid = threadIdx.x % THREADS;
  const RowRoom room = room_of(smem + slot * row_room, a.teacher.k);
  const float c      = 1.4426950408889634f / a.temperature;
  const double inv_t = 1.0 / a.temperature;
  double sum = 0, count = 0;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + slot; row < a.n_rows;
       row += static_cast<int64_t>(gridDim.x) * ROWS) {
    const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
    const TeacherRow t =
      read_teacher<THREADS>(a.teacher, row, a.n_cols, inv_t, tid, room.p, room.at, room.room);
    Running<float> r;
    if (segs > 0) {
      for (int i = tid; i < segs; i += THREADS) r.join(parts[row * segs + i].x, parts[row * segs + i].y, c);
    } else {
      if (REST) mark_named<THREADS>(a.teacher, row, a.n_cols, 0, a.n_cols, lead_of(x, a.n_cols), tid, room.bits);
      r = visit_logits<T, REST>(x, a.n_cols, tid, THREADS, c, room.bits);
    }
    join_row<THREADS>(r, c, reinterpret_cast<float*>(room.room));
    const Running<float> others = r;
    if (REST) {
      Running<float> mine;
      for (int j = tid; j < a.teacher.k; j += THREADS)
        if (room.at[j] >= 0) mine.take(widen(x[room.at[j]]), c);
      join_row<THREADS>(mine, c, reinterpret_cast<float*>(room.room));
      r.join(mine.m, mine.s, c);
    }
    const double log_s = log(static_cast<double>(r.s));
    const bool counts  = t.counts && !(r.s == 0.f);  // (no class has a finite logit: no softmax)
    double loss        = 0;
    for (int j = tid; j < a.teacher.k; j += THREADS) {
      const int at  = room.at[j];
      const float p = room.p[j];
      if (at < 0 || p == 0.f) continue;
      const double log_p = t.merged ? log(static_cast<double>(p))
                                    : (a.teacher.values ? a.teacher.values[row * a.teacher.values_stride + j] * inv_t : 0.0) - t.log_norm;
      const double log_q = (static_cast<double>(widen(x[at])) - r.m) * inv_t - log_s;
      loss += p * (log_p - log_q);
    }
    loss         = sum_row<THREADS>(loss, room.room);
    float factor = 1.f;
    if (REST && t.rest != 0.0) {
      const double log_rest = (static_cast<double>(others.m) - r.m) * inv_t + log(static_cast<double>(others.s)) - log_s;
      loss += t.rest * (log(t.rest) - log_rest);
      factor = static_cast<float>(1.0 - t.rest / exp(log_rest));
    }
    if (!counts) loss = 0;
    loss *= static_cast<double>(a.temperature) * a.temperature;
    if (tid == 0) {
      a.row_loss[row]  = static_cast<float>(loss);
      a.row_stats[row] = make_float4(r.m, 1.f / r.s, factor, counts ? 1.f : 0.f);
      sum += loss;
      count += counts;
    }
  }
  // sums of the block's rows, in a fixed order
  __shared__ double2 sums[ROWS];
  if (tid == 0) sums[slot] = make_double2(sum, count);
  __syncthreads();
  if (threadIdx.x == 0) {
    double2 all = sums[0];
    for (int i = 1; i < ROWS; ++i) {
      all.x += sums[i].x;
      all.y += sums[i].y;
    }
    block_sums[blockIdx.x] = all;
  }
}

// Sum, or mean over the rows that count (0 if none does).
__global__ void __launch_bounds__(kThreads) reduce_loss(const double2* block_sums, int n, Reduced out)
{
  __shared__ double room[32];
  double sum = 0, count = 0;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    sum += block_sums[i].x;
    count += block_sums[i].y;
  }
  sum   = sum_row<kThreads>(sum, room);
  count = sum_row<kThreads>(count, room);
  if (threadIdx.x == 0) {
    const double f = out.reduction == 1 ? 1.0 : count > 0 ? 1.0 / count : 0.0;
    *out.loss      = static_cast<float>(count > 0 ? sum * f : 0.0);
    *out.factor    = static_cast<float>(f);
  }
}

// Gradient of a part of a row; blockIdx.y: the part.
template <class T, int THREADS, bool REST>
__global__ void __launch_bounds__(kThreads) loss_grad(LossGradArgs g, int64_t seg_cols, size_t row_room)
{
  extern __shared__ __align__(16) char smem[];
  constexpr int ROWS = kThreads / THREADS, N = Piece<T>::N;
  const LossArgs& a = g.fwd;
  const int slot = threadIdx.x / THREADS, tid = threadIdx.x % THREADS;
  const RowRoom room  = room_of(smem + slot * row_room, a.teacher.k);
  const float c       = 1.4426950408889634f / a.temperature;
  const double inv_t  = 1.0 / a.temperature;
  const int64_t begin = blockIdx.y * seg_cols;
  const int64_t n     = min(seg_cols, a.n_cols - begin);
  const float scale   = (g.factor ? *g.factor : 1.f) * a.temperature;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + slot; row < a.n_rows;
       row += static_cast<int64_t>(gridDim.x) * ROWS) {
    const T* x     = static_cast<const T*>(a.logits) + row * a.row_stride + begin;
    T* d           = static_cast<T*>(g.grad) + row * g.grad_stride + begin;
    const float4 s = a.row_stats[row];
    const float up = g.upstream[row * g.upstream_stride] * scale;
    const bool counts = s.w != 0.f;
    const TeacherRow t = read_teacher<THREADS>(a.teacher, row, a.n_cols, inv_t, tid, room.p, room.at, room.room);
    (void)t;
    // zero for rows that do not count, whatever their logits are
    const float base = base_of(s.x), f = s.y * up * (REST ? s.z : 1.f);
    auto one = [&](int64_t i, T v) { d[i] = narrow<T>(counts ? power((widen(v) - base) * c) * f : 0.f); };
    if (((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(d)) & 15) == 0) {
      visit_row<kInFlight>(x, n, tid, THREADS, one, [&](int64_t i, const Piece<T>& v) {
        Piece<T> w;
#pragma unroll
        for (int e = 0; e < N; ++e) w.v[e] = narrow<T>(counts ? power((widen(v.v[e]) - base) * c) * f : 0.f);
        *reinterpret_cast<uint4*>(d + i) = *reinterpret_cast<const uint4*>(&w);
      });
    } else {
      for (int64_t i = tid; i < n; i += THREADS) one(i, x[i]);
    }
    sync_row<THREADS>();
    if (counts) {
      for (int j = tid; j < a.teacher.k; j += THREADS) {
        const int64_t at = room.at[j] - begin;
        if (room.at[j] < 0 || at < 0 || at >= n) continue;
        d[at] = narrow<T>((power((widen(x[at]) - base) * c) * s.y - room.p[j]) * up);
      }
    }
  }
}

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

template <class K>
cudaError_t allow(K kernel, size_t bytes)
{
  return bytes <= 48 * 1024 ? cudaSuccess
                            : cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
}

template <class T, bool REST>
cudaError_t run_loss(const LossArgs& a, const Reduced& out, void* workspace, int n_sms, cudaStream_t s)
{
  int segs           = segments(a.n_rows, a.n_cols, n_sms);
  const int64_t cols = part_cols(a.n_cols, segs);
  segs               = segs == 1 ? 1 : static_cast<int>((a.n_cols + cols - 1) / cols);
  const bool warp    = a.n_cols <= kWarpCols;
  const int per      = warp ? kThreads / 32 : 1;
  const int64_t need = (a.n_rows + per - 1) / per;
  const int blocks   = static_cast<int>(need < 8 * n_sms ? need : 8 * n_sms);
  double2* sums      = static_cast<double2*>(workspace);
  float2* parts      = reinterpret_cast<float2*>(sums + 8 * n_sms);
  int launched       = 1;
  cudaError_t e      = cudaSuccess;
  if (segs > 1) {
    const size_t bytes = row_bytes(a.teacher.k, REST ? cols : 0);
    if ((e = allow(loss_parts<T, REST>, bytes)) != cudaSuccess) return e;
    loss_parts<T, REST><<<dim3(segs, static_cast<unsigned>(a.n_rows)), kThreads, bytes, s>>>(a, cols, parts);
    ++launched;
  }
  const size_t bytes = row_bytes(a.teacher.k, REST && segs == 1 ? a.n_cols : 0);
  if (a.n_rows == 0) {
    launched = 0;
  } else if (warp) {
    if ((e = allow(loss_rows<T, 32, REST>, per * bytes)) != cudaSuccess) return e;
    loss_rows<T, 32, REST><<<blocks, kThreads, per * bytes, s>>>(a, 0, nullptr, bytes, sums);
  } else {
    if ((e = allow(loss_rows<T, kThreads, REST>, bytes)) != cudaSuccess) return e;
    loss_rows<T, kThreads, REST><<<blocks, kThreads, bytes, s>>>(a, segs > 1 ? segs : 0, parts, bytes, sums);
  }
  if (out.reduction != 0) {
    reduce_loss<<<1, kThreads, 0, s>>>(sums, blocks, out);
    ++launched;
  }
  count_launches(launched);
  return cudaGetLastError();
}

template <class T, bool REST>
cudaError_t run_grad(const LossGradArgs& g, int n_sms, cudaStream_t s)
{
  const LossArgs& a  = g.fwd;
  const bool warp    = a.n_cols <= kWarpCols;
  const int per      = warp ? kThreads / 32 : 1;
  int segs           = warp ? 1 : segments(a.n_rows, a.n_cols, n_sms);
  const int64_t cols = part_cols(a.n_cols, segs);
  segs               = segs == 1 ? 1 : static_cast<int>((a.n_cols + cols - 1) / cols);
  const int64_t need = (a.n_rows + per - 1) / per;
  const int blocks   = static_cast<int>(need < 8 * n_sms ? need : 8 * n_sms);
  const size_t bytes = row_bytes(a.teacher.k, 0);
  cudaError_t e;
  if (warp) {
    if ((e = allow(loss_grad<T, 32, REST>, per * bytes)) != cudaSuccess) return e;
    loss_grad<T, 32, REST><<<dim3(blocks, 1), kThreads, per * bytes, s>>>(g, cols, bytes);
  } else {
    loss_grad<T, kThreads, REST><<<dim3(blocks, segs), kThreads, bytes, s>>>(g, cols, bytes);
  }
  count_launches(1);
  return cudaGetLastError();
}

}  // namespace

size_t loss_workspace(const LossArgs& a, int n_sms)
{
  const int segs = segments(a.n_rows, a.n_cols, n_sms);
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
  const bool rest = g.fwd.teacher.logsumexp != nullptr;
#define B2FIL_CASE(id, T) \
  case id: return rest ? run_grad<T, true>(g, n_sms, s) : run_grad<T, false>(g, n_sms, s);
  switch (dtype) {
    B2FIL_CASE(kF32, float)
    B2FIL_CASE(kBF16, __nv_bfloat16)
    B2FIL_CASE(kF16, __half)
  }
#undef B2FIL_CASE
  return cudaErrorInvalidValue;
}

}  // namespace distill
}  // namespace b2fil
