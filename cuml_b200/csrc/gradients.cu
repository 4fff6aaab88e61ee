// The norm of many tensors together, and the tensors scaled down to a largest norm.
//
//   norm = (sum x^2)^1/2, or sum |x|, or max |x|, over all elements of all tensors
//   x'   = x min(1, most / norm), in place or to tensors of other types; as they are where the norm is not finite
//
// Bound by memory: one pass for the norm, and one that scales (in place: only where the norm is above `most`), which
// takes the pieces in the opposite order, as the last are in L2.  The tensors' addresses are the kernels' parameters:
// nothing is copied to the device first, and a captured graph keeps them.  Squares of 32-bit numbers are added up in 32
// bits over the 16 bytes of a load and in 64 from there on; pieces whose sum leaves the safe range are taken in
// 64 bits.  Blocks' sums are joined in a fixed order.
#include "distill_common.cuh"

namespace b2fil {
namespace distill {
namespace {

constexpr int kThreads  = 256;
constexpr int kChunk    = 1 << 14;  // elements that a block takes at a time
constexpr int kInFlight = 4;        // pieces of a thread
constexpr int kBatch    = 512;      // tensors of a launch (24 KB of parameters)

// One tensor of a launch.  Strided ones: rows of cols elements; others are one row.
struct Part {
  const void* from;
  void* to;
  int64_t n;
};
struct Strides {
  int64_t cols, from_row, from_col, to_row, to_col;
};

template <int N, bool STRIDED>
struct Batch {
  Part part[N];
  int first[N + 1];  // chunk of the launch with which a tensor begins
  uint8_t from_type[N], to_type[N];
  Strides strides[STRIDED ? N : 1];
  int parts;
};

template <int N, bool S>
__device__ __forceinline__ int part_of(const Batch<N, S>& b, int chunk)
{
  int low = 0, high = b.parts - 1;  // the last one that begins at or before the chunk
  while (low < high) {
    const int mid = (low + high + 1) / 2;
    if (b.first[mid] <= chunk)
      low = mid;
    else
      high = mid - 1;
  }
  return low;
}

enum { kLargest = 0, kSum = 1, kSquares = 2 };

// A thread's part of the norm.
template <int KIND>
struct Norm {
  double sum = 0;
  float top  = 0.f;
  template <int E>
  __device__ __forceinline__ void take(const float (&x)[E])
  {
    if (KIND == kLargest) {
#pragma unroll
      for (int e = 0; e < E; ++e) asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(fabsf(x[e])));
      return;
    }
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = KIND == kSum ? s + fabsf(x[e]) : fmaf(x[e], x[e], s);
    // (squares of numbers below 2^-50 or so lose bits, those above 2^60 may overflow; all zero is neither)
    if (KIND == kSquares ? !(s > 0x1p-90f && s < 0x1p120f) : !(s < 0x1p120f)) {
      double d = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) d += KIND == kSum ? fabs(static_cast<double>(x[e])) : static_cast<double>(x[e]) * x[e];
      sum += d;
    } else {
      sum += s;
    }
  }
  __device__ __forceinline__ double value() const { return KIND == kLargest ? static_cast<double>(top) : sum; }
};
template <int KIND>
__device__ __forceinline__ double joined(double a, double b)
{
  return KIND == kLargest ? (a != a || b != b ? NAN : fmax(a, b)) : a + b;
}
// Of all threads of a block, for all of them.
template <int KIND>
__device__ __forceinline__ double join_block(double x, double* room)
{
#pragma unroll
  for (int d = 16; d; d >>= 1) x = joined<KIND>(x, __shfl_xor_sync(~0u, x, d));
  __syncthreads();
  if (threadIdx.x % 32 == 0) room[threadIdx.x / 32] = x;
  __syncthreads();
  x = room[0];
  for (int i = 1; i < kThreads / 32; ++i) x = joined<KIND>(x, room[i]);
  return x;
}

template <class T, int KIND>
__device__ __forceinline__ void norm_row(const T* x, int64_t n, Norm<KIND>& r)
{
  constexpr int N = Piece<T>::N;
  visit_row<kInFlight>(
    x, n, threadIdx.x, kThreads,
    [&](int64_t, T v) {
      const float one[1] = {widen(v)};
      r.take(one);
    },
    [&](int64_t, const Piece<T>& p) {
      float v[N];
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = widen(p.v[e]);
      r.take(v);
    });
}
__device__ __forceinline__ float element(const void* from, int type, int64_t i)
{
  return type == kF32 ? static_cast<const float*>(from)[i]
         : type == kBF16 ? widen(static_cast<const __nv_bfloat16*>(from)[i]) : widen(static_cast<const __half*>(from)[i]);
}
__device__ __forceinline__ void put_element(void* to, int type, int64_t i, float x)
{
  if (type == kF32)
    static_cast<float*>(to)[i] = x;
  else if (type == kBF16)
    static_cast<__nv_bfloat16*>(to)[i] = narrow<__nv_bfloat16>(x);
  else
    static_cast<__half*>(to)[i] = narrow<__half>(x);
}

// One chunk's part of the norm.
template <int KIND, int N, bool STRIDED>
__device__ __forceinline__ void norm_chunk(const Batch<N, STRIDED>& b, int chunk, Norm<KIND>& r)
{
  const int p         = part_of(b, chunk);
  const int64_t begin = static_cast<int64_t>(chunk - b.first[p]) * kChunk, n = min(static_cast<int64_t>(kChunk), b.part[p].n - begin);
  const void* from    = b.part[p].from;
  const int type      = b.from_type[p];
  if constexpr (STRIDED) {
    const Strides& s = b.strides[p];
    for (int64_t i = begin + threadIdx.x; i < begin + n; i += kThreads) {
      const int64_t row  = i / s.cols;
      const float one[1] = {element(from, type, row * s.from_row + (i - row * s.cols) * s.from_col)};
      r.take(one);
    }
  } else if (type == kF32) {
    norm_row(static_cast<const float*>(from) + begin, n, r);
  } else if (type == kBF16) {
    norm_row(static_cast<const __nv_bfloat16*>(from) + begin, n, r);
  } else {
    norm_row(static_cast<const __half*>(from) + begin, n, r);
  }
}

// Norm and factor of all blocks' sums.
template <int KIND>
__device__ __forceinline__ float factor_of(double all, double most, float* norm)
{
  const double n = KIND == kSquares ? sqrt(all) : all;
  if (norm) *norm = static_cast<float>(n);
  return n > most && n < INFINITY ? static_cast<float>(most / n) : 1.f;
}

template <class T, class U>
__device__ __forceinline__ void scale_row(const T* x, U* y, int64_t n, float f)
{
  constexpr int N = Piece<T>::N;
  // whole pieces are stored 16 bytes at a time (or 8, of fewer) where the result lies on such a boundary
  const int lead = lead_of(x, n);
  if ((reinterpret_cast<uintptr_t>(y + lead) & 15) != 0) {
    for (int64_t i = threadIdx.x; i < n; i += kThreads) y[i] = narrow<U>(widen(x[i]) * f);
    return;
  }
  struct alignas(sizeof(U) * N < 16 ? sizeof(U) * N : 16) Out {
    U v[N];
  };
  // (not through the read-only path: x may be y)
  auto load = [&](int64_t p) {
    Piece<T> r;
    *reinterpret_cast<uint4*>(&r) = *reinterpret_cast<const uint4*>(x + lead + p * N);
    return r;
  };
  auto store = [&](int64_t p, const Piece<T>& v) {
    Out o;
#pragma unroll
    for (int e = 0; e < N; ++e) o.v[e] = narrow<U>(widen(v.v[e]) * f);
    *reinterpret_cast<Out*>(y + lead + p * N) = o;
  };
  const int pieces = static_cast<int>((n - lead) / N);
  int p            = threadIdx.x;
  for (; p + (kInFlight - 1) * kThreads < pieces; p += kInFlight * kThreads) {
    Piece<T> r[kInFlight];
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) r[u] = load(p + u * kThreads);
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) store(p + u * kThreads, r[u]);
  }
  for (; p < pieces; p += kThreads) store(p, load(p));
  const int64_t last = lead + static_cast<int64_t>(pieces) * N + threadIdx.x;
  if (threadIdx.x < lead) y[threadIdx.x] = narrow<U>(widen(x[threadIdx.x]) * f);
  if (last < n) y[last] = narrow<U>(widen(x[last]) * f);
}
template <class T>
__device__ __forceinline__ void scale_to(const T* x, void* to, int type, int64_t begin, int64_t n, float f)
{
  if (type == kF32)
    scale_row(x + begin, static_cast<float*>(to) + begin, n, f);
  else if (type == kBF16)
    scale_row(x + begin, static_cast<__nv_bfloat16*>(to) + begin, n, f);
  else
    scale_row(x + begin, static_cast<__half*>(to) + begin, n, f);
}
template <int N, bool STRIDED>
__device__ __forceinline__ void scale_chunk(const Batch<N, STRIDED>& b, int chunk, float f)
{
  const int p         = part_of(b, chunk);
  const int64_t begin = static_cast<int64_t>(chunk - b.first[p]) * kChunk, n = min(static_cast<int64_t>(kChunk), b.part[p].n - begin);
  const void* from    = b.part[p].from;
  void* to            = b.part[p].to;
  const int type      = b.from_type[p];
  if (f == 1.f && from == to) return;
  if constexpr (STRIDED) {
    const Strides& s = b.strides[p];
    for (int64_t i = begin + threadIdx.x; i < begin + n; i += kThreads) {
      const int64_t row = i / s.cols, col = i - row * s.cols;
      put_element(to, b.to_type[p], row * s.to_row + col * s.to_col, element(from, type, row * s.from_row + col * s.from_col) * f);
    }
  } else if (type == kF32) {
    scale_to(static_cast<const float*>(from), to, b.to_type[p], begin, n, f);
  } else if (type == kBF16) {
    scale_to(static_cast<const __nv_bfloat16*>(from), to, b.to_type[p], begin, n, f);
  } else {
    scale_to(static_cast<const __half*>(from), to, b.to_type[p], begin, n, f);
  }
}

// Sums of the blocks of one launch, to sums[blockIdx.x].
template <int KIND, int N, bool STRIDED>
__global__ void __launch_bounds__(kThreads) norm_parts(const __grid_constant__ Batch<N, STRIDED> b, double* sums)
{
  __shared__ double room[kThreads / 32];
  Norm<KIND> r;
  const int chunks = b.first[b.parts];
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) norm_chunk(b, c, r);
  const double all = join_block<KIND>(r.value(), room);
  if (threadIdx.x == 0) sums[blockIdx.x] = all;
}

// Every block joins all launches' sums; the first one of the first launch writes the norm.
template <int KIND, int N, bool STRIDED>
__global__ void __launch_bounds__(kThreads) scale_parts(const __grid_constant__ Batch<N, STRIDED> b, const double* sums, int n_sums,
                                                        double most, float* norm)
{
  __shared__ double room[kThreads / 32];
  double x = 0;
  for (int i = threadIdx.x; i < n_sums; i += kThreads) x = joined<KIND>(x, sums[i]);
  const double all = join_block<KIND>(x, room);
  const bool first = blockIdx.x == 0 && threadIdx.x == 0;
  const float f    = factor_of<KIND>(all, most, first ? norm : nullptr);
  const int chunks = b.first[b.parts];
  // the last chunks first: they were read last
  for (int c = chunks - 1 - static_cast<int>(blockIdx.x); c >= 0; c -= gridDim.x) scale_chunk(b, c, f);
}

template <int KIND>
__global__ void __launch_bounds__(kThreads) join_sums(const double* sums, int n_sums, float* norm)
{
  __shared__ double room[kThreads / 32];
  double x = 0;
  for (int i = threadIdx.x; i < n_sums; i += kThreads) x = joined<KIND>(x, sums[i]);
  const double all = join_block<KIND>(x, room);
  if (threadIdx.x == 0) factor_of<KIND>(all, INFINITY, norm);
}

// How the tensors are cut into launches.
struct Plan {
  int64_t launches, sums;
};
int64_t chunks_of(const Gradient& g) { return (g.rows * g.cols + kChunk - 1) / kChunk; }
bool is_flat(const Gradient& g)
{
  auto dense = [&](int64_t row, int64_t col) { return (col == 1 || g.cols == 1) && (row == g.cols || g.rows == 1); };
  return dense(g.from_row, g.from_col) && (!g.to || dense(g.to_row, g.to_col));
}
int blocks_of(int64_t chunks, int n_sms)
{
  const int64_t most = 8ll * n_sms;
  return static_cast<int>(chunks < most ? chunks : most);
}

// Calls f(batch) for every launch's worth of tensors; sizes only where `fill` is false.
template <int N, bool STRIDED, class F>
cudaError_t each_batch(const Gradient* g, int64_t n, F f)
{
  Batch<N, STRIDED> b;
  b.parts    = 0;
  b.first[0] = 0;
  auto flush = [&]() {
    const cudaError_t e = b.parts ? f(b) : cudaSuccess;
    b.parts             = 0;
    b.first[0]          = 0;
    return e;
  };
  for (int64_t i = 0; i < n; ++i) {
    if (g[i].rows * g[i].cols == 0 || is_flat(g[i]) == STRIDED) continue;
    const int64_t chunks = chunks_of(g[i]);
    if (b.parts == N || (b.parts > 0 && b.first[b.parts] + chunks > INT32_MAX / 2)) {
      const cudaError_t e = flush();
      if (e != cudaSuccess) return e;
    }
    const int p      = b.parts++;
    b.part[p]        = Part{g[i].from, g[i].to, g[i].rows * g[i].cols};
    b.from_type[p]   = static_cast<uint8_t>(g[i].from_type);
    b.to_type[p]     = static_cast<uint8_t>(g[i].to_type);
    b.first[p + 1]   = static_cast<int>(b.first[p] + chunks);
    if (STRIDED) b.strides[p] = Strides{g[i].cols, g[i].from_row, g[i].from_col, g[i].to_row, g[i].to_col};
  }
  return flush();
}
constexpr int kStridedBatch = 256;

template <int KIND>
cudaError_t run_clip(const ClipArgs& a, double* sums, int n_sms, cudaStream_t s)
{
  int n_sums = 0, launched = 0;
  auto add = [&](auto& b) {
    using B = std::remove_reference_t<decltype(b)>;
    const int blocks = blocks_of(b.first[b.parts], n_sms);
    norm_parts<KIND><<<blocks, kThreads, 0, s>>>(static_cast<const B&>(b), sums + n_sums);
    n_sums += blocks;
    ++launched;
    return cudaGetLastError();
  };
  cudaError_t e = each_batch<kBatch, false>(a.gradients, a.n, add);
  if (e == cudaSuccess) e = each_batch<kStridedBatch, true>(a.gradients, a.n, add);
  if (e != cudaSuccess) return e;
  if (!a.scales || n_sums == 0) {
    join_sums<KIND><<<1, kThreads, 0, s>>>(sums, n_sums, a.norm);
    count_launches(launched + 1);
    return cudaGetLastError();
  }
  float* norm = a.norm;
  auto scale  = [&](auto& b) {
    using B = std::remove_reference_t<decltype(b)>;
    scale_parts<KIND><<<blocks_of(b.first[b.parts], n_sms), kThreads, 0, s>>>(static_cast<const B&>(b), sums, n_sums, a.most, norm);
    norm = nullptr;
    ++launched;
    return cudaGetLastError();
  };
  e = each_batch<kBatch, false>(a.gradients, a.n, scale);
  if (e == cudaSuccess) e = each_batch<kStridedBatch, true>(a.gradients, a.n, scale);
  count_launches(launched);
  return e;
}

}  // namespace

size_t clip_workspace(const ClipArgs& a, int n_sms)
{
  // a launch's blocks, counted as if every launch had as many as there can be
  const int64_t most = a.n / kBatch + a.n / kStridedBatch + 2;
  int64_t chunks     = 0;  // (launches end, too, where their chunks are many)
  for (int64_t i = 0; i < a.n; ++i) chunks += chunks_of(a.gradients[i]);
  return (most + 2 * (chunks / (INT32_MAX / 4))) * 8 * n_sms * sizeof(double);
}

cudaError_t launch_clip(const ClipArgs& a, void* workspace, int n_sms, cudaStream_t s)
{
  double* sums = static_cast<double*>(workspace);
  switch (a.kind) {
    case kLargest: return run_clip<kLargest>(a, sums, n_sms, s);
    case kSum: return run_clip<kSum>(a, sums, n_sms, s);
    case kSquares: return run_clip<kSquares>(a, sums, n_sms, s);
  }
  return cudaErrorInvalidValue;
}

}  // namespace distill
}  // namespace b2fil
