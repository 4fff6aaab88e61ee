// The norm of many tensors together, and the tensors scaled down to a largest norm.
//
//   norm = (sum x^2)^1/2, or sum |x|, or max |x|, over all elements of all tensors
//   x'   = x min(1, most / norm), in place or to tensors of other types; as they are where the norm is not finite
//
// Bound by memory: one pass for the norm, and one that scales (in place: only where the norm is above `most`).  The blocks
// take chunks in turn, and in the second pass backwards, as what was read last is in L2.  (1.1 billion bf16: 323 us for the norm and
// 676 to scale to bf16, 6.7 and 6.4 TB/s.)  Few gradients are one cluster's, which does both in one launch.  The tensors' addresses are the kernels'
// parameters: nothing is copied to the device first, and a captured graph keeps them.  Squares of 32-bit numbers
// are added up in 32 bits over the 16 bytes of a load and in 64 from there on; pieces whose sum leaves the safe range are taken
// in 64 bits.  Blocks' sums are joined in a fixed order.
#include <cooperative_groups.h>

#include <algorithm>

#include "score_common.cuh"

namespace b2fil {
namespace distill {
namespace {

constexpr int kThreads   = 256;
constexpr int kUnit      = 2048;  // elements
constexpr int kMostChunk = 8;     // units of a chunk
constexpr int kInFlight  = 4;     // pieces of a thread
constexpr int kBlocks    = 6;     // of an SM, all there at once
constexpr int kCluster   = 8;     // blocks that do everything for few gradients
constexpr int64_t kFewUnits = 32;  // (65,536 fp32 in place, not above: 6.9 us; 110,000 8.4, by two launches 6.5 and the time between them)
constexpr int kBatch     = 512;   // tensors of a launch (15 KB of parameters)
constexpr int kFewParts  = 32;    // ... of one with fewer parameters to bring over
constexpr int kStridedBatch = 256;

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
  int first[N + 1];  // unit of the launch with which a tensor begins
  uint8_t from_type[N], to_type[N];
  Strides strides[STRIDED ? N : 1];
  int parts;
  int chunk;  // units that a block takes at a time
};

template <int N, bool S>
__device__ __forceinline__ int part_of(const Batch<N, S>& b, int unit)
{
  int low = 0, high = b.parts - 1;  // the last one that begins at or before the unit
  while (low < high) {
    const int mid = (low + high + 1) / 2;
    if (b.first[mid] <= unit)
      low = mid;
    else
      high = mid - 1;
  }
  return low;
}
// Visits the elements of a chunk: f(tensor, first element, elements).
template <int N, bool S, class F>
__device__ __forceinline__ void visit_chunk(const Batch<N, S>& b, int chunk, F f)
{
  int unit      = chunk * b.chunk;
  const int end = min(unit + b.chunk, b.first[b.parts]);
  for (int p = part_of(b, unit); unit < end; ++p) {
    const int64_t begin = static_cast<int64_t>(unit - b.first[p]) * kUnit;
    const int next      = min(end, b.first[p + 1]);
    f(p, begin, static_cast<int>(min(static_cast<int64_t>(next - unit) * kUnit, b.part[p].n - begin)));
    unit = next;
  }
}
template <int N, bool S>
__device__ __forceinline__ int chunks_of(const Batch<N, S>& b)
{
  return (b.first[b.parts] + b.chunk - 1) / b.chunk;
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
    // (squares of numbers below 2^-50 or so lose bits, those above 2^60 may overflow; zeros do neither)
    if (KIND == kSquares ? !(s > 0x1p-90f && s < 0x1p120f) : !(s < 0x1p120f)) {
      if (KIND == kSquares) {
        uint32_t bits = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) bits |= __float_as_uint(x[e]);
        if ((bits & 0x7fffffffu) == 0) return;
      }
      double d = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) d += KIND == kSum ? fabs(static_cast<double>(x[e])) : static_cast<double>(x[e]) * x[e];
      sum += d;
    } else {
      sum += s;
    }
  }
  __device__ __forceinline__ void take(const Norm& o)
  {
    sum += o.sum;
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(o.top));
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

// 16 bytes: of memory that this launch does not write, or of any.
template <bool READ_ONLY>
__device__ __forceinline__ uint4 load_words(const uint4* from)
{
  return READ_ONLY ? __ldg(from) : *from;
}

// (a function of its own, called once per tensor of a chunk: inlined for all types it spilled registers)
template <class T, int KIND, bool READ_ONLY>
__device__ __noinline__ Norm<KIND> norm_row(const T* x, int n)
{
  constexpr int N  = Piece<T>::N;
  const int lead   = lead_of(x, n), pieces = (n - lead) / N, last = lead + pieces * N + threadIdx.x;
  const uint4* from = reinterpret_cast<const uint4*>(x + lead);
  Norm<KIND> r;
  auto take = [&](const uint4& w) {
    float v[N];
    numbers_of(piece_of<T>(w), v);
    r.take(v);
  };
  float two[2] = {0.f, 0.f};
  if (threadIdx.x < lead) two[0] = widen(x[threadIdx.x]);
  if (last < n) two[1] = widen(x[last]);
  int p = threadIdx.x;
  for (; p + (kInFlight - 1) * kThreads < pieces; p += kInFlight * kThreads) {
    uint4 w[kInFlight];
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) w[u] = load_words<READ_ONLY>(from + p + u * kThreads);
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) take(w[u]);
  }
  if (p < pieces) {  // (at most kInFlight - 1, in flight together)
    uint4 w[kInFlight - 1];
#pragma unroll
    for (int u = 0; u < kInFlight - 1; ++u) w[u] = p + u * kThreads < pieces ? load_words<READ_ONLY>(from + p + u * kThreads) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int u = 0; u < kInFlight - 1; ++u)
      if (p + u * kThreads < pieces) take(w[u]);
  }
  r.take(two);
  return r;
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

// The norm's part of a block's chunks.  READ_ONLY: this launch does not write the tensors.
template <int KIND, bool READ_ONLY, int N, bool STRIDED>
__device__ __forceinline__ void norm_chunks(const Batch<N, STRIDED>& b, Norm<KIND>& r)
{
  const int chunks = chunks_of(b);
  for (int c = blockIdx.x; c < chunks; c += gridDim.x)
    visit_chunk(b, c, [&](int p, int64_t begin, int n) {
      const void* from = b.part[p].from;
      const int type   = b.from_type[p];
      if constexpr (STRIDED) {
        const Strides& s = b.strides[p];
        for (int64_t i = begin + threadIdx.x; i < begin + n; i += kThreads) {
          const int64_t row  = i / s.cols;
          const float one[1] = {element(from, type, row * s.from_row + (i - row * s.cols) * s.from_col)};
          r.take(one);
        }
      } else if (type == kF32) {
        r.take(norm_row<float, KIND, READ_ONLY>(static_cast<const float*>(from) + begin, n));
      } else if (type == kBF16) {
        r.take(norm_row<__nv_bfloat16, KIND, READ_ONLY>(static_cast<const __nv_bfloat16*>(from) + begin, n));
      } else {
        r.take(norm_row<__half, KIND, READ_ONLY>(static_cast<const __half*>(from) + begin, n));
      }
    });
}

// Norm and factor of all blocks' sums.
template <int KIND>
__device__ __forceinline__ float factor_of(double all, double most, float* norm)
{
  const double n     = KIND == kSquares ? sqrt(all) : all;
  const float answer = static_cast<float>(n);
  if (norm) *norm = answer;
  return n > most && answer < INFINITY ? static_cast<float>(most / n) : 1.f;
}

// E elements of a type at a time: 16 bytes, or 8.
template <class T, int E>
struct Some {
  using Word = std::conditional_t<sizeof(T) * E == 16, uint4, uint2>;
  T v[E];
  static __device__ __forceinline__ Some at(const T* from)  // (not through the read-only path: it may be written meanwhile)
  {
    const Word w = *reinterpret_cast<const Word*>(from);
    Some r;
    memcpy(r.v, &w, sizeof w);
    return r;
  }
  __device__ __forceinline__ void put(T* to) const
  {
    Word w;
    memcpy(&w, v, sizeof w);
    *reinterpret_cast<Word*>(to) = w;
  }
};
// The wider type's elements are taken 16 bytes at a time, so that a warp's loads and stores leave no gaps.
template <class T, class U>
__device__ __noinline__ void scale_row(const T* x, U* y, int n, float f)
{
  constexpr int W = sizeof(T) > sizeof(U) ? sizeof(T) : sizeof(U), E = 16 / W, F = kInFlight;
  const int mis  = sizeof(T) == W ? (reinterpret_cast<uintptr_t>(x) & 15) / W : (reinterpret_cast<uintptr_t>(y) & 15) / W;
  const int lead = min(n, mis ? E - mis : 0);
  if ((reinterpret_cast<uintptr_t>(x + lead) & (sizeof(T) * E - 1)) != 0 || (reinterpret_cast<uintptr_t>(y + lead) & (sizeof(U) * E - 1)) != 0) {
    for (int i = threadIdx.x; i < n; i += kThreads) y[i] = narrow<U>(widen(x[i]) * f);
    return;
  }
  const int pieces = (n - lead) / E, last = lead + pieces * E + threadIdx.x;
  const T* from    = x + lead;
  U* to            = y + lead;
  auto scaled      = [&](const Some<T, E>& a) {
    Some<U, E> b;
#pragma unroll
    for (int e = 0; e < E; ++e) b.v[e] = narrow<U>(widen(a.v[e]) * f);
    return b;
  };
  int p = threadIdx.x;
  for (; p + (F - 1) * kThreads < pieces; p += F * kThreads) {
    Some<T, E> r[F];
#pragma unroll
    for (int u = 0; u < F; ++u) r[u] = Some<T, E>::at(from + (p + u * kThreads) * E);
#pragma unroll
    for (int u = 0; u < F; ++u) scaled(r[u]).put(to + (p + u * kThreads) * E);
  }
  for (; p < pieces; p += kThreads) scaled(Some<T, E>::at(from + p * E)).put(to + p * E);
  if (threadIdx.x < lead) y[threadIdx.x] = narrow<U>(widen(x[threadIdx.x]) * f);
  if (last < n) y[last] = narrow<U>(widen(x[last]) * f);
}
template <class T>
__device__ __forceinline__ void scale_to(const T* x, void* to, int type, int64_t begin, int n, float f)
{
  if (type == kF32)
    scale_row(x + begin, static_cast<float*>(to) + begin, n, f);
  else if (type == kBF16)
    scale_row(x + begin, static_cast<__nv_bfloat16*>(to) + begin, n, f);
  else
    scale_row(x + begin, static_cast<__half*>(to) + begin, n, f);
}
template <int N, bool STRIDED>
__device__ __forceinline__ void scale_chunks(const Batch<N, STRIDED>& b, float f)
{
  const int chunks = chunks_of(b), last = (chunks - 1) / static_cast<int>(gridDim.x) * static_cast<int>(gridDim.x) + static_cast<int>(blockIdx.x);
  for (int c = last; c >= 0; c -= gridDim.x) {
    if (c >= chunks) continue;
    visit_chunk(b, c, [&](int p, int64_t begin, int n) {
      const void* from = b.part[p].from;
      void* to         = b.part[p].to;
      const int type   = b.from_type[p];
      if (f == 1.f && from == to) return;  // as it is
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
    });
  }
}

// Sums of the blocks of one launch, to sums[blockIdx.x].
template <int KIND, int N, bool STRIDED>
__global__ void __launch_bounds__(kThreads, kBlocks) norm_parts(const __grid_constant__ Batch<N, STRIDED> b, double* sums)
{
  __shared__ double room[kThreads / 32];
  Norm<KIND> r;
  norm_chunks<KIND, true>(b, r);
  const double all = join_block<KIND>(r.value(), room);
  if (threadIdx.x == 0) sums[blockIdx.x] = all;
}

// Every block joins all launches' sums; the first one of the first launch writes the norm.
template <int KIND, int N, bool STRIDED>
__global__ void __launch_bounds__(kThreads, kBlocks) scale_parts(const __grid_constant__ Batch<N, STRIDED> b, const double* sums, int n_sums,
                                                        double most, float* norm)
{
  __shared__ double room[kThreads / 32];
  double x = 0;
  for (int i = threadIdx.x; i < n_sums; i += kThreads) x = joined<KIND>(x, sums[i]);
  const double all = join_block<KIND>(x, room);
  const bool first = blockIdx.x == 0 && threadIdx.x == 0;
  const float f    = factor_of<KIND>(all, most, first ? norm : nullptr);
  scale_chunks(b, f);
}

// Everything by one cluster.
template <int KIND, int N>
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kThreads) clip_few(const __grid_constant__ Batch<N, false> b, bool scales,
                                                                                     double most, float* norm)
{
  namespace cg = cooperative_groups;
  __shared__ double room[kThreads / 32], mine;
  Norm<KIND> r;
  norm_chunks<KIND, false>(b, r);
  double all = join_block<KIND>(r.value(), room);
  if (threadIdx.x == 0) mine = all;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  all = 0;
  for (int i = 0; i < kCluster; ++i) all = joined<KIND>(all, *cluster.map_shared_rank(&mine, i));
  cluster.sync();  // the others' sums have been read
  const bool first = blockIdx.x == 0 && threadIdx.x == 0;
  const float f    = factor_of<KIND>(all, most, first ? norm : nullptr);
  if (scales) scale_chunks(b, f);
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

int64_t units_of(const Gradient& g) { return (g.rows * g.cols + kUnit - 1) / kUnit; }
bool is_flat(const Gradient& g)
{
  auto dense = [&](int64_t row, int64_t col) { return (col == 1 || g.cols == 1) && (row == g.cols || g.rows == 1); };
  return dense(g.from_row, g.from_col) && (!g.to || dense(g.to_row, g.to_col));
}
template <class B>
int blocks_of(const B& b, int n_sms)
{
  return std::min((b.first[b.parts] + b.chunk - 1) / b.chunk, kBlocks * n_sms);
}

// Calls f(batch) for every launch's worth of flat or of strided tensors; at_once: blocks.
template <int N, bool STRIDED, class F>
cudaError_t each_batch(const Gradient* g, int64_t n, int64_t at_once, F f)
{
  Batch<N, STRIDED> b;
  b.parts    = 0;
  b.first[0] = 0;
  auto flush = [&]() {
    const int64_t units = b.first[b.parts];  // (few: a chunk for each block)
    b.chunk             = units <= kFewUnits ? static_cast<int>((units + kCluster - 1) / kCluster)
                                             : std::max<int64_t>(1, std::min<int64_t>(kMostChunk, units / (4 * at_once)));
    const cudaError_t e = b.parts ? f(b) : cudaSuccess;
    b.parts             = 0;
    b.first[0]          = 0;
    return e;
  };
  for (int64_t i = 0; i < n; ++i) {
    if (g[i].rows * g[i].cols == 0 || is_flat(g[i]) == STRIDED) continue;
    const int64_t units = units_of(g[i]);
    if (b.parts == N || (b.parts > 0 && b.first[b.parts] + units > INT32_MAX / 2)) {
      const cudaError_t e = flush();
      if (e != cudaSuccess) return e;
    }
    const int p      = b.parts++;
    b.part[p]        = Part{g[i].from, g[i].to, g[i].rows * g[i].cols};
    b.from_type[p]   = static_cast<uint8_t>(g[i].from_type);
    b.to_type[p]     = static_cast<uint8_t>(g[i].to_type);
    b.first[p + 1]   = static_cast<int>(b.first[p] + units);
    if (STRIDED) b.strides[p] = Strides{g[i].cols, g[i].from_row, g[i].from_col, g[i].to_row, g[i].to_col};
  }
  return flush();
}

template <int KIND, int N>
cudaError_t run_few(const ClipArgs& a, cudaStream_t s)
{
  return each_batch<N, false>(a.gradients, a.n, kCluster, [&](const Batch<N, false>& b) {
    clip_few<KIND><<<kCluster, kThreads, 0, s>>>(b, a.scales, a.most, a.norm);
    count_launches(1);
    return cudaGetLastError();
  });
}

template <int KIND, int N>
cudaError_t run_clip(const ClipArgs& a, double* sums, int n_sms, cudaStream_t s)
{
  int n_sums = 0, launched = 0;
  auto add = [&](auto& b) {
    using B = std::remove_reference_t<decltype(b)>;
    const int blocks = blocks_of(b, n_sms);
    norm_parts<KIND><<<blocks, kThreads, 0, s>>>(static_cast<const B&>(b), sums + n_sums);
    n_sums += blocks;
    ++launched;
    return cudaGetLastError();
  };
  cudaError_t e = each_batch<N, false>(a.gradients, a.n, kBlocks * n_sms, add);
  if (e == cudaSuccess) e = each_batch<kStridedBatch, true>(a.gradients, a.n, kBlocks * n_sms, add);
  if (e != cudaSuccess) return e;
  if (!a.scales || n_sums == 0) {
    join_sums<KIND><<<1, kThreads, 0, s>>>(sums, n_sums, a.norm);
    count_launches(launched + 1);
    return cudaGetLastError();
  }
  float* norm = a.norm;
  auto scale  = [&](auto& b) {
    using B = std::remove_reference_t<decltype(b)>;
    scale_parts<KIND><<<blocks_of(b, n_sms), kThreads, 0, s>>>(static_cast<const B&>(b), sums, n_sums, a.most, norm);
    norm = nullptr;
    ++launched;
    return cudaGetLastError();
  };
  e = each_batch<N, false>(a.gradients, a.n, kBlocks * n_sms, scale);
  if (e == cudaSuccess) e = each_batch<kStridedBatch, true>(a.gradients, a.n, kBlocks * n_sms, scale);
  count_launches(launched);
  return e;
}

template <int KIND>
cudaError_t launch_kind(const ClipArgs& a, double* sums, int n_sms, cudaStream_t s)
{
  int64_t parts = 0, units = 0;
  bool flat     = true;
  for (int64_t i = 0; i < a.n; ++i) {
    const int64_t u = units_of(a.gradients[i]);
    parts += u > 0;
    units += u;
    flat &= u == 0 || is_flat(a.gradients[i]);
  }
  if (flat && parts > 0 && parts <= kBatch && units <= kFewUnits)
    return parts <= kFewParts ? run_few<KIND, kFewParts>(a, s) : run_few<KIND, kBatch>(a, s);
  return parts <= kFewParts ? run_clip<KIND, kFewParts>(a, sums, n_sms, s) : run_clip<KIND, kBatch>(a, sums, n_sms, s);
}

}  // namespace

size_t clip_workspace(const ClipArgs& a, int n_sms)
{
  // a launch's blocks, counted as if every launch had as many as there can be
  const int64_t most = a.n / kBatch + a.n / kStridedBatch + 3;
  int64_t units      = 0;  // (launches end, too, where their units are many)
  for (int64_t i = 0; i < a.n; ++i) units += units_of(a.gradients[i]);
  return (most + 2 * (units / (INT32_MAX / 4))) * kBlocks * n_sms * sizeof(double);
}

cudaError_t launch_clip(const ClipArgs& a, void* workspace, int n_sms, cudaStream_t s)
{
  double* sums = static_cast<double*>(workspace);
  switch (a.kind) {
    case kLargest: return launch_kind<kLargest>(a, sums, n_sms, s);
    case kSum: return launch_kind<kSum>(a, sums, n_sms, s);
    case kSquares: return launch_kind<kSquares>(a, sums, n_sms, s);
  }
  return cudaErrorInvalidValue;
}

}  // namespace distill
}  // namespace b2fil
