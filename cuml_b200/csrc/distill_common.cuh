// Device code that the distillation kernels share: reading rows of any alignment in 16-byte pieces,
// running maximum and sum of a softmax, reductions over the threads of a row, the teacher's side.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "distill.hpp"

namespace b2fil {
namespace distill {

// element types of the C ABI
enum { kF32 = 0, kF64 = 1, kBF16 = 2, kF16 = 3 };

template <class T>
struct ValueOf {
  using type = float;
};
template <>
struct ValueOf<double> {
  using type = double;
};

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ double widen(double x) { return x; }
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float widen(__half x) { return __half2float(x); }

template <class T>
__device__ __forceinline__ T narrow(typename ValueOf<T>::type x);
template <>
__device__ __forceinline__ float narrow<float>(float x) { return x; }
template <>
__device__ __forceinline__ double narrow<double>(double x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half narrow<__half>(float x) { return __float2half_rn(x); }

// 16 bytes of elements
template <class T>
struct alignas(16) Piece {
  static constexpr int N = 16 / sizeof(T);
  T v[N];
};

template <class T>
__device__ __forceinline__ Piece<T> load_piece(const T* p)
{
  Piece<T> r;
  *reinterpret_cast<uint4*>(&r) = __ldg(reinterpret_cast<const uint4*>(p));
  return r;
}

// Elements before the first 16-byte boundary of a row of n elements.
template <class T>
__device__ __forceinline__ int lead_of(const T* p, int64_t n)
{
  const int mis  = static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
  const int lead = mis ? Piece<T>::N - mis : 0;
  return lead < n ? lead : static_cast<int>(n);
}

// Visits a row of n elements with `threads` threads: one(i, x) for the elements before the first
// and behind the last 16-byte boundary, many(i, piece) for whole pieces, in ascending order within a
// thread.  U pieces are in flight per thread.
template <int U, class T, class One, class Many>
__device__ __forceinline__ void visit_row(const T* row, int64_t n, int tid, int threads, One one, Many many)
{
  constexpr int N  = Piece<T>::N;
  const int lead   = lead_of(row, n);
  const int pieces = static_cast<int>((n - lead) / N);
  if (tid < lead) one(static_cast<int64_t>(tid), row[tid]);
  const T* body = row + lead;
  int p         = tid;
  for (; p + (U - 1) * threads < pieces; p += U * threads) {
    Piece<T> r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) r[u] = load_piece(body + static_cast<int64_t>(p + u * threads) * N);
#pragma unroll
    for (int u = 0; u < U; ++u) many(lead + static_cast<int64_t>(p + u * threads) * N, r[u]);
  }
  for (; p < pieces; p += threads) {
    const Piece<T> r = load_piece(body + static_cast<int64_t>(p) * N);
    many(lead + static_cast<int64_t>(p) * N, r);
  }
  const int64_t at = lead + static_cast<int64_t>(pieces) * N + tid;
  if (at < n) one(at, row[at]);
}

// ---- running maximum m and sum s of exp((x - m) / T), c = log2(e) / T ------------------------
// The difference is taken before the scale: the scaled lowest value of a type would be -inf.
__device__ __forceinline__ float power(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ double power(double x) { return exp2(x); }
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double larger(double a, double b) { return fmax(a, b); }
template <class V>
__device__ __forceinline__ V lowest()
{
  return -static_cast<V>(INFINITY);
}
// what is subtracted from values whose maximum is m: any finite number where there is none
template <class V>
__device__ __forceinline__ V base_of(V m)
{
  return m == lowest<V>() ? V(0) : m;
}

template <class V>
struct Running {
  V m = lowest<V>(), s = V(0);
  __device__ __forceinline__ void raise(V to, V c)  // to > m
  {
    s = m == lowest<V>() ? s : s * power((m - to) * c);
    m = to;
  }
  __device__ __forceinline__ void take(V x, V c)
  {
    if (x > m) raise(x, c);
    s += power((x - base_of(m)) * c);
  }
  __device__ __forceinline__ void join(V m2, V s2, V c)
  {
    const V to = larger(m, m2);
    const V b  = base_of(to);
    s          = (m == lowest<V>() ? s : s * power((m - b) * c)) + (m2 == lowest<V>() ? s2 : s2 * power((m2 - b) * c));
    m          = to;
  }
  __device__ __forceinline__ void join_lanes(V c)
  {
#pragma unroll
    for (int d = 16; d; d >>= 1) join(__shfl_xor_sync(~0u, m, d), __shfl_xor_sync(~0u, s, d), c);
  }
};

// ---- the threads of one row: a warp or a block -----------------------------------------------
template <int THREADS>
__device__ __forceinline__ void sync_row()
{
  if (THREADS == 32)
    __syncwarp();
  else
    __syncthreads();
}

// All threads of the row get the joined value; `room`: shared, THREADS / 32 values of 2 V for this row.
template <int THREADS, class V>
__device__ __forceinline__ void join_row(Running<V>& r, V c, V* room)
{
  r.join_lanes(c);
  if (THREADS == 32) return;
  constexpr int W = THREADS / 32;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  __syncthreads();
  if (lane == 0) {
    room[2 * warp]     = r.m;
    room[2 * warp + 1] = r.s;
  }
  __syncthreads();
  r = Running<V>();
  if (lane < W) {
    r.m = room[2 * lane];
    r.s = room[2 * lane + 1];
  }
  r.join_lanes(c);
}

template <int THREADS, class V>
__device__ __forceinline__ V sum_row(V x, V* room)
{
#pragma unroll
  for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(~0u, x, d);
  if (THREADS == 32) return x;
  constexpr int W = THREADS / 32;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  __syncthreads();
  if (lane == 0) room[warp] = x;
  __syncthreads();
  x = lane < W ? room[lane] : V(0);
#pragma unroll
  for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(~0u, x, d);
  return x;
}

template <int THREADS>
__device__ __forceinline__ double max_row(double x, double* room)
{
#pragma unroll
  for (int d = 16; d; d >>= 1) x = fmax(x, __shfl_xor_sync(~0u, x, d));
  if (THREADS == 32) return x;
  constexpr int W = THREADS / 32;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  __syncthreads();
  if (lane == 0) room[warp] = x;
  __syncthreads();
  x = lane < W ? room[lane] : -INFINITY;
#pragma unroll
  for (int d = 16; d; d >>= 1) x = fmax(x, __shfl_xor_sync(~0u, x, d));
  return x;
}

// ---- the teacher's side of a row -------------------------------------------------------------
// Entry j names class at[j] (-1: none) with the probability p[j]; a class that is named again adds
// to its first entry and the later one has at -2 - first.  In 64 bits: the two sides' logarithms nearly
// cancel, and what is left of the teacher is a difference from 1.
struct TeacherRow {
  double log_norm;  // log p[j] = values[j] / T - log_norm
  double rest;      // probability of all classes that are not named
  int named;        // different classes named
  bool counts;
  bool merged;      // a class was named twice: log p[j] is that of p[j]
};

__device__ __forceinline__ int64_t teacher_index(const Teacher& t, int64_t row, int j)
{
  return t.index64 ? static_cast<const int64_t*>(t.index)[row * t.index_stride + j]
                   : static_cast<int64_t>(static_cast<const int32_t*>(t.index)[row * t.index_stride + j]);
}

// p, at: shared, k entries of this row; room: shared, at least 32 doubles of this row.
template <int THREADS>
__device__ __forceinline__ TeacherRow read_teacher(const Teacher& t, int64_t row, int64_t n_cols, double inv_t, int tid,
                                                   float* p, int* at, double* room)
{
  TeacherRow r;
  sync_row<THREADS>();  // the last row's entries have been used
  double top = -INFINITY;
  for (int j = tid; j < t.k; j += THREADS) {
    const int64_t c = teacher_index(t, row, j);
    const bool is   = c >= 0 && c < n_cols && c != t.ignore;
    at[j]           = is ? static_cast<int>(c) : -1;
    if (is) top = fmax(top, t.values ? t.values[row * t.values_stride + j] * inv_t : 0.0);
  }
  sync_row<THREADS>();
  if (t.logsumexp) {
    r.log_norm = t.logsumexp[row];
  } else {
    const double most = max_row<THREADS>(top, room);
    double sum        = 0;
    for (int j = tid; j < t.k; j += THREADS)
      if (at[j] >= 0) sum += t.values ? exp(t.values[row * t.values_stride + j] * inv_t - (most == -INFINITY ? 0.0 : most)) : 1.0;
    sum        = sum_row<THREADS>(sum, room);
    r.log_norm = most + log(sum);
  }
  r.counts = !(r.log_norm == -INFINITY);
  // (a NaN among the values is not seen by fmax: it is in the sum)
  double mass = 0;
  int named   = 0;
  for (int j = tid; j < t.k; j += THREADS) {
    double q = 0;
    if (at[j] >= 0 && r.counts) q = exp((t.values ? t.values[row * t.values_stride + j] * inv_t : 0.0) - r.log_norm);
    p[j] = static_cast<float>(q);
    mass += q;
  }
  // classes named twice (top scores name none twice; a caller's list may)
  sync_row<THREADS>();
  bool again = false;
  for (int j = tid; j < t.k; j += THREADS) {
    const int c = at[j];
    if (c < 0) continue;
    bool dup = false;
    for (int i = 0; i < j; ++i) dup |= at[i] == c;
    named += !dup;
    again |= dup;
  }
  double both = sum_row<THREADS>(named + (again ? 65536.0 : 0.0), room);
  r.merged    = both >= 65536.0;
  if (r.merged) {
    sync_row<THREADS>();
    if (tid == 0) {
      for (int j = 1; j < t.k; ++j) {
        if (at[j] < 0) continue;
        for (int i = 0; i < j; ++i)
          if (at[i] == at[j]) {
            p[i] += p[j];
            p[j]  = 0;
            at[j] = -2 - i;
            break;
          }
      }
    }
    sync_row<THREADS>();
    both = both - 65536.0 * floor(both / 65536.0);
  }
  r.named = static_cast<int>(both);
  r.rest  = 0;
  if (t.logsumexp) {
    mass   = sum_row<THREADS>(mass, room);
    // (a log-sum-exp in 32 bits leaves about that much where nothing is left)
    r.rest = r.named < n_cols && !(1.0 - mass < 0x1p-20) ? 1.0 - mass : 0.0;
  }
  return r;
}

}  // namespace distill
}  // namespace b2fil
