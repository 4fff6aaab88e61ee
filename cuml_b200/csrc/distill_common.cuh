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

// ---- reference m and sum s of exp((x - m) / T), c = log2(e) / T -------------------------------
// m is the largest value, or one hardly below it.
// The difference is taken before the scale: the scaled lowest value of a type would be -inf.
__device__ __forceinline__ float power(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ double power(double x) { return exp2(x); }
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double larger(double a, double b) { return fmax(a, b); }
__device__ __forceinline__ float smaller(float a, float b) { return fminf(a, b); }
__device__ __forceinline__ double smaller(double a, double b) { return fmin(a, b); }
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
  __device__ __forceinline__ void join_lanes(V c)  // the maximum first: one power for all steps
  {
    V to = m;
#pragma unroll
    for (int d = 16; d; d >>= 1) to = larger(to, __shfl_xor_sync(~0u, to, d));
    if (m != lowest<V>()) s *= power((m - to) * c);
    m = to;
#pragma unroll
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(~0u, s, d);
  }
};

// The same for a stream of values: the sum's reference is raised only when a value exceeds it by kSlack powers of
// two.  (A warp of 32 maxima is raised for most of a short row's pieces; an exponent of up to kSlack
// is rounded by 2^-22.)
constexpr float kSlack = 6.f;
template <class V>
struct Stream {
  V m = lowest<V>(), s = V(0), b = V(0), limit = lowest<V>();  // b: what is subtracted, limit: m + slack
  __device__ __forceinline__ void raise(V to, V c, V slack)
  {
    s     = m == lowest<V>() ? s : s * power((m - to) * c);
    m = b = to;
    limit = to + slack;
  }
  __device__ __forceinline__ void add(V x, V c) { s += power((x - b) * c); }
  __device__ __forceinline__ void take(V x, V c, V slack)
  {
    if (x > limit) raise(x, c, slack);
    add(x, c);
  }
  __device__ __forceinline__ Running<V> running() const
  {
    Running<V> r;
    r.m = m;
    r.s = s;
    return r;
  }
};

// ---- rows for one thread each, staged in shared memory ---------------------------------------
constexpr int kTileRows = 128;  // and threads of a block

// Rows an odd number of words apart fall into different banks.
template <class T>
struct TileShape {
  int cols, pitch;
  uint32_t inverse;  // i / cols = i * inverse / 2^32 for i < 128 x 512 (exact: i * cols < 2^32)
  __host__ __device__ explicit TileShape(int n)
      : cols(n), pitch(sizeof(T) >= 4 ? n | 1 : (n + 1) / 2 * 2 + ((n + 1) / 2 % 2 ? 0 : 2)), inverse(0xffffffffu / n + 1)
  {
  }
  __host__ __device__ size_t bytes() const { return static_cast<size_t>(pitch) * kTileRows * sizeof(T); }
  // Where element i of the rows one after the other lies in the tile.
  __device__ __forceinline__ int at(uint32_t i) const { return i + __umulhi(i, inverse) * (pitch - cols); }
};

// Whether all rows of a tile lie one after the other from a 16-byte boundary on.
template <class T>
__device__ __forceinline__ bool without_gaps(const void* rows, int64_t stride, int cols)
{
  return stride == cols && (reinterpret_cast<uintptr_t>(rows) & 15) == 0 && cols > 1;
}

// Visits (row, column) of a tile of rows that are not one after the other.
template <class F>
__device__ __forceinline__ void visit_tile(int rows, int cols, F f)
{
  int r = threadIdx.x / cols, i = threadIdx.x % cols;
  const int dr = kTileRows / cols, di = kTileRows % cols;
  while (r < rows) {
    f(r, i);
    r += dr;
    i += di;
    if (i >= cols) {
      i -= cols;
      ++r;
    }
  }
}

// By all threads of a block, which wait for one another afterwards.
template <class T>
__device__ __forceinline__ void load_tile(T* tile, const TileShape<T>& shape, const T* from, int64_t stride, int rows, bool whole)
{
  constexpr int N = Piece<T>::N, U = 4;  // 16 bytes at a time, U of them in flight
  if (whole) {
    const int all = rows * shape.cols, pieces = all / N;
    for (int p = threadIdx.x; p < pieces; p += U * kTileRows) {
      Piece<T> v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (p + u * kTileRows < pieces) v[u] = load_piece(from + (p + u * kTileRows) * N);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (p + u * kTileRows >= pieces) break;
#pragma unroll
        for (int e = 0; e < N; ++e) tile[shape.at((p + u * kTileRows) * N + e)] = v[u].v[e];
      }
    }
    for (int i = pieces * N + threadIdx.x; i < all; i += kTileRows) tile[shape.at(i)] = from[i];
  } else {
    visit_tile(rows, shape.cols, [&](int r, int i) { tile[r * shape.pitch + i] = from[r * stride + i]; });
  }
}
template <class T>
__device__ __forceinline__ void store_tile(T* to, int64_t stride, const T* tile, const TileShape<T>& shape, int rows, bool whole)
{
  constexpr int N = Piece<T>::N;
  if (whole) {
    const int all = rows * shape.cols, pieces = all / N;
    for (int p = threadIdx.x; p < pieces; p += kTileRows) {
      Piece<T> v;
#pragma unroll
      for (int e = 0; e < N; ++e) v.v[e] = tile[shape.at(p * N + e)];
      *reinterpret_cast<uint4*>(to + p * N) = *reinterpret_cast<const uint4*>(&v);
    }
    for (int i = pieces * N + threadIdx.x; i < all; i += kTileRows) to[i] = tile[shape.at(i)];
  } else {
    visit_tile(rows, shape.cols, [&](int r, int i) { to[r * stride + i] = tile[r * shape.pitch + i]; });
  }
}

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

// ---- the teacher's side of a row -------------------------------------------------------------
// ln of a sum of 32-bit numbers, off by 2^-24 of less than 1 whatever its size: the exponent's part is exact.
__device__ __forceinline__ double log_sum(float s)
{
  if (!(s > 0.f) || s == INFINITY) return log(static_cast<double>(s));
  int e;
  float f = frexpf(s, &e);
  if (f < 0.70710678f) {
    f *= 2.f;
    --e;
  }
  return fma(static_cast<double>(e), 0.69314718055994530942, static_cast<double>(logf(f)));
}

template <class V>
__device__ __forceinline__ V sum_lanes(V x)
{
#pragma unroll
  for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(~0u, x, d);
  return x;
}
__device__ __forceinline__ float max_lanes(float x)
{
#pragma unroll
  for (int d = 16; d; d >>= 1) x = fmaxf(x, __shfl_xor_sync(~0u, x, d));
  return x;
}

// What a teacher names in a row.  Entry j is the class at[j] (-1: none) with the score v[j] and the
// probability p[j]; a class that is named again adds to its first entry and the later one has at -1.
struct Entries {
  float *v, *p;
  int* at;
};
__host__ __device__ __forceinline__ size_t entry_bytes(int k) { return static_cast<size_t>(k) * 12; }
__device__ __forceinline__ Entries entries_at(void* base, int k)
{
  float* v = static_cast<float*>(base);
  return {v, v + k, reinterpret_cast<int*>(v + 2 * k)};
}

// log p[j] = v[j] / T - log_norm is taken in 64 bits, as it nearly cancels with the student's logarithm.
struct TeacherRow {
  double log_norm;
  double rest;   // probability of all classes that are not named: where it is nearly 1 what matters is how nearly
  float mass;    // of all of p: 1, or less where the teacher gives some to no class of the student's
  bool counts;
  bool merged;   // a class was named twice: log p[j] is that of p[j]
};

__device__ __forceinline__ int64_t teacher_index(const Teacher& t, int64_t row, int j)
{
  return t.index64 ? static_cast<const int64_t*>(t.index)[row * t.index_stride + j]
                   : static_cast<int64_t>(static_cast<const int32_t*>(t.index)[row * t.index_stride + j]);
}

// What is left of 1 counts from here on: a log-sum-exp L in 32 bits is off by |L| 2^-24 at least and by few times that as it is
// made, p by that part of itself.
__device__ __forceinline__ double least_rest(double logsumexp) { return fmax(0x1p-20, fabs(logsumexp) * 0x1p-22); }

// By one warp; e: shared memory.  REST: the teacher has a logsumexp.
template <bool REST>
__device__ __forceinline__ TeacherRow read_teacher(const Teacher& t, int64_t row, int64_t n_cols, double inv_t, const Entries& e)
{
  TeacherRow r;
  const int lane = threadIdx.x % 32, k = t.k;
  float top      = lowest<float>();
  double mass    = 0;
  r.mass         = 1.f;
  for (int j = lane; j < k; j += 32) {
    const int64_t c = teacher_index(t, row, j);
    const float v   = t.values ? t.values[row * t.values_stride + j] : 0.f;
    const bool is   = c >= 0 && c < n_cols && c != t.ignore;
    e.at[j]         = is ? static_cast<int>(c) : -1;
    e.v[j]          = v;
    if (is) top = fmaxf(top, v);
  }
  __syncwarp();
  if (REST) {
    // what is left of 1 is a difference: in 64 bits
    r.log_norm  = t.logsumexp[row];
    r.counts    = !(r.log_norm == -INFINITY);
    for (int j = lane; j < k; j += 32) {
      const double q = e.at[j] >= 0 && r.counts ? exp(e.v[j] * inv_t - r.log_norm) : 0.0;
      e.p[j]         = static_cast<float>(q);
      mass += q;
    }
    mass = sum_lanes(mass);
    r.rest = 1.0 - mass < least_rest(r.log_norm) ? 0.0 : 1.0 - mass;
  } else {
    const float most = base_of(max_lanes(top));
    const float ti   = static_cast<float>(inv_t);
    float sum        = 0.f;
    for (int j = lane; j < k; j += 32) {
      const float x = e.at[j] >= 0 ? expf((e.v[j] - most) * ti) : 0.f;
      e.p[j]        = x;
      sum += x;
    }
    sum        = sum_lanes(sum);
    r.log_norm = most * inv_t + log_sum(sum);
    r.counts   = !(sum == 0.f);
    r.rest     = 0.0;
    if (r.counts)
      for (int j = lane; j < k; j += 32) e.p[j] = e.p[j] / sum;
  }
  __syncwarp();
  // classes named twice (top scores name none twice; a caller's list may)
  bool again = false;
  int named  = 0;
  if (k <= 32) {
    const int c        = lane < k ? e.at[lane] : -1;
    const unsigned all = __match_any_sync(~0u, c < 0 ? -1 - lane : c);
    again              = __ffs(all) - 1 < lane;
    named              = c >= 0 && !again;
  } else {
    for (int j = lane; j < k; j += 32) {
      const int c = e.at[j];
      bool dup    = false;
      for (int i = 0; i < j; ++i) dup |= e.at[i] == c;
      named += c >= 0 && !dup;
      again |= c >= 0 && dup;
    }
  }
  r.merged = __any_sync(~0u, again);
  if (r.merged) {
    if (lane == 0) {
      for (int j = 1; j < k; ++j) {
        if (e.at[j] < 0) continue;
        for (int i = 0; i < j; ++i)
          if (e.at[i] == e.at[j]) {
            e.p[i] += e.p[j];
            e.at[j] = -1;
            break;
          }
      }
    }
    __syncwarp();
  }
  if (REST) {
    if (__reduce_add_sync(~0u, named) >= n_cols) r.rest = 0.0;  // no class is left
    if (r.rest == 0.0) r.mass = static_cast<float>(mass);
  }
  return r;
}

// Sum over a row's entries of p (log p - log q), q the softmax with the maximum m and the logarithm of the sum
// log_s; logit(j, class).  By one warp.
template <class F>
__device__ __forceinline__ double named_loss(const Entries& e, int k, const TeacherRow& t, double inv_t, float m, double log_s,
                                             F logit)
{
  double loss = 0;
  for (int j = threadIdx.x % 32; j < k; j += 32) {
    const int at  = e.at[j];
    const float p = e.p[j];
    if (at < 0 || p == 0.f) continue;
    const double log_p = t.merged ? log(static_cast<double>(p)) : e.v[j] * inv_t - t.log_norm;
    loss += p * (log_p - ((static_cast<double>(logit(j, at)) - m) * inv_t - log_s));
  }
  return sum_lanes(loss);
}

// ---- sums over the rows ----------------------------------------------------------------------
// {sum of the losses, rows that count} of the rows of a block's threads that have any, in a fixed order;
// for thread 0.
template <int THREADS>
__device__ __forceinline__ double2 sum_block(double loss, double count, double2* room)
{
  loss  = sum_lanes(loss);
  count = sum_lanes(count);
  __syncthreads();
  if (threadIdx.x % 32 == 0) room[threadIdx.x / 32] = make_double2(loss, count);
  __syncthreads();
  double2 all = make_double2(0, 0);
  if (threadIdx.x == 0)
    for (int i = 0; i < THREADS / 32; ++i) {
      all.x += room[i].x;
      all.y += room[i].y;
    }
  return all;
}
// Sum, or mean over the rows that count (0 if none does).
__device__ __forceinline__ void write_reduced(const Reduced& out, double2 all)
{
  const double f = out.reduction == 1 ? 1.0 : all.y > 0 ? 1.0 / all.y : 0.0;
  *out.loss      = static_cast<float>(all.y > 0 ? all.x * f : 0.0);
  *out.factor    = static_cast<float>(f);
}

}  // namespace distill
}  // namespace b2fil
