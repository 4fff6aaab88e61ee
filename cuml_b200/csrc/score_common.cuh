// What the scoring kernels share: a softmax's maximum, sum and mean exponent in one pass, and what follows from them for
// a row.
//
// With a reference m, a_c = (z_c - m) log2(e) / T, s = sum 2^a and u = sum 2^a a:
//   log q_c = ln2 a_c - ln s,   entropy H = -sum q log q = ln s - ln2 u / s
//   d log q_t / dz_c = (1(c = t) - q_c) / T,   dH / dz_c = -q_c (log q_c + H) / T = -q_c ln2 (a_c - u / s) / T
#pragma once

#include "distill_common.cuh"

namespace b2fil {
namespace distill {

constexpr float kLn2 = 0.69314718055994530942f;

// Exponents below this are as good as any: 2^a is 0, and so is 2^a a, which -inf would make NaN.
constexpr float kLeast = -256.f;

// (NaN stays, unlike in fmaxf)
__device__ __forceinline__ float at_least(float x, float least)
{
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(x), "f"(least));
  return y;
}

// m is the largest value, or one that none exceeds by more than kSlack powers of two (Stream).
struct Scored {
  float m = lowest<float>(), s = 0.f, u = 0.f;

  __device__ __forceinline__ void move(float to, float c)  // s and u relative to `to`, which is finite or +inf
  {
    const float a = at_least((m - to) * c, kLeast), f = power(a);
    u = fmaf(s, a, u) * f;
    s = s * f;
    m = to;
  }
  __device__ __forceinline__ void add(float x, float base, float c)
  {
    const float a = at_least((x - base) * c, kLeast), p = power(a);
    s += p;
    u = fmaf(p, a, u);
  }
  __device__ __forceinline__ void join(float m2, float s2, float u2, float c)
  {
    const float to = fmaxf(m, m2);
    if (to == lowest<float>()) {
      s += s2;  // 0, or NaN
      return;
    }
    Scored o;
    o.m = m2;
    o.s = s2;
    o.u = u2;
    o.move(to, c);
    move(to, c);
    s += o.s;
    u += o.u;
  }
  __device__ __forceinline__ void join_lanes(float c)
  {
    float to;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(to) : "f"(m));
    if (to != lowest<float>()) move(to, c);
    s = sum_lanes(s);
    u = sum_lanes(u);
  }
  // The same for every LANES lanes of a warp.
  template <int LANES>
  __device__ __forceinline__ void join_some(float c)
  {
    if (LANES == 32) {
      join_lanes(c);
      return;
    }
    float to = m;
#pragma unroll
    for (int d = LANES / 2; d; d >>= 1) to = fmaxf(to, __shfl_xor_sync(~0u, to, d));
    if (to != lowest<float>()) move(to, c);
#pragma unroll
    for (int d = LANES / 2; d; d >>= 1) {
      s += __shfl_xor_sync(~0u, s, d);
      u += __shfl_xor_sync(~0u, u, d);
    }
  }
};

// The same for a stream of pieces: `limit` is m + slack.
struct ScoredStream : Scored {
  float base = 0.f, limit = lowest<float>();
  __device__ __forceinline__ void reach(float most, float c, float slack)
  {
    if (!(most > limit)) return;
    move(most, c);
    base  = most;
    limit = most + slack;
  }
  template <int N>
  __device__ __forceinline__ void take(const float (&x)[N], float c, float slack)
  {
    float most = x[0];
#pragma unroll
    for (int e = 1; e < N; ++e) most = fmaxf(most, x[e]);
    reach(most, c, slack);
#pragma unroll
    for (int e = 0; e < N; ++e) add(x[e], base, c);
  }
};

// A piece's 16 bytes and back, as the language allows it.  (Elements written through another type's pointer were left out of
// later stores.)
template <class T>
__device__ __forceinline__ uint4 words_of(const Piece<T>& p)
{
  uint4 w;
  memcpy(&w, &p, 16);
  return w;
}
template <class T>
__device__ __forceinline__ Piece<T> piece_of(const uint4& w)
{
  Piece<T> p;
  memcpy(&p, &w, 16);
  return p;
}

// visit_row whose last pieces are in flight together, too, and the elements before and behind them with the first: ends(i, x, k, y) for those that
// a thread has, i or k below 0 where it has none.  A row of a warp may be no more than that.
template <int U, class T, class Ends, class Many>
__device__ __forceinline__ void visit_all(const T* row, int n, int tid, int threads, Ends ends, Many many)
{
  constexpr int N  = Piece<T>::N;
  const int lead   = lead_of(row, n);
  const int pieces = (n - lead) / N;
  const T* body    = row + lead;
  const int at     = lead + pieces * N + tid;
  T before = T(), behind = T();
  if (tid < lead) before = row[tid];
  if (at < n) behind = row[at];
  for (int first = 0; first < pieces; first += U * threads) {  // (the same rounds for all threads: none goes two ways)
    const int left  = pieces - first - tid;
    const bool full = left + tid >= U * threads;
    const T* from   = body + static_cast<int64_t>(first + tid) * N;
    Piece<T> r[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (full || u * threads < left) r[u] = piece_of<T>(__ldg(reinterpret_cast<const uint4*>(from + u * threads * N)));
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (full || u * threads < left) many(lead + (first + tid + u * threads) * N, r[u]);
  }
  if (tid < lead || at < n) ends(tid < lead ? tid : -1, before, at < n ? at : -1, behind);
}

// ---- two numbers at a time ---------------------------------------------------------------------
__device__ __forceinline__ uint64_t pair_of(float lo, float hi)
{
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void split_pair(uint64_t x, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x)); }
__device__ __forceinline__ uint64_t fma_pairs(uint64_t a, uint64_t b, uint64_t c)
{
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_pairs(uint64_t a, uint64_t b)
{
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// What a type's logits are raised to at least, so that no exponent is -inf, and what ordinary ones are above.
template <class T>
struct Ordinary {
  static constexpr float kFloor = -1e30f, kAbove = -1e29f;
};
template <>
struct Ordinary<__half> {
  static constexpr float kFloor = -65504.f, kAbove = -30000.f;
};

__device__ __forceinline__ float2 halves_of(uint32_t w)
{
  __half2 h;
  memcpy(&h, &w, 4);
  return __half22float2(h);
}

// A piece's numbers.
__device__ __forceinline__ void numbers_of(const Piece<float>& p, float (&x)[4])
{
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = p.v[i];
}
__device__ __forceinline__ void numbers_of(const Piece<__nv_bfloat16>& p, float (&x)[8])
{
  const uint4 all     = words_of(p);
  const uint32_t w[4] = {all.x, all.y, all.z, all.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i]     = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void numbers_of(const Piece<__half>& p, float (&x)[8])
{
  const uint4 all     = words_of(p);
  const uint32_t w[4] = {all.x, all.y, all.z, all.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = halves_of(w[i]);
    x[2 * i]       = f.x;
    x[2 * i + 1]   = f.y;
  }
}

// 16 bytes of logits: the largest (NaN left out), and all of them, at least kFloor, in pairs.
__device__ __forceinline__ float largest_of(const Piece<float>& p) { return fmaxf(fmaxf(p.v[0], p.v[1]), fmaxf(p.v[2], p.v[3])); }
__device__ __forceinline__ float largest_of(const Piece<__nv_bfloat16>& p)
{
  const uint4 w = words_of(p);
  uint32_t a, b;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(a) : "r"(w.x), "r"(w.y));
  asm("max.bf16x2 %0, %1, %2;" : "=r"(b) : "r"(w.z), "r"(w.w));
  asm("max.bf16x2 %0, %1, %2;" : "=r"(a) : "r"(a), "r"(b));
  return fmaxf(__uint_as_float(a << 16), __uint_as_float(a & 0xffff0000u));
}
__device__ __forceinline__ float largest_of(const Piece<__half>& p)
{
  const uint4 w = words_of(p);
  uint32_t a, b;
  asm("max.f16x2 %0, %1, %2;" : "=r"(a) : "r"(w.x), "r"(w.y));
  asm("max.f16x2 %0, %1, %2;" : "=r"(b) : "r"(w.z), "r"(w.w));
  asm("max.f16x2 %0, %1, %2;" : "=r"(a) : "r"(a), "r"(b));
  const float2 f = halves_of(a);
  return fmaxf(f.x, f.y);
}
template <class F>
__device__ __forceinline__ void each_pair(const Piece<float>& p, F f)
{
#pragma unroll
  for (int i = 0; i < 4; i += 2)
    f(pair_of(at_least(p.v[i], Ordinary<float>::kFloor), at_least(p.v[i + 1], Ordinary<float>::kFloor)));
}
template <class F>
__device__ __forceinline__ void each_pair(const Piece<__nv_bfloat16>& p, F f)
{
  const uint4 all     = words_of(p);
  const uint32_t w[4] = {all.x, all.y, all.z, all.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t x;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(x) : "r"(w[i]), "r"(0xf149f149u));  // -1e30
    f(pair_of(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u)));
  }
}
template <class F>
__device__ __forceinline__ void each_pair(const Piece<__half>& p, F f)
{
  const uint4 all     = words_of(p);
  const uint32_t w[4] = {all.x, all.y, all.z, all.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t x;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(x) : "r"(w[i]), "r"(0xfbfffbffu));  // -65504
    const float2 v = halves_of(x);
    f(pair_of(v.x, v.y));
  }
}

// Scored of a row of ordinary logits, 6 instead of 9 instructions per logit: exponents are z c - r with r = m c as it is rounded (by at
// most 2^-4, which all of them share and the end takes back), two at a time.  `usable` tells whether the row's
// maximum is such that it holds; others are taken again by ScoredStream.
template <class T>
struct PairedStream {
  float m = lowest<float>(), r = 0.f, limit = Ordinary<T>::kAbove;
  uint64_t s = 0, u = 0;

  __device__ __forceinline__ void reach(float most, float c, float slack)
  {
    if (!(most > limit)) return;
    const float to = most * c, a = at_least(r - to, kLeast), f = m == lowest<float>() ? 0.f : power(a);
    const uint64_t ff = pair_of(f, f);
    u     = fma_pairs(fma_pairs(s, pair_of(a, a), u), ff, 0);
    s     = fma_pairs(s, ff, 0);
    m     = most;
    r     = to;
    limit = most + slack;
  }
  __device__ __forceinline__ void add(uint64_t z, uint64_t cc, uint64_t minus_r)
  {
    const uint64_t a = fma_pairs(z, cc, minus_r);
    float lo, hi;
    split_pair(a, lo, hi);
    const uint64_t p = pair_of(power(lo), power(hi));
    s = add_pairs(s, p);
    u = fma_pairs(p, a, u);
  }
  __device__ __forceinline__ void take(const Piece<T>& p, float most, float c, float slack)
  {
    reach(most, c, slack);
    const uint64_t cc = pair_of(c, c), minus_r = pair_of(-r, -r);
    each_pair(p, [&](uint64_t z) { add(z, cc, minus_r); });
  }
  __device__ __forceinline__ void take(float z, float c, float slack) { take(z, Ordinary<T>::kFloor, c, slack); }
  __device__ __forceinline__ void take(float z, float y, float c, float slack)
  {
    reach(fmaxf(z, y), c, slack);
    constexpr float kFloor = Ordinary<T>::kFloor;
    add(pair_of(at_least(z, kFloor), at_least(y, kFloor)), pair_of(c, c), pair_of(-r, -r));
  }
  // relative to 2^(m c)
  __device__ __forceinline__ Scored scored(float c) const
  {
    Scored o;
    float lo, hi;
    split_pair(s, lo, hi);
    o.s = lo + hi;
    split_pair(u, lo, hi);
    o.u = lo + hi;
    o.m = m;
    if (m == lowest<float>()) return o;  // (no ordinary logit: 0, or NaN)
    const float d = -fmaf(m, c, -r), f = power(d);
    o.u = fmaf(o.s, d, o.u) * f;
    o.s *= f;
    return o;
  }
  // m: of the row, or of all that was taken.  What was not above kAbove may be left out: its exponent is below -160.
  static __device__ __forceinline__ bool usable(float m, float c)
  {
    return fabsf(m) * c <= 0x1p20f && (m - Ordinary<T>::kAbove) * c >= 160.f;
  }
};

// All threads of the row get the joined value; `room`: shared, 3 floats per warp.
template <int THREADS>
__device__ __forceinline__ void join_scored(Scored& r, float c, float* room)
{
  r.join_lanes(c);
  if (THREADS == 32) return;
  constexpr int W = THREADS / 32;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  __syncthreads();
  if (lane == 0) {
    room[3 * warp]     = r.m;
    room[3 * warp + 1] = r.s;
    room[3 * warp + 2] = r.u;
  }
  __syncthreads();
  r = Scored();
  if (lane < W) {
    r.m = room[3 * lane];
    r.s = room[3 * lane + 1];
    r.u = room[3 * lane + 2];
  }
  r.join_lanes(c);
}

// A row of any logits by THREADS threads, joined for all of them; U pieces of a thread are in flight.
template <class T, int THREADS, int U>
__device__ __noinline__ Scored visit_any(const T* row, int64_t n, int tid, float c, float* room)
{
  constexpr int N = Piece<T>::N;
  ScoredStream r;
  const float slack = kSlack / c;
  visit_row<U>(
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

// What is kept of a row for its gradient: m, 1 / s (0: the row does not count), -u / s and the class.
__device__ __forceinline__ float4 kept_row(float m, float inverse, float mean, int at)
{
  return make_float4(m, inverse, mean, __int_as_float(at));
}

// The given class of a row, -1: none, -2: the row does not count.
__device__ __forceinline__ int target_of(const Target& t, int64_t row, int64_t n_cols)
{
  if (!t.index) return -1;
  const int64_t i = t.index64 ? static_cast<const int64_t*>(t.index)[row * t.stride]
                              : static_cast<int64_t>(static_cast<const int32_t*>(t.index)[row * t.stride]);
  return i >= 0 && i < n_cols && i != t.ignore ? static_cast<int>(i) : -2;
}

// Scores of a row, by one thread.  logit: of class `at`.  The difference of logits and the logarithm are joined in 64 bits; neither
// a logarithm of a probability above 0 nor an entropy below it leaves by their roundings.
struct RowScore {
  double log_s;
  bool counts;
};
__device__ __forceinline__ RowScore finish_score(const Scores& out, int64_t row, const Scored& r, double inv_t, int at, float logit)
{
  RowScore o;
  o.log_s  = log_sum(r.s);
  o.counts = at != -2 && !(r.s == 0.f);  // (no finite logit: no softmax)
  const float mean = -r.u / r.s;
  double log_prob  = (static_cast<double>(logit) - r.m) * inv_t - o.log_s;
  double entropy   = o.log_s + mean * 0.69314718055994530942;
  if (log_prob > 0) log_prob = 0;
  if (entropy < 0) entropy = 0;
  if (r.s != r.s) log_prob = NAN;
  if (out.log_prob) out.log_prob[row] = o.counts ? static_cast<float>(log_prob) : 0.f;
  out.entropy[row] = o.counts ? static_cast<float>(entropy) : 0.f;
  out.kept[row]    = o.counts ? kept_row(r.m, 1.f / r.s, mean, at) : kept_row(0.f, 0.f, 0.f, -1);
  return o;
}

// The gradient by the logits of a row: of class c it is 2^a (A + B a), and `add` more for the given one.
struct RowGrad {
  float base, A, B, add;
  int at;
  bool counts;
  __device__ __forceinline__ float operator()(float z, float c) const
  {
    const float a = at_least((z - base) * c, kLeast);
    return power(a) * fmaf(B, a, A);
  }
};
// The same of a piece; none for classes.
template <class T>
__device__ __forceinline__ void grads_of(const RowGrad& r, const Piece<T>& z, float c, float (&y)[Piece<T>::N])
{
  const uint64_t minus_base = pair_of(-r.base, -r.base), cc = pair_of(c, c), AA = pair_of(r.A, r.A), BB = pair_of(r.B, r.B);
  float x[Piece<T>::N];
  numbers_of(z, x);
#pragma unroll
  for (int e = 0; e < Piece<T>::N; e += 2) {
    const uint64_t far = fma_pairs(add_pairs(pair_of(x[e], x[e + 1]), minus_base), cc, 0);
    float lo, hi;
    split_pair(far, lo, hi);
    lo = at_least(lo, kLeast);
    hi = at_least(hi, kLeast);
    split_pair(fma_pairs(pair_of(power(lo), power(hi)), fma_pairs(BB, pair_of(lo, hi), AA), 0), y[e], y[e + 1]);
  }
}
// g, h: gradients by the row's log probability and entropy, times 1 / T (and a scale).
__device__ __forceinline__ RowGrad row_grad(const float4& kept, float g, float h)
{
  RowGrad r;
  r.base   = base_of(kept.x);
  r.at     = __float_as_int(kept.w);
  r.counts = kept.y != 0.f;
  if (r.at < 0) g = 0.f;
  r.add = g;
  r.B   = -kept.y * kLn2 * h;
  r.A   = fmaf(r.B, kept.z, -kept.y * g);
  return r;
}

}  // namespace distill
}  // namespace b2fil
