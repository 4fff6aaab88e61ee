// Loss of a linear layer's output z = H W^T and its gradients without keeping z.
//
//   forward   z tile by tile on the tensor cores; of a tile only each row's maximum and sum of
//             exp((z - max) / T) are kept, then joined per row with the logits of the classes that the
//             teacher names (dot products of their own: k per row)
//   backward  piece by piece of the classes: z again, d = q - p to a buffer of 16-bit values (up to
//             256 MB, twice the L2), then dH += d W and dW = d^T H from it
//
// Bound by the tensor cores: 8 N D V operations for a training step, of which the second z (2 N D V) is the
// price of not keeping it; kept in 16 bits it would be written once and read twice, and its rounding would
// be in q.  d is rounded to the layer's own 16 bits because both operands of a matrix instruction have
// one type: half a step of each d, independent of each other, where the gradient's own rounding
// is as much again.  Where products are so small that they hardly count, d is kept as two numbers of 16 bits
// (two planes), and the sums run over both.  For fp16 d is scaled by 2^14, so that probabilities down to 4e-9 are normal
// numbers.  Sums over classes and rows are in 32 bits; a sum over several pieces stays in 32 bits.
//
// One kernel does all products: a cluster of two CTAs takes 256 x 256 of the output
// (tcgen05.mma.cta_group::2; each CTA holds 128 rows of A, half of B and 128 rows of the result), since
// one CTA alone with 128 x 256 would have to read 96 bytes per cycle from L2 where 64 pass.  Warp 0 brings the
// tiles (TMA, 128-byte swizzle, ring of 6 x 32 KB), warp 1 of the first CTA issues the products, the others
// work on the finished tile while the next one is summed in the other half of TMEM.  All waits are
// bounded: after two seconds a role gives up, sets the status word and leaves by the common exit.  Until the host has read
// the word, losses and gradients are NaN: they may be incomplete.
#include <cooperative_groups.h>
#include <cuda.h>

#include <algorithm>

#include "distill_common.cuh"

namespace b2fil {
namespace distill {
namespace {

constexpr int kTile    = 256;              // rows and columns of a cluster's tile
constexpr int kHalf    = 128;              // of one CTA
constexpr int kDepth   = 64;               // of the inner dimension per stage: 128 bytes
constexpr int kStages  = 6;
constexpr int kStageA  = kHalf * kDepth * 2;
constexpr int kStage   = 2 * kStageA;      // A and B of one CTA
constexpr int kThreads = 256;
constexpr int kEpilogue = 8;               // warps that work on finished tiles: a quarter of the rows and half of the columns each
constexpr int kProductThreads = (4 + kEpilogue) * 32;
constexpr int kSmem    = kStages * kStage + 1024 + 256;
constexpr long long kPatience = 2000000000ll;  // ns
constexpr int64_t kPieceBytes = 256ll << 20;   // of d (8192 x 2048 x 131,072, gradient: 12.8 ms with 64 MB, 10.7 with 256)
constexpr int kMostSplits     = 16;
// Rows x classes x width up to which d has two planes (2048 x 512 x 1000: the errors of the gradients against
// 64 bits are 1.4 times those of their own rounding with one plane and 1.0 with two, which takes 5 us of
// 31; with two classes one plane made them up to twice as large).
constexpr int64_t kSmallProduct = 1ll << 32;
// ... and classes up to which the forward pass takes the logits as dot products in the kernel that reads the
// teacher: a load's latency per 32 classes of a row, against a kernel of 8 us.
constexpr int64_t kSmallLogits  = 1ll << 25;
constexpr int kFewClasses       = 128;
constexpr int kGroup          = 32;            // tiles of rows whose part of H stays in L2 while all of W passes
constexpr float kHalfScale    = 16384.f;       // of d in fp16
// Named classes of a row that the epilogue looks through for each tile; more are put into d by a kernel of their
// own (4096 x 1024 x 50,001, seven pieces: 32 per row cost 290 us in the epilogue and 28 us in the kernel,
// one per row nothing in the epilogue and 3.6 us per piece in the kernel).
constexpr int kFewNamed = 4;
constexpr int kScaleBlocks = 8;

__device__ int g_status;
__device__ __forceinline__ bool incomplete() { return *static_cast<volatile int*>(&g_status) != 0; }

// ---- PTX -------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t shared_of(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ uint32_t rank_in_cluster()
{
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t in_cta(uint32_t shared, uint32_t rank)
{
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(shared), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync()
{
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void bar_init(uint32_t bar, int count)
{
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, int bytes)
{
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive_cluster(uint32_t bar)  // shared::cluster address
{
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity)
{
  uint32_t ok;
  asm volatile(
    "{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
    : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok;
}
// One lane of a converged warp: what it alone executes stays free of per-lane loops around instructions that
// take uniform registers (a TMA load issued by `lane == 0` takes 260 cycles, by the elected lane a tenth).
__device__ __forceinline__ bool elected()
{
  uint32_t yes;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(yes));
  return yes;
}
__device__ __forceinline__ long long now_ns()
{
  long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
// False: the wait ran out (status word set), or another role of the CTA had given up.
__device__ __noinline__ bool bar_wait_long(uint32_t bar, uint32_t parity, volatile int* gave_up, long long patience)
{
  const long long until = now_ns() + patience;
  while (!bar_try(bar, parity)) {
    if (*gave_up) return false;
    if (now_ns() > until) {
      *gave_up = 1;
      atomicExch(&g_status, 1);
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int* gave_up)
{
  return bar_try(bar, parity) || bar_wait_long(bar, parity, gave_up, kPatience);
}
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* gave_up)
{
  return __all_sync(~0u, bar_wait(bar, parity, gave_up));
}
// 2-dimensional box to this CTA's shared memory; the bytes are counted at `bar`, which may be the other CTA's
__device__ __forceinline__ void load_box(uint32_t to, const CUtensorMap* map, uint32_t bar, int x, int y)
{
  asm volatile(
    "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4}], [%2];"
    ::"r"(to), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add)
{
  asm volatile(
    "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}"
    ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(add)) : "memory");
}
// Arrives at `bar` of both CTAs when the products issued so far are done.
__device__ __forceinline__ void commit(uint32_t bar)
{
  asm volatile(
    "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
    ::"r"(bar), "h"(static_cast<uint16_t>(3)) : "memory");
}
__device__ __forceinline__ void load_columns(uint32_t from, float (&x)[32])
{
  uint32_t r[32];
  asm volatile(
    "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
    "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
    "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
    : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
      "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
      "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
      "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
    : "r"(from));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) x[i] = __uint_as_float(r[i]);
}

// Shared-memory descriptor of a tile with 128-byte swizzle (version 1).  Inner dimension contiguous: rows of
// 128 bytes, 1024 bytes from 8 rows to the next.  Outer dimension contiguous: 64 outer by 64 inner elements
// are 64 rows of 128 bytes; 1024 bytes from 8 of the inner dimension to the next, 8192 from one such block to
// that of the next 64 outer elements.
__device__ __forceinline__ uint64_t descriptor(uint32_t at, bool outer)
{
  const uint64_t leading = outer ? 8192 >> 4 : 1, stride = 1024 >> 4;
  return (at >> 4 & 0x3fff) | leading << 16 | stride << 32 | 1ull << 46 | 2ull << 61;
}
// Instruction descriptor: 32-bit sums, A and B of one 16-bit type, 256 x 256.
__device__ __forceinline__ uint32_t instruction(bool bf16, bool a_outer, bool b_outer)
{
  return 1u << 4 | (bf16 ? 1u << 7 | 1u << 10 : 0u) | static_cast<uint32_t>(a_outer) << 15 |
         static_cast<uint32_t>(b_outer) << 16 | (kTile >> 3) << 17 | (kTile >> 4) << 24;
}

// ---- products --------------------------------------------------------------------------------
enum Result { kStats, kDiff, kGrad };

// out (m x n) = A (m x depth) B (n x depth)^T.  *_outer: the matrix lies with its depth outermost.
struct Product {
  CUtensorMap a, b;
  int m, n, depth;
  int m_tiles, n_tiles, splits;  // splits: parts of the depth, each with sums of its own
  int planes, plane_rows;        // the depth is passed once for each plane of A, which are plane_rows rows apart
  int a_outer, b_outer;
  int n_first;  // order of the tiles: all of a row of tiles, else kGroup of a column
  // kGrad: rows of n elements; 32-bit sums, one matrix per split, to which `add` adds, or 16-bit results
  float* sums;
  int add;
  void* out;    // times `scale`
};
// A factor, of what is there of a, b and t, of results that may be used.
struct Scale {
  const float *a, *b;
  float t;
  __device__ __forceinline__ float operator()() const { return incomplete() ? NAN : (a ? *a : 1.f) * (b ? *b : 1.f) * t; }
};
struct Work {
  Product product[2];
  int products;
  int bf16;
  // kStats: (row, half a tile of columns) -> maximum and sum
  float2* parts;
  // kStats, kDiff
  float c;                // log2(e) / T
  // kDiff: d = scale q of the classes from `first` on, columns up to a whole tile
  const float4* stats;
  const float* row_scale; // row_step elements from one row's to the next, or null: 1
  int64_t row_step;
  void* diff;
  int64_t diff_stride;
  float diff_scale;
  int planes, plane_rows;
  Named named;
  int k, first;
  Scale scale;            // kGrad
  int* ticket;            // kStats: set to 0 for linear_rows; kDiff: for the next kernel, which takes its tiles by it
};

struct Tile {
  int which, m, n, split, begin, end;  // begin, end: stages of the depth
};
__device__ __forceinline__ bool tile_of(const Work& w, int t, Tile& r)
{
  for (int i = 0; i < w.products; ++i) {
    const Product& p = w.product[i];
    const int tiles  = p.m_tiles * p.n_tiles * p.splits;
    if (t < tiles) {
      r.which = i;
      r.split = t / (p.m_tiles * p.n_tiles);
      t %= p.m_tiles * p.n_tiles;
      if (p.n_first) {
        r.m = t / p.n_tiles;
        r.n = t % p.n_tiles;
      } else {
        const int first = t / (kGroup * p.n_tiles) * kGroup, rows = min(kGroup, p.m_tiles - first);
        t -= first * p.n_tiles;
        r.m = first + t % rows;
        r.n = t / rows;
      }
      const int steps = (p.depth + kDepth - 1) / kDepth * p.planes;
      r.begin         = static_cast<int>(static_cast<int64_t>(steps) * r.split / p.splits);
      r.end           = static_cast<int>(static_cast<int64_t>(steps) * (r.split + 1) / p.splits);
      return true;
    }
    t -= tiles;
  }
  return false;
}

__device__ __forceinline__ void store32(void* to, const uint32_t (&x)[8])
{
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(to), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]),
               "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7]) : "memory");
}
__device__ __forceinline__ uint32_t two(float lo, float hi, bool bf16)
{
  uint32_t r;
  if (bf16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// 2^x of a logit by the maximum, at most the sum of all of them (NaN stays).  The tensor cores' sums and those of the dot
// products, of which the maximum or the named classes' logits may be, differ by some 1e-6 of their size: over a
// temperature of that size or less, an exponent.
__device__ __forceinline__ float power_within(float x, float sum)
{
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(power(x)), "f"(sum));
  return y;
}

// What rounding x to 16 bits leaves.
__device__ __forceinline__ float left_of(float x, bool bf16)
{
  return bf16 ? x - __bfloat162float(__float2bfloat16_rn(x)) : x - __half2float(__float2half_rn(x));
}

// Part of a row (32 columns from `col` on) of a finished tile.  n: columns of the result.
template <int KIND>
__device__ __forceinline__ void take_columns(const Work& w, const Product& p, int split, int64_t row, int col, float (&x)[32],
                                             Running<float>& r, float base, float sum, float factor)
{
  if (KIND == kStats) {
    if (col + 32 > p.n) {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (col + i >= p.n) x[i] = lowest<float>();
    }
    float most = x[0];
#pragma unroll
    for (int i = 1; i < 32; ++i) most = fmaxf(most, x[i]);
    if (most > r.m) r.raise(most, w.c);
    const float b = base_of(r.m);
    float s[4]    = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 32; ++i) s[i & 3] += power((x[i] - b) * w.c);
    r.s += (s[0] + s[1]) + (s[2] + s[3]);
    return;
  }
  if (KIND == kDiff) {
#pragma unroll
    for (int i = 0; i < 32; ++i) x[i] = col + i < p.n ? power_within((x[i] - base) * w.c, sum) * factor : 0.f;
    if (factor == 0.f) {  // a row that does not count, whatever its logits are
#pragma unroll
      for (int i = 0; i < 32; ++i) x[i] = 0.f;
    }
    for (int plane = 0;;) {
      char* to = static_cast<char*>(w.diff) + ((plane * static_cast<int64_t>(w.plane_rows) + row) * w.diff_stride + col) * 2;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = two(x[16 * h + 2 * i], x[16 * h + 2 * i + 1], w.bf16);
        store32(to + 32 * h, v);
      }
      if (++plane == w.planes) break;
#pragma unroll
      for (int i = 0; i < 32; ++i) x[i] = left_of(x[i], w.bf16);
    }
    return;
  }
  if (p.sums) {
    float* to = p.sums + (split * static_cast<int64_t>(p.m) + row) * p.n + col;
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      if (col + i >= p.n) break;
      float4 v = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
      if (p.add) {
        const float4 o = *reinterpret_cast<const float4*>(to + i);
        v              = make_float4(v.x + o.x, v.y + o.y, v.z + o.z, v.w + o.w);
      }
      *reinterpret_cast<float4*>(to + i) = v;
    }
    return;
  }
  char* to = static_cast<char*>(p.out) + (row * p.n + col) * 2;
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    if (col + i >= p.n) break;
    uint4 v;
    v.x = two(x[i] * factor, x[i + 1] * factor, w.bf16);
    v.y = two(x[i + 2] * factor, x[i + 3] * factor, w.bf16);
    v.z = two(x[i + 4] * factor, x[i + 5] * factor, w.bf16);
    v.w = two(x[i + 6] * factor, x[i + 7] * factor, w.bf16);
    *reinterpret_cast<uint4*>(to + 2 * i) = v;
  }
}

template <int KIND>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kProductThreads, 1) products(const __grid_constant__ Work w)
{
  extern __shared__ char raw[];
  constexpr bool kByTicket = KIND == kGrad;
  constexpr int kReaders   = 3 + 2 * kEpilogue;  // of a ticket: two producers, the issuer, both CTAs' epilogues
  __shared__ __align__(8) uint64_t bars[2 * kStages + 9];
  __shared__ volatile int tickets[2];
  __shared__ uint32_t tmem_at;
  __shared__ volatile int gave_up;
  const uint32_t ring = (shared_of(raw) + 1023) & ~1023u;
  const uint32_t full = shared_of(bars), empty = full + 8 * kStages, done = empty + 8 * kStages, freed = done + 16,
                 last = freed + 16, told = last + 8, heard = told + 16;
  const uint32_t rank = rank_in_cluster();
  const int warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  const int cluster = blockIdx.x / 2, clusters = gridDim.x / 2;
  if (!kByTicket && blockIdx.x == 0 && threadIdx.x == 0) *w.ticket = 0;
  if (threadIdx.x == 0) {
    gave_up = 0;
    for (int i = 0; i < kStages; ++i) {
      bar_init(full + 8 * i, 1);
      bar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      bar_init(done + 8 * i, 1);
      bar_init(freed + 8 * i, 2 * kEpilogue);
      bar_init(told + 8 * i, 1);
      bar_init(heard + 8 * i, kReaders);
    }
    bar_init(last, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(shared_of(&tmem_at)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_at;

  // The tile after tile i: the next in turn, or what the first CTA's fourth warp has drawn for the cluster.
  int drawn       = 0;
  auto next_tile = [&](int& i) {
    if (!kByTicket) {
      i += clusters;
      return true;
    }
    const int slot = drawn & 1;
    if (!warp_wait(told + 8 * slot, drawn >> 1 & 1, &gave_up)) return false;
    i = __shfl_sync(~0u, tickets[slot], 0);
    if (elected()) bar_arrive_cluster(in_cta(heard + 8 * slot, 0));
    ++drawn;
    return true;
  };

  if (warp == 0) {
    // tiles to the ring; the bytes of both CTAs are counted at the first one's barrier
    const uint32_t count_at = in_cta(full, 0);
    int stage = 0, phase = 0, issued = 0;
    bool ok = true;
    Tile t;
    for (int i = cluster; ok && tile_of(w, i, t); ok = ok && next_tile(i)) {
      const Product& p = w.product[t.which];
      const int m0 = t.m * kTile + rank * kHalf, n0 = t.n * kTile + rank * kHalf;
      const int steps = (p.depth + kDepth - 1) / kDepth;
      int plane = t.begin / steps, at = t.begin % steps;  // step of the plane
      for (int k = t.begin; k < t.end; ++k) {
        if (!warp_wait(empty + 8 * stage, phase ^ 1, &gave_up)) {
          ok = false;
          break;
        }
        const uint32_t a = ring + stage * kStage, b = a + kStageA, bar = count_at + 8 * stage;
        if (elected()) {
          if (rank == 0) bar_expect(full + 8 * stage, 2 * kStage);
          const int x = at * kDepth, y = plane * p.plane_rows;
          if (p.a_outer) {
            load_box(a, &p.a, bar, m0, y + x);
            load_box(a + 8192, &p.a, bar, m0 + 64, y + x);
          } else {
            load_box(a, &p.a, bar, x, y + m0);
          }
          if (p.b_outer) {
            load_box(b, &p.b, bar, n0, x);
            load_box(b + 8192, &p.b, bar, n0 + 64, x);
          } else {
            load_box(b, &p.b, bar, x, n0);
          }
        }
        __syncwarp();
        if (++at == steps) {
          at = 0;
          ++plane;
        }
        ++issued;
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    if (!ok && rank == 0) {
      // copies in flight have to land before the CTA ends: the last phase of every stage that was filled
      for (int i = 0; i < kStages && i < issued; ++i) {
        const int n           = issued - 1 - i;
        const long long until = now_ns() + kPatience;
        while (!bar_try(full + 8 * (n % kStages), (n / kStages) & 1) && now_ns() < until) {}
      }
    }
  } else if (warp == 1 && rank == 0) {
    int stage = 0, phase = 0, half = 0, turn = 0;
    bool ok = true;
    Tile t;
    for (int i = cluster; ok && tile_of(w, i, t); ok = ok && next_tile(i)) {
      const Product& p      = w.product[t.which];
      const uint32_t idesc  = instruction(w.bf16, p.a_outer, p.b_outer);
      const uint64_t step_a = (p.a_outer ? 2048 : 32) >> 4, step_b = (p.b_outer ? 2048 : 32) >> 4;
      const uint64_t a0     = descriptor(ring, p.a_outer), b0 = descriptor(ring + kStageA, p.b_outer);
      if (!warp_wait(freed + 8 * half, turn ^ 1, &gave_up)) {
        ok = false;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      for (int k = t.begin; k < t.end; ++k) {
        if (!warp_wait(full + 8 * stage, phase, &gave_up)) {
          ok = false;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint64_t a = a0 + stage * (kStage >> 4), b = b0 + stage * (kStage >> 4);
        if (elected()) {
#pragma unroll
          for (int j = 0; j < kDepth / 16; ++j)
            mma(tmem + half * kTile, a + j * step_a, b + j * step_b, idesc, k > t.begin || j > 0);
          commit(empty + 8 * stage);
          if (k + 1 == t.end) commit(done + 8 * half);
        }
        __syncwarp();
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (!ok) break;
      half ^= 1;
      turn ^= half == 0;
    }
    if (!ok) {  // products in flight have to end before TMEM is given back
      if (elected()) commit(last);
      const long long until = now_ns() + kPatience;
      while (!bar_try(last, 0) && now_ns() < until) {}
    }
  } else if (kByTicket && warp == 3 && lane == 0 && rank == 0) {
    // draws tiles, one ahead, and tells both CTAs
    Tile t;
    int i = 0;
    for (int n = 0; tile_of(w, i, t); ++n) {
      const int slot = n & 1;
      if (!bar_wait(heard + 8 * slot, (n >> 1 & 1) ^ 1, &gave_up)) break;
      i = clusters + atomicAdd(w.ticket, 1);
      for (int cta = 0; cta < 2; ++cta) {
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(in_cta(shared_of(const_cast<int*>(tickets) + slot), cta)), "r"(i) : "memory");
        bar_arrive_cluster(in_cta(told + 8 * slot, cta));
      }
    }
  } else if (warp >= 4) {
    const int quarter = warp % 4, from = (warp - 4) / 4 * (kTile / 2);
    const uint32_t freed0 = in_cta(freed, 0);
    int half = 0, turn = 0;
    Tile t;
    bool ok = true;
    for (int i = cluster; ok && tile_of(w, i, t); ok = next_tile(i)) {
      const Product& p  = w.product[t.which];
      const int64_t row = static_cast<int64_t>(t.m) * kTile + rank * kHalf + quarter * 32 + lane;
      const bool in     = row < (KIND == kDiff ? w.plane_rows : p.m);
      float base = 0.f, sum = 1.f, factor = 1.f;
      if (KIND == kDiff && in) {  // (rows up to a plane's end are zeros: they meet zeros, but not as NaN)
        const float4 s = row < p.m ? w.stats[row] : make_float4(0.f, 0.f, 0.f, 0.f);
        base           = base_of(s.x);
        sum            = 1.f / s.y;
        factor         = s.w == 0.f ? 0.f : s.y * w.diff_scale * (w.row_scale ? w.row_scale[row * w.row_step] : 1.f);
      }
      if (KIND == kGrad && !p.sums) factor = w.scale();
      if (!warp_wait(done + 8 * half, turn, &gave_up)) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      Running<float> r;
#pragma unroll 1
      for (int c = from; c < from + kTile / 2; c += 32) {
        const int col = t.n * kTile + c;
        if (KIND != kDiff && col >= p.n) break;
        float x[32];
        load_columns(tmem + half * kTile + c + (static_cast<uint32_t>(quarter * 32) << 16), x);
        if (in) take_columns<KIND>(w, p, t.split, row, col, x, r, base, sum, factor);
        __syncwarp();
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) bar_arrive_cluster(freed0 + 8 * half);
      if (KIND == kDiff && in && factor != 0.f && w.k <= kFewNamed) {  // over what has just been written
        const float per = w.diff_scale * (w.row_scale ? w.row_scale[row * w.row_step] : 1.f), inv = w.stats[row].y;
        const int low = t.n * kTile + from, high = min(low + kTile / 2, p.n);
        for (int j = 0; j < w.k; ++j) {
          const int64_t e = row * w.k + j;
          const int at    = w.named.at[e] - w.first;
          if (at < low || at >= high) continue;
          float d  = (power_within((w.named.logit[e] - base) * w.c, sum) * inv - w.named.p[e]) * per;
          char* to = static_cast<char*>(w.diff) + (row * w.diff_stride + at) * 2;
          for (int plane = 0; plane < w.planes; ++plane, d = left_of(d, w.bf16), to += w.plane_rows * w.diff_stride * 2)
            *reinterpret_cast<uint16_t*>(to) = static_cast<uint16_t>(two(d, 0.f, w.bf16));
        }
      }
      if (KIND == kStats && in) w.parts[(row * p.n_tiles + t.n) * 2 + (from != 0)] = make_float2(r.m, r.s);
      half ^= 1;
      turn ^= half == 0;
    }
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync();
  if (warp == 2) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

// ---- rows ------------------------------------------------------------------------------------
template <class T>
__device__ __forceinline__ float dot_piece(const Piece<T>& a, const Piece<T>& b, float s)
{
#pragma unroll
  for (int i = 0; i < Piece<T>::N; ++i) s = fmaf(widen(a.v[i]), widen(b.v[i]), s);
  return s;
}

// Dot products of h with n rows of w, those that class_of(j) names, by WARPS warps, four at a time: take(j, sum) for
// lane 0 of the warp that has j.  (A class below 0 has none.)
template <class T, int WARPS, class C, class F>
__device__ __forceinline__ void dots(const LinearArgs& a, const T* h, int n, int warp, C class_of, F take)
{
  constexpr int N = Piece<T>::N;
  const int lane  = threadIdx.x % 32;
  for (int j = 4 * warp; j < n; j += 4 * WARPS) {
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    const T* v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int cls = j + u < n ? class_of(j + u) : -1;
      v[u]          = static_cast<const T*>(a.weight) + (cls < 0 ? 0 : cls) * a.weight_stride;
    }
    const int most = min(4, n - j);
    for (int i = lane * N; i < a.width; i += 32 * N) {
      const Piece<T> x = load_piece(h + i);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (u < most) s[u] = dot_piece(x, load_piece(v[u] + i), s[u]);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (u < most) {
        s[u] = sum_lanes(s[u]);
        if (lane == 0) take(j + u, s[u]);
      }
  }
}

// Loss of a row from the maxima and sums of its tiles, by THREADS threads, of which the first warp does what
// concerns the teacher; the named classes' logits are dot products of their own.  Without tiles (small
// problems: a launch less, and logits whose sums do not go through the tensor cores) all logits are.  The
// block that is last to finish adds up all blocks' losses.
template <class T, int THREADS>
__global__ void __launch_bounds__(kThreads) linear_rows(LinearArgs a, const float2* parts, int tiles, Reduced out,
                                                        double2* block_sums, int* ticket)
{
  constexpr int ROWS = kThreads / THREADS, WARPS = THREADS / 32;
  extern __shared__ __align__(16) char smem[];
  __shared__ double2 room[kThreads / 32];
  __shared__ float joins[2 * kThreads / 32];
  __shared__ bool is_last;
  const int slot = threadIdx.x / THREADS, tid = threadIdx.x % THREADS, lane = threadIdx.x % 32;
  const int k        = a.teacher.k;
  char* mine         = smem + slot * (entry_bytes(k) + static_cast<size_t>(k) * 4);
  const Entries e    = entries_at(mine, k);
  float* logit       = reinterpret_cast<float*>(e.at + k);
  const float c      = a.temperature.c;
  const double inv_t = a.temperature.inverse;
  const bool lost    = tiles > 0 && incomplete();
  double sum = 0, count = 0;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + slot; row < a.n_rows;
       row += static_cast<int64_t>(gridDim.x) * ROWS) {
    TeacherRow t{};
    sync_row<THREADS>();
    if (tid < 32) t = read_teacher<false>(a.teacher, row, a.n_cols, inv_t, e);
    sync_row<THREADS>();
    const T* h = static_cast<const T*>(a.hidden) + row * a.hidden_stride;
    dots<T, WARPS>(a, h, k, tid / 32, [&](int j) { return e.at[j]; }, [&](int j, float s) { logit[j] = s; });
    Running<float> r;
    if (tiles > 0) {
      for (int i = tid; i < tiles; i += THREADS) r.join(parts[row * tiles + i].x, parts[row * tiles + i].y, c);
    } else {
      dots<T, WARPS>(a, h, static_cast<int>(a.n_cols), tid / 32, [](int j) { return j; }, [&](int, float s) { r.take(s, c); });
    }
    join_row<THREADS>(r, c, joins);
    sync_row<THREADS>();
    if (tid < 32) {
      const bool counts = t.counts && !(r.s == 0.f);
      double loss = named_loss(e, k, t, inv_t, r.m, log_sum(r.s), [&](int j, int) { return logit[j]; });
      if (!counts) loss = 0;
      if (lost) loss = NAN;
      loss *= a.temperature.t * a.temperature.t;
      for (int j = lane; j < k; j += 32) {
        a.named.logit[row * k + j] = logit[j];
        a.named.p[row * k + j]     = e.p[j];
        a.named.at[row * k + j]    = e.at[j];
      }
      if (lane == 0) {
        a.row_loss[row]  = static_cast<float>(loss);
        a.row_stats[row] = make_float4(r.m, 1.f / r.s, 1.f, counts ? 1.f : 0.f);
        sum += loss;
        count += counts;
      }
    }
  }
  if (out.reduction == 0) return;
  const double2 all = sum_block<kThreads>(sum, count, room);
  if (threadIdx.x == 0) {
    block_sums[blockIdx.x] = all;
    __threadfence();
    is_last = atomicAdd(ticket, 1) == static_cast<int>(gridDim.x) - 1;
  }
  __syncthreads();
  if (!is_last) return;
  __threadfence();
  sum = count = 0;
  for (int i = threadIdx.x; i < static_cast<int>(gridDim.x); i += kThreads) {  // in a fixed order
    sum += __ldcg(&block_sums[i].x);
    count += __ldcg(&block_sums[i].y);
  }
  const double2 total = sum_block<kThreads>(sum, count, room);
  if (threadIdx.x == 0) write_reduced(out, total);
}

// One upstream value per row of an fp16 layer: the rows' are brought below 1 by a power of two, which *scale takes
// back, so that d stays in range.  By one cluster (one block took 280 us for 2^20 rows).
__global__ void __cluster_dims__(kScaleBlocks, 1, 1) __launch_bounds__(1024) grad_scales(LinearGradArgs g, float* scale, float* row_scale)
{
  namespace cg = cooperative_groups;
  __shared__ float room[32], mine;
  const int64_t from = blockIdx.x * 1024 + threadIdx.x;
  float most = 0.f;
#pragma unroll 4
  for (int64_t i = from; i < g.fwd.n_rows; i += kScaleBlocks * 1024) most = fmaxf(most, fabsf(g.upstream[i * g.upstream_stride]));
  most = max_lanes(most);
  if (threadIdx.x % 32 == 0) room[threadIdx.x / 32] = most;
  __syncthreads();
  most = max_lanes(room[threadIdx.x % 32]);
  if (threadIdx.x == 0) mine = most;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  for (int b = 0; b < kScaleBlocks; ++b) most = fmaxf(most, *cluster.map_shared_rank(&mine, b));
  cluster.sync();  // the others' shared memory has been read
  int e = 0;
  if (most > 0.f && most < INFINITY) frexpf(most, &e);
  e                = max(-100, min(100, e));
  const float down = ldexpf(1.f, -e);
  if (from == 0) *scale = ldexpf(1.f, e);
#pragma unroll 4
  for (int64_t i = from; i < g.fwd.n_rows; i += kScaleBlocks * 1024) row_scale[i] = g.upstream[i * g.upstream_stride] * down;
}

// d of the classes that the teacher names, in a piece of the classes.
template <class T>
__global__ void __launch_bounds__(kThreads) named_diff(Work w, int64_t entries, int n)
{
  for (int64_t i = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x; i < entries; i += gridDim.x * static_cast<int64_t>(kThreads)) {
    const int at = w.named.at[i] - w.first;
    if (at < 0 || at >= n) continue;
    const int64_t row = i / w.k;
    const float4 s    = w.stats[row];
    if (s.w == 0.f) continue;
    const float q = power_within((w.named.logit[i] - base_of(s.x)) * w.c, 1.f / s.y) * s.y;
    float d       = (q - w.named.p[i]) * w.diff_scale * (w.row_scale ? w.row_scale[row * w.row_step] : 1.f);
    for (int plane = 0; plane < w.planes; ++plane, d -= widen(narrow<T>(d)))
      static_cast<T*>(w.diff)[(plane * static_cast<int64_t>(w.plane_rows) + row) * w.diff_stride + at] = narrow<T>(d);
  }
}

// A gradient from the sums of its parts.
template <class T>
__global__ void __launch_bounds__(kThreads) finish_sums(const float* sums, int splits, int64_t n, Scale scale, T* out)
{
  const float f = scale();
  for (int64_t i = 4 * (blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x); i < n; i += 4 * gridDim.x * static_cast<int64_t>(kThreads)) {
    float4 v = *reinterpret_cast<const float4*>(sums + i);
    for (int s = 1; s < splits; ++s) {
      const float4 o = *reinterpret_cast<const float4*>(sums + s * n + i);
      v              = make_float4(v.x + o.x, v.y + o.y, v.z + o.z, v.w + o.w);
    }
    T r[4] = {narrow<T>(v.x * f), narrow<T>(v.y * f), narrow<T>(v.z * f), narrow<T>(v.w * f)};
    *reinterpret_cast<uint2*>(out + i) = *reinterpret_cast<const uint2*>(r);
  }
}

// The same for rows of `width` of `pitch` columns: four results per thread, which may be in two rows (or more).
template <class T>
__global__ void __launch_bounds__(kThreads) finish_rows(const float* sums, int splits, int64_t rows, int pitch, int width,
                                                        Scale scale, T* out)
{
  const float f     = scale();
  const int64_t all = rows * width;
  for (int64_t i = 4 * (blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x); i < all; i += 4 * gridDim.x * static_cast<int64_t>(kThreads)) {
    int64_t r = i / width;
    int c     = static_cast<int>(i - r * width);
    T v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float x = 0.f;
      if (i + j < all)
        for (int s = 0; s < splits; ++s) x += sums[(s * rows + r) * pitch + c];
      v[j] = narrow<T>(x * f);
      if (++c == width) {
        c = 0;
        ++r;
      }
    }
    if (i + 3 < all) {
      *reinterpret_cast<uint2*>(out + i) = *reinterpret_cast<const uint2*>(v);
    } else {
      for (int j = 0; i + j < all; ++j) out[i + j] = v[j];
    }
  }
}

// Rows of `width` elements to rows of `pitch` (a multiple of 8) with zeros behind: 16 bytes per thread.
template <class T>
__global__ void __launch_bounds__(kThreads) pad_rows(const T* from, int64_t stride, int64_t rows, int width, int pitch, T* to)
{
  const int per     = pitch / 8;
  const int64_t all = rows * per;
  for (int64_t i = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x; i < all; i += gridDim.x * static_cast<int64_t>(kThreads)) {
    const int64_t r = i / per;
    const int c     = static_cast<int>(i - r * per) * 8;
    Piece<T> v;
#pragma unroll
    for (int j = 0; j < 8; ++j) v.v[j] = c + j < width ? from[r * stride + c + j] : narrow<T>(0.f);
    *reinterpret_cast<uint4*>(to + i * 8) = *reinterpret_cast<const uint4*>(&v);
  }
}

__global__ void no_rows(Reduced out) { write_reduced(out, make_double2(0, 0)); }

__global__ void wait_for_nothing()
{
  __shared__ __align__(8) uint64_t bar;
  __shared__ volatile int gave_up;
  gave_up = 0;
  bar_init(shared_of(&bar), 1);
  bar_wait_long(shared_of(&bar), 0, &gave_up, 1000000ll);
}

// ---- host ------------------------------------------------------------------------------------
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encoder()
{
  static EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}
// A matrix of `rows` rows of `cols` 16-bit elements, in boxes of 64 columns by box_rows rows.
bool make_map(CUtensorMap* map, bool bf16, const void* base, int64_t rows, int64_t cols, int64_t stride, int box_rows)
{
  const EncodeFn encode    = encoder();
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t step[1] = {static_cast<cuuint64_t>(stride) * 2};
  const cuuint32_t box[2] = {64, static_cast<cuuint32_t>(box_rows)}, one[2] = {1, 1};
  return encode && encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
                          const_cast<void*>(base), dims, step, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
int tiles_of(int64_t n) { return static_cast<int>((n + kTile - 1) / kTile); }

template <int KIND>
cudaError_t run_products(const Work& w, int n_sms, cudaStream_t s)
{
  const cudaError_t e = cudaFuncSetAttribute(products<KIND>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e != cudaSuccess) return e;
  int tiles = 0;
  for (int i = 0; i < w.products; ++i) tiles += w.product[i].m_tiles * w.product[i].n_tiles * w.product[i].splits;
  const int clusters = tiles < n_sms / 2 ? tiles : n_sms / 2;
  products<KIND><<<2 * clusters, kProductThreads, kSmem, s>>>(w);
  return cudaGetLastError();
}

// The kernels read 16 bytes at a time, rows that start on them and end with whole pieces.  Others are copied, with
// zeros behind each row, which change no product; so are large ones off the 32-byte sectors, which are read a
// quarter slower (4096 x 1032 x 16,384, loss and gradient: 501 us, with 1040 or 1024 columns 380).
struct Layer {
  bool copied;
  int64_t width;         // of a row as the kernels read it
  int64_t bytes;         // of the copies
};
int64_t padded(int64_t bytes) { return (bytes + 255) / 256 * 256; }
Layer layer_of(const LinearArgs& a)
{
  Layer l;
  l.copied = a.width % 8 || a.hidden_stride % 8 || a.weight_stride % 8 || reinterpret_cast<uintptr_t>(a.hidden) % 16 ||
             reinterpret_cast<uintptr_t>(a.weight) % 16 ||
             ((a.width % 16 || a.hidden_stride % 16 || a.weight_stride % 16) && a.n_rows * a.n_cols >= (1ll << 36) / a.width);
  l.width = l.copied ? (a.width + 15) / 16 * 16 : a.width;
  l.bytes = l.copied ? padded(a.n_rows * l.width * 2) + padded(a.n_cols * l.width * 2) : 0;
  return l;
}
// `a` with the layer as the kernels read it; copies go to `at`, which is moved behind them.
template <class T>
cudaError_t give_layer(LinearArgs& a, const Layer& l, char*& at, int n_sms, cudaStream_t s)
{
  if (!l.copied) return cudaSuccess;
  T* hidden = reinterpret_cast<T*>(at);
  T* weight = reinterpret_cast<T*>(at + padded(a.n_rows * l.width * 2));
  at += l.bytes;
  auto pad = [&](const void* from, int64_t stride, int64_t rows, T* to) {
    const int64_t need = (rows * l.width / 8 + kThreads - 1) / kThreads, most = 16ll * n_sms;
    pad_rows<T><<<static_cast<unsigned>(need < most ? need : most), kThreads, 0, s>>>(
      static_cast<const T*>(from), stride, rows, static_cast<int>(a.width), static_cast<int>(l.width), to);
  };
  pad(a.hidden, a.hidden_stride, a.n_rows, hidden);
  pad(a.weight, a.weight_stride, a.n_cols, weight);
  a.hidden = hidden;
  a.weight = weight;
  a.width = a.hidden_stride = a.weight_stride = l.width;
  count_launches(2);
  return cudaGetLastError();
}

// z = H W^T of the classes from `first` on
bool logits_product(Product& p, bool bf16, const LinearArgs& a, int64_t first, int64_t n)
{
  p.m       = static_cast<int>(a.n_rows);
  p.n       = static_cast<int>(n);
  p.depth   = static_cast<int>(a.width);
  p.m_tiles = tiles_of(p.m);
  p.n_tiles = tiles_of(p.n);
  p.splits = p.planes = 1;
  p.plane_rows = 0;
  p.a_outer = p.b_outer = 0;
  p.n_first = 0;
  return make_map(&p.a, bf16, a.hidden, a.n_rows, a.width, a.hidden_stride, kHalf) &&
         make_map(&p.b, bf16, static_cast<const char*>(a.weight) + first * a.weight_stride * 2, n, a.width, a.weight_stride, kHalf);
}

template <class T>
cudaError_t run_linear(bool bf16, const LinearArgs& given, const Reduced& out, void* workspace, int n_sms, cudaStream_t s)
{
  LinearArgs a = given;
  if (a.n_rows == 0) {
    if (out.reduction != 0) no_rows<<<1, 1, 0, s>>>(out);
    count_launches(out.reduction != 0);
    return cudaGetLastError();
  }
  char* at      = static_cast<char*>(workspace);
  cudaError_t e = give_layer<T>(a, layer_of(given), at, n_sms, s);
  if (e != cudaSuccess) return e;
  double2* sums = reinterpret_cast<double2*>(at);
  Work w{};
  w.products = 1;
  w.bf16     = bf16;
  w.c        = a.temperature.c;
  w.ticket   = reinterpret_cast<int*>(sums + 8 * n_sms);
  w.parts    = reinterpret_cast<float2*>(sums + 8 * n_sms + 1);
  const bool small = a.n_cols <= kFewClasses && a.n_rows * a.n_cols <= kSmallLogits / a.width;
  if (small) {
    if (out.reduction != 0) e = cudaMemsetAsync(w.ticket, 0, sizeof(int), s);
  } else {
    if (!logits_product(w.product[0], bf16, a, 0, a.n_cols)) return cudaErrorInvalidValue;
    e = run_products<kStats>(w, n_sms, s);
  }
  if (e != cudaSuccess) return e;
  const int tiles = small ? 0 : 2 * w.product[0].n_tiles;
  // a warp per row where there are enough rows (or nothing to share), else a block
  const bool warp    = (a.teacher.k <= 4 && !(small && a.n_cols > 8)) || a.n_rows >= 8 * n_sms;
  const int per      = warp ? kThreads / 32 : 1;
  const int64_t need = (a.n_rows + per - 1) / per;
  const int blocks   = static_cast<int>(need < 8 * n_sms ? need : 8 * n_sms);
  const size_t bytes = per * (entry_bytes(a.teacher.k) + static_cast<size_t>(a.teacher.k) * 4);
  if (warp)
    linear_rows<T, 32><<<blocks, kThreads, bytes, s>>>(a, w.parts, tiles, out, sums, w.ticket);
  else
    linear_rows<T, kThreads><<<blocks, kThreads, bytes, s>>>(a, w.parts, tiles, out, sums, w.ticket);
  count_launches(small ? 1 : 2);
  return cudaGetLastError();
}

// How the classes are cut into pieces and the sums over classes and rows into parts.
struct Plan {
  int pieces;
  int64_t cols;                 // of a piece, a multiple of a tile
  int planes;                   // of d
  int64_t plane_rows;
  int splits_hidden, splits_weight;
  bool sums_hidden, sums_weight;  // in memory
};
Plan plan_of(const LinearGradArgs& g, const Layer& l, int n_sms)
{
  const LinearArgs& a = g.fwd;
  Plan p;
  int64_t most = kPieceBytes / 2 / (a.n_rows > 0 ? a.n_rows : 1) / kTile * kTile;
  if (most < 2 * kTile) most = 2 * kTile;
  p.pieces = static_cast<int>((a.n_cols + most - 1) / most);
  p.cols   = static_cast<int64_t>(tiles_of((a.n_cols + p.pieces - 1) / p.pieces)) * kTile;
  p.pieces = static_cast<int>((a.n_cols + p.cols - 1) / p.cols);
  p.planes     = a.n_rows * a.n_cols <= kSmallProduct / l.width ? 2 : 1;
  p.plane_rows = (a.n_rows + kDepth - 1) / kDepth * kDepth;
  // as many parts as bring a part down to an even share of the machine, 32 stages at least: fewer are not worth
  // the kernel that joins them (2048 x 512 x 1000: 23.0 us with 16, 22.8 with 32 and a launch less)
  const int64_t wide = tiles_of(l.width), dh_tiles = tiles_of(a.n_rows) * wide, dw_tiles = tiles_of(p.cols) * wide;
  const int64_t dh_steps = p.planes * (p.cols / kDepth), dw_steps = p.planes * (p.plane_rows / kDepth);
  int64_t share = ((g.grad_hidden ? dh_tiles * dh_steps : 0) + (g.grad_weight ? dw_tiles * dw_steps : 0)) / (n_sms / 2);
  if (share < 32) share = 32;
  auto parts = [&](int64_t steps) {
    const int64_t n = (steps + share - 1) / share;
    return static_cast<int>(n < 1 ? 1 : n > kMostSplits ? kMostSplits : n);
  };
  p.splits_hidden = parts(dh_steps);
  p.splits_weight = parts(dw_steps);
  p.sums_hidden   = g.grad_hidden && (p.pieces > 1 || p.splits_hidden > 1 || l.width != a.width);
  p.sums_weight   = g.grad_weight && (p.splits_weight > 1 || l.width != a.width);
  return p;
}

template <class T>
cudaError_t finish(const float* sums, int splits, int64_t rows, int64_t pitch, int64_t width, const Scale& scale, void* out,
                   int n_sms, cudaStream_t s)
{
  const int64_t n = rows * width, most = 8ll * n_sms;
  if (pitch == width) {
    const int64_t need = (n / 4 + kThreads - 1) / kThreads;
    finish_sums<T><<<static_cast<unsigned>(need < most ? need : most), kThreads, 0, s>>>(sums, splits, n, scale, static_cast<T*>(out));
  } else {
    const int64_t need = (n / 4 + kThreads) / kThreads;
    finish_rows<T><<<static_cast<unsigned>(need < most ? need : most), kThreads, 0, s>>>(
      sums, splits, rows, static_cast<int>(pitch), static_cast<int>(width), scale, static_cast<T*>(out));
  }
  return cudaGetLastError();
}

template <class T>
cudaError_t run_linear_grad(bool bf16, const LinearGradArgs& g, void* workspace, int n_sms, cudaStream_t s)
{
  LinearArgs a        = g.fwd;
  const int64_t width = a.width;  // of the gradients' rows
  const Layer layer   = layer_of(a);
  const Plan plan     = plan_of(g, layer, n_sms);
  char* at            = static_cast<char*>(workspace);
  cudaError_t e       = give_layer<T>(a, layer, at, n_sms, s);
  if (e != cudaSuccess) return e;
  float* scale         = reinterpret_cast<float*>(at);
  int* ticket          = reinterpret_cast<int*>(at + 16);
  float* row_scale     = reinterpret_cast<float*>(at += 256);
  T* diff              = reinterpret_cast<T*>(at += padded(a.n_rows * 4));
  float* sums_hidden   = reinterpret_cast<float*>(at += padded(plan.planes * plan.plane_rows * plan.cols * 2));
  float* sums_weight   = reinterpret_cast<float*>(at + (plan.sums_hidden ? plan.splits_hidden * a.n_rows * a.width * 4 : 0));
  const float d_scale  = bf16 ? 1.f : kHalfScale;
  const bool per_row   = g.factor == nullptr;
  const bool scaled    = per_row && !bf16;  // (bf16 has the range of the upstream values itself)
  int launched         = scaled;
  if (scaled) grad_scales<<<kScaleBlocks, 1024, 0, s>>>(g, scale, row_scale);
  Work w{};
  w.bf16        = bf16;
  w.c           = a.temperature.c;
  w.stats       = a.row_stats;
  w.row_scale   = scaled ? row_scale : per_row ? g.upstream : nullptr;
  w.row_step    = scaled ? 1 : g.upstream_stride;
  w.diff        = diff;
  w.diff_stride = plan.cols;
  w.diff_scale  = d_scale;
  w.planes      = plan.planes;
  w.plane_rows  = static_cast<int>(plan.plane_rows);
  w.scale       = Scale{scaled ? scale : per_row ? nullptr : g.upstream, g.factor, static_cast<float>(a.temperature.t) / d_scale};
  w.named       = a.named;
  w.k           = a.teacher.k;
  w.ticket      = ticket;
  for (int i = 0; i < plan.pieces; ++i) {
    const int64_t first = i * plan.cols, n = a.n_cols - first < plan.cols ? a.n_cols - first : plan.cols;
    w.products = 1;
    w.first    = static_cast<int>(first);
    if (!logits_product(w.product[0], bf16, a, first, n)) return cudaErrorInvalidValue;
    if ((e = run_products<kDiff>(w, n_sms, s)) != cudaSuccess) return e;
    if (w.k > kFewNamed) {
      const int64_t entries = a.n_rows * w.k, need = (entries + kThreads - 1) / kThreads;
      named_diff<T><<<static_cast<unsigned>(need < 8 * n_sms ? need : 8 * n_sms), kThreads, 0, s>>>(w, entries, static_cast<int>(n));
      ++launched;
    }
    // d ends with the tile that holds its last class: what is behind has not been written
    const int64_t made = static_cast<int64_t>(tiles_of(n)) * kTile;
    const char* weight = static_cast<const char*>(a.weight) + first * a.weight_stride * 2;
    T* grad_weight     = g.grad_weight ? static_cast<T*>(g.grad_weight) + first * width : nullptr;
    w.products         = 0;
    auto hidden = [&] {
      if (!g.grad_hidden) return true;
      Product& p = w.product[w.products++];
      p.m        = static_cast<int>(a.n_rows);
      p.depth    = static_cast<int>(made);
      // (a short last piece adds to the first of them; the first piece has written all)
      p.splits = static_cast<int>(std::min<int64_t>(plan.splits_hidden, plan.planes * (made / kDepth)));
      p.a_outer  = 0;
      p.sums     = plan.sums_hidden ? sums_hidden : nullptr;
      p.add      = i > 0;
      p.out      = g.grad_hidden;
      return make_map(&p.a, bf16, diff, plan.planes * plan.plane_rows, made, plan.cols, kHalf) &&
             make_map(&p.b, bf16, weight, n, a.width, a.weight_stride, 64);
    };
    auto of_weight = [&] {
      if (!g.grad_weight) return true;
      Product& p = w.product[w.products++];
      p.m        = static_cast<int>(n);
      p.depth    = static_cast<int>(a.n_rows);
      p.splits   = plan.splits_weight;
      p.a_outer  = 1;
      p.sums     = plan.sums_weight ? sums_weight : nullptr;
      p.add      = 0;
      p.out      = grad_weight;
      return make_map(&p.a, bf16, diff, plan.planes * plan.plane_rows, made, plan.cols, 64) &&
             make_map(&p.b, bf16, a.hidden, a.n_rows, a.width, a.hidden_stride, 64);
    };
    // the longer sums first: what is left at the end is short
    const bool hidden_first = made / plan.splits_hidden >= a.n_rows / plan.splits_weight;
    if (!(hidden_first ? hidden() && of_weight() : of_weight() && hidden())) return cudaErrorInvalidValue;
    for (int j = 0; j < w.products; ++j) {
      Product& p = w.product[j];
      p.n        = static_cast<int>(a.width);
      p.b_outer  = 1;
      p.m_tiles  = tiles_of(p.m);
      p.n_tiles  = tiles_of(p.n);
      p.planes     = plan.planes;
      p.plane_rows = static_cast<int>(plan.plane_rows);
      p.n_first  = 1;  // d is read once, by all the tiles of a row of them at the same time
    }
    if ((e = run_products<kGrad>(w, n_sms, s)) != cudaSuccess) return e;
    launched += 2;
    if (plan.sums_weight) {
      if ((e = finish<T>(sums_weight, plan.splits_weight, n, a.width, width, w.scale, grad_weight, n_sms, s)) != cudaSuccess) return e;
      ++launched;
    }
  }
  if (plan.sums_hidden) {
    e = finish<T>(sums_hidden, plan.splits_hidden, a.n_rows, a.width, width, w.scale, g.grad_hidden, n_sms, s);
    ++launched;
  }
  count_launches(launched);
  return e;
}

}  // namespace

size_t linear_workspace(const LinearArgs& a, int n_sms)
{
  return layer_of(a).bytes + (8 * n_sms + 1) * sizeof(double2) +
         a.n_rows * static_cast<size_t>(2 * tiles_of(a.n_cols)) * sizeof(float2);
}

size_t linear_grad_workspace(const LinearGradArgs& g, int n_sms)
{
  const LinearArgs& a = g.fwd;
  const Layer l       = layer_of(a);
  const Plan p        = plan_of(g, l, n_sms);
  return l.bytes + 256 + padded(a.n_rows * 4) + padded(p.planes * p.plane_rows * p.cols * 2) +
         (p.sums_hidden ? p.splits_hidden * a.n_rows * l.width * sizeof(float) : 0) +
         (p.sums_weight ? p.splits_weight * p.cols * l.width * sizeof(float) : 0);
}

cudaError_t launch_linear(int dtype, const LinearArgs& a, const Reduced& out, void* workspace, int n_sms, cudaStream_t s)
{
  return dtype == kBF16 ? run_linear<__nv_bfloat16>(true, a, out, workspace, n_sms, s)
                        : run_linear<__half>(false, a, out, workspace, n_sms, s);
}

cudaError_t launch_linear_grad(int dtype, const LinearGradArgs& g, void* workspace, int n_sms, cudaStream_t s)
{
  return dtype == kBF16 ? run_linear_grad<__nv_bfloat16>(true, g, workspace, n_sms, s)
                        : run_linear_grad<__half>(false, g, workspace, n_sms, s);
}

cudaError_t linear_status(int* status)
{
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(status, g_status, sizeof(int));
  if (e == cudaSuccess && *status != 0) {
    const int zero = 0;
    e              = cudaMemcpyToSymbol(g_status, &zero, sizeof(int));
  }
  return e;
}

cudaError_t launch_linear_timeout(cudaStream_t s)
{
  wait_for_nothing<<<1, 1, 0, s>>>();
  return cudaGetLastError();
}

}  // namespace distill
}  // namespace b2fil
