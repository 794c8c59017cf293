// Drawing one entry per row of logits: temperature, top-k, top-p, min-p, inverse of the cumulative sum at a given random number.
//
// With m the row's largest logit and w(l) = exp((l - m) / T), an entry's weight, entries in the order of falling logits (equal
// logits: lower index first): top-k keeps the first k; top-p those ahead of which the weights sum to less than p S, S the sum of what
// top-k kept; min-p those with w >= min_p.  Each cut keeps a front part of the order, so a row is never sorted: a cut is a logit and,
// among the entries that equal it, an index.  The draw runs over the indices: the first kept i with sum_{j <= i, kept} w_j > u W.
//
// The answer is a whole number, so it has to be the one that exact sums give.  Sums of fp32 weights decide where they can: with an
// error of at most e S (SampleParams::slack) a comparison that is closer than e S is open, and what it belongs to, the cut or the
// draw, is done again with weights and sums in 64 bits (spread 1.5: of 1858 logits 0.7 % of the draws and 1.4 % of the top-p cuts, of
// 50257 bf16 logits 7.7 % and 9.4 %).
//
// A row is held in shared memory as fp32 by a group of threads: a warp, a CTA or a cluster of CTAs.  Thread t owns a run of consecutive
// entries (an odd number of 16-byte pieces: no bank conflicts), so that sums over threads run in the order of the indices.
#include <cooperative_groups.h>

#include <atomic>

#include "../../include/b200nn.h"
#include "kernels.cuh"

namespace cg = cooperative_groups;

namespace b200 {
namespace {

constexpr int kMaxCluster = 8;
constexpr int kWide = 256;              // threads of a CTA that has a row, or a part of one
constexpr int kMaxPieces = 33;          // 16-byte pieces per thread there: 132 KB
constexpr int kWarpRows = 4;            // rows of a CTA whose groups are warps
static_assert(kMaxCluster * kWide * kMaxPieces * 4 >= B200_SAMPLE_MAX_WIDTH + 8, "the widest row fits a cluster");

struct SampleParams {
  const void* logits; long long ld;
  int rows, width;
  const unsigned short* ids; const int* counts; int ld_ids;
  const float* temperature; const int* top_k; const float* top_p; const float* min_p; const float* u;
  int* choice; float* prob;
  int pieces;   // 16-byte pieces per thread, odd
  int cluster;  // CTAs per row (kCluster)
  int ahead;    // rows of one round of CTAs
  float slack;  // bound of a sum's error, relative to the sum of all weights
  unsigned long long wait_ns;  // after which a wait for the other CTAs of a cluster gives up
  int give_up_cta, give_up_at;  // for tests: this CTA of each cluster gives up at its wait of this number; -1: none
};

// Larger keys are larger logits; -0 and +0 have one key.
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// The threads of a row: sums, maxima and prefix sums over them in a fixed order.
template <int kThreads, bool kCluster> struct Group {
  static constexpr int kWarps = kThreads / 32;
  static constexpr int kSlots = kCluster ? kMaxCluster * kWarps : kWarps;
  double* slots;  // [2][kSlots], kThreads > 32
  float* wide;    // [2][kSlots][4]
  uint64_t* bars;  // [2] for exchanges, one for meetings; kCluster
  int cluster, crank, turn, meetings;
  unsigned long long wait_ns;
  int give_up_at;
  // A wait for the other CTAs has ended without them: the same in all threads of a CTA, which then make no further exchange (sums are 0,
  // maxima -infinity, whatever has arrived) and leave.  The others' waits end the same way, so that every thread gets to the
  // two cluster barriers of the hardware, which have no limit: one before the first exchange, one before the end.
  bool gave_up;
  int lane, warp;
  __device__ Group(double* s, float* s4, uint64_t* b, const SampleParams& p)
      : slots(s), wide(s4), bars(b), cluster(kCluster ? p.cluster : 1), crank(0), turn(0), meetings(0), wait_ns(p.wait_ns), give_up_at(-1), gave_up(false) {
    lane = threadIdx.x & 31;
    warp = kThreads == 32 ? 0 : threadIdx.x >> 5;
    if (kCluster) {
      crank = (int)cg::this_cluster().block_rank();
      if (crank == p.give_up_cta) give_up_at = p.give_up_at;
      if (threadIdx.x < 3)
        asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(address(bars + threadIdx.x)), "r"(threadIdx.x < 2 ? 1 : cluster) : "memory");
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");  // (the row is read, and a barrier passed, before their first use)
    }
  }
  static __device__ __forceinline__ uint32_t address(const void* q) { return (uint32_t)__cvta_generic_to_shared(q); }
  static __device__ __forceinline__ uint32_t address(const void* q, int cta) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(address(q)), "r"(cta));
    return a;
  }
  // The CTAs of a cluster hand values around by stores that count themselves in at the receiver's barrier: 2 k cycles less per exchange
  // than a cluster barrier, which waits for all the memory traffic of the threads that arrive.  `bytes`: what a CTA receives this turn.
  __device__ __forceinline__ void expect(int bytes) const {
    if (threadIdx.x == 0)
      asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(address(bars + (turn & 1))), "r"(bytes) : "memory");
  }
  __device__ __forceinline__ void wait(const uint64_t* b, uint32_t parity) {
    const uint32_t bar = address(b);
    unsigned long long t0 = 0;
    gave_up = turn + meetings == give_up_at;
    for (int it = 0; !gave_up; ++it) {
      uint32_t ok;
      asm volatile(
          "{\n\t.reg .pred p;\n\t"
          "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
          "selp.u32 %0, 1, 0, p;\n\t}"
          : "=r"(ok)
          : "r"(bar), "r"(parity), "r"(20000u)
          : "memory");
      if (ok) break;
      if ((it & 63) == 63) {
        unsigned long long now;
        asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
        if (t0 == 0) t0 = now;
        gave_up = now - t0 > wait_ns;
      }
    }
    gave_up = __syncthreads_or(gave_up) != 0;
  }
  __device__ __forceinline__ void await() {
    wait(bars + (turn & 1), turn >> 1 & 1);
    ++turn;
  }
  // All threads of the cluster, and what they have written to shared memory: a barrier with a limit.
  __device__ __forceinline__ void meet() {
    __syncthreads();
    if (gave_up) return;
    if ((int)threadIdx.x < cluster)
      asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(address(bars + 2, threadIdx.x)) : "memory");
    wait(bars + 2, meetings & 1);
    ++meetings;
  }
  __device__ __forceinline__ int thread() const { return (crank * kWarps + warp) * 32 + lane; }
  __device__ __forceinline__ int threads() const { return cluster * kThreads; }
  __device__ __forceinline__ void barrier() {
    if (kThreads == 32) __syncwarp();
    else if (kCluster) meet();
    else __syncthreads();
  }
  // One value per warp, seen by all threads of the group afterwards.  Two sets of slots in turn: the barrier of one exchange
  // lies between the reads of the last and the writes of the next.
  __device__ __forceinline__ const double* gather(double v) {
    double* mine = slots + (turn & 1) * kSlots;
    if (kCluster) {
      if (gave_up) return mine;
      expect(cluster * kWarps * 8);
      if (lane < cluster)
        asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b64 [%0], %1, [%2];" ::"r"(address(mine + crank * kWarps + warp, lane)),
                     "l"(__double_as_longlong(v)), "r"(address(bars + (turn & 1), lane))
                     : "memory");
      await();
      return mine;
    }
    ++turn;
    if (lane == 0) mine[warp] = v;
    __syncthreads();
    return mine;
  }
  __device__ __forceinline__ double sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (kThreads == 32) return v;
    const double* s = gather(v);
    if (kCluster && gave_up) return 0.0;
    double t = 0.0;
    for (int i = lane; i < cluster * kWarps; i += 32) t += s[i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    return t;
  }
  __device__ __forceinline__ float max(float v) {
    v = of_key(__reduce_max_sync(0xffffffffu, key_of(v)));
    if (kThreads == 32) return v;
    const double* s = gather((double)v);
    if (kCluster && gave_up) return -INFINITY;
    uint32_t t = 0;
    for (int i = lane; i < cluster * kWarps; i += 32) t = ::max(t, key_of((float)s[i]));
    return of_key(__reduce_max_sync(0xffffffffu, t));
  }
  // Sums of four values at once, in a fixed order, for places to look in.
  __device__ __forceinline__ void sum4(float (&a)[4]) {
    // halving exchange: a lane is left with value lane >> 3 of its warp
    auto halve = [&](bool upper, int o, float& low, float high) {
      const float send = upper ? low : high, keep = upper ? high : low;
      low = keep + __shfl_xor_sync(0xffffffffu, send, o);
    };
    halve((lane & 16) != 0, 16, a[0], a[2]);
    halve((lane & 16) != 0, 16, a[1], a[3]);
    halve((lane & 8) != 0, 8, a[0], a[1]);
    float v = a[0];
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (kThreads > 32) {
      float* mine = wide + (turn & 1) * kSlots * 4;
      const int at = (crank * kWarps + warp) * 4 + (lane >> 3);
      if (kCluster) {
        if (!gave_up) {
          expect(cluster * kWarps * 16);
          if ((lane & 7) < cluster)
            asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(address(mine + at, lane & 7)),
                         "r"(__float_as_uint(v)), "r"(address(bars + (turn & 1), lane & 7))
                         : "memory");
          await();
        }
        if (gave_up) {
          a[0] = a[1] = a[2] = a[3] = 0.f;
          return;
        }
      } else {
        ++turn;
        if ((lane & 7) == 0) mine[at] = v;
        __syncthreads();
      }
      v = 0.f;
      for (int w = lane & 7; w < cluster * kWarps; w += 8) v += mine[w * 4 + (lane >> 3)];
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = __shfl_sync(0xffffffffu, v, j * 8);
  }
  // Sum over the threads before this one; `total` over all.
  __device__ __forceinline__ double before(double v, double& total) {
    double in = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double up = __shfl_up_sync(0xffffffffu, in, o);
      if (lane >= o) in += up;
    }
    const double warp_total = __shfl_sync(0xffffffffu, in, 31);
    double ex = __shfl_up_sync(0xffffffffu, in, 1);
    if (lane == 0) ex = 0.0;
    if (kThreads == 32) {
      total = warp_total;
      return ex;
    }
    const double* s = gather(warp_total);
    if (kCluster && gave_up) {
      total = 0.0;
      return 0.0;
    }
    // every warp scans the warps' sums in the same order, a few per lane
    constexpr int kEach = (kSlots + 31) / 32;
    const int mine = crank * kWarps + warp;
    double part[kEach], sum = 0.0, ahead = 0.0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      part[i] = sum;
      const int at = lane * kEach + i;
      if (at < cluster * kWarps) sum += s[at];
    }
    double run = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double up = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += up;
    }
    total = __shfl_sync(0xffffffffu, run, 31);
    run = __shfl_up_sync(0xffffffffu, run, 1);
    if (lane == 0) run = 0.0;
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (i == mine % kEach) ahead = run + part[i];
    return __shfl_sync(0xffffffffu, ahead, mine / kEach) + ex;
  }
};

// e^x in 64 bits for kN values x <= 0, side by side and without a branch (one after the other each step waits for the last): x = k ln 2 + r
// with ln 2 in two pieces (Cody and Waite), the Taylor series of e^r up to r^13 (|r| <= 0.35: the next term is 1e-17), times 2^k in
// two halves, whose product may be subnormal.
template <int kN> __device__ __forceinline__ void exp_below(double (&x)[kN]) {
  double r[kN], s[kN];
  int n[kN];
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    const double y = fmax(x[i], -760.0), k = rint(y * 1.4426950408889634);
    r[i] = fma(k, -0x1.abc9e3b39803fp-56, fma(k, -0x1.62e42fefa39efp-1, y));
    n[i] = (int)k;
    s[i] = 1.0 / 6227020800.0;
  }
  constexpr double kInverse[13] = {1.0 / 479001600.0, 1.0 / 39916800.0, 1.0 / 3628800.0, 1.0 / 362880.0, 1.0 / 40320.0, 1.0 / 5040.0, 1.0 / 720.0,
                                   1.0 / 120.0, 1.0 / 24.0, 1.0 / 6.0, 0.5, 1.0, 1.0};
#pragma unroll
  for (int c = 0; c < 13; ++c)
#pragma unroll
    for (int i = 0; i < kN; ++i) s[i] = fma(s[i], r[i], kInverse[c]);
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    const int half = n[i] >> 1;
    x[i] = s[i] * __hiloint2double((half + 1023) << 20, 0) * __hiloint2double((n[i] - half + 1023) << 20, 0);
  }
}
// Weights in fp32 or in 64 bits, of a row whose largest logit is finite.  kFine: the rounding of l - m is made good.  The rows of a warp do
// without, at the price of a wider bound: 1.4 % of them have their top-p cut done again in 64 bits.  Wider rows, whose sums have more
// terms, keep it.
template <bool kFine> struct Weight {
  float half_max, c, c_lo, max, temp;
  double inv_t;
  __device__ Weight(float m, float t) : max(m), temp(t) {
    inv_t = 1.0 / (double)t;
    const double e = 2.8853900817779268 * inv_t;  // 2 log2(e) / T
    half_max = 0.5f * m;
    c = (float)fmin(e, 1e37);
    c_lo = (float)(fmin(e, 1e37) - (double)c);
  }
  // (beyond, temperatures of 1e-37 or 1e+30, c or its second piece leaves the range of fp32)
  __device__ bool fp32_usable() const { return c < 1e37f && c > 1e-30f; }
  // 2^((l - m) log2(e) / T), the difference (of halves, since l - m can overflow) and the exponent each in two pieces.  No branch: passes
  // over a row live on several entries being in work at once.
  __device__ __forceinline__ float get(float l, float) const {
    const float a = 0.5f * l, x = a - half_max;
    float x_lo = 0.f;
    if constexpr (kFine) {
      const float b = x - a;
      x_lo = (a - (x - b)) - (half_max + b);
    }
    const float z = x * c;
    float lo = fmaf(x, c_lo, fmaf(x, c, -z));
    if constexpr (kFine) lo = fmaf(x_lo, c, lo);
    float w;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(z));
    w = fmaf(w, lo * 0.69314718f, w);
    return z > -126.f ? w : 0.f;
  }
  // within 1e-5 of it
  __device__ __forceinline__ float quick(float l) const {
    float w;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(fmaf(l, 0.5f, -half_max) * c));
    return l > -INFINITY ? w : 0.f;
  }
  __device__ __forceinline__ double exponent(float l) const { return l > -INFINITY ? ((double)l - (double)max) * inv_t : -1e9; }
  __device__ __forceinline__ double get(float l, double) const {
    double x[1] = {exponent(l)};
    exp_below(x);
    return x[0];
  }
  template <typename W> __device__ __forceinline__ void get4(const float (&l)[4], W (&w)[4]) const {
    if constexpr (sizeof(W) == 4) {
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = get(l[j], 0.f);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = exponent(l[j]);
      exp_below(w);
    }
  }
};

template <typename T> struct Pieces;  // 16 bytes of logits as fp32
template <> struct Pieces<float> {
  static constexpr int n = 4;
  static __device__ __forceinline__ void get(uint4 v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
  }
};
template <> struct Pieces<__half> {
  static constexpr int n = 8;
  static __device__ __forceinline__ void get(uint4 v, float (&f)[8]) {
    const __half2* h = reinterpret_cast<const __half2*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float2 p = __half22float2(h[i]); f[2 * i] = p.x; f[2 * i + 1] = p.y; }
  }
};
template <> struct Pieces<__nv_bfloat16> {
  static constexpr int n = 8;
  static __device__ __forceinline__ void get(uint4 v, float (&f)[8]) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float2 p = __bfloat1622float2(h[i]); f[2 * i] = p.x; f[2 * i + 1] = p.y; }
  }
};

// A row's entries into shared memory; slot `first` + i holds entry i, -inf where there is none.  Whole 16-byte pieces of memory are read
// with one load, eight of a thread on their way at a time, those that reach beyond the row entry by entry.  (NaN stays: every
// comparison that would take it in is false, and its weight is 0.)
template <typename T, int kThreads, bool kCluster>
__device__ int load_row(const SampleParams& p, const Group<kThreads, kCluster>& g, int row, float* v, int cap, int& n) {
  const T* src = static_cast<const T*>(p.logits) + (long long)row * p.ld;
  const int base = g.crank * cap;  // this CTA holds slots [base, base + cap)
  const int tid = kThreads == 32 ? g.lane : (int)threadIdx.x;
  if (p.ids) {
    n = p.counts[row];
    n = n < 0 ? 0 : n > p.ld_ids ? p.ld_ids : n;
    const unsigned short* ids = p.ids + (long long)row * p.ld_ids;
#pragma unroll 2
    for (int i = tid; i < cap; i += kThreads) {
      const int e = base + i;
      const int id = e < n ? ids[e] : 0x7fffffff;
      v[i] = id < p.width ? to_f(src[id]) : -INFINITY;
    }
    return 0;
  }
  n = p.width;
  constexpr int kPer = Pieces<T>::n;
  const int first = (int)((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(T));  // the row's place in its first piece
  const uint4* pieces = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(src) & ~uintptr_t(15)) + base / kPer;
  auto put = [&](int i, const float (&f)[kPer]) {
#pragma unroll
    for (int j = 0; j < kPer; j += 4) *reinterpret_cast<float4*>(v + i * kPer + j) = make_float4(f[j], f[j + 1], f[j + 2], f[j + 3]);
  };
  // of this CTA's pieces: those whole inside the row
  const int whole0 = base == 0 && first > 0 ? 1 : 0, held = cap / kPer;
  int whole1 = (first + n) / kPer - base / kPer;
  whole1 = whole1 < whole0 ? whole0 : whole1 > held ? held : whole1;
  for (int i0 = whole0 + tid; i0 < whole1; i0 += 8 * kThreads) {
    uint4 u[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i0 + j * kThreads < whole1) u[j] = __ldg(pieces + i0 + j * kThreads);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i0 + j * kThreads < whole1) {
        float f[kPer];
        Pieces<T>::get(u[j], f);
        put(i0 + j * kThreads, f);
      }
  }
  auto edge = [&](int i) {
    const int e = base + i * kPer - first;
    float f[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) f[j] = e + j >= 0 && e + j < n ? to_f(src[e + j]) : -INFINITY;
    put(i, f);
  };
  if (tid < whole0) edge(tid);
  for (int i = whole1 + tid; i < held; i += kThreads) edge(i);
  return first;
}

// The end of what stays of a row: entries above `l`, and those equal to it up to `slot`.
struct Cut {
  float l;
  int slot;
};

constexpr int kSort = 64;    // entries that a warp sorts
constexpr int kList = 256;   // entries between two logits that are solved by a warp

template <int kThreads, bool kCluster> struct Shared {
  double slots[2 * Group<kThreads, kCluster>::kSlots];
  float wide[kThreads == 32 ? 1 : 2 * Group<kThreads, kCluster>::kSlots * 4];
  float list_l[kList];
  int list_slot[kList];
  uint64_t sorted[32];
  double weights[kThreads == 32 ? kSort : 1];
  uint64_t bars[3];
  double ahead;
  int count;
  int solved;
  uint64_t cut;
};

// Entries as 64-bit numbers whose order is the row's: by logit, of equal ones the lower slot is larger.  0: none.
__device__ __forceinline__ uint64_t entry_of(float l, int slot) {
  return l > -INFINITY ? (uint64_t)key_of(l) << 32 | (uint32_t)~slot : 0;
}
__device__ __forceinline__ Cut cut_of(uint64_t e) {
  Cut c;
  c.l = of_key((uint32_t)(e >> 32));
  c.slot = (int)~(uint32_t)e;
  return c;
}
// Sorts 32 (b = 0) or 64 entries of a warp, falling: a lane's `a` is number lane, its `b` number 32 + lane.
__device__ __forceinline__ void sort_entries(uint64_t& a, uint64_t& b, bool two, int lane) {
  auto step = [&](uint64_t v, int j, bool larger) {
    const uint64_t o = __shfl_xor_sync(0xffffffffu, v, j);
    return (v > o) == larger ? v : o;
  };
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      a = step(a, j, ((lane & j) == 0) == ((lane & k) == 0));
      // the upper half rises, so that both form one bitonic run of 64
      if (two) b = step(b, j, ((lane & j) == 0) == (k == 32 ? false : (lane & k) == 0));
    }
  if (!two) return;
  if (b > a) { const uint64_t t = a; a = b; b = t; }
#pragma unroll
  for (int j = 16; j > 0; j >>= 1) {
    a = step(a, j, (lane & j) == 0);
    b = step(b, j, (lane & j) == 0);
  }
}
template <typename W> __device__ __forceinline__ W warp_before(W v, W& total, int lane) {
  W in = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const W up = __shfl_up_sync(0xffffffffu, in, o);
    if (lane >= o) in += up;
  }
  total = __shfl_sync(0xffffffffu, in, 31);
  const W ex = __shfl_up_sync(0xffffffffu, in, 1);
  return lane == 0 ? W(0) : ex;
}

// A row in shared memory, seen by one thread of its group.
template <int kThreads, bool kCluster> struct Row {
  Group<kThreads, kCluster>& g;
  Shared<kThreads, kCluster>& sh;
  const SampleParams& p;
  float* mine;   // this thread's entries
  int slot0;     // slot of the first of them
  int count;     // their number
  int row, first;
  Weight<(kThreads > 32)> wt;

  template <typename F> __device__ __forceinline__ void each(F f) const {
#pragma unroll 2
    for (int i = 0; i < count; i += 4) {
      const float4 x = *reinterpret_cast<const float4*>(mine + i);
      f(i, x.x); f(i + 1, x.y); f(i + 2, x.z); f(i + 3, x.w);
    }
  }
  // Sum of f(i, l, w) over this thread's entries, w their weights (not computed where kWeights is false): 8 at a time in W, those sums
  // in 64 bits.  (Longer loop bodies ran slower: instructions that did not arrive in time were half of the warps' stalls.)
  template <typename W, bool kWeights, typename F> __device__ __forceinline__ double sum(F f) const {
    auto quad = [&](int at) -> W {
      const float4 x = *reinterpret_cast<const float4*>(mine + at);
      const float l[4] = {x.x, x.y, x.z, x.w};
      W w[4] = {};
      if (kWeights) wt.get4(l, w);
      const W a = f(at, l[0], w[0]), b = f(at + 1, l[1], w[1]), c = f(at + 2, l[2], w[2]), d = f(at + 3, l[3], w[3]);
      return (a + b) + (c + d);
    };
    double total = 0.0;
    int i = 0;
    if constexpr (sizeof(W) == 4) {
#pragma unroll 1
      for (; i + 8 <= count; i += 8) {
        const W a = quad(i), b = quad(i + 4);
        total += (double)(a + b);
      }
    }
#pragma unroll 1
    for (; i < count; i += 4) total += (double)quad(i);
    return total;
  }
  __device__ __forceinline__ bool keeps(const Cut cut, int i, float l) const { return (l > cut.l) | ((l == cut.l) & (i <= cut.slot - slot0)); }
  __device__ __forceinline__ void keep(const Cut cut) const {
#pragma unroll 2
    for (int i = 0; i < count; i += 4) {
      float4 x = *reinterpret_cast<const float4*>(mine + i);
      x.x = keeps(cut, i, x.x) ? x.x : -INFINITY;
      x.y = keeps(cut, i + 1, x.y) ? x.y : -INFINITY;
      x.z = keeps(cut, i + 2, x.z) ? x.z : -INFINITY;
      x.w = keeps(cut, i + 3, x.w) ? x.w : -INFINITY;
      *reinterpret_cast<float4*>(mine + i) = x;
    }
  }
  __device__ __forceinline__ void give(int slot, float prob) const {
    p.choice[row] = slot < 0 ? -1 : slot - first;
    if (p.prob) p.prob[row] = prob;
  }
  // Slot of the j-th (from 0) entry equal to l.
  __device__ int nth_equal(float l, double j) {
    int same = 0;
    each([&](int, float x) { same += x == l; });
    double all;
    double left = j - g.before((double)same, all);
    int at = -1;
    if (left >= 0.0 && left < (double)same)
      each([&](int i, float x) {
        if (x == l) {
          if (left == 0.0) at = slot0 + i;
          left -= 1.0;
        }
      });
    return (int)g.max((float)at);
  }

  // The end of the front part by bisection over all entries: for what the quicker ways do not find.
  template <typename W, bool kMass> __device__ bool bisect(double target, Cut& out) {
    uint32_t lo_key = key_of(-INFINITY), hi_key = key_of(wt.max);  // measure above lo_key: the target or more; above hi_key: less
    double over = 0.0;
    while (hi_key - lo_key > 1) {
      const uint32_t mid = lo_key + (hi_key - lo_key) / 2;
      const float cut = of_key(mid);
      const double m = g.sum(sum<W, kMass>([&](int, float l, W w) { return l > cut ? (kMass ? w : W(1)) : W(0); }));
      if (kCluster && g.gave_up) return true;
      if (m >= target) lo_key = mid;
      else { hi_key = mid; over = m; }
    }
    out.l = of_key(hi_key);
    const double ties = (target - over) / (kMass ? (double)wt.get(out.l, W()) : 1.0);
    out.slot = nth_equal(out.l, ties <= 1.0 ? 0.0 : ceil(fmin(ties, 1e9)) - 1.0);
    if (out.slot < 0) out.slot = 0x7fffffff;  // all of them
    return true;
  }
  // The end of the front part inside a run of equal entries, ahead of which `front` is found.
  template <typename W, bool kMass> __device__ bool equal_entries(float l, double front, double target, double all, double slack, Cut& out) {
    constexpr bool kOpen = kMass && sizeof(W) == 4;
    const double w = kMass ? (double)wt.get(l, W()) : 1.0, ties = (target - front) / w;
    if (kOpen && (w < 1e-30 || fabs(ties - rint(ties)) <= slack * all / w + 1e-6 * fabs(ties))) return false;
    out.l = l;
    out.slot = nth_equal(l, ties <= 1.0 ? 0.0 : ceil(fmin(ties, 1e9)) - 1.0);
    if (out.slot >= 0) return true;
    return kOpen ? false : bisect<W, kMass>(target, out);  // the run ends before it
  }
  // The end among the n <= kList entries that were gathered, by one warp: bisection by the measure until 32 are left, which are
  // sorted.  1: sh.cut; 2: a comparison was open; 3: in a run of entries equal to sh.cut, ahead of which sh.ahead is found; 0: not here.
  template <typename W, bool kMass> __device__ int solve_list(int n, double front, double target, double slack) {
    constexpr bool kOpen = kMass && sizeof(W) == 4;
    constexpr int kEach = kList / 32;
    const int lane = g.lane;
    uint32_t key[kEach];  // 0: none
    int slot[kEach];
    W w[kEach];
    const int own = kCluster && lane < g.cluster ? *cg::this_cluster().map_shared_rank(&sh.count, lane) : 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      int at = 32 * i + lane < n ? 32 * i + lane : 0, cta = 0;
      if (kCluster)  // a list in each CTA of the cluster, one behind the other
        for (int c = 0; c < kMaxCluster - 1; ++c) {
          const int nc = __shfl_sync(0xffffffffu, own, c);
          const bool behind = cta == c && at >= nc && c < g.cluster - 1;
          at -= behind ? nc : 0;
          cta += behind;
        }
      const float l = kCluster ? cg::this_cluster().map_shared_rank(sh.list_l, cta)[at] : sh.list_l[at];
      slot[i] = kCluster ? cg::this_cluster().map_shared_rank(sh.list_slot, cta)[at] : sh.list_slot[at];
      key[i] = 32 * i + lane < n ? key_of(l) : 0;
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) w[i] = key[i] ? kMass ? wt.get(of_key(key[i]), W()) : W(1) : W(0);
    uint32_t lo = 0, hi = 0xffffffffu;  // above lo the target or more, above hi less
    int left = n;
    bool open = false;
    while (left > 32) {
      // the middle of what is left, in logits
      uint32_t down = 0xffffffffu, up = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const bool in = key[i] > lo && key[i] <= hi;
        down = in ? min(down, key[i]) : down;
        up = in ? max(up, key[i]) : up;
      }
      down = __reduce_min_sync(0xffffffffu, down);
      up = __reduce_max_sync(0xffffffffu, up);
      if (down >= up) {  // equal entries
        double m = 0.0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) m += key[i] > up ? (double)w[i] : 0.0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
        if (lane == 0) { sh.cut = (uint64_t)up << 32; sh.ahead = front + m; }
        return open ? 2 : 3;
      }
      uint32_t at = key_of(0.5f * of_key(down) + 0.5f * of_key(up));
      if (at < down || at >= up) at = down;
      W m = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) m += key[i] > at ? w[i] : W(0);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
      if (kOpen) open |= fabs(front + (double)m - target) <= slack + 13.0 * 0x1p-24 * (double)m;  // (thirteen additions)
      if (front + (double)m >= target) lo = at;
      else hi = at;
      left = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) left += key[i] > lo && key[i] <= hi;
      left = __reduce_add_sync(0xffffffffu, left);
    }
    if (open) return 2;
    double ahead = 0.0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) ahead += key[i] > hi ? (double)w[i] : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
    // those left side by side, through the gathered entries' place
    __syncwarp();
    int pos = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const bool in = key[i] > lo && key[i] <= hi;
      const uint32_t b = __ballot_sync(0xffffffffu, in);
      if (in) sh.sorted[pos + __popc(b & ((1u << lane) - 1))] = (uint64_t)key[i] << 32 | (uint32_t)~slot[i];
      pos += __popc(b);
    }
    __syncwarp();
    uint64_t e = lane < pos ? sh.sorted[lane] : 0, none = 0;
    sort_entries(e, none, false, lane);
    const float mine_l = of_key((uint32_t)(e >> 32));
    double t0;
    const double before = front + ahead + warp_before(!e ? 0.0 : kMass ? (double)wt.get(mine_l, W()) : 1.0, t0, lane);
    const double end = front + ahead + t0;
    // entries that stay: those ahead of which less than the target lies
    const int stay = __popc(__ballot_sync(0xffffffffu, e && before < target));
    if (kOpen && (__any_sync(0xffffffffu, e && fabs(before - target) <= slack) || fabs(end - target) <= slack)) return 2;
    const uint64_t cut = __shfl_sync(0xffffffffu, e, (stay - 1) & 31);
    if (lane == 0) sh.cut = cut;
    return stay > 0 && end >= target ? 1 : 0;
  }

  // The end of the front part: the first entry ahead of which the measure (kMass: weights, else 1 each) sums to the target or more is out,
  // with all behind it; the first of all stays.  kMass: `target` is a share of the sum of all weights.  The end lies between two
  // logits, above the upper of which less than the target is found, above the lower the target or more; three pivots between them
  // per pass, where the last pass makes the end expected, until the entries between them are few enough to be sorted.  What finds
  // the place are sums of quick weights with a margin; what decides is the exact measure above and the sorted entries.  (Counting
  // in bins instead: an addition to shared memory took 64 cycles per warp, twice what the pivots take.)
  // False: a comparison was open.
  // `lo_at`, `hi_at`: the two logits, from a call that left a comparison open to one in 64 bits (hi_at = infinity: none yet).
  template <typename W, bool kMass>
  __device__ bool select(int n_row, double target, float hi, float least, double slack, float& lo_at, float& hi_at, Cut& out) {
    constexpr bool kOpen = kMass && sizeof(W) == 4;
    const int tid = kThreads == 32 ? g.lane : (int)threadIdx.x;
    float lo = -INFINITY, reach_lo = 0.f, reach_hi = 0.f;  // found above them (lo: all, where it is infinite)
    const bool known = hi_at < INFINITY;
    if (known) { lo = lo_at; hi = hi_at; }
    double all = 0.0;
    float x[3];
    {
      constexpr float kSteps[3] = {2.f, 4.5f, 8.f}, kShares[3] = {0.0625f, 0.25f, 0.5f};
#pragma unroll
      for (int j = 0; j < 3; ++j) x[j] = kMass ? hi - kSteps[j] * wt.temp : hi - kShares[j] * fminf(hi - least, 3.4e38f);
    }
    for (int round = 0; round < 16; ++round) {
      float a[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) a[j] = 0.f;
      auto pivots = [&](float l, float w) {
#pragma unroll
        for (int j = 0; j < 3; ++j) a[j] += l > x[j] ? w : 0.f;
        a[3] += l > -INFINITY ? w : 0.f;
      };
      if (kMass && round == 0) {
        if (known) all = sum<W, true>([&](int, float, W w) -> W { return w; });
        else all = sum<W, true>([&](int, float l, W w) -> W { pivots(l, (float)w); return w; });
        all = g.sum(all);
        target *= all;
      } else {
        each([&](int, float l) { pivots(l, kMass ? wt.quick(l) : 1.f); });
      }
      const bool looked = !(known && round == 0);
      if (looked) g.sum4(a);
      if (kCluster && g.gave_up) return true;
      if (round == 0) reach_lo = a[3];
      const float goal = (float)target, margin = kMass ? 2e-5f * (float)all : 0.f;
#pragma unroll
      for (int j = 0; j < 3; ++j)
        if (looked && x[j] < hi && a[j] < goal - margin) { hi = x[j]; reach_hi = a[j]; }
#pragma unroll
      for (int j = 2; j >= 0; --j)
        if (looked && x[j] > lo && x[j] < hi && a[j] >= goal + margin) { lo = x[j]; reach_lo = a[j]; }
      // entries between the two, as many as there would be if all were as light as the lower end
      const float most_here = (reach_lo - reach_hi + margin) / (kMass ? fmaxf(wt.quick(lo), 1e-30f) : 1.f);
      const float low = lo > -INFINITY ? lo : kMass ? fmaxf(hi - 16.f * wt.temp, -3.4e38f) : fminf(least, hi);
      const float f = fminf(fmaxf((goal - reach_hi) / (reach_lo - reach_hi), 0.f), 1.f), width = fminf(hi - low, 3.4e38f);
      const float parts[3] = {0.875f * f, f + 0.015625f * (1.f - f), f + 0.125f * (1.f - f)};
#pragma unroll
      for (int j = 0; j < 3; ++j) x[j] = hi - parts[j] * width;
      if (!(most_here <= (float)kList) && n_row > kList && round < 5 && !(known && round == 0)) continue;
      lo_at = lo;
      hi_at = hi;
      // the exact measure above them, and the entries between them, marked 32 at a time
      g.barrier();  // the others are done with what is cleared
      if (kCluster && g.gave_up) return true;
      if (tid == 0) sh.count = 0;
      if (kThreads == 32) __syncwarp(); else __syncthreads();
      float down = INFINITY, up = -INFINITY;
      double more = 0.0;
#pragma unroll 1
      for (int i0 = 0; i0 < count; i0 += 32) {
        uint32_t hits = 0;
        const int end = count - i0 < 32 ? count - i0 : 32;
#pragma unroll 1
        for (int i = 0; i < end; i += 4) {
          const float4 v = *reinterpret_cast<const float4*>(mine + i0 + i);
          const float l4[4] = {v.x, v.y, v.z, v.w};
          W w4[4] = {1, 1, 1, 1};
          if constexpr (kMass) wt.get4(l4, w4);
          uint32_t four = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            four |= (l4[j] <= hi) & (l4[j] > lo) ? 1u << j : 0u;
            w4[j] = l4[j] > hi ? w4[j] : W(0);
          }
          more += (double)((w4[0] + w4[1]) + (w4[2] + w4[3]));
          hits |= four << i;
        }
        const int own = __popc(hits);
        int pos = own ? atomicAdd(&sh.count, own) : 0;
        for (; hits; hits &= hits - 1, ++pos) {
          const int i = i0 + __ffs((int)hits) - 1;
          const float l = mine[i];
          down = fminf(down, l);
          up = fmaxf(up, l);
          if (pos < kList) { sh.list_l[pos] = l; sh.list_slot[pos] = slot0 + i; }
        }
      }
      const double front = g.sum(more);
      // the lists are read across the warp (whose sum is shuffles alone, which order no memory), the CTA (the sum has a barrier) or the cluster
      if (kThreads == 32 || kCluster) g.barrier();
      if (kCluster && g.gave_up) return true;
      int n = sh.count;
      if (kCluster) {
        n = g.lane < g.cluster ? *cg::this_cluster().map_shared_rank(&sh.count, g.lane) : 0;
        n = __reduce_add_sync(0xffffffffu, n);
      }
      if (n == 0 || front >= target) break;
      if (n > kList) {
        hi = g.max(up);  // the entries' own ends
        const float bottom = -g.max(-down);
        if (kCluster && g.gave_up) return true;
        reach_hi = (float)front;
        if (hi == bottom) return equal_entries<W, kMass>(hi, front, target, all, slack, out);
        // the largest of them is above every next pivot but not above `hi`
#pragma unroll
        for (int j = 0; j < 3; ++j) x[j] = hi - (j + 1) * 0.25f * fminf(hi - bottom, 3.4e38f);
        continue;
      }
      if (kThreads == 32 || g.warp == 0) {
        const int result = solve_list<W, kMass>(n, front, target, slack * all);
        if (g.lane == 0) sh.solved = result;
      }
      if (kThreads == 32) __syncwarp(); else __syncthreads();
      if (sh.solved == 2) return false;
      if (sh.solved == 0) break;
      out = cut_of(sh.cut);
      if (sh.solved == 3) return equal_entries<W, kMass>(out.l, sh.ahead, target, all, slack, out);
      return true;
    }
    // (a few values many decades apart, a target that rounding puts beyond all)
    return kOpen ? false : bisect<W, kMass>(target, out);
  }

  // The draw among what the cut and min-p keep.  False: a comparison was open.
  template <typename W> __device__ bool draw(const Cut cut, float p_min, float u, double slack) {
    constexpr bool kOpen = sizeof(W) == 4;
    const W limit = p_min > 0.f ? (W)fminf(p_min, 1.f) : W(0);
    bool open = false;
    const float near = 4.f * (float)slack * (float)limit;
    double own;
    if (limit > W(0)) {
      own = sum<W, true>([&](int i, float l, W w) -> W {
        if (kOpen) open |= (fabsf((float)w - (float)limit) <= near) & (l != wt.max);
        return keeps(cut, i, l) & (w >= limit) ? w : W(0);
      });
    } else if (cut.l > -INFINITY) {
      own = sum<W, true>([&](int i, float l, W w) -> W { return keeps(cut, i, l) ? w : W(0); });
    } else {
      own = sum<W, true>([&](int, float, W w) -> W { return w; });
    }
    double total;
    const double ahead = g.before(own, total), target = (double)u * total;
    if (kCluster && g.gave_up) return true;
    const bool here = ahead <= target && target < ahead + own;
    // the warp of the thread whose entries the sum passes the target in looks for the entry together
    const float id = (float)g.thread();
    float owner = 0.f;
    bool claims = here;
    if (!kOpen) {  // neighbours' bounds can differ in their last bit: the first that claims it, else the last with a weight
      owner = -g.max(here ? -id : -INFINITY);
      if (owner == INFINITY) owner = g.max(own > 0.0 ? id : -INFINITY);
      if (kCluster && g.gave_up) return true;
      claims = id == owner;
    }
    const uint32_t ballot = __ballot_sync(0xffffffffu, claims);
    int at = -1;
    double w_at = 0.0;
    if (ballot) {
      const int o = __ffs(ballot) - 1;
      const float* theirs = mine + (o - g.lane) * count;
      const int their_slot = slot0 + (o - g.lane) * count;
      double run = __shfl_sync(0xffffffffu, ahead, o);
      const double own_sum = __shfl_sync(0xffffffffu, own, o);
      bool found = false;
      for (int base = 0; base < count; base += 32) {
        W w = 0, sum32;
        const int i = base + g.lane;
        if (i < count && (theirs[i] > cut.l || (theirs[i] == cut.l && their_slot + i <= cut.slot))) {
          const W x = wt.get(theirs[i], W());
          w = x >= limit ? x : W(0);
        }
        const double before = run + (double)warp_before(w, sum32, g.lane);
        const uint32_t any = __ballot_sync(0xffffffffu, w > W(0)), hit = __ballot_sync(0xffffffffu, w > W(0) && before + (double)w > target);
        if (any) {
          const int j = hit ? __ffs(hit) - 1 : 31 - __clz(any);
          at = their_slot + base + j;
          const double b = __shfl_sync(0xffffffffu, before, j);
          w_at = (double)__shfl_sync(0xffffffffu, w, j);
          if (hit) {
            // the sums ahead of this run of entries, and the run's own five additions
            const double near_at = slack * total + 12.0 * 0x1p-24 * own_sum;
            if (kOpen) open |= target - b <= near_at || b + w_at - target <= near_at;
            found = true;
            break;
          }
        }
        run += (double)sum32;
      }
      if (kOpen && !found) open = true;
    }
    if (kOpen) {
      const double one = g.sum((open ? 1048576.0 : 0.0) + (claims ? 1.0 : 0.0));
      if (kCluster && g.gave_up) return true;
      if (one != 1.0) return false;
    }
    if (claims) {
      if (kOpen) w_at = wt.get(mine[at - slot0], 0.0);
      give(at, (float)(w_at / total));
    }
    return true;
  }

  // ---- rows whose kept entries are few: a warp has them all, in the order of their indices, and sums in 64 bits ----
  // l, slot (NULL: from `base` on): n <= 64 entries.
  __device__ void finish(const float* l, const int* slot, int base, int n, int k, float p_top, float p_min, float u) {
    const int lane = g.lane;
    uint64_t own[2];  // entries lane and 32 + lane, by their places here (which rise with the indices)
    double w[2], x[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = 32 * h + lane;
      const float v = i < n ? l[i] : -INFINITY;
      own[h] = entry_of(v, i);
      x[h] = wt.exponent(v);
    }
    exp_below(x);
#pragma unroll
    for (int h = 0; h < 2; ++h) w[h] = own[h] ? x[h] : 0.0;
    uint64_t cut = 1;
    if ((k > 0 && k < n) || p_top < 1.f) {
      uint64_t e[2] = {own[0], own[1]};
      sort_entries(e[0], e[1], n > 32, lane);
      int stay = __popc(__ballot_sync(0xffffffffu, e[0] != 0)) + __popc(__ballot_sync(0xffffffffu, e[1] != 0));
      if (k > 0 && k < stay) stay = k;
      if (p_top < 1.f) {
        sh.weights[lane] = w[0];
        sh.weights[32 + lane] = w[1];
        __syncwarp();
        const double w0 = lane < stay ? sh.weights[~(uint32_t)e[0]] : 0.0, w1 = 32 + lane < stay ? sh.weights[~(uint32_t)e[1]] : 0.0;
        double t0, t1 = 0.0;
        const double b0 = warp_before(w0, t0, lane), b1 = stay > 32 ? t0 + warp_before(w1, t1, lane) : 0.0;
        const double target = (double)p_top * (t0 + t1);
        const int in = __popc(__ballot_sync(0xffffffffu, lane < stay && b0 < target)) +
                       __popc(__ballot_sync(0xffffffffu, 32 + lane < stay && b1 < target));
        stay = in > 1 ? in : 1;
      }
      const uint64_t c0 = __shfl_sync(0xffffffffu, e[0], (stay - 1) & 31), c1 = __shfl_sync(0xffffffffu, e[1], (stay - 1) & 31);
      cut = stay > 32 ? c1 : c0;
    }
    const double limit = p_min > 0.f ? (double)fminf(p_min, 1.f) : 0.0;
    double run = 0.0, total, before[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (own[h] < cut || w[h] < limit) w[h] = 0.0;
      before[h] = 0.0;
      if (h == 0 || n > 32) {
        before[h] = run + warp_before(w[h], total, lane);
        run += total;
      }
    }
    const double target = (double)u * run;
    uint32_t hit0 = __ballot_sync(0xffffffffu, w[0] > 0.0 && before[0] + w[0] > target);
    uint32_t hit1 = __ballot_sync(0xffffffffu, w[1] > 0.0 && before[1] + w[1] > target);
    if (!hit0 && !hit1) {  // rounding: the last with a weight
      hit1 = __ballot_sync(0xffffffffu, w[1] > 0.0);
      if (hit1) hit1 = 1u << (31 - __clz(hit1));
      else hit0 = 1u << (31 - __clz(__ballot_sync(0xffffffffu, w[0] > 0.0)));
    }
    const int half = hit0 ? 0 : 1, j = __ffs(hit0 ? hit0 : hit1) - 1;
    const int i = 32 * half + lane;
    if (lane == j) give(slot ? slot[i] : base + i, (float)((half ? w[1] : w[0]) / run));
  }
  // The entries that top-k can keep, gathered: those not below a logit that k entries reach.  Maxima of the lanes' runs give one: the
  // k-th of them for small k, one of the least else, which more than k entries reach nearly always; from there a bisection over the
  // gathered entries goes on.  Number of entries, 0 if
  // that found none or too many.
  __device__ int gather_top(int n_row, int k, float lane_max) {
    const int lane = g.lane;
    float s = lane_max;
#pragma unroll
    for (int kk = 2; kk <= 32; kk <<= 1)
#pragma unroll
      for (int j = kk >> 1; j > 0; j >>= 1) {
        const float o = __shfl_xor_sync(0xffffffffu, s, j);
        s = ((lane & j) == 0) == ((lane & kk) == 0) ? fmaxf(s, o) : fminf(s, o);
      }
    float floor_l = __shfl_sync(0xffffffffu, s, k <= 24 ? k - 1 : k <= 40 ? 28 : 30);  // (the last run may be empty)
    if (n_row <= kList) floor_l = -3.402823466e38f;
    if (floor_l == -INFINITY) return 0;
    // one row in five hundred has too few or too many above it; another logit is tried there, a row done by all its entries takes
    // twenty times as long and the others wait for it
    uint64_t hits = 0;
    int own = 0, in = 0, n = 0;
    float few = wt.max, many = -INFINITY;
    for (int tries = 0; tries < 6; ++tries) {
      uint32_t hits_lo = 0, hits_hi = 0;
#pragma unroll 4
      for (int i = 0; i < count; i += 4) {
        const float4 x = *reinterpret_cast<const float4*>(mine + i);
        const uint32_t four = (x.x >= floor_l ? 1u : 0u) | (x.y >= floor_l ? 2u : 0u) | (x.z >= floor_l ? 4u : 0u) | (x.w >= floor_l ? 8u : 0u);
        if (i < 32) hits_lo |= four << i;
        else hits_hi |= four << (i - 32);
      }
      hits = (uint64_t)hits_hi << 32 | hits_lo;
      own = __popcll(hits);
      n = __reduce_add_sync(0xffffffffu, own);
      if (n_row <= kList || (n >= k && n <= kList)) break;
      if (n < k) few = floor_l;
      else many = floor_l;
      floor_l = many == -INFINITY ? floor_l - 0.25f * (wt.max - floor_l) : 0.5f * few + 0.5f * many;
    }
    in = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, in, o);
      if (lane >= o) in += up;
    }
    if (n > kList || (n < k && n_row > kList)) return 0;
    for (int pos = in - own; hits; hits &= hits - 1, ++pos) {
      const int i = __ffsll((long long)hits) - 1;
      sh.list_l[pos] = mine[i];
      sh.list_slot[pos] = slot0 + i;
    }
    __syncwarp();
    const int room = k <= 32 ? 32 : kSort;  // half as many are sorted in less than half the steps
    if (n <= room || (n <= kSort && n <= k)) return n;
    float l[kList / 32];
    int slot[kList / 32];
#pragma unroll
    for (int i = 0; i < kList / 32; ++i) {
      l[i] = 32 * i + lane < n ? sh.list_l[32 * i + lane] : -INFINITY;
      slot[i] = 32 * i + lane < n ? sh.list_slot[32 * i + lane] : 0;
    }
    uint32_t lo = key_of(floor_l), hi = key_of(wt.max) + 1;  // too many reach lo, fewer than k reach hi
    float at = 0.f;
    bool found = false;
    while (hi - lo > 1 && !found) {
      const uint32_t mid = lo + (hi - lo) / 2;
      at = of_key(mid);
      int c = 0;
#pragma unroll
      for (int i = 0; i < kList / 32; ++i) c += l[i] >= at;
      c = __reduce_add_sync(0xffffffffu, c);
      if (c > room) lo = mid;
      else if (c < k) hi = mid;
      else found = true;
    }
    if (!found) return n <= kSort ? n : 0;  // equal entries
    __syncwarp();
    n = 0;
#pragma unroll
    for (int i = 0; i < kList / 32; ++i) {
      const bool stays = l[i] >= at;
      const uint32_t b = __ballot_sync(0xffffffffu, stays);
      if (stays) {
        const int pos = n + __popc(b & ((1u << lane) - 1));
        sh.list_l[pos] = l[i];
        sh.list_slot[pos] = slot[i];
      }
      n += __popc(b);
    }
    __syncwarp();
    return n;
  }
};

template <typename T, int kThreads, bool kCluster>
__global__ void __launch_bounds__(kThreads == 32 ? 32 * kWarpRows : kThreads, kThreads == 32 ? 5 : 3)
sample_kernel(const SampleParams p) {
  extern __shared__ float4 smem[];
  __shared__ Shared<kThreads, kCluster> shared[kThreads == 32 ? kWarpRows : 1];
  const int part = kThreads == 32 ? threadIdx.x >> 5 : 0;
  const int cap = kThreads * 4 * p.pieces;
  float* v = reinterpret_cast<float*>(smem) + part * cap;
  Shared<kThreads, kCluster>& sh = shared[part];
  Group<kThreads, kCluster> g(sh.slots, sh.wide, sh.bars, p);
  const int row = kThreads == 32 ? blockIdx.x * kWarpRows + part : blockIdx.x / p.cluster;
  if (row >= p.rows) return;
  float temp = p.temperature ? p.temperature[row] : 1.f;
  const float p_top = p.top_p ? p.top_p[row] : 1.f, p_min = p.min_p ? p.min_p[row] : 0.f;
  const int k = p_top <= 0.f ? 1 : p.top_k ? p.top_k[row] : 0;
  float u = p.u[row];
  u = u >= 0.f ? fminf(u, 1.f - 0x1p-24f) : 0.f;
  if (kThreads == 32 && !p.ids && row + p.ahead < p.rows) {  // a row of the next round of CTAs into L2, while this one is worked on
    const char* next = static_cast<const char*>(p.logits) + (long long)(row + p.ahead) * p.ld * sizeof(T);
    for (int i = g.lane * 128; i < p.width * (int)sizeof(T); i += 32 * 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(next + i));
  }
  int n = 0;
  const int first = load_row<T, kThreads, kCluster>(p, g, row, v, cap, n);
  if (kCluster) cg::this_cluster().sync();  // the barriers of all CTAs are there
  else g.barrier();
  const int local = (kThreads == 32 ? g.lane : (int)threadIdx.x) * 4 * p.pieces;
  Row<kThreads, kCluster> r{g, sh, p, v + local, g.crank * cap + local, 4 * p.pieces, row, first, Weight<(kThreads > 32)>(0.f, 1.f)};
  float own_max = -INFINITY;
  r.each([&](int, float l) { own_max = fmaxf(own_max, l); });
  float m = g.max(own_max);
  bool done = false;
  if (kCluster && g.gave_up) {
    done = true;
  } else if (m == -INFINITY) {
    if (g.thread() == 0) r.give(-1, 0.f);
    done = true;
  } else if (!(temp > 0.f)) {  // the first of the largest
    const int at = r.nth_equal(m, 0.0);
    if (g.thread() == 0) r.give(at, 1.f);
    done = true;
  } else if (m == INFINITY) {  // infinities are equal, and nothing is beside them
    for (int i = 0; i < r.count; ++i) r.mine[i] = r.mine[i] == INFINITY ? 0.f : -INFINITY;
    own_max = own_max == INFINITY ? 0.f : -INFINITY;
    m = 0.f;
    temp = 1.f;
    g.barrier();
    done = g.gave_up;
  }
  if (!done) {
    r.wt = Weight<(kThreads > 32)>(m, temp);
    const bool fp32 = r.wt.fp32_usable();
    const float tp = p_top <= 0.f ? 1.f : p_top;
    if constexpr (kThreads == 32) {
      if (n <= kSort) {
        r.finish(v + first, nullptr, first, n, k, tp, p_min, u);
        done = true;
      } else if (k > 0 && k <= kSort) {
        const int few = r.gather_top(n, k, own_max);
        if (few) {
          r.finish(sh.list_l, sh.list_slot, 0, few, k, tp, p_min, u);
          done = true;
        }
      }
    }
    if (!done) {
      const double slack = (double)p.slack;
      Cut cut{-INFINITY, -1};
      if (k > 0 && k < n) {
        float least = INFINITY;
        int own = 0;
        r.each([&](int, float l) {
          own += l > -INFINITY;
          least = fminf(least, l > -INFINITY ? l : INFINITY);
        });
        if ((double)k < g.sum((double)own)) {
          least = -g.max(-least);  // (without the others: infinity; select finds that out)
          float lo_at = 0.f, hi_at = INFINITY;
          r.template select<float, false>(n, (double)k, m, least, 0.0, lo_at, hi_at, cut);
          if (tp < 1.f) r.keep(cut);
        }
      }
      if (tp < 1.f) {
        float lo_at = 0.f, hi_at = INFINITY;
        if (!fp32 || !r.template select<float, true>(n, (double)tp, m, 0.f, slack, lo_at, hi_at, cut))
          r.template select<double, true>(n, (double)tp, m, 0.f, 0.0, lo_at, hi_at, cut);
      }
      if (!fp32 || !r.template draw<float>(cut, p_min, u, slack)) r.template draw<double>(cut, p_min, u, 0.0);
    }
  }
  if (kCluster) {
    cg::this_cluster().sync();  // no CTA leaves while another may still reach into its shared memory
    if (g.gave_up) {
      for (int i = 0; i < 200; ++i) __nanosleep(1000);  // what others have sent without being waited for lands before the shared memory is released
      if (threadIdx.x == 0) {  // behind the barrier: over what another CTA may have answered
        p.choice[row] = -2;
        if (p.prob) p.prob[row] = 0.f;
      }
    }
  }
}

template <typename T, int kThreads, bool kCluster>
cudaError_t launch_group(const SampleParams& p, cudaStream_t s) {
  const int groups = kThreads == 32 ? kWarpRows : 1;
  cudaError_t e = raise_smem_limit<sample_kernel<T, kThreads, kCluster>>(kThreads == kWide ? kWide * kMaxPieces * 16 : 64 * 1024);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kThreads == 32 ? ceil_div(p.rows, kWarpRows) : p.rows * p.cluster);
  cfg.blockDim = dim3(kThreads * groups);
  cfg.dynamicSmemBytes = (size_t)groups * kThreads * p.pieces * 16;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = kCluster ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, sample_kernel<T, kThreads, kCluster>, p);
}

std::atomic<long long> give_up{-1};  // CTA << 32 | wait, below 0: none (see b200_op_sample_inject_give_up)

template <typename T>
cudaError_t launch_sample(SampleParams p, cudaStream_t s) {
  // a row that does not start on a 16-byte boundary begins inside its first piece
  const int n = p.ids ? p.ld_ids : p.width + Pieces<T>::n - 1;
  auto pieces = [&](int threads) { return ceil_div(ceil_div(n, 4), threads) | 1; };
  p.cluster = 1;
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return e;
  // A warp per row costs the fewest instructions, a CTA the least time: as many rows as there are places for CTAs take these, where the
  // end of top-p is looked for among all entries.  1858 entries with top-p, us, warps / CTAs: 24 rows 28 / 20, 300 29 / 23, 444 29 / 24,
  // 600 29 / 33; 600 entries, 24 rows 9.8 / 9.4, 300 11.4 / 11.5.
  const bool few = p.rows <= 3 * sms && p.top_p && !p.top_k && n > 2 * kList;
  const int threads = pieces(32) <= 15 && !few ? 32 : kWide;
  if (threads == kWide)
    while (p.cluster < kMaxCluster && pieces(kWide * p.cluster) > 9) p.cluster *= 2;
  p.pieces = pieces(threads * p.cluster);
  p.ahead = sms * 5 * kWarpRows;
  // Bound of a sum's error over the sum of all weights, in steps of 2^-24.  A weight: ex2.approx 3, the factor and the second pieces 1;
  // without the rounding of l - m made good |z| more, z = (l - m) / T, and the sum of w |z| is at most ln(n) < 8 times the sum of w
  // (of a warp's rows).  Sums: 8 at a time 3, a total 1.  Twice that, since two sums are compared.
  p.slack = 2.f * (3.f + 1.f + (threads == 32 ? 8.f : 0.f) + 4.f) * 0x1p-24f;
  if (threads == 32) return launch_group<T, 32, false>(p, s);
  return p.cluster == 1 ? launch_group<T, kWide, false>(p, s) : launch_group<T, kWide, true>(p, s);
}

}  // namespace
}  // namespace b200

extern "C" int b200_op_sample(const b200_sample_desc* d, void* stream) {
  using namespace b200;
  return at_c_entry([&]() -> int {
    auto bad = [](const char* what) {
      set_error(std::string("b200_op_sample: ") + what);
      return B200_ERR_INVALID;
    };
    if (!d) return bad("no description");
    if (d->rows < 0 || d->width < 1 || d->width > B200_SAMPLE_MAX_WIDTH) return bad("rows >= 0 and a width of 1 to 262144");
    if (d->precision < B200_PREC_FP32 || d->precision > B200_PREC_BF16) return bad("unknown precision");
    if (d->ld != 0 && d->ld < d->width) return bad("rows overlap");
    if (d->rows > 0x7fffffff / kMaxCluster) return bad("too many rows");
    if (d->move_ids && (!d->n_moves || d->ld_moves < 1 || d->ld_moves > 65536)) return bad("lists of moves need their lengths and a stride of 1 to 65536");
    if (!d->move_ids && d->n_moves) return bad("lengths without lists of moves");
    if (d->rows == 0) return B200_OK;
    if (!d->logits || !d->u || !d->choice) return bad("logits, random numbers and choices are needed");
    auto off = [](const void* q, uintptr_t n) { return reinterpret_cast<uintptr_t>(q) % n != 0; };
    if (off(d->logits, d->precision == B200_PREC_FP32 ? 4 : 2) || off(d->move_ids, 2) || off(d->n_moves, 4) || off(d->temperature, 4) ||
        off(d->top_k, 4) || off(d->top_p, 4) || off(d->min_p, 4) || off(d->u, 4) || off(d->choice, 4) || off(d->prob, 4))
      return bad("an operand is not aligned to its type");
    SampleParams p = {};
    p.logits = d->logits; p.ld = d->ld ? d->ld : d->width; p.rows = d->rows; p.width = d->width;
    p.ids = d->move_ids; p.counts = d->n_moves; p.ld_ids = d->ld_moves;
    p.temperature = d->temperature; p.top_k = d->top_k; p.top_p = d->top_p; p.min_p = d->min_p; p.u = d->u;
    p.choice = d->choice; p.prob = d->prob;
    const long long injected = give_up.load(std::memory_order_relaxed);
    p.wait_ns = injected < 0 ? 2000000000ull : 1000000ull;  // 2 s; 1 ms where one is known not to come
    p.give_up_cta = injected < 0 ? -1 : (int)(injected >> 32);
    p.give_up_at = injected < 0 ? -1 : (int)(injected & 0x7fffffff);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (d->precision == B200_PREC_FP32) B200_CUDA(launch_sample<float>(p, s));
    else if (d->precision == B200_PREC_FP16) B200_CUDA(launch_sample<__half>(p, s));
    else B200_CUDA(launch_sample<__nv_bfloat16>(p, s));
    return B200_OK;
  });
}

extern "C" void b200_op_sample_inject_give_up(int cta, int wait) {
  b200::give_up.store(cta < 0 || wait < 0 ? -1 : (long long)cta << 32 | wait, std::memory_order_relaxed);
}
