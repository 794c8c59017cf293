// Drawing one entry per row of logits: temperature, top-k, top-p, min-p, inverse of the cumulative sum at a given random number.
//
// With m the row's largest logit and w(l) = exp((l - m) / T), an entry's weight, entries in the order of falling logits (equal
// logits: lower index first): top-k keeps the first k; top-p those ahead of which the weights sum to less than p S, S the sum of what
// top-k kept; min-p those with w >= min_p.  Each cut keeps a front part of the order, so a row is never sorted: a cut is a logit and,
// among the entries that equal it, an index.  The draw runs over the indices: the first kept i with sum_{j <= i, kept} w_j > u W.
//
// The answer is a whole number, so it has to be the one that exact sums give.  Sums of fp32 weights decide where they can: with an
// error of at most e S (kSlack below) a comparison that is closer than e S is open, and a row with an open comparison is done
// again with weights and sums in 64 bits (one row in a few thousand for policies).
//
// A row is held in shared memory as fp32 by a group of threads: a warp, a CTA or a cluster of CTAs.  Thread t owns a run of consecutive
// entries (an odd number of 16-byte pieces: no bank conflicts), so that sums over threads run in the order of the indices.
#include <cooperative_groups.h>

#include "../../include/b200nn.h"
#include "kernels.cuh"

namespace cg = cooperative_groups;

namespace b200 {
namespace {

constexpr int kMaxCluster = 8;
constexpr int kWide = 1024;             // threads of the largest CTA
constexpr int kMaxPieces = 13;          // 16-byte pieces per thread there: 208 KB
constexpr int kWarpRows = 4;            // rows of a CTA whose groups are warps
static_assert(kMaxCluster * kWide * kMaxPieces * 4 >= B200_SAMPLE_MAX_WIDTH + 8, "the widest row fits a cluster");

struct SampleParams {
  const void* logits; long long ld;
  int rows, width;
  const unsigned short* ids; const int* counts; int ld_ids;
  const float* temperature; const int* top_k; const float* top_p; const float* min_p; const float* u;
  int* choice; float* prob;
  int pieces;   // 16-byte pieces per thread, odd
  int cluster;  // CTAs per row (kThreads == kWide)
  float slack;  // bound of a sum's error, relative to the sum of all weights
};

// Larger keys are larger logits; -0 and +0 have one key.
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// The threads of a row: sums, maxima and prefix sums over them in a fixed order.
template <int kThreads> struct Group {
  static constexpr int kWarps = kThreads / 32;
  static constexpr int kSlots = kThreads == kWide ? kMaxCluster * kWarps : kWarps;
  double* slots;  // [2][kSlots], kThreads > 32
  int cluster, crank, turn;
  int lane, warp;
  __device__ Group(double* s, int cl) : slots(s), cluster(kThreads == kWide ? cl : 1), crank(0), turn(0) {
    lane = threadIdx.x & 31;
    warp = kThreads == 32 ? 0 : threadIdx.x >> 5;
    if (kThreads == kWide && cluster > 1) crank = (int)cg::this_cluster().block_rank();
  }
  __device__ __forceinline__ int thread() const { return (crank * kWarps + warp) * 32 + lane; }
  __device__ __forceinline__ int threads() const { return cluster * kThreads; }
  __device__ __forceinline__ void barrier() const {
    if (kThreads == 32) __syncwarp();
    else if (kThreads == kWide && cluster > 1) cg::this_cluster().sync();
    else __syncthreads();
  }
  // One value per warp, seen by all threads of the group afterwards.  Two sets of slots in turn: the barrier of one exchange
  // lies between the reads of the last and the writes of the next.
  __device__ __forceinline__ const double* gather(double v) {
    double* mine = slots + (turn & 1) * kSlots;
    ++turn;
    if (kThreads == kWide && cluster > 1) {
      if (lane < cluster) *cg::this_cluster().map_shared_rank(mine + crank * kWarps + warp, lane) = v;
    } else if (lane == 0) {
      mine[warp] = v;
    }
    barrier();
    return mine;
  }
  __device__ __forceinline__ double sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (kThreads == 32) return v;
    const double* s = gather(v);
    double t = 0.0;
    for (int i = lane; i < cluster * kWarps; i += 32) t += s[i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    return t;
  }
  __device__ __forceinline__ float max(float v) {
    v = warp_max(v);
    if (kThreads == 32) return v;
    const double* s = gather((double)v);
    float t = -INFINITY;
    for (int i = lane; i < cluster * kWarps; i += 32) t = fmaxf(t, (float)s[i]);
    return warp_max(t);
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
    double ahead = 0.0, all = 0.0;  // every thread adds the warps in the same order
    for (int i = 0; i < cluster * kWarps; ++i) {
      if (i == crank * kWarps + warp) ahead = all;
      all += s[i];
    }
    total = all;
    return ahead + ex;
  }
};

// Weights in fp32 or, kExact, in 64 bits.
template <bool kExact> struct Weight;
template <> struct Weight<false> {
  using type = float;
  float half_max, c, c_lo, max;
  __device__ Weight(float m, float t) : max(m) {
    const double e = 1.4426950408889634 / (double)t;
    half_max = 0.5f * m;
    c = (float)(2.0 * e);
    c_lo = (float)(2.0 * e - (double)c);
  }
  __device__ bool usable() const { return fabsf(c) < 1e37f; }
  // 2^((l - m) log2(e) / T) with the exponent in two pieces; halves, since l - m can overflow
  __device__ __forceinline__ float operator()(float l) const {
    const float x = 0.5f * l - half_max;
    const float z = x * c;
    const float lo = fmaf(x, c_lo, fmaf(x, c, -z));
    const float w = exp2f(z);
    return l == max ? 1.0f : z < -140.f || max == INFINITY ? 0.0f : fmaf(w, lo * 0.69314718f, w);
  }
};
template <> struct Weight<true> {
  using type = double;
  double t;
  float max;
  __device__ Weight(float m, float temp) : t((double)temp), max(m) {}
  __device__ bool usable() const { return true; }
  __device__ __forceinline__ double operator()(float l) const {
    return l == max ? 1.0 : max == INFINITY ? 0.0 : exp(((double)l - (double)max) / t);
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

// A row's entries into shared memory; slot `first` + i holds entry i, -inf where there is none (NaN counts as none).  Whole 16-byte
// pieces of memory are read with one load, those that reach beyond the row entry by entry.
template <typename T, int kThreads>
__device__ int load_row(const SampleParams& p, const Group<kThreads>& g, int row, float* v, int cap, int& n) {
  const T* src = static_cast<const T*>(p.logits) + (long long)row * p.ld;
  const int base = g.crank * cap;  // this CTA holds slots [base, base + cap)
  const int tid = kThreads == 32 ? g.lane : (int)threadIdx.x;
  auto clean = [](float x) { return x == x ? x : -INFINITY; };
  if (p.ids) {
    n = p.counts[row];
    n = n < 0 ? 0 : n > p.ld_ids ? p.ld_ids : n;
    const unsigned short* ids = p.ids + (long long)row * p.ld_ids;
    for (int i = tid; i < cap; i += kThreads) {
      const int e = base + i;
      const int id = e < n ? ids[e] : 65536;
      v[i] = id < p.width ? clean(to_f(src[id])) : -INFINITY;
    }
    return 0;
  }
  n = p.width;
  constexpr int kPer = Pieces<T>::n;
  const int first = (int)((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(T));  // the row's place in its first piece
  const uint4* pieces = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(src) & ~uintptr_t(15));
  for (int i = tid; i < cap / kPer; i += kThreads) {
    const int e = base + i * kPer - first;  // first entry of the piece
    float f[kPer];
    if (e >= 0 && e + kPer <= n) {
      Pieces<T>::get(__ldg(pieces + base / kPer + i), f);
#pragma unroll
      for (int j = 0; j < kPer; ++j) f[j] = clean(f[j]);
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j) f[j] = e + j >= 0 && e + j < n ? clean(to_f(src[e + j])) : -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < kPer; j += 4) *reinterpret_cast<float4*>(v + i * kPer + j) = make_float4(f[j], f[j + 1], f[j + 2], f[j + 3]);
  }
  return first;
}

// The row in `mine` (this thread's entries, slot0 the first one's slot): cuts and draw.  False: a comparison was open.
template <bool kExact, int kThreads>
__device__ bool draw_row(const SampleParams& p, Group<kThreads>& g, int row, float* mine, int slot0, int first, float temp) {
  const int count = 4 * p.pieces;
  const double slack = kExact ? 0.0 : (double)p.slack;
  auto each = [&](auto f) {
    for (int i = 0; i < count; i += 4) {
      const float4 x = *reinterpret_cast<const float4*>(mine + i);
      f(i, x.x); f(i + 1, x.y); f(i + 2, x.z); f(i + 3, x.w);
    }
  };
  float m = -INFINITY;
  each([&](int, float l) { m = fmaxf(m, l); });
  m = g.max(m);
  auto give = [&](int slot, float prob) {
    p.choice[row] = slot < 0 ? -1 : slot - first;
    if (p.prob) p.prob[row] = prob;
  };
  if (m == -INFINITY) {
    if (g.thread() == 0) give(-1, 0.f);
    return true;
  }
  if (!(temp > 0.f)) {  // the first of the largest
    int at = 0x7fffffff;
    each([&](int i, float l) { if (l == m && at == 0x7fffffff) at = slot0 + i; });
    const int best = -(int)g.max(at == 0x7fffffff ? -INFINITY : -(float)at);
    if (g.thread() == 0) give(best, 1.f);
    return true;
  }
  const Weight<kExact> weight(m, temp);
  if (!weight.usable()) return false;
  using W = typename Weight<kExact>::type;
  auto mass = [&](auto keep) {
    W a[4] = {};
    for (int i = 0; i < count; i += 4) {
      const float4 x = *reinterpret_cast<const float4*>(mine + i);
      if (keep(x.x)) a[0] += weight(x.x);
      if (keep(x.y)) a[1] += weight(x.y);
      if (keep(x.z)) a[2] += weight(x.z);
      if (keep(x.w)) a[3] += weight(x.w);
    }
    return (double)((a[0] + a[1]) + (a[2] + a[3]));
  };
  // Keeps what is larger than `cut` and the first `ties` of the entries that equal it.
  auto cut_at = [&](float cut, long long ties) {
    int same = 0;
    each([&](int, float l) { same += l == cut; });
    double all;
    long long left = ties - (long long)g.before((double)same, all);
    for (int i = 0; i < count; ++i) {
      const float l = mine[i];
      if (l == cut) { if (left <= 0) mine[i] = -INFINITY; --left; }
      else if (l < cut) mine[i] = -INFINITY;
    }
  };
  const uint32_t top = key_of(m), bottom = key_of(-INFINITY);
  const float p_top = p.top_p ? p.top_p[row] : 1.f;
  const int k = p_top <= 0.f ? 1 : p.top_k ? p.top_k[row] : 0;
  if (k > 0 && k < g.threads() * count) {
    // the smallest key above which fewer than k entries lie
    uint32_t lo = bottom, hi = top;  // k or more above lo (else every entry stays), fewer above hi
    auto above = [&](float cut) {
      int c = 0;
      each([&](int, float l) { c += l > cut; });
      return g.sum((double)c);
    };
    if (above(-INFINITY) > (double)k) {
      double over = 0.0;  // above hi
      while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        const double c = above(of_key(mid));
        if (c >= (double)k) lo = mid;
        else { hi = mid; over = c; }
      }
      cut_at(of_key(hi), k - (long long)over);
    }
  }
  if (p_top > 0.f && p_top < 1.f) {
    const double all = g.sum(mass([](float l) { return l > -INFINITY; }));
    const double target = (double)p_top * all;
    uint32_t lo = bottom, hi = top;  // mass above lo: the target or more; above hi: less
    double over = 0.0;
    while (hi - lo > 1) {
      const uint32_t mid = lo + (hi - lo) / 2;
      const float cut = of_key(mid);
      const double above = g.sum(mass([&](float l) { return l > cut; }));
      if (!kExact && fabs(above - target) <= slack * all) return false;
      if (above >= target) lo = mid;
      else { hi = mid; over = above; }
    }
    // of entries equal to the cut the j-th (from 0) stays while over + j w < target; the first of all always does
    const float cut = of_key(hi);
    const double w = (double)weight(cut), ties = (target - over) / w;
    if (!kExact && (w < 1e-30 || fabs(ties - rint(ties)) <= 2.0 * slack * all / w + 1e-6 * fabs(ties))) {
      // open, unless there is a single one
      int same = 0;
      each([&](int, float l) { same += l == cut; });
      if (g.sum((double)same) > 1.0) return false;
    }
    cut_at(cut, ties >= 1e9 ? 1000000000ll : ties <= 1.0 ? 1ll : (long long)ceil(ties));
  }
  const float p_min = p.min_p ? p.min_p[row] : 0.f;
  if (p_min > 0.f) {
    bool open = false;
    const W limit = (W)fminf(p_min, 1.f);
    for (int i = 0; i < count; ++i) {
      const W w = weight(mine[i]);
      if (!kExact && mine[i] > -INFINITY && fabs((double)w - (double)limit) <= slack * (double)limit) open = mine[i] != m;
      if (w < limit) mine[i] = -INFINITY;
    }
    if (!kExact && g.sum(open ? 1.0 : 0.0) > 0.0) return false;
  }
  double total;
  const double own = mass([](float l) { return l > -INFINITY; });
  const double ahead = g.before(own, total);
  float u = p.u[row];
  u = u >= 0.f ? fminf(u, 1.f - 0x1p-24f) : 0.f;
  const double target = (double)u * total;
  // the thread whose entries the running sum passes the target in; the last with a weight where rounding leaves none
  const bool here = ahead <= target && target < ahead + own;
  bool open = false;
  int at = -1;
  if (here) {
    double run = ahead;
    for (int i = 0; i < count; ++i) {
      const double w = mine[i] > -INFINITY ? (double)weight(mine[i]) : 0.0;
      if (w > 0.0) {
        at = i;
        if (run + w > target) break;
      }
      run += w;
    }
    const double w = (double)weight(mine[at]);
    open = !kExact && (target - run <= slack * total || run + w - target <= slack * total);
  }
  if (!kExact) {
    if (g.sum(here ? (open ? 2.0 : 1.0) : 0.0) != 1.0) return false;
    if (here) give(slot0 + at, (float)((double)Weight<true>(m, temp)(mine[at]) / total));
    return true;
  }
  // 64 bits: neighbours' bounds can differ in their last bit, so that two threads claim the draw (the first has it) or none does (the
  // last thread with a weight has it)
  const float id = (float)g.thread();
  float owner = -g.max(here ? -id : -INFINITY);
  if (owner == INFINITY) {
    owner = g.max(own > 0.0 ? id : -INFINITY);
    for (int i = 0; i < count; ++i)
      if (mine[i] > -INFINITY && weight(mine[i]) > (W)0) at = i;
  }
  if (id == owner) give(slot0 + at, (float)((double)weight(mine[at]) / total));
  return true;
}

template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads == 32 ? 32 * kWarpRows : kThreads)
sample_kernel(const SampleParams p) {
  extern __shared__ float4 smem[];
  __shared__ double slots[2 * Group<kThreads>::kSlots];
  const int cap = kThreads * 4 * p.pieces;
  float* v = reinterpret_cast<float*>(smem) + (kThreads == 32 ? (threadIdx.x >> 5) * cap : 0);
  Group<kThreads> g(slots, p.cluster);
  const int row = kThreads == 32 ? blockIdx.x * kWarpRows + (threadIdx.x >> 5) : blockIdx.x / p.cluster;
  if (row >= p.rows) return;
  const float temp = p.temperature ? p.temperature[row] : 1.f;
  const int local = (kThreads == 32 ? g.lane : (int)threadIdx.x) * 4 * p.pieces;
  int n = 0;
  int first = load_row<T, kThreads>(p, g, row, v, cap, n);
  g.barrier();
  if (!draw_row<false, kThreads>(p, g, row, v + local, g.crank * cap + local, first, temp)) {
    g.barrier();
    first = load_row<T, kThreads>(p, g, row, v, cap, n);
    g.barrier();
    draw_row<true, kThreads>(p, g, row, v + local, g.crank * cap + local, first, temp);
  }
  if (kThreads == kWide && p.cluster > 1) g.barrier();  // no CTA leaves while another may write to its slots
}

template <typename T, int kThreads>
cudaError_t launch_group(const SampleParams& p, cudaStream_t s) {
  const int groups = kThreads == 32 ? kWarpRows : 1;
  cudaError_t e = raise_smem_limit<sample_kernel<T, kThreads>>(kThreads == 32 ? 64 * 1024 : kThreads == kWide ? kWide * kMaxPieces * 16 : 64 * 1024);
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
  cfg.numAttrs = p.cluster > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, sample_kernel<T, kThreads>, p);
}

template <typename T>
cudaError_t launch_sample(SampleParams p, cudaStream_t s) {
  // a row that does not start on a 16-byte boundary begins inside its first piece
  const int n = p.ids ? p.ld_ids : p.width + Pieces<T>::n - 1;
  auto pieces = [&](int threads) { return ceil_div(ceil_div(n, 4), threads) | 1; };
  p.cluster = 1;
  int threads = n <= 512 ? 32 : n <= 8192 ? 256 : kWide;
  if (threads == kWide)
    while (pieces(kWide * p.cluster) > kMaxPieces) p.cluster *= 2;
  p.pieces = pieces(threads * p.cluster);
  // Bound of a sum's error over the sum of all weights, in steps of 2^-24.  A weight: its exponent carries the rounding of l - m, at
  // most |z| steps with z = (l - m) / T, and the sum of w |z| is at most ln(n) times the sum of w; exp2f and the factor 6.
  // Sums: a thread's four chains.  Twice that, since a threshold and a sum are compared.
  p.slack = 2.f * (13.f + 6.f + p.pieces + 2.f) * 0x1p-24f;
  if (threads == 32) return launch_group<T, 32>(p, s);
  if (threads == 256) return launch_group<T, 256>(p, s);
  return launch_group<T, kWide>(p, s);
}

}  // namespace
}  // namespace b200

extern "C" int b200_op_sample(const b200_sample_desc* d, void* stream) {
  using namespace b200;
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
  const int size = d->precision == B200_PREC_FP32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(d->logits) % size) return bad("logits are not aligned to their type");
  SampleParams p = {};
  p.logits = d->logits; p.ld = d->ld ? d->ld : d->width; p.rows = d->rows; p.width = d->width;
  p.ids = d->move_ids; p.counts = d->n_moves; p.ld_ids = d->ld_moves;
  p.temperature = d->temperature; p.top_k = d->top_k; p.top_p = d->top_p; p.min_p = d->min_p; p.u = d->u;
  p.choice = d->choice; p.prob = d->prob;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (d->precision == B200_PREC_FP32) B200_CUDA(launch_sample<float>(p, s));
  else if (d->precision == B200_PREC_FP16) B200_CUDA(launch_sample<__half>(p, s));
  else B200_CUDA(launch_sample<__nv_bfloat16>(p, s));
  return B200_OK;
}
