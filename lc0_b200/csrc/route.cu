// The router in front of expert layers: every row's largest logits, their weights, and the choices sorted by expert (a counting sort that
// keeps equal ones in order).  A CTA has a block of rows: it chooses, counts its choices by expert, learns how many of each expert lie
// ahead of its own, and places them.
//   Few rows: the CTAs of one cluster, which write their counts to one another's shared memory (route_cluster_kernel, one launch).
//   Many: route_choose_kernel leaves the counts in the workspace, route_order_kernel reads all of them.
#include "chunk8.cuh"
#include "kernels.cuh"

namespace b200 {
namespace {

constexpr int kThreads = 1024, kClusterThreads = 512, kWarps = kThreads / 32;
constexpr int kMaxBlocks = 148;    // a CTA takes an SM's registers
constexpr int kMaxCluster = 8;
constexpr int kClusterChoices = 4096;  // of a CTA of the cluster, kept in shared memory

struct RouteParams {
  const void* logits; long long ld;
  int rows, experts, top_k, renormalise;
  int* ids; float* weights; int* order; int* offsets;
  int* counts;  // [blocks][stride]
  int stride;   // experts rounded up to whole fours
  int rows_per_block, blocks;
};

// A logit (not NaN) as a whole number of the same order; those below kLeast are minus infinity, which is never chosen.
constexpr uint32_t kLeast = 0x00800000u;
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);  // -0 is 0
  return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

// A logit and its expert as one whole number, larger for the one to be chosen first: equal logits by falling 255 - expert.  16-bit logits leave the
// last 13 bits of a float's key free, which hold the expert.
template <typename T> struct Choice {
  using type = uint32_t;
  static __device__ __forceinline__ type of(float v, int e) { return (key_of(v) & ~0x1fffu) | (uint32_t)(255 - e); }
  static __device__ __forceinline__ bool some(type c) { return c >= kLeast; }
  static __device__ __forceinline__ float logit(type c) { return logit_of(c & 0x80000000u ? c & ~0x1fffu : c | 0x1fffu); }
};
template <> struct Choice<float> {
  using type = unsigned long long;
  static __device__ __forceinline__ type of(float v, int e) { return (type)key_of(v) << 32 | (uint32_t)(255 - e); }
  static __device__ __forceinline__ bool some(type c) { return (uint32_t)(c >> 32) >= kLeast; }
  static __device__ __forceinline__ float logit(type c) { return logit_of((uint32_t)(c >> 32)); }
};
template <typename C> __device__ __forceinline__ C larger(C a, C b) { return a > b ? a : b; }
template <typename C> __device__ __forceinline__ void order_two(C& a, C& b) {
  const C most = larger(a, b);
  b = a > b ? b : a;
  a = most;
}

// kLanes lanes have a row, eight entries each (entry 8 * lane + i), so that a row's logits are one load per lane and all of a warp's shuffles
// serve 32 / kLanes rows.  16-bit logits: each lane sorts its eight (19 exchanges of two instructions) and offers the first of what it has left.
// fp32, whose choices are 64 bits wide: the largest of the eight is looked for anew, which costs the same from there on.  Bound by
// instructions (65536x64 bf16: 412 per warp and its four rows, two thirds of the issue slots).
template <typename T, int kLanes>
__device__ __forceinline__ void choose_row(const RouteParams& p, int row, int first, int lane, bool vec, int* counts, int* kept) {
  using Ch = Choice<T>;
  const int c = lane % kLanes, e0 = 8 * c;
  const bool live = row < p.rows;
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = -INFINITY;
  if (live) {
    const T* x = static_cast<const T*>(p.logits) + row * p.ld + e0;
    if (vec && e0 + 8 <= p.experts) {
      unpack8(load8(x), v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (e0 + i < p.experts) v[i] = to_f(x[i]);
    }
  }
  typename Ch::type mine[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = fmaxf(v[i], -INFINITY);  // NaN becomes minus infinity
    mine[i] = Ch::of(v[i], e0 + i);
  }
  constexpr bool kSorted = sizeof(T) == 2;
  if constexpr (kSorted) {  // odd-even merging
#pragma unroll
    for (int size = 1; size < 8; size *= 2)
#pragma unroll
      for (int gap = size; gap > 0; gap /= 2)
#pragma unroll
        for (int i = gap % size; i + gap < 8; i += 2 * gap)
#pragma unroll
          for (int k = 0; k < gap; ++k)
            if (i + k + gap < 8 && (i + k) / (2 * size) == (i + k + gap) / (2 * size)) order_two(mine[i + k], mine[i + k + gap]);
  }
  constexpr int kMost = 8 * kLanes < B200_MAX_TOP_K ? 8 * kLanes : B200_MAX_TOP_K, kKeep = (kMost + kLanes - 1) / kLanes;
  typename Ch::type keep[kKeep], head = 0;  // lane c of the row keeps the choices c, c + kLanes, ...
#pragma unroll
  for (int q = 0; q < kKeep; ++q) keep[q] = 0;
  for (int j = 0; j < p.top_k; ++j) {
    typename Ch::type best = mine[0];
    if constexpr (!kSorted) {
#pragma unroll
      for (int i = 1; i < 8; ++i) best = larger(best, mine[i]);
    }
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) best = larger(best, __shfl_xor_sync(0xffffffffu, best, o));
    if constexpr (kSorted) {
      const bool pop = mine[0] == best;
#pragma unroll
      for (int i = 0; i < 7; ++i) mine[i] = pop ? mine[i + 1] : mine[i];
      if (pop) mine[7] = 0;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) mine[i] = mine[i] == best ? 0 : mine[i];
    }
    if (j == 0) head = best;
#pragma unroll
    for (int q = 0; q < kKeep; ++q)
      if (q * kLanes + c == j) keep[q] = best;
  }
  const float top = Ch::some(head) ? Ch::logit(head) : 0.f;
  // 16-bit logits: the sum takes the quick exponential, whose term e^x is off by (|x| 2^-24.5 + 2^-22) e^x, far less than the logit's own rounding
  // makes of it.  fp32 logits: expf, as elsewhere (65536x64, four choices 25.3 us with the quick one, 25.7).
  float total = 0.f, weight[kKeep];
  if (p.weights) {
#pragma unroll
    for (int q = 0; q < kKeep; ++q) {
      const float l = Ch::logit(keep[q]);
      weight[q] = !Ch::some(keep[q]) ? 0.f : l == top ? 1.f : top < INFINITY ? expf(l - top) : 0.f;
    }
    if (p.renormalise) {
#pragma unroll
      for (int q = 0; q < kKeep; ++q) total += weight[q];
    } else if (top < INFINITY) {
#pragma unroll
      for (int i = 0; i < 8; ++i) total += sizeof(T) == 4 ? expf(v[i] - top) : __expf(v[i] - top);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) total += v[i] == top ? 1.f : 0.f;
    }
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  if (!live) return;
#pragma unroll
  for (int q = 0; q < kKeep; ++q) {
    const int j = q * kLanes + c;
    if (j >= p.top_k) continue;
    const long long r = (long long)row * p.top_k + j;
    const int id = Ch::some(keep[q]) ? 255 - (int)(keep[q] & 0xffu) : -1;
    p.ids[r] = id;
    if (kept) kept[(row - first) * p.top_k + j] = id;
    if (p.weights) p.weights[r] = id >= 0 ? weight[q] / total : 0.f;
    if (id >= 0) atomicAdd(counts + id, 1);
  }
}

// All rows of a block; kLanes 0: the ids are given.  `kept` (may be nullptr) gets the block's choices.
template <typename T, int kLanes>
__device__ __forceinline__ void choose_block(const RouteParams& p, int first, int end, bool vec, int* counts, int* kept) {
  const int threads = blockDim.x;
  for (int e = threadIdx.x; e < p.stride; e += threads) counts[e] = 0;
  __syncthreads();
  if constexpr (kLanes > 0) {
    const int lane = threadIdx.x & 31;
    for (int row0 = first; row0 < end; row0 += threads / kLanes) {
      const int row = row0 + (int)threadIdx.x / kLanes;
      choose_row<T, kLanes>(p, row < end ? row : p.rows, first, lane, vec, counts, kept);
    }
  } else {
    const long long from = (long long)first * p.top_k;
    const int n = (end - first) * p.top_k;
    for (int i = threadIdx.x; i < n; i += threads) {
      const int id = p.ids[from + i];
      if (kept) kept[i] = id;
      if (id >= 0 && id < p.experts) atomicAdd(counts + id, 1);
    }
  }
  __syncthreads();
}

template <int kWarps> struct PlaceMemory {
  int of_warp[kWarps][B200_MAX_EXPERTS];  // an expert's choices of each warp, then the place of the warp's next one
  int total[B200_MAX_EXPERTS], before[B200_MAX_EXPERTS];  // choices of an expert: in all blocks, in the blocks ahead of this one
  int scan[8];
};
// Places this block's choices, given total and before.
template <int kWarps> __device__ __forceinline__ void place_block(const RouteParams& p, int first, int end, bool first_block, const int* kept, PlaceMemory<kWarps>& m) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = threadIdx.x;
  const long long from = (long long)first * p.top_k;
  const int n = (end - first) * p.top_k, per_warp = ((n + kWarps - 1) / kWarps + 31) & ~31;
  const int w0 = warp * per_warp, w1 = min(w0 + per_warp, n);
  auto id_of = [&](int i) {
    const int id = i < w1 ? (kept ? kept[i] : p.ids[from + i]) : -1;
    return id >= 0 && id < p.experts ? id : -1;
  };
  for (int w = 0; w < kWarps; ++w)
    if (threadIdx.x < (unsigned)p.experts) m.of_warp[w][threadIdx.x] = 0;
  __syncthreads();
  for (int i = w0 + lane; i < w1; i += 32) {
    const int id = id_of(i);
    if (id >= 0) atomicAdd(&m.of_warp[warp][id], 1);
  }
  int upto = 0;
  if (e < 256) {
    upto = e < p.experts ? m.total[e] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int k = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += k;
    }
    if (lane == 31) m.scan[warp] = upto;
  }
  __syncthreads();
  if (e < p.experts) {
    for (int w = 0; w < warp; ++w) upto += m.scan[w];
    const int begin = upto - m.total[e];
    if (first_block) {
      p.offsets[e] = begin;
      if (e == p.experts - 1) p.offsets[p.experts] = upto;
    }
    int at = begin + m.before[e];
#pragma unroll 8
    for (int w = 0; w < kWarps; ++w) {
      const int k = m.of_warp[w][e];
      m.of_warp[w][e] = at;
      at += k;
    }
  }
  __syncthreads();
  for (int i0 = w0; i0 < w1; i0 += 32) {
    const int id = id_of(i0 + lane);
    const uint32_t same = __match_any_sync(0xffffffffu, id);
    const int rank = __popc(same & ((1u << lane) - 1u)), at = id >= 0 ? m.of_warp[warp][id] : 0;
    __syncwarp();
    if (id >= 0) {
      p.order[at + rank] = (int)(from + i0 + lane);
      if (rank == 0) m.of_warp[warp][id] = at + __popc(same);
    }
    __syncwarp();
  }
}

template <typename T, int kLanes>
__global__ void __launch_bounds__(kThreads) route_choose_kernel(const RouteParams p, bool vec) {
  __shared__ int counts[B200_MAX_EXPERTS];
  grid_launch_dependents();
  grid_dependency_wait();
  const int first = blockIdx.x * p.rows_per_block;
  choose_block<T, kLanes>(p, first, min(first + p.rows_per_block, p.rows), vec, counts, nullptr);
  for (int e = threadIdx.x; e < p.stride; e += kThreads) p.counts[blockIdx.x * p.stride + e] = counts[e];
}

// Four experts' counts per load, all loads of a thread on their way together.
__global__ void __launch_bounds__(kThreads) route_order_kernel(const RouteParams p) {
  __shared__ PlaceMemory<kWarps> m;
  grid_launch_dependents();
  for (int e = threadIdx.x; e < B200_MAX_EXPERTS; e += kThreads) m.total[e] = m.before[e] = 0;
  __syncthreads();
  grid_dependency_wait();
  const int fours = p.stride / 4, groups = kThreads / fours, q = threadIdx.x % fours, g = threadIdx.x / fours;
  if (g < groups) {
    int4 total = make_int4(0, 0, 0, 0), before = total;
#pragma unroll 10
    for (int b = g; b < p.blocks; b += groups) {
      const int4 n = reinterpret_cast<const int4*>(p.counts)[b * fours + q];
      total = make_int4(total.x + n.x, total.y + n.y, total.z + n.z, total.w + n.w);
      if (b < (int)blockIdx.x) before = make_int4(before.x + n.x, before.y + n.y, before.z + n.z, before.w + n.w);
    }
    const int t[4] = {total.x, total.y, total.z, total.w}, u[4] = {before.x, before.y, before.z, before.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (t[i]) atomicAdd(m.total + 4 * q + i, t[i]);
      if (u[i]) atomicAdd(m.before + 4 * q + i, u[i]);
    }
  }
  __syncthreads();
  const int first = blockIdx.x * p.rows_per_block;
  place_block(p, first, min(first + p.rows_per_block, p.rows), blockIdx.x == 0, nullptr, m);
}

// All of it by one cluster.
template <typename T, int kLanes>
__global__ void __launch_bounds__(kClusterThreads) route_cluster_kernel(const RouteParams p, bool vec) {
  __shared__ PlaceMemory<kClusterThreads / 32> m;
  __shared__ int all[kMaxCluster][B200_MAX_EXPERTS];  // counts of each CTA
  __shared__ int counts[B200_MAX_EXPERTS];
  __shared__ int kept[kClusterChoices];
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  grid_launch_dependents();
  grid_dependency_wait();
  const int first = min(blockIdx.x * p.rows_per_block, p.rows), end = min(first + p.rows_per_block, p.rows);
  choose_block<T, kLanes>(p, first, end, vec, counts, kept);
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // all CTAs run
  for (int i = threadIdx.x; i < p.blocks * p.stride; i += kClusterThreads) {
    const int cta = i / p.stride, e = i - cta * p.stride;
    uint32_t to;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"((uint32_t)__cvta_generic_to_shared(&all[blockIdx.x][e])), "r"(cta));
    asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(to), "r"(counts[e]) : "memory");
  }
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (threadIdx.x < (unsigned)p.experts) {
    int total = 0, before = 0;
    for (int b = 0; b < p.blocks; ++b) {
      if (b == (int)blockIdx.x) before = total;
      total += all[b][threadIdx.x];
    }
    m.total[threadIdx.x] = total;
    m.before[threadIdx.x] = before;
  }
  __syncthreads();
  place_block(p, first, end, blockIdx.x == 0, kept, m);
}

int lanes_of(int experts) {
  int l = 1;
  while (8 * l < experts) l *= 2;
  return l;
}

// Rows to a block: whole passes of its threads.  A cluster where its eight CTAs have few passes (us, one cluster / two launches: 1536x16 4.8 / 8.4, 4000x16 7.0 / 8.6, 512x64
// 4.6 / 6.7, 1024x64 6.2 / 6.9; four passes, 2048x64, 9.5 / 7.0).
bool plan_blocks(RouteParams& p, int lanes) {
  const long long small = kClusterThreads / lanes, few = (p.rows + kMaxCluster * small - 1) / (kMaxCluster * small);
  const bool cluster = few <= 2 && few * small * p.top_k <= kClusterChoices;
  const long long pass = cluster ? small : kThreads / lanes, passes = (p.rows + pass - 1) / pass;
  const long long most = cluster ? kMaxCluster : kMaxBlocks, per = (passes + most - 1) / most;
  p.rows_per_block = (int)(per * pass);
  p.blocks = (int)((p.rows + per * pass - 1) / (per * pass));
  p.stride = (p.experts + 3) & ~3;
  return cluster;
}

template <typename T, int kLanes>
cudaError_t launch_route(RouteParams p, cudaStream_t s) {
  const bool vec = reinterpret_cast<uintptr_t>(p.logits) % 16 == 0 && p.ld % (16 / (int)sizeof(T)) == 0;
  cudaError_t e;
  if (plan_blocks(p, kLanes ? kLanes : 1)) {
    int size = 1;
    while (size < p.blocks) size *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(size);
    cfg.blockDim = dim3(kClusterThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = size;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    p.blocks = size;
    return cudaLaunchKernelEx(&cfg, route_cluster_kernel<T, kLanes>, static_cast<const RouteParams&>(p), vec);
  }
  if ((e = launch_dependent(route_choose_kernel<T, kLanes>, dim3(p.blocks), dim3(kThreads), 0, s, p, vec)) != cudaSuccess) return e;
  return launch_dependent(route_order_kernel, dim3(p.blocks), dim3(kThreads), 0, s, p);
}
template <typename T>
cudaError_t launch_lanes(const RouteParams& p, cudaStream_t s) {
  switch (lanes_of(p.experts)) {
    case 1: return launch_route<T, 1>(p, s);
    case 2: return launch_route<T, 2>(p, s);
    case 4: return launch_route<T, 4>(p, s);
    case 8: return launch_route<T, 8>(p, s);
    case 16: return launch_route<T, 16>(p, s);
    default: return launch_route<T, 32>(p, s);
  }
}

__global__ void route_none_kernel(int* offsets, int n) {
  grid_launch_dependents();
  grid_dependency_wait();
  for (int i = threadIdx.x; i < n; i += blockDim.x) offsets[i] = 0;
}

const char* check_shape(const b200_route_desc* d) {
  if (!d) return "no description";
  if (d->n_experts < 1 || d->n_experts > B200_MAX_EXPERTS) return "n_experts 1 to 256";
  if (d->top_k < 1 || d->top_k > B200_MAX_TOP_K || (d->top_k > d->n_experts && d->logits)) return "top_k 1 to 16 and at most n_experts";
  if (d->rows < 0 || (long long)d->rows * d->top_k > 1 << 30) return "rows * top_k of 0 to 2^30";
  if (d->precision < B200_PREC_FP32 || d->precision > B200_PREC_BF16) return "unknown precision";
  if (d->ld && d->ld < d->n_experts) return "rows overlap";
  return nullptr;
}
size_t route_bytes(const b200_route_desc& d) {
  return ((size_t)kMaxBlocks * ((d.n_experts + 3) / 4 * 4) * 4 + 255) & ~size_t(255);
}

}  // namespace
}  // namespace b200

extern "C" int b200_op_route_workspace(const b200_route_desc* d, size_t* bytes) {
  using namespace b200;
  return at_c_entry([&]() -> int {
    const char* wrong = check_shape(d);
    if (!wrong && !bytes) wrong = "nowhere to put the size";
    if (wrong) {
      set_error(std::string("b200_op_route_workspace: ") + wrong);
      return B200_ERR_INVALID;
    }
    *bytes = route_bytes(*d);
    return B200_OK;
  });
}

extern "C" int b200_op_route(const b200_route_desc* d, void* stream) {
  using namespace b200;
  return at_c_entry([&]() -> int {
    const char* wrong = check_shape(d);
    if (!wrong) {
      auto off = [](const void* q, uintptr_t n) { return reinterpret_cast<uintptr_t>(q) % n != 0; };
      if (!d->offsets || off(d->offsets, 4)) wrong = "offsets are needed, aligned to their type";
      else if (d->rows > 0 && (!d->ids || !d->order)) wrong = "ids and order are needed";
      else if (!d->logits && d->weights) wrong = "weights come from logits";
      else if (off(d->logits, d->precision == B200_PREC_FP32 ? 4 : 2) || off(d->ids, 4) || off(d->weights, 4) || off(d->order, 4))
        wrong = "an operand is not aligned to its type";
      else if (d->rows > 0 && (!d->workspace || off(d->workspace, 256) || d->workspace_bytes < route_bytes(*d)))
        wrong = "the workspace is missing, too small or not on a 256-byte boundary";
    }
    if (wrong) {
      set_error(std::string("b200_op_route: ") + wrong);
      return B200_ERR_INVALID;
    }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    DependentLaunches dependent;
    if (d->rows == 0) {
      B200_CUDA(launch_dependent(route_none_kernel, dim3(1), dim3(256), 0, s, d->offsets, d->n_experts + 1));
      return B200_OK;
    }
    RouteParams p = {};
    p.logits = d->logits; p.ld = d->ld ? d->ld : d->n_experts;
    p.rows = d->rows; p.experts = d->n_experts; p.top_k = d->top_k; p.renormalise = d->renormalise;
    p.ids = d->ids; p.weights = d->weights; p.order = d->order; p.offsets = d->offsets;
    p.counts = static_cast<int*>(d->workspace);
    if (!d->logits) B200_CUDA((launch_route<float, 0>(p, s)));
    else if (d->precision == B200_PREC_FP32) B200_CUDA(launch_lanes<float>(p, s));
    else if (d->precision == B200_PREC_FP16) B200_CUDA(launch_lanes<__half>(p, s));
    else B200_CUDA(launch_lanes<__nv_bfloat16>(p, s));
    return B200_OK;
  });
}
