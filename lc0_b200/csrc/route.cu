// The router in front of expert layers: every row's largest logits, their weights, and the choices sorted by expert (a counting sort that
// keeps equal ones in order).
//   1. route_choose_kernel: a CTA per block of rows chooses and counts its choices by expert.
//   2. route_order_kernel: the counts of all blocks give each block its first place among an expert's choices; it places its own.
#include "chunk8.cuh"
#include "kernels.cuh"

namespace b200 {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxBlocks = 296;  // two per SM

struct RouteParams {
  const void* logits; long long ld;
  int rows, experts, top_k, renormalise;
  int* ids; float* weights; int* order; int* offsets;
  int* counts;  // [blocks][experts]
  int rows_per_block, blocks;
};

// A logit as a whole number of the same order; 0 for what is never chosen.
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);  // -0 is 0
  return v > -INFINITY ? (u & 0x80000000u ? ~u : u | 0x80000000u) : 0u;
}
__device__ __forceinline__ float logit_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

// kLanes lanes have a row, eight entries each (entry 8 * lane + i), so that a row's logits are one load per lane and all of a warp's shuffles
// serve 32 / kLanes rows.
template <typename T, int kLanes>
__device__ __forceinline__ void choose_row(const RouteParams& p, int row, int lane, bool vec, int* counts) {
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
  uint32_t key[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) key[i] = key_of(v[i]);
  constexpr int kKeep = (B200_MAX_TOP_K + kLanes - 1) / kLanes;
  float top = 0.f, total = 0.f, weight[kKeep];  // lane c of the row keeps the choices c, c + kLanes, ...
  int id[kKeep];
#pragma unroll
  for (int q = 0; q < kKeep; ++q) {
    weight[q] = 0.f;
    id[q] = -1;
  }
  for (int j = 0; j < p.top_k; ++j) {
    uint32_t best = 0;
    int at = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (key[i] > best) {
        best = key[i];
        at = e0 + i;
      }
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) {
      const uint32_t b = __shfl_xor_sync(0xffffffffu, best, o);
      const int a = __shfl_xor_sync(0xffffffffu, at, o);
      if (b > best || (b == best && a < at)) {
        best = b;
        at = a;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (at == e0 + i) key[i] = 0;
    const float l = logit_of(best);
    if (j == 0) {
      top = l;
      if (!p.renormalise) {
#pragma unroll
        for (int i = 0; i < 8; ++i) total += v[i] == top ? 1.f : (v[i] > -INFINITY && top < INFINITY ? expf(v[i] - top) : 0.f);
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
      }
    }
    const float w = best == 0 ? 0.f : l == top ? 1.f : top < INFINITY ? expf(l - top) : 0.f;
    if (p.renormalise) total += w;
#pragma unroll
    for (int q = 0; q < kKeep; ++q)
      if (q * kLanes + c == j) {
        weight[q] = w;
        id[q] = best ? at : -1;
      }
  }
  if (!live) return;
#pragma unroll
  for (int q = 0; q < kKeep; ++q) {
    const int j = q * kLanes + c;
    if (j >= p.top_k) continue;
    const long long r = (long long)row * p.top_k + j;
    p.ids[r] = id[q];
    if (p.weights) p.weights[r] = total > 0.f ? weight[q] / total : 0.f;
    if (id[q] >= 0) atomicAdd(counts + id[q], 1);
  }
}

template <typename T, int kLanes>
__global__ void __launch_bounds__(kThreads) route_choose_kernel(const RouteParams p, bool vec) {
  __shared__ int counts[B200_MAX_EXPERTS];
  grid_launch_dependents();
  for (int e = threadIdx.x; e < p.experts; e += kThreads) counts[e] = 0;
  __syncthreads();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, first = blockIdx.x * p.rows_per_block;
  const int end = min(first + p.rows_per_block, p.rows);
  for (int row0 = first; row0 < end; row0 += kThreads / kLanes) {
    const int row = row0 + (int)threadIdx.x / kLanes;
    choose_row<T, kLanes>(p, row < end ? row : p.rows, lane, vec, counts);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.experts; e += kThreads) p.counts[blockIdx.x * p.experts + e] = counts[e];
}

// Given ids: counts alone.
__global__ void __launch_bounds__(kThreads) route_count_kernel(const RouteParams p) {
  __shared__ int counts[B200_MAX_EXPERTS];
  grid_launch_dependents();
  for (int e = threadIdx.x; e < p.experts; e += kThreads) counts[e] = 0;
  __syncthreads();
  grid_dependency_wait();
  const long long first = (long long)blockIdx.x * p.rows_per_block * p.top_k;
  const long long end = min(first + (long long)p.rows_per_block * p.top_k, (long long)p.rows * p.top_k);
  for (long long r = first + threadIdx.x; r < end; r += kThreads) {
    const int id = p.ids[r];
    if (id >= 0 && id < p.experts) atomicAdd(counts + id, 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.experts; e += kThreads) p.counts[blockIdx.x * p.experts + e] = counts[e];
}

__global__ void __launch_bounds__(kThreads) route_order_kernel(const RouteParams p) {
  __shared__ int of_warp[kWarps][B200_MAX_EXPERTS];  // an expert's choices of each warp, then the place of the warp's next one
  __shared__ int scan[kWarps];
  grid_launch_dependents();
  for (int i = threadIdx.x; i < kWarps * B200_MAX_EXPERTS; i += kThreads) (&of_warp[0][0])[i] = 0;
  __syncthreads();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = threadIdx.x;
  // place of this block's first choice of expert e
  int total = 0, before = 0;
  if (e < p.experts) {
#pragma unroll 8
    for (int b = 0; b < p.blocks; ++b) {
      const int n = p.counts[b * p.experts + e];
      total += n;
      before += b < (int)blockIdx.x ? n : 0;
    }
  }
  int upto = total;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int n = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += n;
  }
  if (lane == 31) scan[warp] = upto;
  // this block's choices by warp
  const long long first = (long long)blockIdx.x * p.rows_per_block * p.top_k;
  const long long end = min(first + (long long)p.rows_per_block * p.top_k, (long long)p.rows * p.top_k);
  const long long per_warp = (end - first + kWarps - 1) / kWarps;
  const long long w0 = first + warp * per_warp, w1 = min(w0 + per_warp, end);
  for (long long r = w0 + lane; r < w1; r += 32) {
    const int id = p.ids[r];
    if (id >= 0 && id < p.experts) atomicAdd(&of_warp[warp][id], 1);
  }
  __syncthreads();
  for (int w = 0; w < warp; ++w) upto += scan[w];
  if (e < p.experts) {
    int at = upto - total + before;
    if (blockIdx.x == 0) {
      p.offsets[e] = upto - total;
      if (e == p.experts - 1) p.offsets[p.experts] = upto;
    }
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const int n = of_warp[w][e];
      of_warp[w][e] = at;
      at += n;
    }
  }
  __syncthreads();
  for (long long r0 = w0; r0 < w1; r0 += 32) {
    const long long r = r0 + lane;
    int id = r < w1 ? p.ids[r] : -1;
    if (id >= p.experts) id = -1;
    const uint32_t same = __match_any_sync(0xffffffffu, id);
    const int rank = __popc(same & ((1u << lane) - 1u));
    const int at = id >= 0 ? of_warp[warp][id] : 0;
    __syncwarp();
    if (id >= 0) {
      p.order[at + rank] = (int)r;
      if (rank == 0) of_warp[warp][id] = at + __popc(same);
    }
    __syncwarp();
  }
}

int lanes_of(int experts) {
  int l = 1;
  while (8 * l < experts) l *= 2;
  return l;
}

// Blocks of rows: enough for every SM to have some, none without a full pass of its threads.
void plan_blocks(RouteParams& p) {
  const int pass = kThreads / lanes_of(p.experts);
  const long long passes = ((long long)p.rows + pass - 1) / pass;
  const long long blocks = passes < kMaxBlocks ? passes : kMaxBlocks;
  const long long per = (passes + blocks - 1) / blocks;
  p.rows_per_block = (int)(per * pass);
  p.blocks = (int)((p.rows + per * pass - 1) / (per * pass));
}

template <typename T>
cudaError_t launch_choose(const RouteParams& p, cudaStream_t s) {
  const bool vec = reinterpret_cast<uintptr_t>(p.logits) % 16 == 0 && p.ld % (16 / (int)sizeof(T)) == 0;
  const int lanes = lanes_of(p.experts);
  auto kernel = lanes == 1 ? route_choose_kernel<T, 1>
                : lanes == 2 ? route_choose_kernel<T, 2>
                : lanes == 4 ? route_choose_kernel<T, 4>
                : lanes == 8 ? route_choose_kernel<T, 8>
                : lanes == 16 ? route_choose_kernel<T, 16>
                              : route_choose_kernel<T, 32>;
  return launch_dependent(kernel, dim3(p.blocks), dim3(kThreads), 0, s, p, vec);
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
  if (d->rows < 0 || (long long)d->rows * d->top_k > 0x7fffffffll) return "rows * top_k of 0 to 2^31 - 1";
  if (d->precision < B200_PREC_FP32 || d->precision > B200_PREC_BF16) return "unknown precision";
  if (d->ld && d->ld < d->n_experts) return "rows overlap";
  return nullptr;
}
size_t route_bytes(const b200_route_desc& d) {
  return ((size_t)kMaxBlocks * d.n_experts * 4 + 255) & ~size_t(255);
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
    plan_blocks(p);
    if (!d->logits) B200_CUDA(launch_dependent(route_count_kernel, dim3(p.blocks), dim3(kThreads), 0, s, p));
    else if (d->precision == B200_PREC_FP32) B200_CUDA(launch_choose<float>(p, s));
    else if (d->precision == B200_PREC_FP16) B200_CUDA(launch_choose<__half>(p, s));
    else B200_CUDA(launch_choose<__nv_bfloat16>(p, s));
    B200_CUDA(launch_dependent(route_order_kernel, dim3(p.blocks), dim3(kThreads), 0, s, p));
    return B200_OK;
  });
}
