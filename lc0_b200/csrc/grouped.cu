// b200_op_gemm_int8 and b200_op_gemm_experts: entry points, the kernel for operands of any size and alignment, and the sum over a token's
// choices.
#include "chunk8.cuh"
#include "grouped.cuh"

namespace b200 {
namespace {

template <typename T> struct SumOf { using type = float; };
template <> struct SumOf<int8_t> { using type = int; };
__device__ __forceinline__ float operand(__half v) { return __half2float(v); }
__device__ __forceinline__ float operand(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ int operand(int8_t v) { return v; }
__device__ __forceinline__ float plus_product(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ int plus_product(int a, int b, int c) { return a * b + c; }

// ---- any size and alignment -------------------------------------------------------------------------------------
constexpr int kTile = 64, kDepth = 16;

// A CTA per 64 slots of an expert and 64 columns; sums in one chain per element, k rising.
template <typename TIn, typename TOut>
__global__ void __launch_bounds__(256) grouped_any_kernel(const GroupedParams p) {
  using Sum = typename SumOf<TIn>::type;
  __shared__ Sum sx[kDepth][kTile + 1], sw[kDepth][kTile + 1];
  __shared__ int x_row[kTile], c_row[kTile], choice_of[kTile];
  grid_launch_dependents();
  grid_dependency_wait();
  const int tid = threadIdx.x, tx = tid % 16, ty = tid / 16, n0 = blockIdx.x * kTile;
  for (long long block = blockIdx.y;; block += gridDim.y) {
    // the block's expert and first slot
    long long left = block;
    int e = 0, begin = 0, end = expert_begin(p, 0);
    for (; e < p.experts; ++e) {
      begin = end;
      end = max(begin, expert_begin(p, e + 1));
      const int blocks = (end - begin + kTile - 1) / kTile;
      if (left < blocks) break;
      left -= blocks;
    }
    if (e == p.experts) return;
    const int s0 = begin + (int)left * kTile;
    __syncthreads();
    if (tid < kTile) {
      SlotRows r = {-1, -1, 0};
      if (s0 + tid < end) r = rows_of_slot(p, s0 + tid);
      if (n0 == 0) keep_place(p, r, s0 + tid);
      x_row[tid] = r.x; c_row[tid] = r.c; choice_of[tid] = r.choice;
    }
    __syncthreads();
    Sum acc[4][4] = {};
    const TIn* W = static_cast<const TIn*>(p.W) + (long long)e * p.N * p.ldw;
    for (int k0 = 0; k0 < p.K; k0 += kDepth) {
      for (int i = tid; i < kTile * kDepth; i += 256) {
        const int r = i / kDepth, k = i % kDepth;
        const bool in = k0 + k < p.K;
        sx[k][r] = in && x_row[r] >= 0 ? operand(static_cast<const TIn*>(p.X)[x_row[r] * p.ldx + k0 + k]) : Sum(0);
        sw[k][r] = in && n0 + r < p.N ? operand(W[(n0 + r) * p.ldw + k0 + k]) : Sum(0);
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kDepth; ++k) {
        Sum a[4], b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          a[i] = sx[k][ty * 4 + i];
          b[i] = sw[k][tx + 16 * i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] = plus_product(a[i], b[j], acc[i][j]);
      }
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = ty * 4 + i, c = c_row[r];
      if (c < 0) continue;
      const float weight = p.weights ? p.alpha * p.weights[choice_of[r]] : p.alpha;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = n0 + tx + 16 * j;
        if (n >= p.N) continue;
        float v = (float)acc[i][j];
        if (p.w_scales) v *= p.x_scales[x_row[r]] * p.w_scales[e * (long long)p.N + n];
        if (p.bias) v += p.bias[e * (long long)p.N + n];
        v = activate<sizeof(TOut) == 2>(v, p.act) * weight;
        if (p.res) v += to_f(static_cast<const TOut*>(p.res)[c * p.ldres + n]);
        static_cast<TOut*>(p.C)[c * p.ldc + n] = one_of<TOut>(v);
      }
    }
  }
}

template <typename TIn, typename TOut>
cudaError_t launch_any(const GroupedParams& p, cudaStream_t s) {
  const long long blocks = ((long long)p.slots + kTile - 1) / kTile + p.experts - 1;
  return launch_dependent(grouped_any_kernel<TIn, TOut>, dim3(ceil_div(p.N, kTile), (unsigned)(blocks < 65535 ? blocks : 65535)), dim3(256), 0, s, p);
}

// ---- the sum over a token's choices -----------------------------------------------------------------------------
struct CombineParams {
  const float* Y;    // [tokens * top_k][N] by slot
  const int* place;  // of each choice, in requests
  const int* ids;
  const void* res; long long ldres;
  void* C; long long ldc;
  int tokens, N, experts, top_k, group;
};

// The place of a request's choice, -1 where it has no expert (or order does not name it, which is the caller's to rule out).
__device__ __forceinline__ int place_of(const CombineParams& p, int request, int j) {
  const long long choice = (long long)request * p.top_k + j;
  const int id = p.ids[choice], at = p.place[choice];
  return id >= 0 && id < p.experts && at >= 0 && at < p.tokens / p.group * p.top_k ? at : -1;
}

// A warp per token and 512 columns: two pieces of eight columns per lane, whose rows of all choices are on their way together; the choices are
// added in order.
template <typename TOut>
__global__ void __launch_bounds__(256) combine_kernel(const CombineParams p, int vec) {
  grid_launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, parts = (p.N + 511) / 512;
  const long long all = (long long)p.tokens * parts;
  for (long long i = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); i < all; i += (long long)gridDim.x * 8) {
    const int t = (int)(i / parts), n0 = (int)(i - (long long)t * parts) * 512 + lane * 8, request = t / p.group, inside = t - request * p.group;
    const TOut* res = p.res ? static_cast<const TOut*>(p.res) + t * p.ldres : nullptr;
    TOut* c = static_cast<TOut*>(p.C) + t * p.ldc;
    if (vec) {
      Chunk<TOut> more[2];
      float v[2][8] = {};
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (res && n0 + 256 * h < p.N) more[h] = load8(res + n0 + 256 * h);
      bool any = false;
#pragma unroll 2
      for (int j = 0; j < p.top_k; ++j) {
        const int at = place_of(p, request, j);
        if (at < 0) continue;
        any = true;
        const float* y = p.Y + ((long long)at * p.group + inside) * p.N + n0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (n0 + 256 * h >= p.N) continue;
          const float4 a = __ldcs(reinterpret_cast<const float4*>(y + 256 * h)), b = __ldcs(reinterpret_cast<const float4*>(y + 256 * h) + 1);
          v[h][0] += a.x; v[h][1] += a.y; v[h][2] += a.z; v[h][3] += a.w;
          v[h][4] += b.x; v[h][5] += b.y; v[h][6] += b.z; v[h][7] += b.w;
        }
      }
      if (!any) continue;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (n0 + 256 * h >= p.N) continue;
        if (res) {
          float w[8];
          unpack8(more[h], w);
#pragma unroll
          for (int k = 0; k < 8; ++k) v[h][k] += w[k];
        }
        store8(c + n0 + 256 * h, pack8<TOut>(v[h]));
      }
    } else {
      bool any = false;
      for (int j = 0; j < p.top_k; ++j) any |= place_of(p, request, j) >= 0;
      if (!any) continue;
      for (int n = n0 - 7 * lane; n < min(n0 - 8 * lane + 512, p.N); n += 32) {  // column by column
        float v = 0.f;
        for (int j = 0; j < p.top_k; ++j) {
          const int at = place_of(p, request, j);
          if (at >= 0) v += p.Y[((long long)at * p.group + inside) * p.N + n];
        }
        c[n] = one_of<TOut>(res ? v + to_f(res[n]) : v);
      }
    }
  }
}

template <typename TOut>
cudaError_t launch_combine(const CombineParams& p, cudaStream_t s) {
  auto fine = [&](const void* q, long long ld) { return reinterpret_cast<uintptr_t>(q) % 16 == 0 && ld % (16 / (int)sizeof(TOut)) == 0; };
  const int vec = p.N % 8 == 0 && fine(p.C, p.ldc) && (!p.res || fine(p.res, p.ldres));
  const long long blocks = ((long long)p.tokens * ((p.N + 511) / 512) + 7) / 8;
  return launch_dependent(combine_kernel<TOut>, dim3((unsigned)(blocks < 148 * 64 ? blocks : 148 * 64)), dim3(256), 0, s, p, vec);
}

// ---- rows in the order of their slots ---------------------------------------------------------------------------
// The pair kernel reads X by boxes of 128 rows, or of 64 where requests are whole 64 rows (1344 rows over 8 experts 13.1 us, copied 18.1); other
// rows that the order names are copied into their order first, once for all tiles of columns, which then find them in L2.
// Fetched in place by TMA's gather4, 33 cycles for four rows and anew for each tile of columns, the product takes half as long again (us, 32768
// slots x 1024 to 1536 columns: 136, in order with the copy 102; by cp.async into the swizzled tiles 318, as the proxy fence ahead of each
// hand-over waits for all copies in flight).
__global__ void __launch_bounds__(256) spread_rows_kernel(const GroupedParams p, uint8_t* to, int row_bytes, int size) {
  grid_launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, pieces = row_bytes / 16;
  int end = 0;
  for (int e = lane; e <= p.experts; e += 32) end = max(end, expert_begin(p, e));
  end = __reduce_max_sync(0xffffffffu, end);
  for (long long slot = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); slot < end; slot += (long long)gridDim.x * 8) {
    const int x = rows_of_slot(p, (int)slot).x;
    if (x < 0) continue;
    const uint4* from = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p.X) + x * p.ldx * size);
    uint4* at = reinterpret_cast<uint4*>(to + slot * row_bytes);
#pragma unroll 4
    for (int i = lane; i < pieces; i += 32) at[i] = from[i];
  }
}

// Rows of X and W that TMA can read.
bool tma_rows(int K, long long ldx, long long ldw, int size) { return K * (long long)size % 16 == 0 && ldx * size % 16 == 0 && ldw * size % 16 == 0; }
// The pair kernel's 256 slots pay from a quarter of a tile per expert on, and where the other kernel's tiles of 64 slots x 128 columns are more than
// a quarter of the SMs (us, pair kernel / the other; int8, K 1024, to 1024 columns: 256 rows, 32 tiles, 7.0 / 6.3, 320 rows, 40 tiles, 7.0 / 7.3,
// 512 rows 7.1 / 7.7, 1024 rows 7.2 / 8.2; K 1536, to 512 columns: 512 rows, 32 tiles, 7.6 / 6.5, 768 rows, 48 tiles, 7.7 / 7.8; 16 bits: 300 rows over 4
// experts, copied into order, to 1024 columns, 48 tiles, 11.1 / 12.4, eight positions over 4 experts to 768 columns, 60 tiles, 9.5 / 10.0).
bool many_rows(const GroupedParams& p, int sms) {
  const int used = p.experts < p.slots ? p.experts : p.slots;
  return p.slots / used > 64 && ((long long)p.slots / 64 + used / 2) * ceil_div(p.N, 128) > sms / 4;
}
// Beyond 16 rows per expert the other kernel, too, is ahead with rows in order, although the copy is a launch more (333 rows over 12 experts to 1858
// columns 25.1 in place, 20.2).
bool spreads(int slots, int experts) { return slots / (experts < slots ? experts : slots) > 16; }

template <typename TIn, typename TOut>
int run_grouped(GroupedParams p, bool exact_sums, void* spread, cudaStream_t s) {
  if (!tma_rows(p.K, p.ldx, p.ldw, sizeof(TIn)) || reinterpret_cast<uintptr_t>(p.X) % 16 != 0 || reinterpret_cast<uintptr_t>(p.W) % 16 != 0) {
    B200_CUDA((launch_any<TIn, TOut>(p, s)));
    return B200_OK;
  }
  int dev = 0, sms = 0;
  B200_CUDA(gemm_tc_init());
  B200_CUDA(cudaGetDevice(&dev));
  B200_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  p.x_by_blocks = p.order && !p.x_by_slot && p.group % 64 == 0;
  const bool pairs = !exact_sums && many_rows(p, sms), in_order_already = !p.order || p.x_by_slot || p.x_by_blocks;
  const bool in_place = in_order_already || (!pairs && !spreads(p.slots, p.experts));
  if (!in_place) {
    const long long blocks = ((long long)p.slots + 7) / 8;
    B200_CUDA(launch_dependent(spread_rows_kernel, dim3((unsigned)(blocks < sms * 8 ? blocks : sms * 8)), dim3(256), 0, s, p, static_cast<uint8_t*>(spread),
                               p.K * (int)sizeof(TIn), (int)sizeof(TIn)));
    p.X = spread;
    p.ldx = p.K;
  }
  const bool in_order = in_order_already || !in_place;
  if (pairs) B200_CUDA((launch_grouped_pair<TIn, TOut>(p, sms, s)));
  else B200_CUDA((launch_grouped_rows<TIn, TOut>(p, in_order, exact_sums, sms, s)));
  return B200_OK;
}

bool off(const void* q, uintptr_t n) { return reinterpret_cast<uintptr_t>(q) % n != 0; }
size_t round256(size_t n) { return (n + 255) & ~size_t(255); }
int size_of(int precision) { return precision == B200_PREC_FP32 ? 4 : 2; }

// Choices are summed by a launch of their own, from fp32 rows in the workspace.
bool sums_choices(const b200_experts_desc& d) { return !d.c_by_slot && d.top_k > 1; }
size_t place_bytes(const b200_experts_desc& d) { return round256((size_t)(d.M / d.group) * d.top_k * 4); }
size_t sums_bytes(const b200_experts_desc& d) { return sums_choices(d) ? round256((size_t)d.M * d.top_k * d.N * 4) + place_bytes(d) : 0; }
// X in the order of the slots.
size_t spread_bytes(const b200_experts_desc& d) {
  const int size = d.int8 ? 1 : 2;
  const bool spread = !d.x_by_slot && d.group % 64 != 0 && d.M > 0 && spreads(d.M * d.top_k, d.n_experts) &&
                      tma_rows(d.K, d.ldx ? d.ldx : d.K, d.ldw ? d.ldw : d.K, size);
  return spread ? round256((size_t)d.M * d.top_k * d.K * size) : 0;
}
size_t experts_bytes(const b200_experts_desc& d) { return sums_bytes(d) + spread_bytes(d); }

const char* check_shape(const b200_experts_desc* d) {
  if (!d) return "no description";
  if (d->N < 1 || d->K < 1 || d->K > B200_INT8_MAX_K) return "N >= 1 and K of 1 to 131071";
  if (d->n_experts < 1 || d->n_experts > B200_MAX_EXPERTS) return "n_experts 1 to 256";
  if (d->top_k < 1 || d->top_k > B200_MAX_TOP_K) return "top_k 1 to 16";
  if (d->group < 1 || d->M < 0 || d->M % d->group != 0) return "M is a multiple of group, which is at least 1";
  if ((long long)d->M * d->top_k > 1 << 30) return "M * top_k of at most 2^30";
  if ((long long)d->n_experts * d->N > 0x7fffffff) return "n_experts * N below 2^31";
  if (d->precision < B200_PREC_FP32 || d->precision > B200_PREC_BF16) return "unknown precision";
  if (d->precision == B200_PREC_FP32 && !d->int8) return "fp16, bf16 or int8";
  if (d->activation < ACT_MISH || d->activation > ACT_RELU_2) return "unknown activation";
  if ((d->ldx && d->ldx < d->K) || (d->ldw && d->ldw < d->K) || (d->ldc && d->ldc < d->N) || (d->res && d->ldres && d->ldres < d->N)) return "rows overlap";
  if (d->c_by_slot && (d->weights || d->res)) return "weights and res are for results by token";
  return nullptr;
}

}  // namespace
}  // namespace b200

extern "C" int b200_op_gemm_int8(const b200_gemm_int8_desc* d, void* stream) {
  using namespace b200;
  return at_c_entry([&]() -> int {
    const char* wrong = nullptr;
    if (!d) wrong = "no description";
    else if (d->M < 0 || d->M > 1 << 30 || d->N < 1 || d->K < 1 || d->K > B200_INT8_MAX_K) wrong = "M of 0 to 2^30, N >= 1, K of 1 to 131071";
    else if (d->precision < B200_PREC_FP32 || d->precision > B200_PREC_BF16) wrong = "unknown precision";
    else if (d->activation < ACT_MISH || d->activation > ACT_RELU_2) wrong = "unknown activation";
    else if ((d->ldx && d->ldx < d->K) || (d->ldw && d->ldw < d->K) || (d->ldc && d->ldc < d->N) || (d->res && d->ldres && d->ldres < d->N))
      wrong = "rows overlap";
    else if (d->M > 0) {
      const uintptr_t size = size_of(d->precision);
      if (!d->X || !d->W || !d->C || !d->x_scales || !d->w_scales) wrong = "X, W, C and both scales are needed";
      else if (off(d->C, size) || off(d->res, size) || off(d->x_scales, 4) || off(d->w_scales, 4) || off(d->bias, 4) || off(d->status, 4))
        wrong = "an operand is not aligned to its type";
      else if (d->res == d->C && (d->ldres ? d->ldres : d->N) != (d->ldc ? d->ldc : d->N)) wrong = "res in place has C's leading dimension";
    }
    if (wrong) {
      set_error(std::string("b200_op_gemm_int8: ") + wrong);
      return B200_ERR_INVALID;
    }
    if (d->M == 0) return B200_OK;
    GroupedParams p = {};
    p.X = d->X; p.ldx = d->ldx ? d->ldx : d->K; p.x_rows = d->M;
    p.W = d->W; p.ldw = d->ldw ? d->ldw : d->K;
    p.bias = d->bias; p.x_scales = d->x_scales; p.w_scales = d->w_scales;
    p.C = d->C; p.ldc = d->ldc ? d->ldc : d->N; p.res = d->res; p.ldres = d->ldres ? d->ldres : d->N;
    p.alpha = d->alpha; p.slots = d->M; p.N = d->N; p.K = d->K; p.experts = 1; p.top_k = 1; p.group = 1; p.act = d->activation;
    p.status = d->status;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    DependentLaunches dependent;
    if (d->precision == B200_PREC_FP32) return run_grouped<int8_t, float>(p, false, nullptr, s);
    if (d->precision == B200_PREC_FP16) return run_grouped<int8_t, __half>(p, false, nullptr, s);
    return run_grouped<int8_t, __nv_bfloat16>(p, false, nullptr, s);
  });
}

extern "C" int b200_op_gemm_experts_workspace(const b200_experts_desc* d, size_t* bytes) {
  using namespace b200;
  return at_c_entry([&]() -> int {
    const char* wrong = check_shape(d);
    if (!wrong && !bytes) wrong = "nowhere to put the size";
    if (wrong) {
      set_error(std::string("b200_op_gemm_experts_workspace: ") + wrong);
      return B200_ERR_INVALID;
    }
    *bytes = experts_bytes(*d);
    return B200_OK;
  });
}

extern "C" int b200_op_gemm_experts(const b200_experts_desc* d, void* stream) {
  using namespace b200;
  return at_c_entry([&]() -> int {
    const char* wrong = check_shape(d);
    if (!wrong && d->M > 0) {
      const uintptr_t in = d->int8 ? 1 : size_of(d->precision), out = d->out_f32 ? 4 : size_of(d->precision);
      if (!d->X || !d->W || !d->C || !d->order || !d->offsets) wrong = "X, W, C, order and offsets are needed";
      else if (d->int8 && (!d->x_scales || !d->w_scales)) wrong = "int8 needs both scales";
      else if (sums_choices(*d) && !d->ids) wrong = "the sum over choices needs ids";
      else if (off(d->X, in) || off(d->W, in) || off(d->C, out) || off(d->res, out) || off(d->bias, 4) || off(d->x_scales, 4) || off(d->w_scales, 4) ||
               off(d->ids, 4) || off(d->order, 4) || off(d->offsets, 4) || off(d->weights, 4) || off(d->status, 4))
        wrong = "an operand is not aligned to its type";
      else if (d->res == d->C && (d->ldres ? d->ldres : d->N) != (d->ldc ? d->ldc : d->N)) wrong = "res in place has C's leading dimension";
      else if (experts_bytes(*d) && (!d->workspace || off(d->workspace, 256) || d->workspace_bytes < experts_bytes(*d)))
        wrong = "the workspace is missing, too small or not on a 256-byte boundary";
    }
    if (wrong) {
      set_error(std::string("b200_op_gemm_experts: ") + wrong);
      return B200_ERR_INVALID;
    }
    if (d->M == 0) return B200_OK;
    const bool sums = sums_choices(*d), f32 = d->out_f32 || d->precision == B200_PREC_FP32;
    GroupedParams p = {};
    p.X = d->X; p.ldx = d->ldx ? d->ldx : d->K; p.x_rows = d->x_by_slot ? d->M * d->top_k : d->M;
    p.W = d->W; p.ldw = d->ldw ? d->ldw : d->K; p.bias = d->bias;
    if (d->int8) { p.x_scales = d->x_scales; p.w_scales = d->w_scales; }
    p.C = sums ? d->workspace : d->C; p.ldc = !sums && d->ldc ? d->ldc : d->N;
    if (!sums) { p.res = d->res; p.ldres = d->ldres ? d->ldres : d->N; }
    p.alpha = 1.f; p.weights = d->weights; p.order = d->order; p.offsets = d->offsets;
    p.slots = d->M * d->top_k; p.N = d->N; p.K = d->K; p.experts = d->n_experts; p.top_k = d->top_k; p.group = d->group; p.act = d->activation;
    p.x_by_slot = d->x_by_slot; p.c_by_slot = d->c_by_slot || sums;
    if (sums) p.place = reinterpret_cast<int*>(static_cast<char*>(d->workspace) + sums_bytes(*d) - place_bytes(*d));
    p.status = d->status;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    DependentLaunches dependent;
    int rc = B200_OK;
    const bool wide = f32 || sums;
    void* spread = static_cast<char*>(d->workspace) + sums_bytes(*d);
    if (d->int8) {
      rc = wide                              ? run_grouped<int8_t, float>(p, false, spread, s)
           : d->precision == B200_PREC_FP16 ? run_grouped<int8_t, __half>(p, false, spread, s)
                                             : run_grouped<int8_t, __nv_bfloat16>(p, false, spread, s);
    } else if (d->precision == B200_PREC_FP16) {
      rc = wide ? run_grouped<__half, float>(p, f32, spread, s) : run_grouped<__half, __half>(p, false, spread, s);
    } else {
      rc = wide ? run_grouped<__nv_bfloat16, float>(p, f32, spread, s) : run_grouped<__nv_bfloat16, __nv_bfloat16>(p, false, spread, s);
    }
    if (rc != B200_OK || !sums) return rc;
    CombineParams c = {};
    c.Y = static_cast<const float*>(d->workspace); c.place = p.place; c.ids = d->ids; c.res = d->res; c.ldres = d->ldres ? d->ldres : d->N;
    c.C = d->C; c.ldc = d->ldc ? d->ldc : d->N; c.tokens = d->M; c.N = d->N; c.experts = d->n_experts; c.top_k = d->top_k; c.group = d->group;
    if (f32) B200_CUDA(launch_combine<float>(c, s));
    else if (d->precision == B200_PREC_FP16) B200_CUDA(launch_combine<__half>(c, s));
    else B200_CUDA(launch_combine<__nv_bfloat16>(c, s));
    return B200_OK;
  });
}
