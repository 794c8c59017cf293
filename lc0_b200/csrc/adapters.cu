// A product that all requests of a batch share, with a low-rank adapter per request beside it:
//   C[m] = act(X[m] W^T + bias + s_a (X[m] A_a^T) B_a^T),  a = ids[m / group].
// The narrow product H[m] = s_a X[m] A_a^T [M][rank] comes first (fp32, in the caller's workspace), then the shared product, which
// meets H and B in fp32.
#include "../../include/b200nn.h"
#include "kernels.cuh"

namespace b200 {
namespace {

struct AdapterParams {
  const void* X; const void* A; const void* B;
  const float* scales; const int* ids;
  const float* bias;
  float* H;          // [M][rank]
  const float* acc;  // [M][N] sums of the shared product and the bias
  long long ldacc;
  void* C; long long ldc;
  long long ldx;
  int M, N, K, rank, group, n_adapters, act, out_f32;
};

__device__ __forceinline__ int adapter_of(const AdapterParams& p, int m) {
  const int a = p.ids[m / p.group];
  return a >= 0 && a < p.n_adapters ? a : -1;
}

// H: a warp per row.
template <typename T>
__global__ void __launch_bounds__(256) adapters_shrink_kernel(const AdapterParams p) {
  const int m = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (m >= p.M) return;
  const int a = adapter_of(p, m);
  if (a < 0) return;  // never read
  const T* x = static_cast<const T*>(p.X) + (long long)m * p.ldx;
  const T* w = static_cast<const T*>(p.A) + (long long)a * p.rank * p.K;
  const float scale = p.scales ? p.scales[a] : 1.f;
  for (int r = 0; r < p.rank; ++r) {
    float s = 0.f;
    for (int k = lane; k < p.K; k += 32) s = fmaf(to_f(x[k]), to_f(w[(long long)r * p.K + k]), s);
    s = warp_sum(s);
    if (lane == 0) p.H[(long long)m * p.rank + r] = scale * s;
  }
}

// C = act(acc + H B^T): a thread per output.
template <typename T>
__global__ void __launch_bounds__(256) adapters_expand_kernel(const AdapterParams p) {
  const int n = blockIdx.x * 256 + threadIdx.x;
  if (n >= p.N) return;
  for (int m = blockIdx.y; m < p.M; m += gridDim.y) {
    float v = p.acc[(long long)m * p.ldacc + n];
    const int a = adapter_of(p, m);
    if (a >= 0) {
      const T* b = static_cast<const T*>(p.B) + ((long long)a * p.N + n) * p.rank;
      const float* h = p.H + (long long)m * p.rank;
      float s = 0.f;
      for (int r = 0; r < p.rank; ++r) s = fmaf(h[r], to_f(b[r]), s);
      v += s;
    }
    v = p.out_f32 ? activate<false>(v, p.act) : activate<true>(v, p.act);
    if (p.out_f32) static_cast<float*>(p.C)[(long long)m * p.ldc + n] = v;
    else static_cast<T*>(p.C)[(long long)m * p.ldc + n] = from_f<T>(v);
  }
}

size_t round256(size_t n) { return (n + 255) & ~size_t(255); }

struct AdapterPlan {
  size_t h_bytes, acc_bytes;
  size_t bytes() const { return h_bytes + acc_bytes; }
};
AdapterPlan plan_of(const b200_adapters_desc& d) {
  AdapterPlan p;
  p.h_bytes = round256((size_t)d.M * d.rank * 4);
  // sums of the shared product: in C itself where it holds floats
  p.acc_bytes = d.out_f32 || d.precision == B200_PREC_FP32 ? 0 : round256((size_t)d.M * d.N * 4);
  return p;
}

template <typename T>
int run_adapters(const b200_adapters_desc& d, cudaStream_t s) {
  const AdapterPlan plan = plan_of(d);
  AdapterParams p = {};
  p.X = d.X; p.ldx = d.ldx ? d.ldx : d.K; p.A = d.A; p.B = d.B; p.scales = d.scales; p.ids = d.ids; p.bias = d.bias;
  p.C = d.C; p.ldc = d.ldc ? d.ldc : d.N;
  p.M = d.M; p.N = d.N; p.K = d.K; p.rank = d.rank; p.group = d.group; p.n_adapters = d.n_adapters; p.act = d.activation;
  p.out_f32 = sizeof(T) == 4 || d.out_f32;
  char* ws = static_cast<char*>(d.workspace);
  p.H = reinterpret_cast<float*>(ws);
  float* acc = plan.acc_bytes ? reinterpret_cast<float*>(ws + plan.h_bytes) : static_cast<float*>(d.C);
  p.acc = acc;
  p.ldacc = plan.acc_bytes ? d.N : p.ldc;
  GemmParams g;
  g.A = d.X; g.lda = p.ldx; g.W = d.W; g.ldw = d.ldw ? d.ldw : d.K; g.bias = d.bias;
  g.C = acc; g.ldc = p.ldacc; g.out_f32 = true;
  g.M = d.M; g.N = d.N; g.K = d.K; g.act = ACT_NONE; g.w_const = true;
  g.split_k = d.M < 64;
  bool tc = false;
  if constexpr (sizeof(T) == 2) {
    tc = gemm_tc_supported(g);
    if (tc) {
      B200_CUDA(gemm_tc_init());
      int dev = 0, sms = 0;
      B200_CUDA(cudaGetDevice(&dev));
      B200_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
      B200_CUDA(launch_gemm_tc<T>(g, d.status, sms, s));
    }
  }
  if (!tc) B200_CUDA(launch_gemm_fma<T>(g, s));
  adapters_shrink_kernel<T><<<ceil_div(d.M, 8), 256, 0, s>>>(p);
  B200_CUDA(cudaGetLastError());
  adapters_expand_kernel<T><<<dim3(ceil_div(d.N, 256), d.M < 32768 ? d.M : 32768), 256, 0, s>>>(p);
  B200_CUDA(cudaGetLastError());
  return B200_OK;
}

// What does not depend on the pointers.
const char* check_shape(const b200_adapters_desc* d) {
  if (!d) return "no description";
  if (d->M < 0 || d->N < 1 || d->K < 1) return "M >= 0, N >= 1 and K >= 1";
  if (d->rank < 1 || d->rank > B200_ADAPTERS_MAX_RANK) return "rank 1 to 128";
  if (d->n_adapters < 1 || d->group < 1) return "n_adapters and group are at least 1";
  if (d->precision < B200_PREC_FP32 || d->precision > B200_PREC_BF16) return "unknown precision";
  if (d->activation < ACT_MISH || d->activation > ACT_RELU_2) return "unknown activation";
  if ((d->ldx && d->ldx < d->K) || (d->ldw && d->ldw < d->K) || (d->ldc && d->ldc < d->N)) return "rows overlap";
  return nullptr;
}

}  // namespace
}  // namespace b200

extern "C" int b200_op_gemm_adapters_workspace(const b200_adapters_desc* d, size_t* bytes) {
  using namespace b200;
  const char* wrong = check_shape(d);
  if (!wrong && !bytes) wrong = "nowhere to put the size";
  if (wrong) {
    set_error(std::string("b200_op_gemm_adapters_workspace: ") + wrong);
    return B200_ERR_INVALID;
  }
  *bytes = plan_of(*d).bytes();
  return B200_OK;
}

extern "C" int b200_op_gemm_adapters(const b200_adapters_desc* d, void* stream) {
  using namespace b200;
  const char* wrong = check_shape(d);
  if (!wrong && d->M > 0) {
    const uintptr_t size = d->precision == B200_PREC_FP32 ? 4 : 2, csize = d->out_f32 ? 4 : size;
    auto off = [](const void* q, uintptr_t n) { return reinterpret_cast<uintptr_t>(q) % n != 0; };
    if (!d->X || !d->W || !d->C || !d->A || !d->B || !d->ids) wrong = "X, W, C, A, B and ids are needed";
    else if (off(d->X, size) || off(d->W, size) || off(d->A, size) || off(d->B, size) || off(d->C, csize) || off(d->bias, 4) ||
             off(d->scales, 4) || off(d->ids, 4) || off(d->status, 4))
      wrong = "an operand is not aligned to its type";
    else if (!d->workspace || off(d->workspace, 256) || d->workspace_bytes < plan_of(*d).bytes())
      wrong = "the workspace is missing, too small or not on a 256-byte boundary";
  }
  if (wrong) {
    set_error(std::string("b200_op_gemm_adapters: ") + wrong);
    return B200_ERR_INVALID;
  }
  if (d->M == 0) return B200_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (d->precision == B200_PREC_FP32) return run_adapters<float>(*d, s);
  if (d->precision == B200_PREC_FP16) return run_adapters<__half>(*d, s);
  return run_adapters<__nv_bfloat16>(*d, s);
}
