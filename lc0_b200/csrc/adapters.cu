// A product that all requests of a batch share, with a low-rank adapter per request beside it:
//   C[m] = act(X[m] W^T + bias + s_a (X[m] A_a^T) B_a^T),  a = ids[m / group].
// Two launches: the narrow product H[m] = s_a X[m] A_a^T [M][rank], and the shared product, which takes H and B in.  The second is
// made dependent on the first early: it loads and multiplies X and W while H is computed.
//
// H, 16-bit, requests of whole 64-row blocks: adapters_shrink.cu, on tensor cores.
// H otherwise: adapters_shrink_rows_kernel.
// The shared product, 16-bit: kernels of gemm_tc.cu (H and B as further k-blocks) and gemm_split.cu (added in the epilogue), see
//   launch_gemm_tc; operands that TMA cannot read: gemm_fma.cu, fp32: gemm_f32.cu or gemm_fma.cu, into fp32 sums, to which
//   adapters_expand_kernel adds.
#include "../../include/b200nn.h"
#include "kernels.cuh"
#include "tma_mma.cuh"

namespace b200 {
namespace {

struct AdapterParams {
  const void* X; const void* A; const void* B;
  const float* scales; const int* ids;
  float* H;      // [M][rank]
  void* pieces;  // [M][2 * rp] or nullptr: H as two values of the type
  const float* acc;  // [M][N] sums of the shared product and the bias
  long long ldacc;
  void* C; long long ldc;
  long long ldx;
  int M, N, K, rank, rp, group, n_adapters, act, out_f32;
  int* status;
};

__device__ __forceinline__ int adapter_of(const AdapterParams& p, int m) {
  const int a = p.ids[m / p.group];
  return a >= 0 && a < p.n_adapters ? a : -1;
}

// ---- H row by row -----------------------------------------------------------------------------------------------
// A warp per rank, eight of a row to a CTA: what a lane reads of the row and of A is on its way together, and the row's other readers find
// it in L1 (the row in shared memory first: a second trip to memory, fp32 64x1536x1536 40 us for 37).  Bound by latency at few rows, by
// what L2 delivers of A, which is read once per row, at many: rank 32 of 4096 rows of 2048, 540 MB.
template <typename T>
__global__ void __launch_bounds__(256) adapters_shrink_rows_kernel(const AdapterParams p, int vec) {
  constexpr int kPer = 16 / sizeof(T);
  grid_launch_dependents();
  const int lane = threadIdx.x & 31, r = blockIdx.y * 8 + (threadIdx.x >> 5);
  if (r >= p.rp) return;
  for (int m = blockIdx.x; m < p.M; m += gridDim.x) {
    const int a = adapter_of(p, m);
    if (a < 0) continue;  // never read
    T* q = p.pieces ? static_cast<T*>(p.pieces) + (long long)m * 2 * p.rp + r : nullptr;
    if (r >= p.rank) {  // zeros beyond the rank
      if (q && lane < 2) q[lane * p.rp] = from_f<T>(0.f);
      continue;
    }
    const T* x = static_cast<const T*>(p.X) + (long long)m * p.ldx;
    const T* w = static_cast<const T*>(p.A) + ((long long)a * p.rank + r) * p.K;
    float s = 0.f;
    if (vec) {
      const uint4* x4 = reinterpret_cast<const uint4*>(x);
      const uint4* w4 = reinterpret_cast<const uint4*>(w);
      const int n = p.K / kPer;
#pragma unroll 4
      for (int i = lane; i < n; i += 32) {
        const uint4 u = __ldg(w4 + i), v = __ldg(x4 + i);
        const T* e = reinterpret_cast<const T*>(&u);
        const T* f = reinterpret_cast<const T*>(&v);
#pragma unroll
        for (int j = 0; j < kPer; ++j) s = fmaf(to_f(e[j]), to_f(f[j]), s);
      }
    } else {
#pragma unroll 4
      for (int i = lane; i < p.K; i += 32) s = fmaf(to_f(w[i]), to_f(x[i]), s);
    }
    s = warp_sum(s) * (p.scales ? p.scales[a] : 1.f);
    if (lane == 0) {
      p.H[(long long)m * p.rank + r] = s;
      if constexpr (sizeof(T) == 2) {
        if (q) {
          const uint32_t hi = pack2<T>(s, 0.f);
          const uint32_t lo = pack2<T>((s - unpack2<T>(hi).x) * (1 << LowPiece<T>::shift), 0.f);
          q[0] = *reinterpret_cast<const T*>(&hi);
          q[p.rp] = *reinterpret_cast<const T*>(&lo);
        }
      }
    }
  }
}

// ---- fp32 sums + H B^T ------------------------------------------------------------------------------------------
// A warp has 32 columns of 8 rows: eight ranks of a lane's row of B stay in registers for as many rows as have that adapter, H is the
// same for the whole warp.  Sums are read and results written as whole lines.
constexpr int kExpandRows = 8;

template <typename T>
__global__ void __launch_bounds__(256) adapters_expand_kernel(const AdapterParams p, int vec) {
  grid_dependency_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = blockIdx.x * 64 + (warp & 1) * 32 + lane;
  const bool mine = n < p.N;
  for (long long m0 = ((long long)blockIdx.y * 4 + (warp >> 1)) * kExpandRows; m0 < p.M; m0 += (long long)gridDim.y * 4 * kExpandRows) {
    int a[kExpandRows];
    float v[kExpandRows], d[kExpandRows];
#pragma unroll
    for (int i = 0; i < kExpandRows; ++i) {
      const long long m = m0 + i;
      a[i] = m < p.M ? adapter_of(p, (int)m) : -1;
      v[i] = mine && m < p.M ? p.acc[m * p.ldacc + n] : 0.f;
      d[i] = 0.f;
    }
    for (int r0 = 0; r0 < p.rank; r0 += 8) {
      float b[8];
#pragma unroll
      for (int i = 0; i < kExpandRows; ++i) {
        if (a[i] < 0) continue;
        if (i == 0 || a[i] != a[i - 1]) {
          const T* src = static_cast<const T*>(p.B) + ((long long)a[i] * p.N + (mine ? n : 0)) * p.rank + r0;
          if (vec) {  // a multiple of eight ranks on 16-byte boundaries
            constexpr int kPer = 16 / sizeof(T);
#pragma unroll
            for (int j = 0; j < 8; j += kPer) {
              const uint4 u = __ldg(reinterpret_cast<const uint4*>(src + j));
              const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
              for (int q = 0; q < kPer; ++q) b[j + q] = to_f(e[q]);
            }
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) b[j] = r0 + j < p.rank ? to_f(src[j]) : 0.f;
          }
        }
        const float* h = p.H + (m0 + i) * p.rank + r0;
        if (vec) {
          const float4 h0 = *reinterpret_cast<const float4*>(h), h1 = *reinterpret_cast<const float4*>(h + 4);
          d[i] = fmaf(h0.x, b[0], fmaf(h0.y, b[1], fmaf(h0.z, b[2], fmaf(h0.w, b[3], d[i]))));
          d[i] = fmaf(h1.x, b[4], fmaf(h1.y, b[5], fmaf(h1.z, b[6], fmaf(h1.w, b[7], d[i]))));
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (r0 + j < p.rank) d[i] = fmaf(h[j], b[j], d[i]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kExpandRows; ++i) {
      const long long m = m0 + i;
      if (!mine || m >= p.M) continue;
      const float x = v[i] + d[i], y = p.out_f32 ? activate<false>(x, p.act) : activate<true>(x, p.act);
      if (p.out_f32) static_cast<float*>(p.C)[m * p.ldc + n] = y;
      else static_cast<T*>(p.C)[m * p.ldc + n] = from_f<T>(y);
    }
  }
}

// ---- host -------------------------------------------------------------------------------------------------------
size_t round256(size_t n) { return (n + 255) & ~size_t(255); }
bool aligned16(const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; }

// fp32: whether a product is worth cutting its weights into pieces for the tensor cores, which every call does.  us with rank 16, FMA /
// tensor cores: 64x512x256 20.7 / 19.0, 256x512x256 25.6 / 20.4, 1024x512x256 28.1 / 23.4, 512x1024x1024 51 / 32,
// 64x1536x1536 40 / 36, 1024x1536x1536 187 / 91.  Fewer rows than a tile's share W among less than the pieces cost.
bool worth_pieces(const b200_adapters_desc& d) { return d.M >= 64 && (long long)d.M * d.N * d.K >= 1 << 23; }

// What a description is computed by, and its workspace: H, its pieces, the fp32 sums, the pieces of fp32 weights.  Nothing here depends on the device.
struct AdapterPlan {
  GemmParams g;
  bool tensor = false, mma = false;
  size_t h_bytes = 0, piece_bytes = 0, acc_bytes = 0, w_bytes = 0;
  size_t bytes() const { return h_bytes + piece_bytes + acc_bytes + w_bytes; }
};
AdapterPlan plan_of(const b200_adapters_desc& d) {
  AdapterPlan out;
  GemmParams& g = out.g;
  g.A = d.X; g.lda = d.ldx ? d.ldx : d.K; g.W = d.W; g.ldw = d.ldw ? d.ldw : d.K; g.bias = d.bias;
  g.C = d.C; g.ldc = d.ldc ? d.ldc : d.N; g.out_f32 = d.out_f32 != 0 || d.precision == B200_PREC_FP32;
  g.M = d.M; g.N = d.N; g.K = d.K; g.act = d.activation; g.w_const = true; g.split_k = true;
  g.ad_ids = d.ids; g.ad_b = d.B; g.ad_group = d.group; g.ad_n = d.n_adapters; g.ad_rank = d.rank; g.ad_rp = (d.rank + 15) / 16 * 16;
  out.tensor = d.precision != B200_PREC_FP32 && gemm_tc_supported(g);
  out.mma = out.tensor && d.group % 64 == 0 && aligned16(d.A) && (long long)d.n_adapters * d.rank < 0x7fffff00;
  out.h_bytes = round256((size_t)d.M * d.rank * 4);
  // (a result in fp32 would show what the two pieces of H leave out)
  if (out.mma && !g.out_f32 && gemm_adapters_pieces(g)) out.piece_bytes = round256((size_t)d.M * 2 * g.ad_rp * 2);
  // sums of the shared product: in C itself where it holds floats
  if (!out.tensor && !g.out_f32) out.acc_bytes = round256((size_t)d.M * d.N * 4);
  // fp32 on tensor cores: W is cut into pieces by every call.  The question needs the address of pieces, which are laid out after it is
  // answered: any aligned one, none of the description's, which need not be set yet.
  g.W3 = reinterpret_cast<const void*>(uintptr_t(256));
  if (d.precision == B200_PREC_FP32 && worth_pieces(d) && gemm_f32_supported(g)) out.w_bytes = round256((size_t)d.N * d.K * 6);
  g.W3 = nullptr;
  return out;
}

// Few long rows: a CTA for each of them spreads over more SMs than one for every 64 does, which has K / 64 steps one after the other, at
// the price of reading A once per row.  Whole call (512 columns), us, tensor cores / by rows: 64x1024 rank 16 9.7 / 7.3, 128x1024 rank 16
// 9.6 / 8.5, 256x1024 rank 16 10.2 / 10.2, 512x1024 rank 16 11.8 / 11.6, 192x1536 rank 8 11.8 / 9.7; short rows: 512x256 rank 8
// 6.2 / 7.2, 1024x256 rank 16 7.9 / 10.2.
bool shrink_by_rows(const b200_adapters_desc& d) { return d.K >= 512 && (long long)d.M * d.rank * d.K <= 4 << 20; }

template <typename T>
cudaError_t launch_shrink_rows(const AdapterParams& p, cudaStream_t s) {
  const int per = 16 / (int)sizeof(T);
  const int vec = p.K % per == 0 && p.ldx % per == 0 && aligned16(p.X) && aligned16(p.A);
  adapters_shrink_rows_kernel<T><<<dim3(p.M < 65536 ? p.M : 65536, ceil_div(p.pieces ? p.rp : p.rank, 8)), 256, 0, s>>>(p, vec);
  return cudaGetLastError();
}

// The second launch made dependent on the first.
struct DependentScope {
  bool before;
  DependentScope() : before(t_dependent_launch) { t_dependent_launch = true; }
  ~DependentScope() { t_dependent_launch = before; }
};

template <typename T>
int run_adapters(const b200_adapters_desc& d, cudaStream_t s) {
  AdapterPlan plan = plan_of(d);
  GemmParams& g = plan.g;
  char* ws = static_cast<char*>(d.workspace);
  AdapterParams p = {};
  p.X = d.X; p.ldx = g.lda; p.A = d.A; p.B = d.B; p.scales = d.scales; p.ids = d.ids;
  p.H = reinterpret_cast<float*>(ws);
  p.C = d.C; p.ldc = g.ldc; p.status = d.status;
  p.M = d.M; p.N = d.N; p.K = d.K; p.rank = d.rank; p.rp = g.ad_rp; p.group = d.group; p.n_adapters = d.n_adapters; p.act = d.activation;
  p.out_f32 = g.out_f32;
  if constexpr (sizeof(T) == 2) {
    if (plan.tensor) {
      B200_CUDA(gemm_tc_init());
      int dev = 0, sms = 0;
      B200_CUDA(cudaGetDevice(&dev));
      B200_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
      g.ad_h = p.H;
      if (plan.piece_bytes) g.ad_pieces = p.pieces = ws + plan.h_bytes;
      if (!plan.mma || shrink_by_rows(d)) B200_CUDA(launch_shrink_rows<T>(p, s));
      else B200_CUDA(launch_adapters_shrink<T>(g, d.A, d.scales, p.H, p.pieces, d.status, s));
      DependentScope dependent;
      B200_CUDA(launch_gemm_tc<T>(g, d.status, sms, s));
      return B200_OK;
    }
  }
  void* acc = plan.acc_bytes ? ws + plan.h_bytes : d.C;
  g.C = acc; g.ldc = plan.acc_bytes ? d.N : g.ldc; g.out_f32 = true; g.act = ACT_NONE; g.ad_ids = nullptr;
  p.acc = static_cast<const float*>(acc); p.ldacc = g.ldc;
  if (plan.w_bytes) {
    // (the product fetches the pieces ahead of its dependency: what it depends on is the launch after the one that writes them)
    B200_CUDA(gemm_tc_init());
    int dev = 0, sms = 0;
    B200_CUDA(cudaGetDevice(&dev));
    B200_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    g.W3 = ws + plan.h_bytes;
    B200_CUDA(launch_split_weights(static_cast<const float*>(d.W), (long long)d.N * d.K, ws + plan.h_bytes, s));
    B200_CUDA(launch_shrink_rows<T>(p, s));
    DependentScope dependent;
    B200_CUDA(launch_gemm_f32(g, d.status, sms, s));
  } else {
    B200_CUDA(launch_shrink_rows<T>(p, s));
    DependentScope dependent;
    B200_CUDA(launch_gemm_fma<T>(g, s));
  }
  DependentScope dependent;
  const int row_blocks = ceil_div(d.M, 4 * kExpandRows);
  const int vec = d.rank % 8 == 0 && aligned16(d.B);
  B200_CUDA(launch_dependent(adapters_expand_kernel<T>, dim3(ceil_div(d.N, 64), row_blocks < 65535 ? row_blocks : 65535), dim3(256), 0, s, p,
                             vec));
  return B200_OK;
}

// What does not depend on the pointers.
const char* check_shape(const b200_adapters_desc* d) {
  if (!d) return "no description";
  if (d->M < 0 || d->M > 64 * 65535 || d->N < 1 || d->K < 1) return "M of 0 to 4194240, N >= 1 and K >= 1";
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
  return at_c_entry([&]() -> int {
    const char* wrong = check_shape(d);
    if (!wrong && !bytes) wrong = "nowhere to put the size";
    if (wrong) {
      set_error(std::string("b200_op_gemm_adapters_workspace: ") + wrong);
      return B200_ERR_INVALID;
    }
    *bytes = plan_of(*d).bytes();
    return B200_OK;
  });
}

extern "C" int b200_op_gemm_adapters(const b200_adapters_desc* d, void* stream) {
  using namespace b200;
  return at_c_entry([&]() -> int {
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
  });
}
