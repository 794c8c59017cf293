// Norms of queries and keys for each head with the position rotation in the same pass.
#include "chunk8.cuh"
#include "kernels.cuh"

namespace b200 {
namespace {

struct QkParams {
  const void* in[2]; void* out[2];  // queries, keys
  long long ld_in[2], ld_out[2];
  const float* gamma[2];
  int rows, heads_q, heads, depth;  // heads: of queries and keys together
  int norm; float eps;
  int rotate, interleaved, n_positions;
  const float2* table; const int* positions;
};

__device__ __forceinline__ int position_of(const QkParams& p, int row) {
  if (p.rotate == 0) return -1;
  const int at = p.positions ? p.positions[row] : (int)((unsigned)row % (unsigned)p.n_positions);
  return at >= 0 && at < p.n_positions ? at : -1;
}

// Eight floats, with 16-byte loads where their address allows.
__device__ __forceinline__ void load_eight(const float* from, bool aligned, float (&v)[8]) {
  if (aligned) {
    const float4 a = reinterpret_cast<const float4*>(from)[0], b = reinterpret_cast<const float4*>(from)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = from[i];
  }
}

// kLanes lanes hold one head, eight entries each, a warp 32 / kLanes heads of the queries or of the keys at a time and kIter times as many of one
// row: gamma and the row's angles stay in registers over all of them, and that many loads are on their way together.
// Bound by memory: 65536 rows of 24 + 24 heads of 32, bf16, 403 MB in 71 us, 5.6 TB/s (75 with the
// index of a warp's row and unit divided in 64 bits).
template <typename T, int kLanes, int kIter>
__global__ void __launch_bounds__(128) qk_norm_rotate_kernel(const QkParams p, int q_units, int units) {
  grid_launch_dependents();
  grid_dependency_wait();
  constexpr int kHeads = 32 / kLanes;
  const int lane = threadIdx.x & 31, c = lane % kLanes, sub = lane / kLanes;
  const unsigned all = blockIdx.x * 4u + (threadIdx.x >> 5);  // (rows times heads are below 2^31)
  const int row = (int)(all / (unsigned)units), unit = (int)(all - (unsigned)row * (unsigned)units), k = unit >= q_units;
  if (row >= p.rows) return;
  const int heads = k ? p.heads - p.heads_q : p.heads_q, h0 = (k ? unit - q_units : unit) * (kHeads * kIter) + sub;
  const bool inside = 8 * c < p.depth;
  const T* in = static_cast<const T*>(p.in[k]) + row * p.ld_in[k] + 8 * c;
  Chunk<T> raw[kIter];
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const int h = h0 + i * kHeads;
    if (inside && h < heads) raw[i] = load8(in + h * p.depth);
#pragma unroll
    for (int j = 0; j < Chunk<T>::kLoads; ++j)
      if (!(inside && h < heads)) raw[i].raw[j] = make_uint4(0u, 0u, 0u, 0u);
  }
  float gamma[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) gamma[j] = 1.f;
  if (p.norm && p.gamma[k] && inside) load_eight(p.gamma[k] + 8 * c, (reinterpret_cast<uintptr_t>(p.gamma[k]) & 15) == 0, gamma);
  const int at = position_of(p, row);
  const bool turned = at >= 0 && 8 * c < p.rotate;
  const bool second = !p.interleaved && 8 * c >= p.rotate / 2;  // of the halves
  float cs[8], sn[8];                                           // with interleaved pairs the first four alone
  int partner = lane;
  if (turned) {
    const float* angles = reinterpret_cast<const float*>(p.table + (long long)at * (p.rotate / 2) + (p.interleaved ? 4 * c : second ? 8 * c - p.rotate / 2 : 8 * c));
    const bool aligned = (reinterpret_cast<uintptr_t>(angles) & 15) == 0;
    float a[8];
    load_eight(angles, aligned, a);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      cs[i] = a[2 * i];
      sn[i] = a[2 * i + 1];
    }
    if (!p.interleaved) {
      load_eight(angles + 8, aligned, a);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        cs[4 + i] = a[2 * i];
        sn[4 + i] = a[2 * i + 1];
      }
      partner = second ? lane - p.rotate / 16 : lane + p.rotate / 16;
      if (!second) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sn[i] = -sn[i];
      }
    }
  }
  const float inv_depth = 1.f / (float)p.depth;
  T* out = static_cast<T*>(p.out[k]) + row * p.ld_out[k] + 8 * c;
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const int h = h0 + i * kHeads;
    float v[8];
    unpack8(raw[i], v);
    if (p.norm) {
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fmaf(v[j], v[j], sum);
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      // fp32 results: rounded to nearest, as in the kernel below; rsqrtf, off by two steps, does not show in 16 bits.
      const float mean = fmaf(sum, inv_depth, p.eps), r = sizeof(T) == 4 ? __frsqrt_rn(mean) : rsqrtf(mean);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= r * gamma[j];
    }
    if (p.rotate) {
      if (p.interleaved) {
        if (turned) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float a = v[2 * j], b = v[2 * j + 1];
            v[2 * j] = a * cs[j] - b * sn[j];
            v[2 * j + 1] = a * sn[j] + b * cs[j];
          }
        }
      } else {
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = __shfl_sync(0xffffffffu, v[j], partner);
        if (turned) {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = v[j] * cs[j] + w[j] * sn[j];
        }
      }
    }
    if (inside && h < heads) store8(out + h * p.depth, pack8<T>(v));
  }
}

// Any depth, rotation, stride and alignment: a warp per row and head, entry by entry; each lane reads its entries and their partners ahead of
// the first store of the warp.
template <typename T>
__global__ void __launch_bounds__(128) qk_norm_rotate_any_kernel(const QkParams p) {
  grid_launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const unsigned unit = blockIdx.x * 4u + (threadIdx.x >> 5);
  const int row = (int)(unit / (unsigned)p.heads), h = (int)(unit % (unsigned)p.heads), k = h >= p.heads_q;
  if (row >= p.rows) return;
  const T* x = static_cast<const T*>(p.in[k]) + row * p.ld_in[k] + (long long)(k ? h - p.heads_q : h) * p.depth;
  T* y = static_cast<T*>(p.out[k]) + row * p.ld_out[k] + (long long)(k ? h - p.heads_q : h) * p.depth;
  const int at = position_of(p, row);
  const float* gamma = p.gamma[k];
  float v[8], sum = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int e = lane + 32 * i;
    v[i] = e < p.depth ? to_f(x[e]) : 0.f;
    sum = fmaf(v[i], v[i], sum);
  }
  const float r = p.norm ? __frsqrt_rn(warp_sum(sum) / (float)p.depth + p.eps) : 1.f;
  auto scaled = [&](float u, int e) { return p.norm ? u * (gamma ? r * gamma[e] : r) : u; };
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int e = lane + 32 * i;
    if (e >= p.depth) continue;
    v[i] = scaled(v[i], e);
    if (at >= 0 && e < p.rotate) {
      const int half = p.rotate / 2;
      const bool second = p.interleaved ? (e & 1) : e >= half;
      const int other = p.interleaved ? (e ^ 1) : (second ? e - half : e + half);
      const float2 a = p.table[(long long)at * half + (p.interleaved ? e / 2 : e % half)];
      const float w = scaled(to_f(x[other]), other);
      v[i] = second ? w * a.y + v[i] * a.x : v[i] * a.x - w * a.y;
    }
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (lane + 32 * i < p.depth) y[lane + 32 * i] = one_of<T>(v[i]);
}

template <typename T, int kLanes>
cudaError_t launch_lanes(const QkParams& p, cudaStream_t s) {
  constexpr int kHeads = 32 / kLanes;
  // As many heads per warp as leave warps for every SM: the iterations with the fewest empty places, the most of equal ones.
  const int q_steps = (p.heads_q + kHeads - 1) / kHeads, k_steps = (p.heads - p.heads_q + kHeads - 1) / kHeads;
  auto units_of = [&](int i) { return (q_steps + i - 1) / i + (k_steps + i - 1) / i; };
  int iter = 1;
  for (int i = 2; i <= 4; ++i)
    if ((long long)p.rows * units_of(i) >= 148 * 16 && units_of(i) * i <= units_of(iter) * iter) iter = i;
  const int q_units = (q_steps + iter - 1) / iter, units = units_of(iter);
  const long long blocks = ((long long)p.rows * units + 3) / 4;
  auto kernel = iter == 1 ? qk_norm_rotate_kernel<T, kLanes, 1>
                : iter == 2 ? qk_norm_rotate_kernel<T, kLanes, 2>
                : iter == 3 ? qk_norm_rotate_kernel<T, kLanes, 3>
                            : qk_norm_rotate_kernel<T, kLanes, 4>;
  return launch_dependent(kernel, dim3((unsigned)blocks), dim3(128), 0, s, p, q_units, units);
}

template <typename T>
cudaError_t launch_qk(const QkParams& p, cudaStream_t s) {
  DependentLaunches dependent;
  const int per16 = 16 / (int)sizeof(T);
  auto fine = [&](int k) {
    return reinterpret_cast<uintptr_t>(p.in[k]) % 16 == 0 && reinterpret_cast<uintptr_t>(p.out[k]) % 16 == 0 && p.ld_in[k] % per16 == 0 &&
           p.ld_out[k] % per16 == 0;
  };
  const bool vec = p.depth % 8 == 0 && fine(0) && (p.heads == p.heads_q || fine(1)) && p.rotate % (p.interleaved ? 8 : 16) == 0;
  if (!vec)
    return launch_dependent(qk_norm_rotate_any_kernel<T>, dim3((unsigned)(((long long)p.rows * p.heads + 3) / 4)), dim3(128), 0, s, p);
  const int chunks = p.depth / 8;
  if (chunks <= 1) return launch_lanes<T, 1>(p, s);
  if (chunks <= 2) return launch_lanes<T, 2>(p, s);
  if (chunks <= 4) return launch_lanes<T, 4>(p, s);
  if (chunks <= 8) return launch_lanes<T, 8>(p, s);
  if (chunks <= 16) return launch_lanes<T, 16>(p, s);
  return launch_lanes<T, 32>(p, s);
}

}  // namespace
}  // namespace b200

extern "C" int b200_op_qk_norm_rotate(const b200_qk_norm_desc* d, void* stream) {
  using namespace b200;
  return at_c_entry([&]() -> int {
    const char* wrong = nullptr;
    QkParams p = {};
    if (!d) wrong = "no description";
    else if (d->rows < 0 || d->q_heads < 0 || d->k_heads < 0) wrong = "rows, q_heads and k_heads are at least 0";
    else if (d->depth < 1 || d->depth > 256) wrong = "depth 1 to 256";
    else if (d->precision < B200_PREC_FP32 || d->precision > B200_PREC_BF16) wrong = "unknown precision";
    else if (d->q_heads + (long long)d->k_heads > 65536) wrong = "at most 65536 heads";
    else if ((long long)d->rows * (d->q_heads + d->k_heads) > 0x7fffffffll) wrong = "rows times heads below 2^31";
    else if (d->norm && !(d->eps >= 0.f)) wrong = "eps is at least 0";
    else if (d->rotate < 0 || d->rotate > d->depth || d->rotate % 2 != 0) wrong = "rotate is even and at most depth";
    else if (d->rotate > 0 && d->n_positions < 1) wrong = "n_positions is at least 1";
    else {
      const long long wq = (long long)d->q_heads * d->depth, wk = (long long)d->k_heads * d->depth;
      p.ld_in[0] = d->ldq ? d->ldq : wq; p.ld_in[1] = d->ldk ? d->ldk : wk;
      p.ld_out[0] = d->ldq_out ? d->ldq_out : wq; p.ld_out[1] = d->ldk_out ? d->ldk_out : wk;
      if (p.ld_in[0] < wq || p.ld_in[1] < wk || p.ld_out[0] < wq || p.ld_out[1] < wk) wrong = "rows overlap";
    }
    if (!wrong && d->rows > 0 && d->q_heads + d->k_heads > 0) {
      const uintptr_t size = d->precision == B200_PREC_FP32 ? 4 : 2;
      auto off = [](const void* q, uintptr_t n) { return reinterpret_cast<uintptr_t>(q) % n != 0; };
      if ((d->q_heads > 0 && (!d->q || !d->q_out)) || (d->k_heads > 0 && (!d->k || !d->k_out))) wrong = "queries, keys and their outputs are needed";
      else if (d->rotate > 0 && !d->table) wrong = "the table is needed";
      else if (off(d->q, size) || off(d->k, size) || off(d->q_out, size) || off(d->k_out, size) || off(d->gamma_q, 4) || off(d->gamma_k, 4) ||
               off(d->table, 8) || off(d->positions, 4))
        wrong = "an operand is not aligned to its type (the table to 8 bytes)";
      else if ((d->q_heads > 0 && d->q == d->q_out && p.ld_in[0] != p.ld_out[0]) || (d->k_heads > 0 && d->k == d->k_out && p.ld_in[1] != p.ld_out[1]))
        wrong = "in place, the leading dimensions are the same";
    }
    if (wrong) {
      set_error(std::string("b200_op_qk_norm_rotate: ") + wrong);
      return B200_ERR_INVALID;
    }
    if (d->rows == 0 || d->q_heads + d->k_heads == 0) return B200_OK;
    p.in[0] = d->q; p.in[1] = d->k; p.out[0] = d->q_out; p.out[1] = d->k_out;
    p.gamma[0] = d->gamma_q; p.gamma[1] = d->gamma_k;
    p.rows = d->rows; p.heads_q = d->q_heads; p.heads = d->q_heads + d->k_heads; p.depth = d->depth;
    p.norm = d->norm; p.eps = d->eps;
    p.rotate = d->rotate; p.interleaved = d->interleaved; p.n_positions = d->n_positions;
    p.table = reinterpret_cast<const float2*>(d->table); p.positions = d->positions;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (d->precision == B200_PREC_FP32) B200_CUDA(launch_qk<float>(p, s));
    else if (d->precision == B200_PREC_FP16) B200_CUDA(launch_qk<__half>(p, s));
    else B200_CUDA(launch_qk<__nv_bfloat16>(p, s));
    return B200_OK;
  });
}
