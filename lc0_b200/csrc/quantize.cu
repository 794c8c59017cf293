// Rows in 8 bits with a scale each: s = max |x| (1 / 127) in fp32, q = x / s to the nearest whole number, ties to even.
#include "chunk8.cuh"
#include "kernels.cuh"

namespace b200 {
namespace {

constexpr int kWarps = 4;

// Sizes compared as whole numbers, so that a NaN is above infinity and infinity above all else.
__device__ __forceinline__ uint32_t size_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t largest8(const Chunk<float>& c) {
  float v[8];
  unpack8(c, v);
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, size_bits(v[i]));
  return m;
}
template <typename T> __device__ __forceinline__ uint32_t largest8(const Chunk<T>& c) {  // two 16-bit sizes at a time
  const uint32_t k = 0x7fff7fffu;
  const uint32_t m = __vmaxu2(__vmaxu2(c.raw[0].x & k, c.raw[0].y & k), __vmaxu2(c.raw[0].z & k, c.raw[0].w & k));
  const float2 f = pair_f<T>(m);
  return max(size_bits(f.x), size_bits(f.y));
}

// x / s to the nearest whole number as the exact quotient has it: the sign of x - (r +- 1/2) s, which one fma gives without a rounding that
// could change it, says on which side of a tie x lies.
__device__ __noinline__ int exact_q(float x, float s) {
  if (s < 1e-30f) return (int)fmin(fmax(rint((double)x / (double)s), -127.0), 127.0);  // the reciprocal and the fma may leave fp32's range
  float r = rintf(x / s);
  const float up = fmaf(-(r + 0.5f), s, x), down = fmaf(-(r - 0.5f), s, x);
  const bool odd = ((int)r & 1) != 0;
  if (up > 0.f || (up == 0.f && odd)) r += 1.f;
  else if (down < 0.f || (down == 0.f && odd)) r -= 1.f;
  return (int)fminf(fmaxf(r, -127.f), 127.f);
}

// Adding 1.5 2^23 rounds to a whole number and leaves it in the low byte.  The product with the reciprocal is off by 2e-5 at most: chunks
// with a quotient that close to a tie are done again exactly.
__device__ __forceinline__ uint2 quantize8(const float (&v)[8], float s, float inv) {
  uint32_t b[8];
  float far = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float t = fmaf(v[i], inv, 12582912.f);
    b[i] = __float_as_uint(t);
    far = fmaxf(far, fabsf(fmaf(v[i], inv, 12582912.f - t)));
  }
  if (far > 0.4999f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = (uint32_t)exact_q(v[i], s);
  }
  uint2 q;
  q.x = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
  q.y = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
  return q;
}

struct RowScale {
  float s, inv;
  bool zero;   // all entries become 0
  bool exact;  // the reciprocal is not usable
};
__device__ __forceinline__ RowScale scale_of(uint32_t largest) {
  RowScale r;
  r.s = __fmul_rn(__uint_as_float(largest), 1.f / 127.f);
  if (largest >= 0x7f800000u) r.s = __uint_as_float(0x7fffffffu);
  r.zero = !(r.s > 0.f);
  r.exact = r.s < 1e-30f;
  r.inv = r.zero || r.exact ? 0.f : 1.f / r.s;
  return r;
}

// A warp per row, which stays in registers (kPer chunks of eight entries per lane) where it fits, and is read again where it does not.
template <typename T, int kPer>
__global__ void __launch_bounds__(32 * kWarps) quantize_rows_kernel(const T* X, long long ldx, int M, int K, int8_t* Q, long long ldq, float* scales) {
  grid_launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, chunks = K / 8;
  for (long long m = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5); m < M; m += (long long)gridDim.x * kWarps) {
    const T* x = X + m * ldx;
    Chunk<T> held[kPer > 0 ? kPer : 1];
    uint32_t largest = 0;
    if constexpr (kPer > 0) {
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (lane + 32 * i < chunks) held[i] = load8(x + 8 * (lane + 32 * i));
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (lane + 32 * i < chunks) largest = max(largest, largest8(held[i]));
    } else {
#pragma unroll 4
      for (int c = lane; c < chunks; c += 32) largest = max(largest, largest8(load8(x + 8 * c)));
    }
    const RowScale r = scale_of(__reduce_max_sync(0xffffffffu, largest));
    if (lane == 0) scales[m] = r.s;
    auto put = [&](const Chunk<T>& c, int at) {
      float v[8];
      unpack8(c, v);
      uint2 q = make_uint2(0u, 0u);
      if (r.exact && !r.zero) {
        int8_t b[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = (int8_t)exact_q(v[i], r.s);
        q = make_uint2((uint8_t)b[0] | (uint8_t)b[1] << 8 | (uint8_t)b[2] << 16 | (uint32_t)(uint8_t)b[3] << 24,
                       (uint8_t)b[4] | (uint8_t)b[5] << 8 | (uint8_t)b[6] << 16 | (uint32_t)(uint8_t)b[7] << 24);
      } else if (!r.zero) {
        q = quantize8(v, r.s, r.inv);
      }
      *reinterpret_cast<uint2*>(Q + m * ldq + 8 * at) = q;
    };
    if constexpr (kPer > 0) {
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (lane + 32 * i < chunks) put(held[i], lane + 32 * i);
    } else {
#pragma unroll 4
      for (int c = lane; c < chunks; c += 32) put(load8(x + 8 * c), c);
    }
  }
}

// Any width and alignment, entry by entry.
template <typename T>
__global__ void __launch_bounds__(32 * kWarps) quantize_rows_any_kernel(const T* X, long long ldx, int M, int K, int8_t* Q, long long ldq, float* scales) {
  grid_launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  for (long long m = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5); m < M; m += (long long)gridDim.x * kWarps) {
    uint32_t largest = 0;
    for (int k = lane; k < K; k += 32) largest = max(largest, size_bits(to_f(X[m * ldx + k])));
    const RowScale r = scale_of(__reduce_max_sync(0xffffffffu, largest));
    if (lane == 0) scales[m] = r.s;
    for (int k = lane; k < K; k += 32) Q[m * ldq + k] = r.zero ? (int8_t)0 : (int8_t)exact_q(to_f(X[m * ldx + k]), r.s);
  }
}

template <typename T>
cudaError_t launch_quantize(const void* X, long long ldx, int M, int K, int8_t* Q, long long ldq, float* scales, cudaStream_t s) {
  const T* x = static_cast<const T*>(X);
  const long long blocks = ((long long)M + kWarps - 1) / kWarps;
  const dim3 grid((unsigned)(blocks < 0x7fffffff ? blocks : 0x7fffffff)), block(32 * kWarps);
  const bool vec = K % 8 == 0 && ldx % (16 / (int)sizeof(T)) == 0 && ldq % 8 == 0 && reinterpret_cast<uintptr_t>(X) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(Q) % 8 == 0;
  auto kernel = !vec         ? quantize_rows_any_kernel<T>
                : K <= 256   ? quantize_rows_kernel<T, 1>
                : K <= 512   ? quantize_rows_kernel<T, 2>
                : K <= 1024  ? quantize_rows_kernel<T, 4>
                : K <= 2048  ? quantize_rows_kernel<T, 8>
                             : quantize_rows_kernel<T, 0>;
  DependentLaunches dependent;
  return launch_dependent(kernel, grid, block, 0, s, x, ldx, M, K, Q, ldq, scales);
}

}  // namespace
}  // namespace b200

extern "C" int b200_op_quantize_rows(const void* X, long long ldx, int M, int K, int precision, int8_t* Q, long long ldq, float* scales, void* stream) {
  using namespace b200;
  return at_c_entry([&]() -> int {
    const char* wrong = nullptr;
    if (M < 0 || K < 1) wrong = "M >= 0 and K >= 1";
    else if (precision < B200_PREC_FP32 || precision > B200_PREC_BF16) wrong = "unknown precision";
    else if ((ldx && ldx < K) || (ldq && ldq < K)) wrong = "rows overlap";
    else if (M > 0) {
      auto off = [](const void* q, uintptr_t n) { return reinterpret_cast<uintptr_t>(q) % n != 0; };
      if (!X || !Q || !scales) wrong = "X, Q and scales are needed";
      else if (off(X, precision == B200_PREC_FP32 ? 4 : 2) || off(scales, 4)) wrong = "an operand is not aligned to its type";
    }
    if (wrong) {
      set_error(std::string("b200_op_quantize_rows: ") + wrong);
      return B200_ERR_INVALID;
    }
    if (M == 0) return B200_OK;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const long long lx = ldx ? ldx : K, lq = ldq ? ldq : K;
    if (precision == B200_PREC_FP32) B200_CUDA(launch_quantize<float>(X, lx, M, K, Q, lq, scales, s));
    else if (precision == B200_PREC_FP16) B200_CUDA(launch_quantize<__half>(X, lx, M, K, Q, lq, scales, s));
    else B200_CUDA(launch_quantize<__nv_bfloat16>(X, lx, M, K, Q, lq, scales, s));
    return B200_OK;
  });
}
