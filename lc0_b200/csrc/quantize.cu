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

// x / s where the reciprocal of s, or what the steps below need, may leave fp32's range.
__device__ __noinline__ uint32_t tiny_q(float x, float s) { return (uint32_t)(int)fmin(fmax(rint((double)x / (double)s), -127.0), 127.0); }

// x / s to the nearest whole number, in the low byte.  Adding 1.5 2^23 rounds the product with the reciprocal, which is off by 1e-5 at most, to r
// or, beside a tie, to its neighbour.  e = x - r s is exact (r s and x are multiples of half an ulp of s or more, and beside a tie e is about s / 2), so
// r + e / s is the quotient, and a second fma rounds r + e (1 / s): off by |e| 2^-24 < ulp(s) / 2 with the reciprocal's rounding, while what is
// no tie is at least ulp(s) / 2 away from one.  Ties proper, |e| = s / 2, are told by comparing and go to the even of the two.
// us at 65536x1536 bf16: remainders only for chunks beside a tie, which bf16's eight bits bring about in most 127; remainders compared with s / 2
// entry by entry 60; now 51 (6.0 TB/s).
__device__ __forceinline__ uint32_t nearer(uint32_t b, float e, float half) {  // b: r in its low byte
  const float limit = __uint_as_float(__float_as_uint(half) + (~b & 1u));      // an even r keeps the tie
  return fabsf(e) >= limit ? b + (uint32_t)((__float_as_int(e) >> 31) | 1) : b;
}
__device__ __forceinline__ uint32_t exact_q(float x, float s, float inv) {
  const float t = fmaf(x, inv, 12582912.f);
  return nearer(__float_as_uint(t), fmaf(12582912.f - t, s, x), 0.5f * s);
}
// Two at a time where the arithmetic comes in pairs.
__device__ __forceinline__ uint64_t two(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint2 quantize8(const float (&v)[8], float s, float inv) {
  uint32_t b[8];
  const uint64_t inv2 = two(inv, inv), s2 = two(s, s), magic = two(12582912.f, 12582912.f), minus = two(-1.f, -1.f);
  const float half = 0.5f * s;
  bool tie = inv == 0.f;  // (no usable reciprocal)
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const uint64_t x2 = two(v[i], v[i + 1]), t2 = fma2(x2, inv2, magic), e2 = fma2(fma2(t2, minus, magic), s2, x2), u2 = fma2(e2, inv2, t2);
    float e0, e1;
    asm("mov.b64 {%0, %1}, %2;" : "=r"(b[i]), "=r"(b[i + 1]) : "l"(u2));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(e0), "=f"(e1) : "l"(e2));
    tie = tie || fabsf(e0) == half || fabsf(e1) == half;
  }
  if (tie) {
    asm volatile("");
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = inv == 0.f ? tiny_q(v[i], s) : exact_q(v[i], s, inv);
  }
  uint2 q;
  q.x = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
  q.y = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
  return q;
}

struct RowScale {
  float s, inv;
  bool zero;  // all entries become 0
};
__device__ __forceinline__ RowScale scale_of(uint32_t largest) {
  RowScale r;
  r.s = __fmul_rn(__uint_as_float(largest), 1.f / 127.f);
  if (largest >= 0x7f800000u) r.s = __uint_as_float(0x7fffffffu);
  r.zero = !(r.s > 0.f);
  r.inv = r.zero || r.s < 1e-30f ? 0.f : 1.f / r.s;
  return r;
}

template <typename T> __device__ __forceinline__ Chunk<T> load8_once(const T* p) {  // read once: leaves L2 ahead of what is written
  Chunk<T> c;
#pragma unroll
  for (int i = 0; i < Chunk<T>::kLoads; ++i) c.raw[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
  return c;
}

// A row in the registers of kThreads threads, kPer chunks of eight entries each; the next row is on its way meanwhile.
//   Many rows: a warp each, as many as fit, each walking over its rows (us, a warp for one row and the next CTA behind it / now: 65536x1536 bf16
//   57 / 51, 65536x1024 fp32 62 / 53: 6.0 and 6.3 TB/s of 6.55).
//   Up to 2048 rows: four warps each, so that a thread has one or two chunks (bf16 in a chain of launches, us, four warps / one: 64x1024 1.2 / 1.8,
//   1024x1024 2.2 / 2.7, 2048x1024 3.3 / 3.4, 2560x1024 3.6 / 3.5, 4096x1024 4.8 / 3.9; rows of 2048 entries turn later, 4096 of them 6.3 / 7.6, rows
//   of 512 earlier, 1024 of them 2.0 / 1.9).
template <typename T, int kPer, int kThreads>
__global__ void __launch_bounds__(128) quantize_rows_kernel(const T* X, long long ldx, int M, int K, int8_t* Q, long long ldq, float* scales) {
  __shared__ uint32_t of_warp[4];
  grid_launch_dependents();
  grid_dependency_wait();
  const int at = threadIdx.x % kThreads, chunks = K / 8;
  const long long step = (long long)gridDim.x * (128 / kThreads);
  long long m = (long long)blockIdx.x * (128 / kThreads) + threadIdx.x / kThreads;
  Chunk<T> next[kPer];
  auto fetch = [&](long long row) {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (row < M && at + kThreads * i < chunks) next[i] = load8_once(X + row * ldx + 8 * (at + kThreads * i));
  };
  fetch(m);
  for (; m < M; m += step) {
    Chunk<T> held[kPer];
    uint32_t largest = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      held[i] = next[i];
      if (at + kThreads * i < chunks) largest = max(largest, largest8(held[i]));
    }
    fetch(m + step);
    largest = __reduce_max_sync(0xffffffffu, largest);
    if constexpr (kThreads > 32) {
      if (threadIdx.x % 32 == 0) of_warp[threadIdx.x / 32] = largest;
      __syncthreads();
      largest = max(max(of_warp[0], of_warp[1]), max(of_warp[2], of_warp[3]));
      __syncthreads();
    }
    const RowScale r = scale_of(largest);
    if (at == 0) scales[m] = r.s;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int c = at + kThreads * i;
      if (c >= chunks) continue;
      float v[8];
      unpack8(held[i], v);
      *reinterpret_cast<uint2*>(Q + m * ldq + 8 * c) = r.zero ? make_uint2(0u, 0u) : quantize8(v, r.s, r.inv);
    }
  }
}

// Rows too long for that: a CTA reads each twice.
template <typename T>
__global__ void __launch_bounds__(256) quantize_long_rows_kernel(const T* X, long long ldx, int M, int K, int8_t* Q, long long ldq, float* scales) {
  __shared__ uint32_t of_warp[8];
  grid_launch_dependents();
  grid_dependency_wait();
  const int chunks = K / 8;
  for (long long m = blockIdx.x; m < M; m += gridDim.x) {
    const T* x = X + m * ldx;
    uint32_t largest = 0;
#pragma unroll 4
    for (int c = threadIdx.x; c < chunks; c += 256) largest = max(largest, largest8(load8(x + 8 * c)));
    largest = __reduce_max_sync(0xffffffffu, largest);
    if (threadIdx.x % 32 == 0) of_warp[threadIdx.x / 32] = largest;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) largest = max(largest, of_warp[w]);
    __syncthreads();
    const RowScale r = scale_of(largest);
    if (threadIdx.x == 0) scales[m] = r.s;
#pragma unroll 2
    for (int c = threadIdx.x; c < chunks; c += 256) {
      float v[8];
      unpack8(load8_once(x + 8 * c), v);
      *reinterpret_cast<uint2*>(Q + m * ldq + 8 * c) = r.zero ? make_uint2(0u, 0u) : quantize8(v, r.s, r.inv);
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
    for (int k = lane; k < K; k += 32) {
      const float v = to_f(X[m * ldx + k]);
      Q[m * ldq + k] = r.zero ? (int8_t)0 : (int8_t)(r.inv == 0.f ? tiny_q(v, r.s) : exact_q(v, r.s, r.inv));
    }
  }
}

template <typename T, int kPer, int kThreads>
cudaError_t launch_rows(const T* x, long long ldx, int M, int K, int8_t* Q, long long ldq, float* scales, cudaStream_t s) {
  auto kernel = quantize_rows_kernel<T, kPer, kThreads>;
  const long long blocks = ((long long)M + 128 / kThreads - 1) / (128 / kThreads);
  int per_sm = 0, dev = 0, sms = 0;
  cudaError_t e = cudaSuccess;
  if (kThreads == 32) {
    if ((e = cudaGetDevice(&dev)) != cudaSuccess || (e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess ||
        (e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, 128, 0)) != cudaSuccess)
      return e;
  }
  const long long most = kThreads == 32 ? (long long)sms * per_sm : 0x7fffffff;
  return launch_dependent(kernel, dim3((unsigned)(blocks < most ? blocks : most)), dim3(128), 0, s, x, ldx, M, K, Q, ldq, scales);
}

template <typename T>
cudaError_t launch_quantize(const void* X, long long ldx, int M, int K, int8_t* Q, long long ldq, float* scales, cudaStream_t s) {
  const T* x = static_cast<const T*>(X);
  DependentLaunches dependent;
  const bool vec = K % 8 == 0 && ldx % (16 / (int)sizeof(T)) == 0 && ldq % 8 == 0 && reinterpret_cast<uintptr_t>(X) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(Q) % 8 == 0;
  if (!vec)
    return launch_dependent(quantize_rows_any_kernel<T>, dim3((unsigned)(((long long)M + kWarps - 1) / kWarps)), dim3(32 * kWarps), 0, s, x, ldx, M, K, Q, ldq,
                            scales);
  const int chunks = K / 8;
  if (M <= 2048 && chunks > 32) {
    if (chunks <= 128) return launch_rows<T, 1, 128>(x, ldx, M, K, Q, ldq, scales, s);
    if (chunks <= 256) return launch_rows<T, 2, 128>(x, ldx, M, K, Q, ldq, scales, s);
    if (chunks <= 512) return launch_rows<T, 4, 128>(x, ldx, M, K, Q, ldq, scales, s);
  }
  if (chunks <= 32) return launch_rows<T, 1, 32>(x, ldx, M, K, Q, ldq, scales, s);
  if (chunks <= 64) return launch_rows<T, 2, 32>(x, ldx, M, K, Q, ldq, scales, s);
  if (chunks <= 128) return launch_rows<T, 4, 32>(x, ldx, M, K, Q, ldq, scales, s);
  if (chunks <= 192) return launch_rows<T, 6, 32>(x, ldx, M, K, Q, ldq, scales, s);
  if (chunks <= 256) return launch_rows<T, 8, 32>(x, ldx, M, K, Q, ldq, scales, s);
  if (chunks <= 512) return launch_rows<T, 4, 128>(x, ldx, M, K, Q, ldq, scales, s);
  return launch_dependent(quantize_long_rows_kernel<T>, dim3((unsigned)(M < 65536 ? M : 65536)), dim3(256), 0, s, x, ldx, M, K, Q, ldq, scales);
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
