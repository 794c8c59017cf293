// What the tensor-core kernels of grouped and 8-bit products share.
#pragma once
#include "chunk8.cuh"
#include "grouped.cuh"
#include "tcgen05.cuh"

namespace b200 {
namespace {

template <typename T> struct Operand {
  static constexpr int prec = TypeTag<T>::prec, k = 64;
  static constexpr uint32_t idesc = (1u << 4) | (FmtCode<T>::v << 7) | (FmtCode<T>::v << 10);
};
// D format s32 (bits 4-5 = 2), A and B signed (bits 7-9, 10-12 = 1)
template <> struct Operand<int8_t> {
  static constexpr int prec = 3, k = 128;
  static constexpr uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10);
};


// A wait whose answer is the same in the whole warp.
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity, volatile int* abort_flag, int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, code));
}

// Row tiles of kRows slots ahead of each expert's, and the experts' first slots; by all threads of a CTA of at least 256.
template <int kRows>
__device__ __forceinline__ void list_tiles(const GroupedParams& p, int* first, int* begin, int* scan) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = threadIdx.x;
  int upto = 0;
  if (e < 256) {
    if (e < p.experts) {
      const int b = expert_begin(p, e), n = expert_begin(p, e + 1) - b;
      begin[e] = b;
      if (e == p.experts - 1) begin[p.experts] = b + max(n, 0);
      upto = n > 0 ? (n + kRows - 1) / kRows : 0;
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int n = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += n;
    }
    if (lane == 31) scan[warp] = upto;
  }
  __syncthreads();
  if (e < 256) {
    for (int w = 0; w < warp; ++w) upto += scan[w];
    if (e < p.experts) first[e + 1] = upto;
    if (e == 0) first[0] = 0;
  }
  __syncthreads();
}

// The tiles in the order they are computed: row tile by row tile, its column tiles of kCols.  Those from `split` on count twice, as a left and a right
// half.
template <int kRows, int kCols> struct TileWalk {
  const int* first;  // [experts + 1] row tiles ahead of each expert's
  const int* begin;  // [experts + 1] slots
  int experts, n_tiles, split = 0x7fffffff;
  int e = 0, s0 = 0, end = 0, n0 = 0, width = kCols;  // of the tile last asked for: its expert, slots from s0 on below `end`, columns
  __device__ __forceinline__ int whole() const { return first[experts] * n_tiles; }
  __device__ __forceinline__ void at(int t) {  // t may only grow
    int right = 0;
    if (t >= split) {
      right = (t - split) & 1;
      t = split + ((t - split) >> 1);
      width = kCols / 2;
    }
    const int mt = t / n_tiles;
    while (first[e + 1] <= mt) ++e;
    s0 = begin[e] + (mt - first[e]) * kRows;
    end = begin[e + 1];
    n0 = (t - mt * n_tiles) * kCols + right * (kCols / 2);
  }
};

// v e / (e + 1) with e = exp(v), and v n / (n + 2) with n = e (e + 2): four at a time share one reciprocal.  exp is held to exp(10) (Mish) and
// exp(20), beyond which the quotient is 1 to 2^-27, so that the four denominators' product stays finite.  An epilogue of 65536x1024 columns
// with a reciprocal each spent 121 us where one without an activation took 80.
template <bool kMish> __device__ __forceinline__ void gate4(float* v) {
  float n[4], d[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float e = __expf(fminf(v[i], kMish ? 10.f : 20.f));
    n[i] = kMish ? e * (e + 2.f) : e;
    d[i] = n[i] + (kMish ? 2.f : 1.f);
  }
  const float d01 = d[0] * d[1], d23 = d[2] * d[3], r = __fdividef(1.f, d01 * d23), r01 = r * d23, r23 = r * d01;
  v[0] *= n[0] * (r01 * d[1]);  // (a row's columns share it, whose number does not depend on the batch)
  v[1] *= n[1] * (r01 * d[0]);
  v[2] *= n[2] * (r23 * d[3]);
  v[3] *= n[3] * (r23 * d[2]);
}

// The same with the four columns in neighbouring lanes: the same products, so the same bits.
template <bool kMish> __device__ __forceinline__ float gate_lane(float v) {
  const float e = __expf(fminf(v, kMish ? 10.f : 20.f)), n = kMish ? e * (e + 2.f) : e, d = n + (kMish ? 2.f : 1.f);
  const float other = __shfl_xor_sync(0xffffffffu, d, 1), both = d * other, far = __shfl_xor_sync(0xffffffffu, both, 2);
  return v * (n * (__fdividef(1.f, both * far) * far * other));
}

// By all lanes of a warp, four neighbours having columns 4i .. 4i + 3 of each of kN rows (0 behind the last column).
template <typename TOut, int kN> __device__ __forceinline__ void activate_lanes(float (&v)[kN], int act) {
  if (sizeof(TOut) == 2 && act == ACT_MISH) {
#pragma unroll
    for (int j = 0; j < kN; ++j) v[j] = gate_lane<true>(v[j]);
  } else if (sizeof(TOut) == 2 && act == ACT_SWISH) {
#pragma unroll
    for (int j = 0; j < kN; ++j) v[j] = gate_lane<false>(v[j]);
  } else if (act != ACT_NONE) {
#pragma unroll
    for (int j = 0; j < kN; ++j) v[j] = activate<sizeof(TOut) == 2>(v[j], act);
  }
}

// Columns of a row, the first a multiple of 4 and 0 behind the last column.
template <typename TOut, int kN> __device__ __forceinline__ void activate_columns(float (&v)[kN], int act) {
  if constexpr (sizeof(TOut) == 2) {
    if (act == ACT_MISH) {
#pragma unroll
      for (int j = 0; j < kN; j += 4) gate4<true>(v + j);
    } else if (act == ACT_SWISH) {
#pragma unroll
      for (int j = 0; j < kN; j += 4) gate4<false>(v + j);
    } else {
      apply_activation(v, act);
    }
  } else if (act != ACT_NONE) {
#pragma unroll
    for (int j = 0; j < kN; ++j) v[j] = activate<false>(v[j], act);
  }
}

inline bool aligned16(const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; }

}  // namespace
}  // namespace b200
