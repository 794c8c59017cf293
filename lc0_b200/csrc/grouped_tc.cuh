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

// A tile of the walk: its expert, the first slot and column.
template <int kRows> struct TileWalk {
  const int* first;  // [experts + 1] row tiles ahead of each expert's
  const int* begin;  // [experts + 1] slots
  int experts, n_tiles, e = 0;
  __device__ __forceinline__ int total() const { return first[experts] * n_tiles; }
  // t may only grow
  __device__ __forceinline__ void at(int t, int bn, int& s0, int& end, int& n0) {
    const int mt = t / n_tiles;
    while (first[e + 1] <= mt) ++e;
    s0 = begin[e] + (mt - first[e]) * kRows;
    end = begin[e + 1];
    n0 = (t - mt * n_tiles) * bn;
  }
};

template <typename TOut> __device__ __forceinline__ void activate32(float (&v)[32], int act) {
  if constexpr (sizeof(TOut) == 2) {
    apply_activation(v, act);
  } else if (act != ACT_NONE) {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = activate<false>(v[j], act);
  }
}

inline bool aligned16(const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; }

}  // namespace
}  // namespace b200
