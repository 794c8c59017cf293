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
  int b = 0, n = 0, upto = 0;
  if (e < p.experts) {
    b = expert_begin(p, e);
    n = expert_begin(p, e + 1) - b;
  }
  auto list = [&]() {
    if (e >= 256) return;
    if (e < p.experts) begin[e] = b;
    if (e == p.experts - 1) begin[p.experts] = b + n;
    upto = (n + kRows - 1) / kRows;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int ahead = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += ahead;
    }
    if (lane == 31) scan[warp] = upto;
  };
  list();
  if (__syncthreads_or(n < 0)) {  // falling offsets: an entry counts as the largest ahead of it, so that no slot has two experts
    if (e < p.experts) {
      for (int i = 0; i < e; ++i) b = max(b, expert_begin(p, i));
      n = max(expert_begin(p, e + 1) - b, 0);
    }
    list();
    __syncthreads();
  }
  if (e < 256) {
    for (int w = 0; w < warp; ++w) upto += scan[w];
    if (e < p.experts) first[e + 1] = upto;
    if (e == 0) first[0] = 0;
  }
  __syncthreads();
}

// The tiles in the order they are computed, row tile by row tile, every `step`th of them.  Those from `split` on count twice, as a left and a right half of
// their kCols columns.
template <int kRows, int kCols> struct TileWalk {
  const int* first;  // [experts + 1] row tiles ahead of each expert's
  const int* begin;  // [experts + 1] slots
  int n_tiles, step, split, tiles;
  int t, e = 0, s0 = 0, end = 0, n0 = 0, width = kCols;  // the tile at hand: its expert, slots from s0 on below `end`, columns
  int mt, nt;
  // split_pairs: a last round that at most half of these have a tile of is computed in half tiles; 0: never.
  __device__ __forceinline__ TileWalk(const int* first_, const int* begin_, int experts, int n_tiles_, int start, int step_, int split_pairs)
      : first(first_), begin(begin_), n_tiles(n_tiles_), step(step_), t(start) {
    const int whole = first[experts] * n_tiles, last = split_pairs > 0 ? whole % split_pairs : 0;
    const bool halves = split_pairs > 0 && 2 * last <= split_pairs;
    split = halves ? whole - last : 0x7fffffff;
    tiles = halves ? whole + last : whole;
    mt = t / n_tiles;
    nt = t - mt * n_tiles;
    locate();
  }
  __device__ __forceinline__ bool valid() const { return t < tiles; }
  __device__ __forceinline__ void next() {
    t += step;
    nt += step % n_tiles;
    mt += step / n_tiles;
    if (nt >= n_tiles) {
      nt -= n_tiles;
      ++mt;
    }
    locate();
  }
  __device__ __forceinline__ void locate() {
    if (t >= tiles) return;
    if (t < split) {
      n0 = nt * kCols;
    } else {
      const int whole = split + ((t - split) >> 1);
      mt = whole / n_tiles;
      n0 = (whole - mt * n_tiles) * kCols + ((t - split) & 1) * (kCols / 2);
      width = kCols / 2;
    }
    while (first[e + 1] <= mt) ++e;
    s0 = begin[e] + (mt - first[e]) * kRows;
    end = begin[e + 1];
  }
};

// v e / (e + 1) with e = exp(v), and v n / (n + 2) with n = e (e + 2): four at a time share one reciprocal.  exp is held to exp(10) (Mish) and
// exp(20), beyond which the quotient is 1 to 2^-27, so that the four denominators' product stays finite; arithmetic in pairs.  us, 65536x1536x1024
// int8 with Mish: a reciprocal each, one by one 133, now 120; without an activation 88.
// (Results below 2^-126 are 0, and with them Mish and Swish of less than -87, which are up to 1e-36 in size: what bf16 could hold, and the quick Swish of
// the other products, whose denominator passes 2^126 there, does not give either.)
__device__ __forceinline__ float exp2_quick(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float reciprocal_quick(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
struct Two {
  uint64_t v;
  __device__ __forceinline__ Two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  __device__ __forceinline__ void parts(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
};
__device__ __forceinline__ Two operator*(Two a, Two b) {
  asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(a.v) : "l"(b.v));
  return a;
}
__device__ __forceinline__ Two operator+(Two a, Two b) {
  asm("add.rn.f32x2 %0, %0, %1;" : "+l"(a.v) : "l"(b.v));
  return a;
}
constexpr float kLog2e = 1.44269504f;
template <bool kMish> __device__ __forceinline__ void gate4(float* v) {
  constexpr float kMost = kMish ? 10.f : 20.f;
  float d[4];
  Two n[2] = {Two(0.f, 0.f), Two(0.f, 0.f)};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float a, b;
    (Two(fminf(v[2 * i], kMost), fminf(v[2 * i + 1], kMost)) * Two(kLog2e, kLog2e)).parts(a, b);
    const Two e(exp2_quick(a), exp2_quick(b));
    n[i] = kMish ? e * (e + Two(2.f, 2.f)) : e;
    (n[i] + (kMish ? Two(2.f, 2.f) : Two(1.f, 1.f))).parts(d[2 * i], d[2 * i + 1]);
  }
  const float d01 = d[0] * d[1], d23 = d[2] * d[3], r = reciprocal_quick(d01 * d23), r01 = r * d23, r23 = r * d01;
  // (a row's columns share it, whose number does not depend on the batch)
  (Two(v[0], v[1]) * (n[0] * (Two(r01, r01) * Two(d[1], d[0])))).parts(v[0], v[1]);
  (Two(v[2], v[3]) * (n[1] * (Two(r23, r23) * Two(d[3], d[2])))).parts(v[2], v[3]);
}

// The same with the four columns in neighbouring lanes: the same products, so the same bits.
template <bool kMish> __device__ __forceinline__ float gate_lane(float v) {
  const float e = exp2_quick(fminf(v, kMish ? 10.f : 20.f) * kLog2e), n = kMish ? __fmul_rn(e, __fadd_rn(e, 2.f)) : e, d = __fadd_rn(n, kMish ? 2.f : 1.f);
  const float other = __shfl_xor_sync(0xffffffffu, d, 1), both = d * other, far = __shfl_xor_sync(0xffffffffu, both, 2);
  return v * (n * (reciprocal_quick(both * far) * far * other));
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
