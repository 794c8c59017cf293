// The narrow product of the adapters, H[m] = s_a X[m] A_a^T, on tensor cores, for requests of whole blocks of 64 rows.
//
// What it cannot do without is one pass through X; a tile is 128 rows, i.e. at most two requests, and its B operand is the A of both, side by
// side: every row meets both and keeps its own.  That doubles multiplications which cost nothing (256 of a k-block's columns at most)
// and needs no masks.  X's and A's k-blocks arrive by TMA in a ring of about 100 KB, two CTAs to an SM; one thread issues
// tcgen05.mma (cta_group::1, 128 x 2 rank x 16), the accumulator is in tensor memory, and a thread of the epilogue has a row: H as
// fp32 (for a product with fp32 results, which shows that the tensor core truncates its sums, from two accumulators in turn that leave
// tensor memory after every k-block and are added in registers) and, where the shared product takes it as k-blocks, as two values of the type: the second holds what the first rounds off
// (fp16, where it is scaled by 2^11, 22 bits of the 24 in all, down to 2^-36; bf16 16).
#include "../../include/b200nn.h"
#include "kernels.cuh"
#include "tcgen05.cuh"

namespace b200 {
namespace {

constexpr int kShrinkThreads = 192;  // warps 0-3 epilogue, 4 TMA, 5 MMA
constexpr int kShrinkRing = 100 * 1024;

struct ShrinkParams {
  const float* scales; const int* ids;
  float* H; void* pieces;
  int M, K, rank, rp, group, n_adapters, stages, tmem_cols;
  int* status;
};

// Without saturation: an H beyond the range of fp16 is infinite, which the shared product notices.
__device__ __forceinline__ __half narrow(float v, __half) { return __float2half_rn(v); }
__device__ __forceinline__ __nv_bfloat16 narrow(float v, __nv_bfloat16) { return __float2bfloat16_rn(v); }
template <typename T> __device__ __forceinline__ uint32_t both(T lo, T hi) {
  return (uint32_t)*reinterpret_cast<const uint16_t*>(&lo) | (uint32_t)*reinterpret_cast<const uint16_t*>(&hi) << 16;
}

template <typename T, bool kRounded>
__global__ void __launch_bounds__(kShrinkThreads, 2)
adapters_shrink_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_a, const ShrinkParams p) {
  constexpr int kMaxStages = 8;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages], done[2], taken[2];  // kRounded: an accumulator each, else done[0]
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  const int warp = warp_index(), lane = threadIdx.x & 31, S = p.stages;
  const int m0 = blockIdx.x * BM;
  auto adapter = [&](int m) {
    const int a = m < p.M ? p.ids[m / p.group] : -1;
    return a >= 0 && a < p.n_adapters ? a : -1;
  };
  const int a0 = adapter(m0), a1 = adapter(m0 + 64);
  if (a0 < 0 && a1 < 0) return;
  // the adapters of the tile's columns: [0, rp) the first, [rp, 2 rp) the second where there are two
  const int first = a0 >= 0 ? a0 : a1;
  const bool two = a0 >= 0 && a1 >= 0 && a1 != a0;
  const int n = two ? 2 * p.rp : p.rp;
  const int a_bytes = p.rp * 128, stage_bytes = BM * 128 + 2 * a_bytes;
  if (threadIdx.x == 128) {
    tma_prefetch_map(&map_x);
    tma_prefetch_map(&map_a);
    for (int i = 0; i < S; ++i) {
      mbar_init(smem_u32(&full[i]), 1);
      mbar_init(smem_u32(&empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&done[i]), 1);
      mbar_init(smem_u32(&taken[i]), 4);
    }
    abort_word = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 5) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"((uint32_t)p.tmem_cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  // After the allocation: the shared product's CTAs, which wait for this launch's end, must not hold the tensor memory that it waits for.
  // (What they read ahead of that was written before this launch began.)
  grid_launch_dependents();
  const uint32_t tmem = tmem_slot;
  const int k_blocks = (p.K + BK - 1) / BK;
  if (warp == 4) {
    if (elect_one()) {
      int s = 0;
      uint32_t ph = 0;
      for (int kb = 0; kb < k_blocks; ++kb) {
        if (!mbar_wait(smem_u32(&empty[s]), ph ^ 1, abort_flag, 1)) break;
        const uint32_t fb = smem_u32(&full[s]), dst = smem_u32(smem + s * stage_bytes);
        mbar_expect_tx(fb, BM * 128 + (two ? 2 : 1) * p.rank * 128);
        tma_load_2d(dst, &map_x, kb * BK, m0, fb);
        tma_load_2d(dst + BM * 128, &map_a, kb * BK, first * p.rank, fb);
        if (two) tma_load_2d(dst + BM * 128 + a_bytes, &map_a, kb * BK, a1 * p.rank, fb);
        if (++s == S) { s = 0; ph ^= 1; }
      }
    }
    __syncwarp();
  } else if (warp == 5) {
    if (elect_one()) {
      const uint32_t idesc = (1u << 4) | (FmtCode<T>::v << 7) | (FmtCode<T>::v << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int kb = 0; kb < k_blocks; ++kb) {
        if (kRounded && !mbar_wait(smem_u32(&taken[kb & 1]), (kb >> 1 & 1) ^ 1, abort_flag, 4)) { ok = false; break; }
        if (!mbar_wait(smem_u32(&full[s]), ph, abort_flag, 2)) { ok = false; break; }
        tcgen05_fence_after();
        const uint32_t sa = smem_u32(smem + s * stage_bytes), sums = tmem + (kRounded ? (kb & 1) * 2 * p.rp : 0);
        const uint64_t adesc = make_smem_desc(sa), bdesc = make_smem_desc(sa + BM * 128);
#pragma unroll
        for (int k = 0; k < BK / 16; ++k) tcgen05_mma_f16(sums, adesc + 2 * k, bdesc + 2 * k, idesc, ((!kRounded && kb > 0) || k > 0) ? 1u : 0u);
        tcgen05_commit(smem_u32(&empty[s]));
        if (kRounded) tcgen05_commit(smem_u32(&done[kb & 1]));
        if (++s == S) { s = 0; ph ^= 1; }
      }
      if (ok && !kRounded) tcgen05_commit(smem_u32(&done[0]));
    }
    __syncwarp();
  } else {
    const int row = warp * 32 + lane, m = m0 + row;
    const int a = warp < 2 ? a0 : a1;  // the same in the whole warp
    const float scale = a >= 0 && p.scales ? p.scales[a] : 1.f;
    const uint32_t from = tmem + ((uint32_t)(warp * 32) << 16) + (two && a == a1 ? p.rp : 0);
    float* h = p.H + (long long)m * p.rank;
    T* q = static_cast<T*>(p.pieces) + (long long)m * 2 * p.rp;
    // sixteen ranks of the row, from r0 on
    auto finish = [&](int r0, float (&x)[16]) {
      // beyond the rank what lay behind A's rows was multiplied
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = r0 + j < p.rank ? scale * x[j] : 0.f;
      if (m >= p.M) return;
      if (p.rank % 4 == 0) {
#pragma unroll
        for (int j = 0; j < 16; j += 4)
          if (r0 + j < p.rank) *reinterpret_cast<float4*>(h + r0 + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (r0 + j < p.rank) h[r0 + j] = x[j];
      }
      if (!kRounded && p.pieces) {
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const T c0 = narrow(x[2 * j], T()), c1 = narrow(x[2 * j + 1], T());
          hi[j] = both(c0, c1);
          constexpr float kUp = 1 << LowPiece<T>::shift;
          lo[j] = both(narrow((x[2 * j] - to_f(c0)) * kUp, T()), narrow((x[2 * j + 1] - to_f(c1)) * kUp, T()));
        }
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
          *reinterpret_cast<uint4*>(q + r0 + 2 * j) = make_uint4(hi[j], hi[j + 1], hi[j + 2], hi[j + 3]);
          *reinterpret_cast<uint4*>(q + p.rp + r0 + 2 * j) = make_uint4(lo[j], lo[j + 1], lo[j + 2], lo[j + 3]);
        }
      }
    };
    if constexpr (kRounded) {
      constexpr int kMost = (B200_ADAPTERS_MAX_RANK + 15) / 16;
      float x[kMost][16];
#pragma unroll
      for (int i = 0; i < kMost; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) x[i][j] = 0.f;
      bool there = true;
#pragma unroll 1
      for (int kb = 0; kb < k_blocks && there; ++kb) {
        there = mbar_wait(smem_u32(&done[kb & 1]), kb >> 1 & 1, abort_flag, 3);
        tcgen05_fence_after();
        if (there && a >= 0) {
#pragma unroll
          for (int i = 0; i < kMost; ++i) {
            if (i * 16 >= p.rp) break;
            uint32_t v[16];
            tmem_ld16(from + (kb & 1) * 2 * p.rp + i * 16, v);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j) x[i][j] += __uint_as_float(v[j]);
          }
        }
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&taken[kb & 1]));
      }
      if (there && a >= 0) {
#pragma unroll
        for (int i = 0; i < kMost; ++i)
          if (i * 16 < p.rp) finish(i * 16, x[i]);
      }
    } else {
      const bool there = mbar_wait(smem_u32(&done[0]), 0, abort_flag, 3);
      tcgen05_fence_after();
      if (there && a >= 0) {
        for (int r0 = 0; r0 < p.rp; r0 += 16) {
          uint32_t v[16];
          tmem_ld16(from + r0, v);
          tmem_ld_wait();
          float x[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) x[j] = __uint_as_float(v[j]);
          finish(r0, x);
        }
      }
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 5) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)p.tmem_cols) : "memory");
  }
  if (abort_word) {
    for (int i = 0; i < 200; ++i) __nanosleep(1000);  // copies in flight land before the shared memory is released
    if (threadIdx.x == 0 && p.status) atomicCAS(p.status, 0, 800 + abort_word);
  }
}

}  // namespace

template <typename T>
cudaError_t launch_adapters_shrink(const GemmParams& g, const void* a, const float* scales, float* h, void* pieces, int* status, cudaStream_t s) {
  ShrinkParams p;
  p.scales = scales; p.ids = g.ad_ids; p.H = h; p.pieces = pieces;
  p.M = g.M; p.K = g.K; p.rank = g.ad_rank; p.rp = g.ad_rp; p.group = g.ad_group; p.n_adapters = g.ad_n; p.status = status;
  const int stage = BM * 128 + 2 * p.rp * 128, k_blocks = ceil_div(g.K, BK);
  p.stages = kShrinkRing / stage;
  if (p.stages > 8) p.stages = 8;
  if (p.stages > k_blocks) p.stages = k_blocks;
  p.tmem_cols = 32;
  while (p.tmem_cols < (g.out_f32 ? 4 : 2) * p.rp) p.tmem_cols *= 2;
  cudaError_t e = g.out_f32 ? raise_smem_limit<adapters_shrink_kernel<T, true>>(kShrinkRing + 1024)
                            : raise_smem_limit<adapters_shrink_kernel<T, false>>(kShrinkRing + 1024);
  CUtensorMap mx, ma;
  if (e == cudaSuccess) e = gemm_tensor_map(g.A, g.lda, g.M, g.K, BM, TypeTag<T>::prec, &mx);
  if (e == cudaSuccess) e = gemm_tensor_map(a, g.K, g.ad_n * g.ad_rank, g.K, g.ad_rank, TypeTag<T>::prec, &ma);
  if (e != cudaSuccess) return e;
  auto* kernel = g.out_f32 ? adapters_shrink_kernel<T, true> : adapters_shrink_kernel<T, false>;
  kernel<<<ceil_div(g.M, BM), kShrinkThreads, p.stages * stage + 1024, s>>>(mx, ma, p);
  return cudaGetLastError();
}
template cudaError_t launch_adapters_shrink<__half>(const GemmParams&, const void*, const float*, float*, void*, int*, cudaStream_t);
template cudaError_t launch_adapters_shrink<__nv_bfloat16>(const GemmParams&, const void*, const float*, float*, void*, int*, cudaStream_t);

}  // namespace b200
