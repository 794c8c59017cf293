// Grouped and 8-bit products of few rows per expert, and fp32 results of 16-bit operands: tcgen05 with W's rows on the 128 lanes of tensor
// memory and up to 64 slots as its columns.
//
// Such products are bound by how fast W arrives, so a tile takes 128 rows of W and whatever slots an expert has, 24 KB per k-block of 128
// bytes, and a CTA has up to eight of them in flight.  The other way round (128 slots on the lanes) most of what arrives would be room for
// slots that do not exist.  Results leave row by row: a thread has one column of 32 slots, a warp writes 32 consecutive columns.
//   warp 0      TMA producer of W, and of X where its rows lie in order
//   warp 1      tcgen05.mma issuer, kind::f16 or kind::i8
//   warp 2      gather4 of X's rows that the order names
//   warps 4-11  epilogue: four warps per half of the slots
// With fewer tiles than SMs the k-blocks of a tile are cut over the CTAs of a cluster (`ks`), which add their sums from one another's
// shared memory, in the order of their ranks, each a part of the slots.
// The tensor core truncates its sums, the more the longer they are; results of 16 bits hide it.  For fp32 results of 16-bit operands (kRounded)
// the accumulators leave tensor memory after every k-block and are added in registers, rounded to nearest.
// Every wait is bounded by wall-clock time like those of gemm_tc.cu; the cluster barriers are reached by all threads whatever happened before.
#include "grouped_tc.cuh"

namespace b200 {
namespace {

constexpr int kRows = 64;  // slots of a tile
constexpr int kStageBytes = (BM + kRows) * 128;
constexpr int kMaxStages = 8;
constexpr int kThreads = 384;
constexpr int kTmemCols = 2 * kRows;
constexpr int kListBytes = (2 * (B200_MAX_EXPERTS + 1) * 4 + 15) / 16 * 16;
constexpr int smem_bytes(int stages) { return stages * kStageBytes + kListBytes + kRows * 4 + 256 + 1024; }

template <typename T>
__device__ __forceinline__ void mma_one(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (sizeof(T) == 1) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  } else {
    tcgen05_mma_f16(d, a, b, idesc, accumulate);
  }
}
__device__ __forceinline__ void tma_gather4(uint32_t dst, const CUtensorMap* map, int x, const int4 row, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(row.x), "r"(row.y), "r"(row.z), "r"(row.w), "r"(bar)
      : "memory");
}
__device__ __forceinline__ uint32_t ld_cluster(uint32_t addr, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(v) : "r"(mapa(addr, rank)) : "memory");
  return v;
}

// A sum in tensor memory's type with its scales and bias.
template <typename TIn> __device__ __forceinline__ float scaled_sum(uint32_t sum, float sx, float sw, float bias) {
  return sizeof(TIn) == 1 ? fmaf((float)(int)sum, sx * sw, bias) : __uint_as_float(sum) + bias;
}
template <typename TIn> __device__ __forceinline__ uint32_t plus(uint32_t a, uint32_t b) {
  return sizeof(TIn) == 1 ? a + b : __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
}

template <typename TIn, typename TOut, bool kGather, bool kRounded>
__global__ void __launch_bounds__(kThreads, 1)
grouped_rows_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const GroupedParams p, int stages, int ks) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  int* first = reinterpret_cast<int*>(smem + stages * kStageBytes);
  int* begin = first + B200_MAX_EXPERTS + 1;
  int* gathered = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(first) + kListBytes);  // [64] rows of X
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(gathered + kRows);  // [stages]
  uint64_t* empty_bar = full_bar + kMaxStages;                          // [stages]
  uint64_t* tfull_bar = empty_bar + kMaxStages;                         // [2]
  uint64_t* tempty_bar = tfull_bar + 2;                                 // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty_bar + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* scan = reinterpret_cast<int*>(tmem_slot + 2);  // [8]

  const int warp = warp_index(), lane = threadIdx.x & 31;
  const uint32_t rank = ks > 1 ? cluster_ctarank() : 0;
  const int unit = blockIdx.x / ks, units = gridDim.x / ks;
  const int n_tiles = (p.N + BM - 1) / BM, k_blocks = (p.K + Operand<TIn>::k - 1) / Operand<TIn>::k;
  const int kb0 = k_blocks * (int)rank / ks, kb1 = k_blocks * ((int)rank + 1) / ks;

  if (threadIdx.x == 64) {
    tma_prefetch_map(&map_x);
    tma_prefetch_map(&map_w);
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(smem_u32(&full_bar[i]), 1);
      mbar_init(smem_u32(&empty_bar[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&tfull_bar[i]), 1);
      mbar_init(smem_u32(&tempty_bar[i]), 8);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  grid_dependency_wait();
  tcgen05_fence_before();
  list_tiles<kRows>(p, first, begin, scan);
  tcgen05_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  grid_launch_dependents();  // not ahead of the tensor memory: a dependent that took it would hold it while it waits for this kernel
  TileWalk<kRows> walk{first, begin, p.experts, n_tiles};
  const int tiles = walk.total();
  int s0 = 0, end = 0, n0 = 0;

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    if (elect_one()) {
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int t = unit; t < tiles && ok; t += units) {
        walk.at(t, BM, s0, end, n0);
        const int x_bytes = kGather ? (min(kRows, end - s0) + 3) / 4 * 512 : kRows * 128;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(smem_u32(&empty_bar[s]), ph ^ 1, abort_flag, 1)) { ok = false; break; }
          const uint32_t fb = smem_u32(&full_bar[s]), sa = smem_u32(smem + s * kStageBytes);
          mbar_expect_tx(fb, BM * 128 + x_bytes);
          tma_load_2d(sa, &map_w, kb * Operand<TIn>::k, walk.e * p.N + n0, fb);
          if constexpr (!kGather) tma_load_2d(sa + BM * 128, &map_x, kb * Operand<TIn>::k, s0, fb);
          if (++s == stages) { s = 0; ph ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    if (elect_one()) {
      int s = 0;
      uint32_t ph = 0, it = 0;  // it: accumulators filled
      bool ok = true;
      for (int t = unit; t < tiles && ok; t += units) {
        walk.at(t, BM, s0, end, n0);
        const uint32_t idesc = Operand<TIn>::idesc | ((uint32_t)(BM >> 4) << 24) | ((uint32_t)(((min(kRows, end - s0) + 15) & ~15) >> 3) << 17);
        uint32_t d = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (kRounded || kb == kb0) {
            if (!mbar_wait(smem_u32(&tempty_bar[it & 1]), ((it >> 1) & 1) ^ 1, abort_flag, 2)) { ok = false; break; }
            tcgen05_fence_after();
            d = tmem_base + (it & 1) * kRows;
          }
          if (!mbar_wait(smem_u32(&full_bar[s]), ph, abort_flag, 3)) { ok = false; break; }
          tcgen05_fence_after();
          const uint32_t sa = smem_u32(smem + s * kStageBytes);
          const uint64_t adesc = make_smem_desc(sa), bdesc = make_smem_desc(sa + BM * 128);
#pragma unroll
          for (int k = 0; k < 4; ++k) mma_one<TIn>(d, adesc + 2 * k, bdesc + 2 * k, idesc, ((!kRounded && kb > kb0) || k > 0) ? 1u : 0u);
          tcgen05_commit(smem_u32(&empty_bar[s]));
          if (kRounded || kb + 1 == kb1) {
            tcgen05_commit(smem_u32(&tfull_bar[it & 1]));
            ++it;
          }
          if (++s == stages) { s = 0; ph ^= 1; }
        }
      }
    }
  } else if (warp == 2) {
    // ---------------- gather ----------------
    if constexpr (kGather) {
      uint32_t done = 0;  // k-blocks before this tile's
      bool ok = true;
      for (int t = unit; t < tiles && ok; t += units, done += kb1 - kb0) {
        walk.at(t, BM, s0, end, n0);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int slot = s0 + 32 * i + lane, x = slot < end ? rows_of_slot(p, slot).x : 0;
          gathered[32 * i + lane] = x < 0 ? 0 : x;  // whatever lies there: its results are not stored
        }
        __syncwarp();
        if (elect_one()) {
          int s = (int)(done % stages);
          uint32_t ph = (done / stages) & 1;
          const int fours = (min(kRows, end - s0) + 3) / 4;
          for (int kb = kb0; kb < kb1; ++kb) {
            if (!mbar_wait(smem_u32(&empty_bar[s]), ph ^ 1, abort_flag, 5)) { ok = false; break; }
            const uint32_t fb = smem_u32(&full_bar[s]), sa = smem_u32(smem + s * kStageBytes) + BM * 128;
#pragma unroll 4
            for (int i = 0; i < fours; ++i) tma_gather4(sa + i * 512, &map_x, kb * Operand<TIn>::k, reinterpret_cast<const int4*>(gathered)[i], fb);
            if (++s == stages) { s = 0; ph ^= 1; }
          }
        }
        ok = __all_sync(0xffffffffu, ok);
      }
    }
  }
  // ---------------- epilogue ----------------
  const int quarter = warp & 3, half = warp >= 8 ? 1 : 0, column = quarter * 32 + lane;
  uint32_t* part = reinterpret_cast<uint32_t*>(smem);  // [64][128] sums of this CTA, once its stages are used up (ks > 1: one tile)
  int rows = 0;
  if (warp >= 4) {
    uint32_t it = 0;
    for (int t = unit; t < tiles; t += units) {
      walk.at(t, BM, s0, end, n0);
      rows = min(kRows, end - s0);
      const int n = n0 + column, slot = s0 + half * 32 + lane;
      const bool mine = half * 32 < rows;  // the same in the whole warp
      float bias = 0.f, sw = 1.f, sx = 1.f, weight = p.alpha;
      SlotRows r = {-1, -1, 0};
      if (ks == 1) {
        if (n < p.N) {
          if (p.bias) bias = __ldg(p.bias + (long long)walk.e * p.N + n);
          if (sizeof(TIn) == 1) sw = __ldg(p.w_scales + (long long)walk.e * p.N + n);
        }
        if (slot < end) r = rows_of_slot(p, slot);
        if (r.c >= 0) {
          if (sizeof(TIn) == 1) sx = p.x_scales[r.x];
          if (p.weights) weight *= p.weights[r.choice];
        }
      }
      uint32_t sum[32];
      bool ok = true;
      for (int kb = kb0; kb < kb1; kb = kRounded ? kb + 1 : kb1, ++it) {
        if (!mbar_wait(smem_u32(&tfull_bar[it & 1]), (it >> 1) & 1, abort_flag, 4)) { ok = false; break; }
        tcgen05_fence_after();
        if (mine) {
          uint32_t a[32];
          tmem_ld32(tmem_base + ((uint32_t)(quarter * 32) << 16) + (it & 1) * kRows + half * 32, a);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; ++j) sum[j] = kRounded && kb > kb0 ? plus<TIn>(sum[j], a[j]) : a[j];
        }
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&tempty_bar[it & 1]));
      }
      if (!ok) break;
      if (!mine) continue;
      if (ks > 1) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (half * 32 + j < rows) part[(half * 32 + j) * 128 + column] = sum[j];
        continue;
      }
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        if (half * 32 + j >= rows) break;
        const int c = __shfl_sync(0xffffffffu, r.c, j);
        const float w = __shfl_sync(0xffffffffu, weight, j);
        float v = scaled_sum<TIn>(sum[j], sizeof(TIn) == 1 ? __shfl_sync(0xffffffffu, sx, j) : 1.f, sw, bias);
        v = activate_lane<TOut>(n < p.N ? v : 0.f, p.act) * w;
        if (c >= 0 && n < p.N) {
          if (p.res) v += to_f(static_cast<const TOut*>(p.res)[c * p.ldres + n]);
          static_cast<TOut*>(p.C)[c * p.ldc + n] = one_of<TOut>(v);
        }
      }
    }
  }

  __syncwarp();
  tcgen05_fence_before();
  __syncthreads();
  if (*abort_flag) {
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
    if (threadIdx.x == 0 && p.status) atomicCAS(p.status, 0, 800 + *abort_flag);
    __syncthreads();
  }
  if (warp == 1) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)kTmemCols) : "memory");
  }
  if (ks == 1) return;
  cluster_sync_all();  // the sums of all CTAs are in their shared memory
  if (warp >= 4 && unit < tiles) {
    const int n = n0 + column;
    float bias = 0.f, sw = 1.f;
    if (n < p.N) {
      if (p.bias) bias = __ldg(p.bias + (long long)walk.e * p.N + n);
      if (sizeof(TIn) == 1) sw = __ldg(p.w_scales + (long long)walk.e * p.N + n);
    }
    const int m0 = rows * (int)rank / ks, m1 = rows * ((int)rank + 1) / ks;
#pragma unroll 2
    for (int m = m0 + half; m < m1; m += 2) {
      const uint32_t at = smem_u32(part + m * 128 + column);
      uint32_t from[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) from[k] = k < ks ? ld_cluster(at, k) : 0u;
      const SlotRows r = rows_of_slot(p, s0 + m);
      if (r.c < 0) continue;
      uint32_t sum = from[0];
#pragma unroll
      for (int k = 1; k < 8; ++k)
        if (k < ks) sum = plus<TIn>(sum, from[k]);
      float v = scaled_sum<TIn>(sum, sizeof(TIn) == 1 ? p.x_scales[r.x] : 1.f, sw, bias);
      v = activate_lane<TOut>(n < p.N ? v : 0.f, p.act) * (p.weights ? p.alpha * p.weights[r.choice] : p.alpha);
      if (n >= p.N) continue;
      if (p.res) v += to_f(static_cast<const TOut*>(p.res)[r.c * p.ldres + n]);
      static_cast<TOut*>(p.C)[r.c * p.ldc + n] = one_of<TOut>(v);
    }
  }
  cluster_sync_all();  // no CTA leaves while another may read its sums
}

template <typename TIn, typename TOut, bool kGather, bool kRounded>
cudaError_t launch_rows(const GroupedParams& p, int sm_count, cudaStream_t s) {
  CUtensorMap mx, mw;
  cudaError_t e = tma_encode_rows(p.X, p.ldx, p.x_rows, p.K, kGather ? 1 : kRows, Operand<TIn>::prec, &mx);
  if (e == cudaSuccess) e = tma_encode_rows(p.W, p.ldw, (long long)p.experts * p.N, p.K, BM, Operand<TIn>::prec, &mw);
  if (e == cudaSuccess) e = raise_smem_limit<grouped_rows_kernel<TIn, TOut, kGather, kRounded>>(smem_bytes(kMaxStages));
  if (e != cudaSuccess) return e;
  const int n_tiles = ceil_div(p.N, BM), k_blocks = ceil_div(p.K, Operand<TIn>::k);
  const int used = p.experts < p.slots ? p.experts : p.slots;
  const long long most = ((long long)p.slots + kRows - 1) / kRows + used - 1;  // row tiles there can be
  // Row tiles to expect: one per expert, or what the slots fill.  A tile is cut over as many CTAs as leave each of them an SM.
  const long long expected = ((long long)p.slots / kRows > used ? (long long)p.slots / kRows : used) * n_tiles;
  int ks = 1;
  while (ks < 8 && expected * ks * 2 <= sm_count && 2 * ks <= k_blocks) ks *= 2;
  const long long tiles = most * n_tiles;
  const int per_cta = ceil_div(k_blocks, ks);
  const int stages = ks > 1 && per_cta < kMaxStages ? (per_cta < 2 ? 2 : per_cta) : kMaxStages;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(ks > 1 ? tiles * ks : tiles < sm_count ? tiles : sm_count));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem_bytes(stages);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ks;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ks > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, grouped_rows_kernel<TIn, TOut, kGather, kRounded>, mx, mw, p, stages, ks);
}

}  // namespace

template <typename TIn, typename TOut>
cudaError_t launch_grouped_rows(const GroupedParams& p, bool rounded, int sm_count, cudaStream_t s) {
  const bool gather = p.order && !p.x_by_slot;
  if constexpr (sizeof(TIn) == 2 && sizeof(TOut) == 4) {
    if (rounded) return gather ? launch_rows<TIn, TOut, true, true>(p, sm_count, s) : launch_rows<TIn, TOut, false, true>(p, sm_count, s);
  }
  return gather ? launch_rows<TIn, TOut, true, false>(p, sm_count, s) : launch_rows<TIn, TOut, false, false>(p, sm_count, s);
}
#define INSTANCE(TIn, TOut) template cudaError_t launch_grouped_rows<TIn, TOut>(const GroupedParams&, bool, int, cudaStream_t)
INSTANCE(__half, __half);
INSTANCE(__half, float);
INSTANCE(__nv_bfloat16, __nv_bfloat16);
INSTANCE(__nv_bfloat16, float);
INSTANCE(int8_t, __half);
INSTANCE(int8_t, __nv_bfloat16);
INSTANCE(int8_t, float);

}  // namespace b200
