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
// With fewer tiles than SMs the k-blocks of a tile are cut over the CTAs of a cluster (`ks`), which send their sums of each CTA's part of the slots
// to its shared memory, where they are added in the order of the ranks.
// The tensor core truncates its sums, the more the longer they are; results of 16 bits hide it.  For fp32 results of 16-bit operands (kRounded)
// the accumulators leave tensor memory after every k-block and are added in registers, rounded to nearest.
// Every wait is bounded by wall-clock time like those of gemm_tc.cu; the cluster barriers are reached by all threads whatever happened before.
#include <type_traits>

#include "grouped_tc.cuh"

namespace b200 {
namespace {

constexpr int kRows = 64;  // slots of a tile
constexpr int kStageBytes = (BM + kRows) * 128;
constexpr int kMaxStages = 8;
constexpr int kThreads = 384;
constexpr int kAccs = 4;  // accumulators
constexpr int kTmemCols = kAccs * kRows;
constexpr int kListBytes = (2 * (B200_MAX_EXPERTS + 1) * 4 + 15) / 16 * 16;
// ks > 1: 32 KB for the sums that the CTAs of the cluster send to one another
constexpr int kMaxSplitStages = 6;
constexpr int kPartBytes = 8 * 128 * 8 * 4;
constexpr int smem_bytes(int stages, bool split) { return stages * kStageBytes + (split ? kPartBytes : 0) + kListBytes + kRows * 4 + 256 + 1024; }

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
__device__ __forceinline__ void st_cluster4(uint32_t addr, uint32_t rank, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(mapa(addr, rank)), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// Slots that each CTA of a cluster finishes: whole fours.
__device__ __forceinline__ int slots_each(int rows, int log_ks) { return (((rows + (1 << log_ks) - 1) >> log_ks) + 3) & ~3; }

// A sum in tensor memory's type with its scales and bias.
template <typename TIn> __device__ __forceinline__ float scaled_sum(uint32_t sum, float sx, float sw, float bias) {
  return sizeof(TIn) == 1 ? fmaf((float)(int)sum, sx * sw, bias) : __uint_as_float(sum) + bias;
}
template <typename TIn> __device__ __forceinline__ uint32_t plus(uint32_t a, uint32_t b) {
  return sizeof(TIn) == 1 ? a + b : __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
}

template <typename TIn, typename TOut, bool kGather, bool kRounded>
__global__ void __launch_bounds__(kThreads, 1)
grouped_rows_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const GroupedParams p, int stages, int log_ks) {
  const int ks = 1 << log_ks;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint32_t* part = reinterpret_cast<uint32_t*>(smem + stages * kStageBytes);  // ks > 1: [ks][slots_each / 4][128][4] sums of this CTA's slots from each CTA
  int* first = reinterpret_cast<int*>(smem + stages * kStageBytes + (ks > 1 ? kPartBytes : 0));
  int* begin = first + B200_MAX_EXPERTS + 1;
  int* gathered = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(first) + kListBytes);  // [64] rows of X
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(gathered + kRows);  // [stages]
  uint64_t* empty_bar = full_bar + kMaxStages;                          // [stages]
  uint64_t* tfull_bar = empty_bar + kMaxStages;                         // [kAccs]
  uint64_t* tempty_bar = tfull_bar + kAccs;                             // [kAccs]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty_bar + kAccs);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* scan = reinterpret_cast<int*>(tmem_slot + 2);  // [8]

  const int warp = warp_index(), lane = threadIdx.x & 31;
  const uint32_t rank = ks > 1 ? cluster_ctarank() : 0;
  const int unit = blockIdx.x >> log_ks, units = gridDim.x >> log_ks;
  const int n_tiles = (p.N + BM - 1) / BM, k_blocks = (p.K + Operand<TIn>::k - 1) / Operand<TIn>::k;
  const int kb0 = k_blocks * (int)rank >> log_ks, kb1 = k_blocks * ((int)rank + 1) >> log_ks;

  // Waited for ahead of the first store to another CTA: that it runs.  Not behind the tensor memory, which a CTA then holds for no longer than its own
  // products take: clusters that each wait for what another holds would wait for ever.
  if (ks > 1) cluster_arrive();
  if (threadIdx.x == 64) {
    tma_prefetch_map(&map_x);
    tma_prefetch_map(&map_w);
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(smem_u32(&full_bar[i]), 1);
      mbar_init(smem_u32(&empty_bar[i]), 1);
    }
    for (int i = 0; i < kAccs; ++i) {
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
  TileWalk<kRows, BM> walk(first, begin, p.experts, n_tiles, unit, units, 0);
  const int &s0 = walk.s0, &end = walk.end, &n0 = walk.n0;

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    if (elect_one()) {
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (; walk.valid() && ok; walk.next()) {
        const int x_row = p.x_by_blocks ? row_of_block(p, s0, end) : s0;
        const int x_bytes = kGather ? (min(kRows, end - s0) + 3) / 4 * 512 : kRows * 128;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(smem_u32(&empty_bar[s]), ph ^ 1, abort_flag, 1)) { ok = false; break; }
          const uint32_t fb = smem_u32(&full_bar[s]), sa = smem_u32(smem + s * kStageBytes);
          mbar_expect_tx(fb, BM * 128 + x_bytes);
          tma_load_2d(sa, &map_w, kb * Operand<TIn>::k, walk.e * p.N + n0, fb);
          if constexpr (!kGather) tma_load_2d(sa + BM * 128, &map_x, kb * Operand<TIn>::k, x_row, fb);
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
      for (; walk.valid() && ok; walk.next()) {
        const uint32_t idesc = Operand<TIn>::idesc | ((uint32_t)(BM >> 4) << 24) | ((uint32_t)(((min(kRows, end - s0) + 15) & ~15) >> 3) << 17);
        uint32_t d = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (kRounded || kb == kb0) {
            if (!mbar_wait(smem_u32(&tempty_bar[it % kAccs]), ((it / kAccs) & 1) ^ 1, abort_flag, 2)) { ok = false; break; }
            tcgen05_fence_after();
            d = tmem_base + (it % kAccs) * kRows;
          }
          if (!mbar_wait(smem_u32(&full_bar[s]), ph, abort_flag, 3)) { ok = false; break; }
          tcgen05_fence_after();
          const uint32_t sa = smem_u32(smem + s * kStageBytes);
          const uint64_t adesc = make_smem_desc(sa), bdesc = make_smem_desc(sa + BM * 128);
#pragma unroll
          for (int k = 0; k < 4; ++k) mma_one<TIn>(d, adesc + 2 * k, bdesc + 2 * k, idesc, ((!kRounded && kb > kb0) || k > 0) ? 1u : 0u);
          tcgen05_commit(smem_u32(&empty_bar[s]));
          if (kRounded || kb + 1 == kb1) {
            tcgen05_commit(smem_u32(&tfull_bar[it % kAccs]));
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
      for (; walk.valid() && ok; walk.next(), done += kb1 - kb0) {
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
  const TOut* res = static_cast<const TOut*>(p.res);
  TOut* C = static_cast<TOut*>(p.C);
  const bool scaled = p.weights != nullptr || p.alpha != 1.f;
  int rows = 0, n = 0;
  bool met = false;  // this thread has waited for the cluster's start
  float bias = 0.f, sw = 1.f, sx = 1.f, weight = p.alpha;  // of this thread's column, of the warp's slot `lane`
  SlotRows r = {-1, -1, 0};
  // Scales, activation and residual of kN slots of this warp's, the first `j0`, and their rows written; by all lanes.
  auto finish = [&](auto sum_of, int j0, int count, auto kN) {
    float v[kN.value], x[kN.value];
    int c[kN.value];
#pragma unroll
    for (int j = 0; j < kN.value; ++j) {
      c[j] = __shfl_sync(0xffffffffu, r.c, j0 + j);
      v[j] = scaled_sum<TIn>(sum_of(j), sizeof(TIn) == 1 ? __shfl_sync(0xffffffffu, sx, j0 + j) : 1.f, sw, bias);
      if (n >= p.N) v[j] = 0.f;
      x[j] = res && j < count && c[j] >= 0 && n < p.N ? to_f(res[c[j] * p.ldres + n]) : 0.f;
    }
    activate_lanes<TOut>(v, p.act);
#pragma unroll
    for (int j = 0; j < kN.value; ++j) {
      if (scaled) v[j] *= __shfl_sync(0xffffffffu, weight, j0 + j);
      if (j < count && c[j] >= 0 && n < p.N) C[c[j] * p.ldc + n] = one_of<TOut>(res ? v[j] + x[j] : v[j]);
    }
  };
  if (warp >= 4) {
    uint32_t it = 0;
    for (; walk.valid(); walk.next()) {
      rows = min(kRows, end - s0);
      n = n0 + column;
      // ks > 1: the slots that this CTA finishes; else all 64
      const int slot = s0 + (ks > 1 ? (int)rank * slots_each(rows, log_ks) + lane : half * 32 + lane);
      bias = n < p.N && p.bias ? p.bias[(long long)walk.e * p.N + n] : 0.f;
      if (sizeof(TIn) == 1) sw = n < p.N ? p.w_scales[(long long)walk.e * p.N + n] : 0.f;
      r = {-1, -1, 0};
      sx = 1.f;
      weight = p.alpha;
      if (slot < end) r = rows_of_slot(p, slot);
      if (n0 == 0 && quarter == 0) keep_place(p, r, slot);
      if (r.c >= 0) {
        if (sizeof(TIn) == 1) sx = p.x_scales[r.x];
        if (p.weights) weight *= p.weights[r.choice];
      }
      const bool mine = half * 32 < rows;  // the same in the whole warp
      uint32_t sum[32];
      bool ok = true;
      for (int kb = kb0; kb < kb1; kb = kRounded ? kb + 1 : kb1, ++it) {
        ok = mbar_wait_warp(smem_u32(&tfull_bar[it % kAccs]), (it / kAccs) & 1, abort_flag, 4);
        if (!ok) break;
        tcgen05_fence_after();
        if (mine) {
          uint32_t a[32];
          tmem_ld32(tmem_base + ((uint32_t)(quarter * 32) << 16) + (it % kAccs) * kRows + half * 32, a);
          tmem_ld_wait();
          tcgen05_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&tempty_bar[it % kAccs]));
#pragma unroll
          for (int j = 0; j < 32; ++j) sum[j] = kRounded && kb > kb0 ? plus<TIn>(sum[j], a[j]) : a[j];
        } else if (lane == 0) {
          mbar_arrive(smem_u32(&tempty_bar[it % kAccs]));
        }
      }
      if (!ok) break;
      if (ks > 1) {  // (one tile)
        cluster_wait();
        met = true;
        const int each = slots_each(rows, log_ks);
        int k = 0, k0 = 0;  // the CTA whose slots they are, its first
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          const int m = half * 32 + j;
          if (m >= rows) break;
          for (; m >= k0 + each; ++k) k0 += each;
          st_cluster4(smem_u32(part + (((int)rank * each + m - k0) * 128 + column * 4)), k, sum[j], sum[j + 1], sum[j + 2], sum[j + 3]);
        }
        break;
      }
      if (!mine) continue;
      const int count = min(rows - half * 32, 32);
#pragma unroll 1
      for (int j0 = 0; j0 < count; j0 += 8) {  // one copy of the code, whose fetching took longer than its running
        finish([&](int j) { return sum[j]; }, j0, count - j0, std::integral_constant<int, 8>());
#pragma unroll
        for (int j = 0; j < 24; ++j) sum[j] = sum[j + 8];
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
  if (!met) cluster_wait();
  cluster_sync_all();  // all sums have arrived
  if (warp >= 4 && rows > 0) {
    const int each = slots_each(rows, log_ks), count = min(each, rows - (int)rank * each);
    for (int j0 = half * 4; j0 < count; j0 += 8) {  // four slots of a warp at a time
      const uint4* from = reinterpret_cast<const uint4*>(part) + j0 * 32 + column;
      uint4 four = *from;
      for (int k = 1; k < ks; ++k) {
        const uint4 more = from[k * 32 * each];
        four = make_uint4(plus<TIn>(four.x, more.x), plus<TIn>(four.y, more.y), plus<TIn>(four.z, more.z), plus<TIn>(four.w, more.w));
      }
      finish([&](int j) { return j == 0 ? four.x : j == 1 ? four.y : j == 2 ? four.z : four.w; }, j0, count - j0, std::integral_constant<int, 4>());
    }
  }
}

template <typename TIn, typename TOut, bool kGather, bool kRounded>
cudaError_t launch_rows(const GroupedParams& p, int sm_count, cudaStream_t s) {
  CUtensorMap mx, mw;
  cudaError_t e = tma_encode_rows(p.X, p.ldx, kGather || p.x_by_blocks ? p.x_rows : p.slots, p.K, kGather ? 1 : kRows, Operand<TIn>::prec, &mx);
  if (e == cudaSuccess) e = tma_encode_rows(p.W, p.ldw, (long long)p.experts * p.N, p.K, BM, Operand<TIn>::prec, &mw);
  if (e == cudaSuccess) e = raise_smem_limit<grouped_rows_kernel<TIn, TOut, kGather, kRounded>>(smem_bytes(kMaxStages, false) > smem_bytes(kMaxSplitStages, true) ? smem_bytes(kMaxStages, false) : smem_bytes(kMaxSplitStages, true));
  if (e != cudaSuccess) return e;
  const int n_tiles = ceil_div(p.N, BM), k_blocks = ceil_div(p.K, Operand<TIn>::k);
  const int used = p.experts < p.slots ? p.experts : p.slots;
  const long long full = ((long long)p.slots + kRows - 1) / kRows, most = full + used - 1;  // row tiles: all full, and as many as there can be
  // A tile is cut over as many CTAs as leave each of them an SM of its own, going by one row tile per expert, or what the slots fill.  Clusters
  // of eight do not all find eight free SMs of a GPC: sixteen of them took two turns (128x1024x1024 int8 11.8 us, by four CTAs 5.3), so fifteen at
  // most; of four, 32 at most (64 rows, K 1024, us by four CTAs / by two: 32 tiles 6.3, 33 tiles 6.4 / 7.5, 34 tiles 11.6 / 7.5).
  const long long expected = (full > used ? full : used) * n_tiles;
  int ks = 1;
  while (ks < 8 && expected * ks * 2 <= (ks == 4 ? 120 : ks == 2 ? 128 : sm_count) && 2 * ks <= k_blocks) ks *= 2;
  const long long tiles = most * n_tiles;
  const int per_cta = ceil_div(k_blocks, ks), room = ks > 1 ? kMaxSplitStages : kMaxStages;
  const int stages = per_cta < room && ks > 1 ? (per_cta < 2 ? 2 : per_cta) : room;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(ks > 1 ? tiles * ks : tiles < sm_count ? tiles : sm_count));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem_bytes(stages, ks > 1);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ks;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ks > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, grouped_rows_kernel<TIn, TOut, kGather, kRounded>, mx, mw, p, stages, ks == 8 ? 3 : ks / 2);
}

}  // namespace

template <typename TIn, typename TOut>
cudaError_t launch_grouped_rows(const GroupedParams& p, bool in_order, bool rounded, int sm_count, cudaStream_t s) {
  const bool gather = !in_order;
  if constexpr (sizeof(TIn) == 2 && sizeof(TOut) == 4) {
    if (rounded) return gather ? launch_rows<TIn, TOut, true, true>(p, sm_count, s) : launch_rows<TIn, TOut, false, true>(p, sm_count, s);
  }
  return gather ? launch_rows<TIn, TOut, true, false>(p, sm_count, s) : launch_rows<TIn, TOut, false, false>(p, sm_count, s);
}
#define INSTANCE(TIn, TOut) template cudaError_t launch_grouped_rows<TIn, TOut>(const GroupedParams&, bool, bool, int, cudaStream_t)
INSTANCE(__half, __half);
INSTANCE(__half, float);
INSTANCE(__nv_bfloat16, __nv_bfloat16);
INSTANCE(__nv_bfloat16, float);
INSTANCE(int8_t, __half);
INSTANCE(int8_t, __nv_bfloat16);
INSTANCE(int8_t, float);

}  // namespace b200
