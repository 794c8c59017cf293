// Grouped and 8-bit products of many rows: CTA pairs (tcgen05, cta_group::2) over 256 slots x 256 columns.
//
// A persistent grid of pairs walks the tiles of all experts (256 slots of one expert each; how many an expert has is read on the device).  Per
// k-block of 128 bytes each CTA fetches its 128 rows of X and half of the tile's rows of W:
//   warp 0      TMA producer of W, and of X where its rows lie in order
//   warps 2, 3  gather4 of X's rows that the order names, 64 rows each
//   warp 1      tcgen05.mma issuer (even CTA), kind::f16 or kind::i8, two accumulators in tensor memory
//   warps 4-11  epilogue: two groups of four warps, 128 bytes of each of a warp's 32 rows at a time: tensor memory -> scales, bias, activation,
//               weight, residual -> the warp's own staging buffer -> whole 128-byte pieces of the rows.  Rows behind the expert's last are not
//               stored, which a TMA store of the tile could not leave out.
// Every wait is bounded by wall-clock time like those of gemm_tc.cu.
#include "chunk8.cuh"
#include "grouped_tc.cuh"

namespace b200 {
namespace {

template <typename T>
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (sizeof(T) == 1) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  } else {
    tcgen05_mma_f16_pair(d, a, b, idesc, accumulate);
  }
}
// Four rows of a matrix, 128 bytes of each, one below the other; counted on a barrier of either CTA of the pair.
__device__ __forceinline__ void tma_gather4_pair(uint32_t dst, const CUtensorMap* map, int x, const int4 row, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(row.x), "r"(row.y), "r"(row.z), "r"(row.w), "r"(bar)
      : "memory");
}

template <int BN> struct GroupedPairCfg {
  static constexpr int kStageBytes = (BM + BN / 2) * 128;
  static constexpr int kStages = BN == 256 ? 5 : 6;
  static constexpr int kThreads = 384;
  static constexpr int kTmemCols = 2 * BN;
  static constexpr int kStagingBytes = 8 * 32 * 128;
  static constexpr int kVecBytes = 8 * 128 * 4;                    // per epilogue warp: bias and scale of 64 columns
  static constexpr int kListBytes = (2 * (B200_MAX_EXPERTS + 1) * 4 + 15) / 16 * 16;  // first tile and first slot of each expert
  static constexpr int kSmemBytes = kStages * kStageBytes + kStagingBytes + kVecBytes + kListBytes + BM * 4 + 256 + 1024;
};

template <typename TIn, typename TOut, int BN, bool kGather>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(GroupedPairCfg<BN>::kThreads, 1)
grouped_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const GroupedParams p, int vec) {
  using Cfg = GroupedPairCfg<BN>;
  constexpr int S = Cfg::kStages;
  constexpr int kCols = 128 / (int)sizeof(TOut);  // columns of a 128-byte piece of an output row
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* staging = smem + S * Cfg::kStageBytes;
  float* vectors = reinterpret_cast<float*>(staging + Cfg::kStagingBytes);
  int* first = reinterpret_cast<int*>(staging + Cfg::kStagingBytes + Cfg::kVecBytes);
  int* begin = first + B200_MAX_EXPERTS + 1;
  int* gathered = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(first) + Cfg::kListBytes);  // [128] rows of X of this CTA's half tile
  uint8_t* bar_mem = reinterpret_cast<uint8_t*>(gathered + BM);
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(bar_mem);  // [S]  waited on by the even CTA only
  uint64_t* empty_bar = full_bar + S;                          // [S]  per CTA
  uint64_t* tfull_bar = empty_bar + S;                         // [2]  per CTA
  uint64_t* tempty_bar = tfull_bar + 2;                        // [2]  even CTA: one arrival per epilogue warp of both CTAs
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty_bar + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* scan = reinterpret_cast<int*>(tmem_slot + 2);  // [8]

  const int warp = warp_index(), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int n_tiles = (p.N + BN - 1) / BN, k_blocks = (p.K + Operand<TIn>::k - 1) / Operand<TIn>::k;

  if (threadIdx.x == 64) {
    tma_prefetch_map(&map_x);
    tma_prefetch_map(&map_w);
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(smem_u32(&full_bar[i]), 1);
      mbar_init(smem_u32(&empty_bar[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&tfull_bar[i]), 1);
      mbar_init(smem_u32(&tempty_bar[i]), 16);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)Cfg::kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  grid_dependency_wait();
  tcgen05_fence_before();
  list_tiles<2 * BM>(p, first, begin, scan);
  cluster_sync_all();  // the peer's barriers are initialised before anything arrives on them
  tcgen05_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  grid_launch_dependents();  // not ahead of the tensor memory: a dependent that took it would hold it while it waits for this kernel
  TileWalk<2 * BM> walk{first, begin, p.experts, n_tiles};
  const int tiles = walk.total();
  int s0, end, n0;

  if (warp == 0) {
    // ---------------- TMA producer (both CTAs): W, and X where its rows lie in order ----------------
    if (elect_one()) {
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int t = pair; t < tiles && ok; t += pairs) {
        walk.at(t, BN, s0, end, n0);
        s0 += (int)rank * BM;
        const int w_row = walk.e * p.N + n0 + (int)rank * (min(BN, (p.N - n0 + 31) & ~31) / 2);
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait(smem_u32(&empty_bar[s]), ph ^ 1, abort_flag, 1)) { ok = false; break; }
          const uint32_t fb_local = smem_u32(&full_bar[s]);
          const uint32_t fb = mapa(fb_local, 0), sa = smem_u32(smem + s * Cfg::kStageBytes);
          if (rank == 0) mbar_expect_tx(fb_local, 2 * Cfg::kStageBytes);
          if constexpr (!kGather) tma_load_2d_pair(sa, &map_x, kb * Operand<TIn>::k, s0, fb);
          tma_load_2d_pair(sa + BM * 128, &map_w, kb * Operand<TIn>::k, w_row, fb);
          if (++s == S) { s = 0; ph ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer (even CTA) ----------------
    if (rank == 0 && elect_one()) {
      int s = 0;
      uint32_t ph = 0, tile_it = 0;
      bool ok = true;
      for (int t = pair; t < tiles && ok; t += pairs, ++tile_it) {
        const int left = p.N - (t % n_tiles) * BN;
        const uint32_t idesc = Operand<TIn>::idesc | ((uint32_t)((2 * BM) >> 4) << 24) | ((uint32_t)(min(BN, (left + 31) & ~31) >> 3) << 17);
        const uint32_t acc = tile_it & 1, aph = (tile_it >> 1) & 1;
        if (!mbar_wait(smem_u32(&tempty_bar[acc]), aph ^ 1, abort_flag, 2)) break;
        tcgen05_fence_after();
        const uint32_t d = tmem_base + acc * BN;
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait(smem_u32(&full_bar[s]), ph, abort_flag, 3)) { ok = false; break; }
          tcgen05_fence_after();
          const uint32_t sa = smem_u32(smem + s * Cfg::kStageBytes);
          const uint64_t adesc = make_smem_desc(sa), bdesc = make_smem_desc(sa + BM * 128);
#pragma unroll
          for (int k = 0; k < 4; ++k) mma_pair<TIn>(d, adesc + 2 * k, bdesc + 2 * k, idesc, (kb > 0 || k > 0) ? 1u : 0u);
          tcgen05_commit_both(smem_u32(&empty_bar[s]));
          if (++s == S) { s = 0; ph ^= 1; }
        }
        if (ok) tcgen05_commit_both(smem_u32(&tfull_bar[acc]));
      }
    }
  } else if (warp < 4) {
    // ---------------- gather (both CTAs): half of the CTA's rows of X each ----------------
    if constexpr (kGather) {
      int* rows = gathered + (warp - 2) * 64;
      uint32_t done = 0;  // k-blocks before this tile's
      bool ok = true;
      for (int t = pair; t < tiles && ok; t += pairs, done += k_blocks) {
        walk.at(t, BN, s0, end, n0);
        s0 += (int)rank * BM + (warp - 2) * 64;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int slot = s0 + 32 * i + lane, x = slot < end ? rows_of_slot(p, slot).x : 0;
          rows[32 * i + lane] = x < 0 ? 0 : x;  // whatever lies there: its results are not stored
        }
        __syncwarp();
        if (elect_one()) {
          int s = (int)(done % S);
          uint32_t ph = (done / S) & 1;
          for (int kb = 0; kb < k_blocks; ++kb) {
            if (!mbar_wait(smem_u32(&empty_bar[s]), ph ^ 1, abort_flag, 5)) { ok = false; break; }
            const uint32_t fb = mapa(smem_u32(&full_bar[s]), 0), sa = smem_u32(smem + s * Cfg::kStageBytes) + (warp - 2) * 64 * 128;
#pragma unroll
            for (int i = 0; i < 16; ++i) tma_gather4_pair(sa + i * 512, &map_x, kb * Operand<TIn>::k, reinterpret_cast<const int4*>(rows)[i], fb);
            if (++s == S) { s = 0; ph ^= 1; }
          }
        }
        ok = __all_sync(0xffffffffu, ok);
      }
    }
  } else {
    // ---------------- epilogue ----------------
    const int quarter = warp & 3, group = (warp - 4) >> 2;
    uint8_t* mine_bytes = staging + (warp - 4) * 4096;
    float* vec_b = vectors + (warp - 4) * 128;
    float* vec_w = vec_b + 64;
    uint32_t tile_it = 0;
    const TOut* res = static_cast<const TOut*>(p.res);
    TOut* C = static_cast<TOut*>(p.C);
    for (int t = pair; t < tiles; t += pairs, ++tile_it) {
      const uint32_t acc = tile_it & 1, aph = (tile_it >> 1) & 1;
      walk.at(t, BN, s0, end, n0);
      const int slot = s0 + (int)rank * BM + quarter * 32 + lane;
      SlotRows r = {-1, -1, 0};
      if (slot < end) r = rows_of_slot(p, slot);
      float sx = 1.f, weight = p.alpha;
      if (r.c >= 0) {
        if (sizeof(TIn) == 1) sx = p.x_scales[r.x];
        if (p.weights) weight *= p.weights[r.choice];
      }
      const bool scaled = p.weights != nullptr || p.alpha != 1.f;
      const bool any = __any_sync(0xffffffffu, r.c >= 0);
      const long long wb = (long long)walk.e * p.N;
      float b0, b1, w0 = 1.f, w1 = 1.f;  // bias and scale of columns lane and 32 + lane of a slab, fetched one slab ahead
      auto fetch = [&](int c0) {
        const int a = n0 + c0 + lane, b = a + 32;
        b0 = p.bias && a < p.N ? __ldg(p.bias + wb + a) : 0.f;
        b1 = p.bias && b < p.N ? __ldg(p.bias + wb + b) : 0.f;
        if (sizeof(TIn) == 1) {
          w0 = a < p.N ? __ldg(p.w_scales + wb + a) : 0.f;
          w1 = b < p.N ? __ldg(p.w_scales + wb + b) : 0.f;
        }
      };
      fetch(group * 64);
      if (!mbar_wait(smem_u32(&tfull_bar[acc]), aph, abort_flag, 4)) break;
      tcgen05_fence_after();
      const uint32_t trow = tmem_base + ((uint32_t)(quarter * 32) << 16) + acc * BN;
#pragma unroll 1
      for (int c0 = group * 64; c0 < BN && n0 + c0 < p.N && any; c0 += 128) {
        vec_b[lane] = b0;
        vec_b[32 + lane] = b1;
        if (sizeof(TIn) == 1) {
          vec_w[lane] = w0;
          vec_w[32 + lane] = w1;
        }
        __syncwarp();
        if (c0 + 128 < BN) fetch(c0 + 128);
#pragma unroll 1
        for (int half = 0; half < 64; half += kCols) {  // pieces of 128 bytes: one of 64 columns, or two of 32
          const int n = n0 + c0 + half;
          if (n >= p.N) break;
          if (res) {
            if (vec) {
              uint4 piece[8];
#pragma unroll
              for (int it = 0; it < 8; ++it) {
                const int c = __shfl_sync(0xffffffffu, r.c, it * 4 + (lane >> 3)), col = n + (lane & 7) * (kCols / 8);
                piece[it] = make_uint4(0u, 0u, 0u, 0u);
                if (c >= 0 && col < p.N) piece[it] = *reinterpret_cast<const uint4*>(res + c * p.ldres + col);
              }
#pragma unroll
              for (int it = 0; it < 8; ++it) {
                const int rr = it * 4 + (lane >> 3);
                *reinterpret_cast<uint4*>(mine_bytes + rr * 128 + (((lane & 7) ^ (rr & 7)) << 4)) = piece[it];
              }
            } else {
#pragma unroll 1
              for (int rr = 0; rr < 32; ++rr) {
                const int c = __shfl_sync(0xffffffffu, r.c, rr);
                for (int j = lane; j < kCols; j += 32)
                  if (c >= 0 && n + j < p.N)
                    reinterpret_cast<TOut*>(mine_bytes + rr * 128 + (((j / (kCols / 8)) ^ (rr & 7)) << 4))[j % (kCols / 8)] = res[c * p.ldres + n + j];
              }
            }
            __syncwarp();
          }
#pragma unroll
          for (int q = 0; q < kCols; q += 32) {
            uint32_t a[32];
            tmem_ld32(trow + c0 + half + q, a);
            tmem_ld_wait();
            float v[32];
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              const float4 b = *reinterpret_cast<const float4*>(vec_b + half + q + j);
              if constexpr (sizeof(TIn) == 1) {
                const float4 w = *reinterpret_cast<const float4*>(vec_w + half + q + j);
                v[j] = fmaf((float)(int)a[j], sx * w.x, b.x);
                v[j + 1] = fmaf((float)(int)a[j + 1], sx * w.y, b.y);
                v[j + 2] = fmaf((float)(int)a[j + 2], sx * w.z, b.z);
                v[j + 3] = fmaf((float)(int)a[j + 3], sx * w.w, b.w);
              } else {
                v[j] = __uint_as_float(a[j]) + b.x;
                v[j + 1] = __uint_as_float(a[j + 1]) + b.y;
                v[j + 2] = __uint_as_float(a[j + 2]) + b.z;
                v[j + 3] = __uint_as_float(a[j + 3]) + b.w;
              }
            }
            activate32<TOut>(v, p.act);
            if (scaled) {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] *= weight;
            }
            constexpr int kPer = 16 / (int)sizeof(TOut);  // entries of a 16-byte piece
#pragma unroll
            for (int j = 0; j < 32; j += kPer) {
              uint4* at = reinterpret_cast<uint4*>(mine_bytes + lane * 128 + ((((q + j) / kPer) ^ (lane & 7)) << 4));
              uint4 out;
              uint32_t* o = &out.x;
              if (res) {
                const uint4 have = *at;
                const uint32_t* h = &have.x;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  if constexpr (sizeof(TOut) == 2) {
                    const float2 f = pair_f<TOut>(h[i]);
                    v[j + 2 * i] += f.x;
                    v[j + 2 * i + 1] += f.y;
                  } else {
                    v[j + i] += __uint_as_float(h[i]);
                  }
                }
              }
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                if constexpr (sizeof(TOut) == 2) o[i] = two_of<TOut>(v[j + 2 * i], v[j + 2 * i + 1]);
                else o[i] = __float_as_uint(v[j + i]);
              }
              *at = out;
            }
          }
          __syncwarp();
          if (vec) {
#pragma unroll
            for (int it = 0; it < 8; ++it) {
              const int rr = it * 4 + (lane >> 3), c = __shfl_sync(0xffffffffu, r.c, rr), col = n + (lane & 7) * (kCols / 8);
              const uint4 piece = *reinterpret_cast<const uint4*>(mine_bytes + rr * 128 + (((lane & 7) ^ (rr & 7)) << 4));
              if (c >= 0 && col < p.N) *reinterpret_cast<uint4*>(C + c * p.ldc + col) = piece;
            }
          } else {
#pragma unroll 1
            for (int rr = 0; rr < 32; ++rr) {
              const int c = __shfl_sync(0xffffffffu, r.c, rr);
              for (int j = lane; j < kCols; j += 32)
                if (c >= 0 && n + j < p.N)
                  C[c * p.ldc + n + j] = reinterpret_cast<const TOut*>(mine_bytes + rr * 128 + (((j / (kCols / 8)) ^ (rr & 7)) << 4))[j % (kCols / 8)];
            }
          }
          __syncwarp();
        }
      }
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(mapa(smem_u32(&tempty_bar[acc]), 0));
    }
  }

  __syncwarp();
  tcgen05_fence_before();
  __syncthreads();
  if (*abort_flag) {
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
    if (threadIdx.x == 0 && p.status) atomicCAS(p.status, 0, 700 + *abort_flag);
    __syncthreads();
  }
  cluster_sync_all();  // neither CTA releases tensor or shared memory while its peer may still touch it
  if (warp == 1) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)Cfg::kTmemCols) : "memory");
  }
}

template <typename TIn, typename TOut, int BN, bool kGather>
cudaError_t launch_tiles(const GroupedParams& p, int sm_count, cudaStream_t s) {
  using Cfg = GroupedPairCfg<BN>;
  CUtensorMap mx, mw;
  cudaError_t e = tma_encode_rows(p.X, p.ldx, p.x_rows, p.K, kGather ? 1 : BM, Operand<TIn>::prec, &mx);
  if (e == cudaSuccess) e = tma_encode_rows(p.W, p.ldw, (long long)p.experts * p.N, p.K, BN / 2, Operand<TIn>::prec, &mw);
  if (e == cudaSuccess) e = raise_smem_limit<grouped_pair_kernel<TIn, TOut, BN, kGather>>(Cfg::kSmemBytes);
  if (e != cudaSuccess) return e;
  const int per = 16 / (int)sizeof(TOut);
  const int vec = p.N % per == 0 && p.ldc % per == 0 && aligned16(p.C) && (!p.res || (p.ldres % per == 0 && aligned16(p.res)));
  const long long row_tiles = ((long long)p.slots + 2 * BM - 1) / (2 * BM) + (p.experts < p.slots ? p.experts : p.slots) - 1;
  const long long tiles = row_tiles * ceil_div(p.N, BN);
  const int pairs = (int)(tiles < sm_count / 2 ? tiles : sm_count / 2);
  return launch_dependent(grouped_pair_kernel<TIn, TOut, BN, kGather>, dim3(2 * pairs), dim3(Cfg::kThreads), Cfg::kSmemBytes, s, mx, mw, p, vec);
}

}  // namespace

template <typename TIn, typename TOut>
cudaError_t launch_grouped_pair(const GroupedParams& p, int sm_count, cudaStream_t s) {
  const bool gather = p.order && !p.x_by_slot;
  if (p.N <= 128) return gather ? launch_tiles<TIn, TOut, 128, true>(p, sm_count, s) : launch_tiles<TIn, TOut, 128, false>(p, sm_count, s);
  return gather ? launch_tiles<TIn, TOut, 256, true>(p, sm_count, s) : launch_tiles<TIn, TOut, 256, false>(p, sm_count, s);
}
#define INSTANCE(TIn, TOut) template cudaError_t launch_grouped_pair<TIn, TOut>(const GroupedParams&, int, cudaStream_t)
INSTANCE(__half, __half);
INSTANCE(__half, float);
INSTANCE(__nv_bfloat16, __nv_bfloat16);
INSTANCE(__nv_bfloat16, float);
INSTANCE(int8_t, __half);
INSTANCE(int8_t, __nv_bfloat16);
INSTANCE(int8_t, float);

}  // namespace b200
