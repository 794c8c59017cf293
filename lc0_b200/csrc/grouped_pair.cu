// Grouped and 8-bit products of many rows: CTA pairs (tcgen05, cta_group::2) over 256 slots x 256 columns.
//
// A persistent grid of pairs walks the tiles of all experts (256 slots of one expert each; how many an expert has is read on the device).  Per
// k-block of 128 bytes each CTA fetches its 128 rows of X and half of the tile's rows of W:
//   warp 0      TMA producer; requests of whole 64 rows are fetched where they lie, two boxes for one
//   warp 1      tcgen05.mma issuer (even CTA), kind::f16 or kind::i8, two accumulators in tensor memory
//   warps 4-19  epilogue: four groups of four warps, 64 bytes of each of a warp's 32 rows at a time: tensor memory -> scales, bias, activation,
//               weight, residual -> the warp's own staging buffer -> a TMA store where the 32 rows lie in order and are all this expert's, else
//               64-byte pieces of those rows that are.  A TMA store spares it reading the buffer and writing line by line
//               (65536x1536x1024 int8, us: 104 without, 94 with).
// us and what they are of 1.65 PFLOP/s (int8: of twice that), on the device: 32768 slots over 16 experts, 1024x1536 columns by slot 90, 69 %;
// 65536x1536x1024 int8 86 - 88, 71 %; without an epilogue 81 and 62.
// No unit is full: the epilogue is bound by latency, four warps per scheduler that wait for each 16 columns of tensor memory and for their residual
// before they compute.  Counters, % of the tensor pipe, of the issue slots, of shared memory's wavefronts (the epilogue's and the operands'):
// 65536x1024x1536 int8 65, 38, 41 + 33; with a residual 50, 41, 36 + 25; 18000 slots of int8 over 16 experts, 1536x1024, 38, 37, 34 + 20; with
// Mish 29, 41, 25 + 15.
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
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }

template <int BN> struct GroupedPairCfg {
  static constexpr int kStageBytes = (BM + BN / 2) * 128;
  static constexpr int kMaxStages = BN == 256 ? 5 : 6;
  static constexpr int kThreads = 640;
  static constexpr int kTmemCols = 2 * BN;
  static constexpr int kStagingBytes = 16 * 32 * 64;  // per epilogue warp: 64 bytes of its 32 rows
  static constexpr int kVecBytes = 16 * 128 * 4;      // ... and bias and scale of up to 64 columns
  static constexpr int kListBytes = (2 * (B200_MAX_EXPERTS + 1) * 4 + 15) / 16 * 16;  // first tile and first slot of each expert
  // With a residual the epilogue warps have two staging buffers each, which the 32 KB of a pipeline stage make room for.
  static constexpr int stages(bool res) { return kMaxStages - res; }
  static constexpr int smem_bytes(bool res) {
    return stages(res) * kStageBytes + (1 + res) * kStagingBytes + kVecBytes + kListBytes + 256 + 1024;
  }
};

template <typename TIn, typename TOut, int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(GroupedPairCfg<BN>::kThreads, 1)
grouped_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_c,
                    const GroupedParams p, int vec, int boxes) {
  using Cfg = GroupedPairCfg<BN>;
  const int S = Cfg::kMaxStages - (p.res ? 1 : 0);
  constexpr int kCols = 64 / (int)sizeof(TOut);  // columns of a 64-byte piece of an output row
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* staging = smem + S * Cfg::kStageBytes;
  float* vectors = reinterpret_cast<float*>(staging + (p.res ? 2 : 1) * Cfg::kStagingBytes);
  int* first = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(vectors) + Cfg::kVecBytes);
  int* begin = first + B200_MAX_EXPERTS + 1;
  uint8_t* bar_mem = reinterpret_cast<uint8_t*>(first) + Cfg::kListBytes;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(bar_mem);  // [S]  waited on by the even CTA only
  uint64_t* empty_bar = full_bar + Cfg::kMaxStages;                          // [S]  per CTA
  uint64_t* tfull_bar = empty_bar + Cfg::kMaxStages;                         // [2]  per CTA
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
    if (boxes) tma_prefetch_map(&map_c);
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(smem_u32(&full_bar[i]), 1);
      mbar_init(smem_u32(&empty_bar[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&tfull_bar[i]), 1);
      mbar_init(smem_u32(&tempty_bar[i]), 32);
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
  TileWalk<2 * BM, BN> walk(first, begin, p.experts, n_tiles, pair, pairs, BN == 256 ? pairs : 0);
  // columns that the MMA computes: the tile's, or what is left of N rounded up to 32
  auto columns = [&]() { return max(32, min(walk.width, (p.N - walk.n0 + 31) & ~31)); };

  if (warp == 0) {
    // ---------------- TMA producer (both CTAs): W, and X where its rows lie in order ----------------
    if (elect_one()) {
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (; walk.valid() && ok; walk.next()) {
        const int x0 = walk.s0 + (int)rank * BM;
        const int x_row = p.x_by_blocks ? row_of_block(p, x0, walk.end) : x0, x_next = p.x_by_blocks ? row_of_block(p, x0 + 64, walk.end) : 0;
        const int w_row = walk.e * p.N + walk.n0 + (int)rank * (columns() / 2);
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait(smem_u32(&empty_bar[s]), ph ^ 1, abort_flag, 1)) { ok = false; break; }
          const uint32_t fb_local = smem_u32(&full_bar[s]);
          const uint32_t fb = mapa(fb_local, 0), sa = smem_u32(smem + s * Cfg::kStageBytes);
          if (rank == 0) mbar_expect_tx(fb_local, 2 * Cfg::kStageBytes);
          tma_load_2d_pair(sa, &map_x, kb * Operand<TIn>::k, x_row, fb);
          if (p.x_by_blocks) tma_load_2d_pair(sa + 64 * 128, &map_x, kb * Operand<TIn>::k, x_next, fb);
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
      for (; walk.valid() && ok; walk.next(), ++tile_it) {
        const uint32_t idesc = Operand<TIn>::idesc | ((uint32_t)((2 * BM) >> 4) << 24) | ((uint32_t)(columns() >> 3) << 17);
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
  } else if (warp >= 4) {
    // ---------------- epilogue ----------------
    // Four groups of four warps, a quarter of the columns each, in pieces of 64 bytes of each of the warp's rows.  The residual of the piece
    // after this one is copied to the warp's other staging buffer meanwhile (65536x1024x1536 int8, us: 151 with loads at the start of each
    // piece, 97 ahead of it; 80 without a residual).  Eight
    // warps with pieces of 128 bytes had too little to do while they waited: 18000 slots of int8 with Mish 71, now 58; without an activation 102, 105.
    constexpr int kSlab = BN / 4, kPieces = kSlab / kCols, kPer = 16 / (int)sizeof(TOut);  // kPer: entries of 16 bytes
    const int quarter = warp & 3, group = (warp - 4) >> 2, sub = lane >> 2, part = lane & 3;
    const TOut* res = static_cast<const TOut*>(p.res);
    TOut* C = static_cast<TOut*>(p.C);
    uint8_t* buffers = staging + (warp - 4) * 2048 * (res ? 2 : 1);
    float* vec_b = vectors + (warp - 4) * 128;
    float* vec_w = vec_b + 64;
    const bool scaled = p.weights != nullptr || p.alpha != 1.f;
    auto at = [&](uint8_t* buffer, int row, int q) { return buffer + row * 64 + ((q ^ ((row >> 1) & 3)) << 4); };  // 16 bytes, swizzled
    // Rows that are no whole 16 bytes but whole words leave by two rows of 16 words at a time (16384x1858x512 int8, fp16
    // results, us: 70 entry by entry, 45; with a residual, copied ahead like the others, 231, 67; fp32 124, 61).
    constexpr int kWord = 4 / (int)sizeof(TOut);
    auto word_at = [&](uint8_t* buffer, int row) { return reinterpret_cast<uint32_t*>(at(buffer, row, (lane & 15) >> 2) + (lane & 3) * 4); };
    auto copy_res = [&](uint8_t* buffer, int c_row, int n) {  // the residual's piece that begins at column n
      if (vec == 2) {
#pragma unroll
        for (int it = 0; it < 4; ++it) {
          const int c = __shfl_sync(0xffffffffu, c_row, it * 8 + sub), col = n + part * kPer;
          if (c >= 0 && col < p.N) cp_async16(smem_u32(at(buffer, it * 8 + sub, part)), res + c * p.ldres + col);
        }
      } else {
#pragma unroll 4
        for (int rr = lane >> 4; rr < 32; rr += 2) {
          const int c = __shfl_sync(0xffffffffu, c_row, rr), col = n + (lane & 15) * kWord;
          if (c >= 0 && col < p.N) cp_async4(smem_u32(word_at(buffer, rr)), res + c * p.ldres + col);
        }
      }
    };
    float b0 = 0.f, b1 = 0.f, w0 = 1.f, w1 = 1.f;  // bias and scale of columns lane and 32 + lane of the next tile's slab
    auto fetch_vectors = [&](int wb, int n) {
      const bool first = n + lane < p.N, second = kSlab > 32 && n + 32 + lane < p.N;
      b0 = p.bias && first ? p.bias[wb + n + lane] : 0.f;
      b1 = p.bias && second ? p.bias[wb + n + 32 + lane] : 0.f;
      if (sizeof(TIn) == 1) {
        w0 = first ? p.w_scales[wb + n + lane] : 0.f;
        w1 = second ? p.w_scales[wb + n + 32 + lane] : 0.f;
      }
    };
    struct Tile {
      SlotRows r;
      float sx, weight;
      int n;     // the first column of the group's slab
      int row0;  // the first of the warp's slots
      int wb;    // where the expert's vectors begin
    };
    auto tile_at_hand = [&]() {
      Tile x = {{-1, -1, 0}, 1.f, p.alpha, p.N, 0, 0};
      if (!walk.valid()) return x;
      const int slot = walk.s0 + (int)rank * BM + quarter * 32 + lane;
      if (slot < walk.end) x.r = rows_of_slot(p, slot);
      if (walk.n0 == 0 && group == 0) keep_place(p, x.r, slot);
      if (x.r.c >= 0) {
        if (sizeof(TIn) == 1) x.sx = p.x_scales[x.r.x];
        if (p.weights) x.weight *= p.weights[x.r.choice];
      }
      x.n = group * kSlab < walk.width ? walk.n0 + group * kSlab : p.N;  // (half a tile is two groups')
      x.row0 = slot - lane;
      x.wb = walk.e * p.N;
      return x;
    };
    uint32_t tile_it = 0;
    int buf = 0;
    bool copied = false;  // the residual of the next piece is in, or on its way to, its buffer
    bool more = walk.valid();
    Tile next = tile_at_hand();
    fetch_vectors(next.wb, next.n);
    for (; more; ++tile_it) {
      const uint32_t acc = tile_it & 1, aph = (tile_it >> 1) & 1;
      const Tile x = next;
      const bool any = __any_sync(0xffffffffu, x.r.c >= 0) && x.n < p.N;
      const bool box = boxes && __all_sync(0xffffffffu, x.r.c >= 0);  // the warp's rows are 32 in order, all of them this expert's
      vec_b[lane] = b0;
      vec_b[32 + lane] = b1;
      if (sizeof(TIn) == 1) {
        vec_w[lane] = w0;
        vec_w[32 + lane] = w1;
      }
      walk.next();
      more = walk.valid();
      next = tile_at_hand();
      fetch_vectors(next.wb, next.n);
      const bool any_next = __any_sync(0xffffffffu, next.r.c >= 0) && next.n < p.N;
      if (res && vec && any && !copied) {
        copy_res(buffers + buf * 2048, x.r.c, x.n);
        cp_async_commit();
      }
      copied = false;
      if (!mbar_wait_warp(smem_u32(&tfull_bar[acc]), aph, abort_flag, 4)) break;
      tcgen05_fence_after();
      const uint32_t trow = tmem_base + ((uint32_t)(quarter * 32) << 16) + acc * BN + group * kSlab;
#pragma unroll 1
      for (int i = 0; i < kPieces && any; ++i) {
        const int n = x.n + i * kCols;
        if (n >= p.N) break;
        uint8_t* buffer = buffers + buf * 2048;
        if (res) {
          if (vec) {
            uint8_t* other = buffers + (buf ^ 1) * 2048;
            if (lane == 0) tma_store_wait_read0();  // (of the piece before this one)
            __syncwarp();
            const bool here = i + 1 < kPieces && n + kCols < p.N;
            if (here) copy_res(other, x.r.c, n + kCols);
            else if (any_next) copy_res(other, next.r.c, next.n), copied = true;
            cp_async_commit();
            cp_async_wait<1>();
            buf ^= 1;
          } else {
#pragma unroll 1
            for (int rr = 0; rr < 32; ++rr) {
              const int c = __shfl_sync(0xffffffffu, x.r.c, rr);
              if (c >= 0 && lane < kCols && n + lane < p.N) reinterpret_cast<TOut*>(at(buffer, rr, lane / kPer))[lane % kPer] = res[c * p.ldres + n + lane];
            }
          }
        }
        __syncwarp();
#pragma unroll
        for (int q = 0; q < kCols; q += 16) {
          uint32_t a[16];
          tmem_ld16(trow + i * kCols + q, a);
          tmem_ld_wait();
          float v[16];
#pragma unroll
          for (int j = 0; j < 16; j += 4) {
            const float4 b = *reinterpret_cast<const float4*>(vec_b + i * kCols + q + j);
            if constexpr (sizeof(TIn) == 1) {
              const float4 w = *reinterpret_cast<const float4*>(vec_w + i * kCols + q + j);
              v[j] = fmaf((float)(int)a[j], x.sx * w.x, b.x);
              v[j + 1] = fmaf((float)(int)a[j + 1], x.sx * w.y, b.y);
              v[j + 2] = fmaf((float)(int)a[j + 2], x.sx * w.z, b.z);
              v[j + 3] = fmaf((float)(int)a[j + 3], x.sx * w.w, b.w);
            } else {
              v[j] = __uint_as_float(a[j]) + b.x;
              v[j + 1] = __uint_as_float(a[j + 1]) + b.y;
              v[j + 2] = __uint_as_float(a[j + 2]) + b.z;
              v[j + 3] = __uint_as_float(a[j + 3]) + b.w;
            }
          }
          if ((p.N & 3) != 0 && n + q + 16 > p.N) {  // (each branch here is one: as predicated instructions they cost what they do either way)
            asm volatile("");
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if (n + q + j >= p.N) v[j] = 0.f;
          }
          if (p.act != ACT_NONE) {
            asm volatile("");
            activate_columns<TOut>(v, p.act);
          }
          if (scaled) {
            asm volatile("");
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] *= x.weight;
          }
          if (res) {
            asm volatile("");
#pragma unroll
            for (int j = 0; j < 16; j += kPer) {
              const uint4 have = *reinterpret_cast<const uint4*>(at(buffer, lane, (q + j) / kPer));
              const uint32_t* h = &have.x;
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                if constexpr (sizeof(TOut) == 2) {
                  const float2 f = pair_f<TOut>(h[k]);
                  v[j + 2 * k] += f.x;
                  v[j + 2 * k + 1] += f.y;
                } else {
                  v[j + k] += __uint_as_float(h[k]);
                }
              }
            }
          } else if (q == 0) {
            if (lane == 0) tma_store_wait_read0();  // the piece before this one has left the buffer
            __syncwarp();
          }
#pragma unroll
          for (int j = 0; j < 16; j += kPer) {
            uint4 out;
            uint32_t* o = &out.x;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if constexpr (sizeof(TOut) == 2) o[k] = two_of<TOut>(v[j + 2 * k], v[j + 2 * k + 1]);
              else o[k] = __float_as_uint(v[j + k]);
            }
            *reinterpret_cast<uint4*>(at(buffer, lane, (q + j) / kPer)) = out;
          }
        }
        if (box) fence_async_smem();
        __syncwarp();
        if (box) {
          if (lane == 0) {
            tma_store_2d(&map_c, n, x.row0, smem_u32(buffer));
            tma_store_commit();
          }
        } else if (vec == 2) {
#pragma unroll
          for (int it = 0; it < 4; ++it) {
            const int c = __shfl_sync(0xffffffffu, x.r.c, it * 8 + sub), col = n + part * kPer;
            const uint4 out = *reinterpret_cast<const uint4*>(at(buffer, it * 8 + sub, part));
            if (c >= 0 && col < p.N) *reinterpret_cast<uint4*>(C + c * p.ldc + col) = out;
          }
        } else if (vec == 1) {
#pragma unroll 8
          for (int rr = lane >> 4; rr < 32; rr += 2) {
            const int c = __shfl_sync(0xffffffffu, x.r.c, rr), col = n + (lane & 15) * kWord;
            if (c >= 0 && col < p.N) *reinterpret_cast<uint32_t*>(C + c * p.ldc + col) = *word_at(buffer, rr);
          }
        } else {
#pragma unroll 1
          for (int rr = 0; rr < 32; ++rr) {
            const int c = __shfl_sync(0xffffffffu, x.r.c, rr);
            if (c >= 0 && lane < kCols && n + lane < p.N) C[c * p.ldc + n + lane] = reinterpret_cast<const TOut*>(at(buffer, rr, lane / kPer))[lane % kPer];
          }
        }
        __syncwarp();
      }
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(mapa(smem_u32(&tempty_bar[acc]), 0));
    }
    cp_async_wait<0>();
    if (lane == 0) tma_store_wait_all0();
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

template <typename TIn, typename TOut, int BN>
cudaError_t launch_tiles(const GroupedParams& p, int sm_count, cudaStream_t s) {
  using Cfg = GroupedPairCfg<BN>;
  CUtensorMap mx, mw, mc = {};
  constexpr int kMostBytes = Cfg::smem_bytes(false) > Cfg::smem_bytes(true) ? Cfg::smem_bytes(false) : Cfg::smem_bytes(true);
  cudaError_t e = tma_encode_rows(p.X, p.ldx, p.x_by_blocks ? p.x_rows : p.slots, p.K, p.x_by_blocks ? 64 : BM, Operand<TIn>::prec, &mx);
  if (e == cudaSuccess) e = tma_encode_rows(p.W, p.ldw, (long long)p.experts * p.N, p.K, BN / 2, Operand<TIn>::prec, &mw);
  if (e == cudaSuccess) e = raise_smem_limit<grouped_pair_kernel<TIn, TOut, BN>>(kMostBytes);
  if (e != cudaSuccess) return e;
  const int per = 16 / (int)sizeof(TOut);
  // pieces that rows of C and res can be read and written in: 2: 16 bytes, 1: words, 0: entries
  auto pieces_of = [&](int n, uintptr_t bytes) {
    return p.N % n == 0 && p.ldc % n == 0 && reinterpret_cast<uintptr_t>(p.C) % bytes == 0 &&
           (!p.res || (p.ldres % n == 0 && reinterpret_cast<uintptr_t>(p.res) % bytes == 0));
  };
  const int vec = pieces_of(per, 16) ? 2 : pieces_of(per / 4, 4) ? 1 : 0;
  const int boxes = vec == 2 && (!p.order || p.c_by_slot);  // rows of C in the order of the slots
  if (boxes && (e = tma_encode_out(p.C, p.ldc, p.slots, p.N, TypeTag<TOut>::prec, &mc)) != cudaSuccess) return e;
  const long long row_tiles = ((long long)p.slots + 2 * BM - 1) / (2 * BM) + (p.experts < p.slots ? p.experts : p.slots) - 1;
  const long long tiles = row_tiles * ceil_div(p.N, BN);
  const int pairs = (int)(tiles < sm_count / 2 ? tiles : sm_count / 2);
  return launch_dependent(grouped_pair_kernel<TIn, TOut, BN>, dim3(2 * pairs), dim3(Cfg::kThreads), Cfg::smem_bytes(p.res != nullptr), s, mx, mw, mc, p, vec, boxes);
}

}  // namespace

template <typename TIn, typename TOut>
cudaError_t launch_grouped_pair(const GroupedParams& p, int sm_count, cudaStream_t s) {
  // Narrow tiles where whole ones leave half of the pairs without any (2048x1024x1024 int8, us: 9.6 with wide ones, 7.5).
  const long long row_tiles = ((long long)p.slots + 2 * BM - 1) / (2 * BM) + ((p.experts < p.slots ? p.experts : p.slots) - 1) / 2;
  return p.N <= 128 || 4 * row_tiles * ceil_div(p.N, 256) <= sm_count ? launch_tiles<TIn, TOut, 128>(p, sm_count, s) : launch_tiles<TIn, TOut, 256>(p, sm_count, s);
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
