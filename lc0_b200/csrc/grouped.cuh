// Products grouped by expert, and those of 8-bit integers, which have one group: what their kernels share.
#pragma once
#include "kernels.cuh"

namespace b200 {

// v[slot][n] = act(scales * (X[x_row(slot)] . W[e]^T) + bias[e][n]) with the slot's expert e; see b200_op_gemm_experts and b200_op_gemm_int8.
// The output is alpha * weight * v + res, stored by token or by slot.  Where a token's choices are summed they are stored by slot in fp32, and
// `place` learns the slot of each choice for combine_kernel.
struct GroupedParams {
  const void* X; long long ldx; int x_rows;
  const void* W; long long ldw;
  const float* bias; const float* x_scales; const float* w_scales;
  void* C; long long ldc;
  const void* res; long long ldres;
  float alpha;
  const float* weights;
  const int* order; const int* offsets;  // null: one group, all slots in order
  int slots;                             // rows of choices there may be (M * top_k)
  int N, K, experts, top_k, group, act;
  int x_by_slot, c_by_slot;
  int x_by_blocks;  // tensor-core kernels: X in the tokens' order, requests of whole 64 rows, which are fetched where they lie
  int* place;  // [choices] or nullptr
  int* status;
};

// The rows of a slot.  x: of X; c: of C (and res); choice: in `weights`.  c < 0: no row.
struct SlotRows {
  int x, c, choice;
};
__device__ __forceinline__ SlotRows rows_of_slot(const GroupedParams& p, int slot) {
  SlotRows r;
  if (!p.order) {
    r.x = r.c = slot;
    r.choice = 0;
    return r;
  }
  const int s = p.group == 1 ? slot : slot / p.group, i = p.group == 1 ? 0 : slot - s * p.group;
  const int choice = p.order[s];
  if (choice < 0 || choice >= p.slots / p.group) return {-1, -1, 0};
  const int token = (p.top_k == 1 ? choice : choice / p.top_k) * p.group + i;
  r.x = p.x_by_slot ? slot : token;
  r.c = p.c_by_slot ? slot : token;
  r.choice = choice;
  return r;
}
// Kept by whichever thread has the slot's rows in hand for the first column.
__device__ __forceinline__ void keep_place(const GroupedParams& p, const SlotRows& r, int slot) {
  if (p.place && r.c >= 0) p.place[r.choice] = slot / p.group;
}
// The first row of X of the 64 slots from `slot` on, a multiple of 64 behind the expert's first (x_by_blocks).
__device__ __forceinline__ int row_of_block(const GroupedParams& p, int slot, int end) {
  const int x = slot < end ? rows_of_slot(p, slot).x : 0;
  return x < 0 ? 0 : x;  // whatever lies there: its results are not stored
}
// offsets[e] in slots, held within what there is.  (An entry below one ahead of it counts as that one; it is the callers that see to it.)
__device__ __forceinline__ int expert_begin(const GroupedParams& p, int e) {
  if (!p.offsets) return e == 0 ? 0 : p.slots;
  const int most = p.slots / p.group, at = p.offsets[e];
  return (at < 0 ? 0 : at < most ? at : most) * p.group;
}

// Many rows (grouped_pair.cu): operands that TMA can read, X [slots][K] in the order of the slots, or x_by_blocks.
template <typename TIn, typename TOut> cudaError_t launch_grouped_pair(const GroupedParams& p, int sm_count, cudaStream_t s);

// Few rows per expert (grouped_rows.cu): operands that TMA can read.  in_order: X is [slots][K] in the order of the slots, or x_by_blocks.  rounded: fp32 results of 16-bit operands as exact as a plain fp32 product.
template <typename TIn, typename TOut> cudaError_t launch_grouped_rows(const GroupedParams& p, bool in_order, bool rounded, int sm_count, cudaStream_t s);

}  // namespace b200
