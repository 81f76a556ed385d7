// Host launchers of the norms around a block (no counterpart in the reference):
//   u = rmsnorm(T) * PW,  H = alpha * X + G u,  Y = rmsnorm(H) * W      with r1, r2 the two rows' 1 / rms.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

namespace fo {

constexpr int kMaxNormBlockRows = INT32_MAX - 3;  // the number of a row that is loaded three ahead stays an int

// One call's operands: 16-bit row-major [rows, dim], weights [dim], gate [lines, dim] (lines consecutive groups of
// rows / lines rows share a line; nullptr: no gate), stats [rows][2] fp32 = (r1, r2).
struct NormBlock {
  const void *X, *T, *PW, *W, *G;
  int rows, dim, lines;
  float alpha, eps;
  bool bf16;
};

// stats may be nullptr.
cudaError_t norm_block_launch(const NormBlock& p, void* H, void* Y, float* stats, int sm_count, cudaStream_t stream);

// The backward pass: the CTAs that share the rows, or the clusters where a row takes one, and the scratch for their sums.
struct NormBlockPlan {
  int at_once;
  size_t workspace;  // floats
};
NormBlockPlan norm_block_plan(const NormBlock& p, int sm_count);

// GH, GY: gradients of H and Y (either may be nullptr: zero).  DX, DT [rows, dim], DPW, DW [dim], DG like G
// (ignored without a gate).  `workspace`: plan.workspace floats.
cudaError_t norm_block_backward_launch(const NormBlock& p, const float* stats, const void* GH, const void* GY, void* DX,
                                       void* DT, void* DPW, void* DW, void* DG, float* workspace,
                                       const NormBlockPlan& plan, cudaStream_t stream);

}  // namespace fo
