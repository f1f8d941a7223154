// Tensor-core attention -- host interface (attn_tc.cu).
#pragma once
#include "attnops_dev.cuh"

namespace cw {

// Query rows of one tile, slots of one tile, most CTAs of a tree call.
constexpr int TC_ROWS = 128, TC_KEYS = 128, TC_CTAS = 148;

cudaError_t tc_configure();
cudaError_t tc_prompt(const AttnOp &a, int type, int hd, cudaStream_t st);
cudaError_t tc_tree(const AttnOp &a, int type, int hd, cudaStream_t st);

}  // namespace cw
