// The transfer rule of a denoise step (fastdllm_engine.py:2146-2157 of the reference engine), by one wave for one block of the
// batch: over the positions that still hold the mask token, the most confident one (lowest index on ties) always, the others
// when their confidence reaches the threshold.
#pragma once

#include "pdllm_common.h"

namespace pdllm {

__device__ __forceinline__ void unmask_block(const float* conf, const long* token, long* block_ids, long b, long block_len,
                                             long mask_token_id, float threshold, uint8_t* transfer, int* n_left) {
  const int lane = threadIdx.x & 63;
  const long base = b * block_len;
  // pass 1: most confident masked position (lowest index on ties)
  float best = -INFINITY;
  long besti = 0x7fffffffffffffffL;
  int n_masked = 0;
  for (long i = lane; i < block_len; i += 64) {
    if (block_ids[base + i] == mask_token_id) {
      ++n_masked;
      const float c = conf[base + i];
      if (c > best || besti == 0x7fffffffffffffffL) { best = c; besti = i; }
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float ob = __shfl_xor(best, o, 64);
    const long oi = __shfl_xor(besti, o, 64);
    n_masked += __shfl_xor(n_masked, o, 64);
    const bool o_valid = oi != 0x7fffffffffffffffL, s_valid = besti != 0x7fffffffffffffffL;
    const bool take = o_valid && (!s_valid || ob > best || (ob == best && oi < besti));
    if (take) { best = ob; besti = oi; }
  }
  int moved = 0;
  for (long i = lane; i < block_len; i += 64) {
    const bool masked = block_ids[base + i] == mask_token_id;
    const bool t = masked && (i == besti || conf[base + i] >= threshold);
    transfer[base + i] = t ? 1 : 0;
    if (t) { block_ids[base + i] = token[base + i]; ++moved; }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) moved += __shfl_xor(moved, o, 64);
  if (lane == 0 && n_left) n_left[b] = n_masked - moved;
}

}  // namespace pdllm
