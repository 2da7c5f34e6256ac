// The transfer rule of a denoise step (fastdllm_engine.py:2146-2157 of the reference engine), by one wave for one block of the
// batch: over the positions that still hold the mask token, the most confident one (lowest index on ties) always, the others
// when their confidence reaches the threshold.  A NaN counts as more confident than every number, as in the reference's
// torch.topk, and reaches no threshold.
#pragma once

#include "pdllm_common.h"

namespace pdllm {

// The most confident masked position so far.  Positions are ordered by (key, lowest index): a total order, so that all lanes
// arrive at the same one whatever the confidences are.
struct BestMasked {
  int key = -0x7fffffff - 1;  // below the key of every confidence: no masked position
  long idx = 0x7fffffffffffffffL;
  int n_masked = 0;
};

// order-preserving integer image of a confidence: NaN on top, -0 as 0
__device__ __forceinline__ int conf_key(float c) {
  if (c != c) return 0x7fffffff;
  const int b = __float_as_int(c + 0.f);
  return b ^ ((b >> 31) & 0x7fffffff);
}

// a lane's positions in ascending order
__device__ __forceinline__ void best_push(BestMasked& a, float c, long i) {
  const int k = conf_key(c);
  ++a.n_masked;
  if (k > a.key) {
    a.key = k;
    a.idx = i;
  }
}

__device__ __forceinline__ void best_join_wave(BestMasked& a) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const int ok = __shfl_xor(a.key, o, 64);
    const long oi = __shfl_xor(a.idx, o, 64);
    a.n_masked += __shfl_xor(a.n_masked, o, 64);
    if (ok > a.key || (ok == a.key && oi < a.idx)) {
      a.key = ok;
      a.idx = oi;
    }
  }
}

// second pass: the transfers of the block whose first position is `base`
__device__ __forceinline__ void unmask_transfer(const BestMasked& best, const float* conf, const long* token, long* block_ids,
                                                long b, long base, long block_len, long mask_token_id, float threshold,
                                                uint8_t* transfer, int* n_left) {
  const int lane = threadIdx.x & 63;
  int moved = 0;
  for (long i = lane; i < block_len; i += 64) {
    const bool masked = block_ids[base + i] == mask_token_id;
    const bool t = masked && (i == best.idx || conf[base + i] >= threshold);
    transfer[base + i] = t ? 1 : 0;
    if (t) { block_ids[base + i] = token[base + i]; ++moved; }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) moved += __shfl_xor(moved, o, 64);
  if (lane == 0 && n_left) n_left[b] = best.n_masked - moved;
}

__device__ __forceinline__ void unmask_block(const float* conf, const long* token, long* block_ids, long b, long block_len,
                                             long mask_token_id, float threshold, uint8_t* transfer, int* n_left) {
  const long base = b * block_len;
  BestMasked best;
  for (long i = threadIdx.x & 63; i < block_len; i += 64)
    if (block_ids[base + i] == mask_token_id) best_push(best, conf[base + i], i);
  best_join_wave(best);
  unmask_transfer(best, conf, token, block_ids, b, base, block_len, mask_token_id, threshold, transfer, n_left);
}

}  // namespace pdllm
