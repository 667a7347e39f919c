// cross_attention.cuh - what the two cross-attention kernels share: the
// checked arguments and how rows, heads and keys are numbered.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "sam3cu_internal.h"

namespace s3 {

// Queries of the g heads that share a key head are rows of one matrix: row r
// of (batch, key head) is head r % g of query r / g, so that one pass over K
// and V serves them all.
struct CrossParams {
  const uint16_t *q, *k, *v;
  uint16_t* o;
  int64_t qb, qs, qh, kb, ks, kh, vb, vs, vh, ob, os, oh;  // element strides
  int batch, sq, sk, kv_heads, group, head_dim;
  int rows;          // sq * group
  float scale;       // of the scores
  float scale_log2;  // scale * log2(e)
  const int32_t* k_lens;
  const uint8_t* key_mask;
  int64_t mask_stride;
  const float* bias;
  int64_t bb, bh, bs;
};

// Keys of a sequence that may count.
__device__ __forceinline__ int cross_len(const CrossParams& p, int b) {
  return p.k_lens ? max(0, min(p.k_lens[b], p.sk)) : p.sk;
}

int launch_cross_mma(const CrossParams& p, int dtype, cudaStream_t st);

}  // namespace s3
