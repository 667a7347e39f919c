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

// Distributed shared memory of the cluster.
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster_f2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

int launch_cross_mma(const CrossParams& p, int dtype, cudaStream_t st);
// cross_attention_sm100.cu: whether the tensor maps can describe the call.
bool cross_tc_takes(const CrossParams& p);
int launch_cross_tc(const CrossParams& p, int dtype, cudaStream_t st);
unsigned int dev_error_cross();

}  // namespace s3
