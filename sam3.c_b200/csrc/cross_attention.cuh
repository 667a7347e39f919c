// cross_attention.cuh - what the cross-attention kernels share: the
// checked arguments and how rows, heads and keys are numbered.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <initializer_list>

#include "cluster_table.h"
#include "sam3cu_internal.h"
#include "tma_host.cuh"

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

// Which dimensions of K and V a batch or its heads share: factors of the
// coordinates, 0 or 1.
struct KvShare {
  int kb, kh, vb, vh;
};

// One dimension of a tensor map; one of stride 0 (shared data) or a single
// element becomes one of extent 1 (*mul 0).
struct TensorDim {
  int64_t extent, stride;
  int* mul;
};
// A tensor [d2][d1][d0][head_dim] of 16-bit elements by element strides, boxes
// of box[2] x box[1] x box[0] rows of 64 elements (128-byte swizzle), or of 32
// (64-byte swizzle) for head_dim <= 32; what lies past head_dim reads zeros.
inline bool make_cross_map(CUtensorMap* m, const void* base, int dtype, int head_dim, const TensorDim (&d)[3],
                           const int (&box)[3]) {
  EncodeTiledFn fn = get_encode_tiled();
  if (!fn) return false;
  const bool small = head_dim <= 32;
  cuuint64_t dims[4] = {static_cast<cuuint64_t>(head_dim), 1, 1, 1};
  cuuint64_t strides[3] = {16, 16, 16};
  cuuint32_t bx[4] = {small ? 32u : 64u, 1, 1, 1}, es[4] = {1, 1, 1, 1};
  for (int i = 0; i < 3; ++i) {
    bx[i + 1] = static_cast<cuuint32_t>(box[i]);
    if (d[i].mul) *d[i].mul = d[i].stride != 0;
    if (d[i].stride == 0) continue;
    dims[i + 1] = static_cast<cuuint64_t>(d[i].extent);
    strides[i] = static_cast<cuuint64_t>(d[i].stride) * 2;
  }
  return fn(m, dtype == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
            const_cast<void*>(base), dims, strides, bx, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
            small ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
inline bool make_kv_maps(const CrossParams& p, int dtype, int keys, CUtensorMap* mk, CUtensorMap* mv, KvShare* share) {
  const TensorDim dk[3] = {{p.sk, p.ks, nullptr}, {p.kv_heads, p.kh, &share->kh}, {p.batch, p.kb, &share->kb}};
  const TensorDim dv[3] = {{p.sk, p.vs, nullptr}, {p.kv_heads, p.vh, &share->vh}, {p.batch, p.vb, &share->vb}};
  const int box[3] = {keys, 1, 1};
  return make_cross_map(mk, p.k, dtype, p.head_dim, dk, box) && make_cross_map(mv, p.v, dtype, p.head_dim, dv, box);
}
// Whether tensor maps can describe K and V: strides below 2^40 bytes, and no
// key shared (stride 0 cannot be part of a box).
inline bool cross_kv_maps(const CrossParams& p) {
  constexpr int64_t kMost = 1ll << 39;
  for (int64_t x : {p.kb, p.ks, p.kh, p.vb, p.vs, p.vh})
    if (x >= kMost) return false;
  return p.sk > 0 && (p.sk == 1 || (p.ks != 0 && p.vs != 0));
}

// CTAs of a cluster that share an item's keys: the most, up to `most` (<= 16),
// of which all items' clusters run at once and each has `tiles_each` key tiles.
// (Clusters are placed within a GPC: 16 items of 8 are two waves, 15 fit.)
// table: the kernel's own, of what fits on each device.
template <class K>
int cluster_splits(K kernel, int threads, int smem, int64_t items, int key_tiles, int tiles_each, int most,
                   ClusterTable& table) {
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess) cudaGetLastError();
  for (int n = most; n > 1; --n) {
    if (key_tiles < tiles_each * n || items * n > 4 * num_sms()) continue;
    const int fit = table.fit(dev, n, [&](int* f) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(n);
      cfg.blockDim = dim3(threads);
      cfg.dynamicSmemBytes = smem;
      cudaLaunchAttribute at[1];
      at[0].id = cudaLaunchAttributeClusterDimension;
      at[0].val.clusterDim.x = n;
      at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
      cfg.attrs = at;
      cfg.numAttrs = 1;
      const cudaError_t e = cudaOccupancyMaxActiveClusters(f, kernel, &cfg);
      if (e != cudaSuccess) cudaGetLastError();  // the next call's own check must not see it
      return static_cast<int>(e);
    });
    if (items <= fit) return n;
  }
  return 1;
}

int launch_cross_mma(const CrossParams& p, int dtype, cudaStream_t st);
// cross_attention_sm100.cu: whether the tensor maps can describe the call.
bool cross_tc_takes(const CrossParams& p);
// Launches, or returns kCrossTcSpills where the compiler spilled registers of
// the kernel: launch_cross_mma takes every call that this one takes.
constexpr int kCrossTcSpills = 1;
int cross_tc_as_if_spilled(bool on);  // for the self test
int launch_cross_tc(const CrossParams& p, int dtype, cudaStream_t st);
unsigned int dev_error_cross();
unsigned int dev_error_cross_few();

}  // namespace s3
