// cross_attention.cu - attention of queries over states of another length,
// for few query rows, few keys or a bias (and the entry point, which sends the
// rest to cross_attention_sm100.cu).
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(s_j - max s),
//   s_j = scale q.k_j + bias_j, over the keys that count
//
// One pass over the keys with the running maximum and sum of each row; a warp
// computes 16 rows with m16n8k16 MMAs (fp32 accumulate).  With few rows to a
// key head a call reads K and V once and does little with them, with few keys
// it reads Q and writes O: HBM bounds both, and what matters is that enough
// loads are under way on every SM.  Three kernels:
//   * cross_few_kernel, up to 16 rows of a key head: one warp fetches 128-key
//     tiles by TMA, four compute.  2 x 4 key heads of 128 under 32, one query,
//     65521 and 49141 keys: 45 us, 0.80 of the measured copy rate (49 us a call);
//   * cross_keep_kernel, few keys: K and V stay in shared memory, the warps
//     walk the rows.  4 x 8 heads of 32, 5184 rows, 77 keys: 17 us;
//   * cross_rows_kernel, the rest: 64 rows to a CTA, 16 to a warp, K, V and the
//     bias through a ring of cp.async.  4 x 8 heads of 32, 201 rows, 5184 keys
//     with a bias: 50 us, 0.47 of the copy rate for reading the bias once, and 50
//     with one bias for all heads (shared memory bounds it: every 16 rows read
//     all of K and V there).
// Where that leaves SMs idle the keys are split over the CTAs of a cluster,
// which exchange (max, sum, partial O) through distributed shared memory: no
// workspace, no second launch, a fixed order of sums.  Few items over long
// states need more CTAs than a cluster has: those leave their parts in a
// workspace, which cross_join_kernel adds up, in a fixed order too.
// A key that does not count is never multiplied: its score is -inf, and its V
// row becomes zeros (so what it holds cannot reach the sums as 0 * NaN).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <cstring>

#include "../../include/sam3cu.h"
#include "attention_math.cuh"
#include "cross_attention.cuh"
#include "sam3cu_internal.h"
#include "sm100_ptx.cuh"
#include "tma_host.cuh"

namespace s3 {

S3_DEV_ERROR_ACCESSOR(dev_error_cross_few)

namespace {

constexpr int kThreads = 128;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxKeep = 256;  // keys that cross_keep_kernel may hold

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr)
               : "memory");
}
template <bool kBf16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (kBf16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if (kBf16) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}
// kD: head_dim rounded up to 32, 64 or 128 (the copies fill the rest with
// zeros).
template <int kD, bool kBias>
struct RowsCfg {
  static constexpr int kRows = 64;                     // query rows of a CTA, 16 to a warp
  static constexpr int kKT = 64;                       // keys of a tile
  static constexpr int kChunks = kD / 8;               // 16-byte pieces of a row
  static constexpr int kTileBytes = kKT * kD * 2;      // K or V
  static constexpr int kBiasBytes = kBias ? kRows * kKT * 4 : 0;
  static constexpr int kStageBytes = 2 * kTileBytes + kBiasBytes;
  // (with a bias two, so that more CTAs fit: 201 x 5184 x 8 heads of 16, 32, 64
  // and 128, batch 4: 50, 50, 72 and 114 us, with three stages 60, 60, 81 and
  // 161; 8 x 40 rows, heads of 64: 42 and 45; 8 x 100 x 1024, heads of 64: even)
  static constexpr int kStages = kBias ? 2 : kD == 32 ? 4 : kD == 128 ? 2 : 3;
  static constexpr int kQBytes = kRows * kD * 2;
  static constexpr int kPitch = kD + 4;                // floats of a partial row
  static constexpr int kPartBytes = kRows * kPitch * 4;  // over the ring
  static constexpr int kRing = kStages * kStageBytes;
  static constexpr int kSmem = kQBytes + (kRing > kPartBytes ? kRing : kPartBytes);
};
template <int kD>
struct FewCfg {
  static constexpr int kRows = 16;                     // query rows of a CTA
  static constexpr int kWarps = 4;                     // each 32 keys of a tile
  static constexpr int kThreads = 32 * (kWarps + 1);   // and one that loads
  static constexpr int kKT = 32 * kWarps;
  static constexpr int kTileBytes = kKT * kD * 2;
  static constexpr int kStages = kD == 32 ? 4 : 3;
  static constexpr int kQBytes = kRows * kD * 2;
  static constexpr int kPitch = kD + 4;
  static constexpr int kPartBytes = kWarps * kRows * kPitch * 4;  // over the ring
  static constexpr int kRing = 2 * kStages * kTileBytes;
  static_assert(kPartBytes <= kRing, "partial rows fit over the ring");
  static constexpr int kSmem = kRing + kQBytes;
};

// Byte offset of 16-byte piece c of row r in a tile of kChunks pieces a row,
// permuted within each 128-byte line so that ldmatrix (8 rows, one piece)
// and the copies (consecutive pieces) touch all banks.
template <int kChunks>
__device__ __forceinline__ uint32_t tile_at(int r, int c) {
  const int at = r * kChunks + c;
  const int key = kChunks == 4 ? (r >> 1) & 3 : r & 7;
  return static_cast<uint32_t>((at ^ key) << 4);
}

// A warp's 16 rows (a lane: rows lane / 4 and + 8): running maximum, sum (this
// lane's share) and O.
template <int kD>
struct RowState {
  float acc[kD / 8][4];
  float m[2], l[2];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < kD / 8; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
  }
  // Scores to P, against the maximum with them in it; sum and O rescaled.
  // f16 P are times 2^14, which cancels in O / sum: below 2^-14 the type has
  // no full precision left.  The maximum is taken off before the factor: their
  // product would be rounded, by 4 at 2^26, and exp2 of that is past f16's
  // range; a bias of the type's lowest value would overflow with it.
  template <int kKeys, bool kBf16>
  __device__ __forceinline__ void softmax(float (&s)[kKeys / 8][4], float to_log2) {
    const float shift = kBf16 ? 0.f : 14.f;
    float top[2], corr[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < kKeys / 8; ++j) mx = max3(mx, s[j][2 * h], s[j][2 * h + 1]);
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      top[h] = fmaxf(m[h], mx);
    }
    const bool grew = __any_sync(0xffffffffu, top[0] != m[0] || top[1] != m[1]);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float base = top[h] == -INFINITY ? 0.f : top[h];  // nothing counted yet: every p is 0
      corr[h] = ex2((m[h] - base) * to_log2);
      m[h] = top[h];
      const uint64_t c2 = f2pack(to_log2, to_log2);
      const uint64_t sh2 = f2pack(shift, shift), b2 = f2pack(-base, -base);
      uint64_t sum2 = f2pack(0.f, 0.f);
#pragma unroll
      for (int j = 0; j < kKeys / 8; ++j) {
        const uint64_t x = fadd2(f2pack(s[j][2 * h], s[j][2 * h + 1]), b2);
        float e0, e1;
        f2unpack(kBf16 ? fmul2(x, c2) : ffma2(x, c2, sh2), e0, e1);
        s[j][2 * h] = ex2(e0);
        s[j][2 * h + 1] = ex2(e1);
        sum2 = fadd2(sum2, f2pack(s[j][2 * h], s[j][2 * h + 1]));
      }
      float s0, s1;
      f2unpack(sum2, s0, s1);
      l[h] = fmaf(l[h], corr[h], s0 + s1);
    }
    if (grew) {
      const uint64_t c2[2] = {f2pack(corr[0], corr[0]), f2pack(corr[1], corr[1])};
#pragma unroll
      for (int j = 0; j < kD / 8; ++j) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float a0, a1;
          f2unpack(fmul2(f2pack(acc[j][2 * h], acc[j][2 * h + 1]), c2[h]), a0, a1);
          acc[j][2 * h] = a0;
          acc[j][2 * h + 1] = a1;
        }
      }
    }
  }
};

// 8 elements of an output row, scaled by what they were summed with.
template <bool kBf16>
__device__ __forceinline__ void store_row(const CrossParams& p, int b, int kvh, int row, int c, const float (&o)[8],
                                          float l) {
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // no key: zeros; NaN stays NaN
  const int q = row / p.group;
  uint4 w4;
  w4.x = pack2<kBf16>(o[0] * inv, o[1] * inv);
  w4.y = pack2<kBf16>(o[2] * inv, o[3] * inv);
  w4.z = pack2<kBf16>(o[4] * inv, o[5] * inv);
  w4.w = pack2<kBf16>(o[6] * inv, o[7] * inv);
  *reinterpret_cast<uint4*>(p.o + b * p.ob + q * p.os + static_cast<int64_t>(kvh * p.group + row - q * p.group) * p.oh +
                            c) = w4;
}

// Adds up what the key warps of a CTA left for its kRows rows: (max, sum) in ml
// [kWK][kRows] and the unscaled partial O in part [kWK][kRows][kD + 4]; the
// sums take the place of the first warp's.  wgt: [kWK][kRows].
template <int kD, int kRows, int kWK, int kN>
__device__ __forceinline__ void join_warps(float* part, float2* ml, float* wgt, float to_log2) {
  constexpr int kPitch = kD + 4;
  const int tid = threadIdx.x;
  __syncthreads();
  // the weight of each warp's partial row against the row's maximum
  if (tid < kRows) {
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int w = 0; w < kWK; ++w) m = fmaxf(m, ml[w * kRows + tid].x);
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int w = 0; w < kWK; ++w) {
      const float f = ex2((ml[w * kRows + tid].x - base) * to_log2);
      wgt[w * kRows + tid] = f;
      l = fmaf(f, ml[w * kRows + tid].y, l);
    }
    ml[tid] = make_float2(m, l);
  }
  __syncthreads();
  for (int i = tid; i < kRows * kD / 4; i += kN) {
    const int r = i / (kD / 4), c = (i % (kD / 4)) * 4;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWK; ++w) {
      const float f = wgt[w * kRows + r];
      const float4 x = *reinterpret_cast<const float4*>(part + (w * kRows + r) * kPitch + c);
      a.x = fmaf(f, x.x, a.x);
      a.y = fmaf(f, x.y, a.y);
      a.z = fmaf(f, x.z, a.z);
      a.w = fmaf(f, x.w, a.w);
    }
    *reinterpret_cast<float4*>(part + r * kPitch + c) = a;
  }
}

// The end of a kernel that left ml [kRows] and part [kRows][kD + 4]: the rows to
// the output, with splits > 1 added up over the cluster's CTAs (each takes a
// share of the rows over all of them, in rank order).
template <bool kBf16, int kD, int kRows, int kN>
__device__ __forceinline__ void join_cluster(const CrossParams& p, float* part, float2* ml, int row0, int b, int kvh,
                                             int split, int splits, float to_log2) {
  constexpr int kPitch = kD + 4;
  const int tid = threadIdx.x;
  if (splits > 1) cluster_sync();
  else __syncthreads();
  // Rows to the output, 8 elements a thread.
  const int out_chunks = p.head_dim / 8;
  const uint32_t part_s = smem_u32(part), ml_s = smem_u32(ml);
  for (int i = tid + kN * split; i < kRows * out_chunks; i += kN * splits) {
    const int r = i / out_chunks, c = (i % out_chunks) * 8;
    if (row0 + r >= p.rows) break;
    float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, l = 0.f;
    if (splits > 1) {
      float m = -INFINITY;
      for (int w = 0; w < splits; ++w) m = fmaxf(m, ld_cluster_f2(mapa_shared(ml_s + r * 8, w)).x);
      const float base = m == -INFINITY ? 0.f : m;
      for (int w = 0; w < splits; ++w) {
        const float2 s = ld_cluster_f2(mapa_shared(ml_s + r * 8, w));
        const float f = ex2((s.x - base) * to_log2);
        l = fmaf(f, s.y, l);
        const uint32_t src = mapa_shared(part_s + (r * kPitch + c) * 4, w);
        const float4 x = ld_cluster_f4(src), y = ld_cluster_f4(src + 16);
        const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = fmaf(f, v[e], o[e]);
      }
    } else {
      l = ml[r].y;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = part[r * kPitch + c + e];
    }
    store_row<kBf16>(p, b, kvh, row0 + r, c, o, l);
  }
  if (splits > 1) cluster_sync();  // the others may still read this CTA's partial rows
}

template <bool kBf16, int kD, bool kBias>
__global__ void __launch_bounds__(kThreads) cross_rows_kernel(const __grid_constant__ CrossParams p, int row_tiles,
                                                              int splits, int bias_step) {
  using Cf = RowsCfg<kD, kBias>;
  constexpr int kKT = Cf::kKT, kCh = Cf::kChunks, kStages = Cf::kStages;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ float2 ml[Cf::kRows];  // (max, sum) of each row
  __shared__ const float* brow[kBias ? Cf::kRows : 1];
  const uint32_t sq = smem_u32(smem), ring = sq + Cf::kQBytes;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int split = blockIdx.x % splits, item = blockIdx.x / splits;
  const int rt = item % row_tiles, bh = item / row_tiles;
  const int kvh = bh % p.kv_heads, b = bh / p.kv_heads;
  const int row0 = rt * Cf::kRows;
  const int len = cross_len(p, b);
  const uint16_t* kg = p.k + b * p.kb + kvh * p.kh;
  const uint16_t* vg = p.v + b * p.vb + kvh * p.vh;
  const uint8_t* mg = p.key_mask ? p.key_mask + b * p.mask_stride : nullptr;

  const int n_tiles = (len + kKT - 1) / kKT;
  const int t0 = static_cast<int>(static_cast<int64_t>(n_tiles) * split / splits);
  const int t1 = static_cast<int>(static_cast<int64_t>(n_tiles) * (split + 1) / splits);

  // the rows' queries, zero-filled past the last row and past head_dim
  for (int i = tid; i < Cf::kRows * kCh; i += kThreads) {
    const int r = i / kCh, c = i % kCh;
    const bool ok = row0 + r < p.rows && c * 8 < p.head_dim;
    const int s = ok ? (row0 + r) / p.group : 0, h = ok ? (row0 + r) % p.group : 0;
    const uint16_t* src = p.q + b * p.qb + s * p.qs + static_cast<int64_t>(kvh * p.group + h) * p.qh + (ok ? c * 8 : 0);
    cp_async16(sq + tile_at<kCh>(r, c), src, ok);
  }
  cp_async_commit();

  // Tile t into its ring slot.
  auto load = [&](int t) {
    const uint32_t sk = ring + (t % kStages) * Cf::kStageBytes, sv = sk + Cf::kTileBytes;
#pragma unroll 4
    for (int i = 0; i < kKT * kCh / kThreads; ++i) {
      const int idx = tid + i * kThreads;
      const int r = idx / kCh, c = idx % kCh;
      const int key = t * kKT + r;
      bool ok = key < len && c * 8 < p.head_dim;
      if (mg && ok) ok = mg[key] != 0;
      const int64_t at = ok ? key : 0;
      const int cc = ok ? c * 8 : 0;
      cp_async16(sk + tile_at<kCh>(r, c), kg + at * p.ks + cc, ok);
      cp_async16(sv + tile_at<kCh>(r, c), vg + at * p.vs + cc, ok);
    }
    if constexpr (kBias) {
      // the tile's bias, a row by 16 lanes of 4 keys; bias_step 4: its rows
      // start on 16 bytes, 1: key by key.  Piece c of row r lies at c ^ 2 (r % 4),
      // so that the 8-byte reads of four rows touch all banks (rows with 4
      // floats between them: two reads to a bank, 53 us instead of 50 for the
      // case at kStages).
      const uint32_t sb = sv + Cf::kTileBytes;
#pragma unroll 2
      for (int r = tid / 16; r < Cf::kRows; r += kThreads / 16) {
        const float* src = brow[kBias ? r : 0];
        const int key = t * kKT + tid % 16 * 4;
        const uint32_t dst = sb + r * kKT * 4 + ((tid % 16) ^ (2 * (r & 3))) * 16;
        if (bias_step == 4) {
          cp_async16(dst, src + (key < len ? key : 0), key < len);  // (sk is a multiple of 4)
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) cp_async4(dst + 4 * e, src + (key + e < len ? key + e : 0), key + e < len);
        }
      }
    }
  };
  if constexpr (kBias) {
    if (tid < Cf::kRows) {
      const int row = min(row0 + tid, p.rows - 1), q = row / p.group;
      brow[tid] = p.bias + b * p.bb + static_cast<int64_t>(kvh * p.group + row - q * p.group) * p.bh + q * p.bs;
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
    if (t0 + i < t1) load(t0 + i);
    cp_async_commit();
  }

  RowState<kD> st;
  st.clear();
  uint32_t qf[kD / 16][4];
  // with a bias the scores are in natural units (its lowest finite values
  // would overflow in base 2), without one they stay unscaled dot products
  const float to_log2 = kBias ? kLog2e : p.scale_log2;
  cp_async_wait<kStages - 1>();  // the queries
  __syncthreads();
#pragma unroll
  for (int kk = 0; kk < kD / 16; ++kk) {
    const int r = warp * 16 + (lane & 15);
    ldsm_x4(sq + tile_at<kCh>(r, kk * 2 + (lane >> 4)), qf[kk][0], qf[kk][1], qf[kk][2], qf[kk][3]);
  }

  for (int t = t0; t < t1; ++t) {
    cp_async_wait<kStages - 2>();
    __syncthreads();
    if (t + kStages - 1 < t1) load(t + kStages - 1);  // into the slot of tile t - 1, which all have left
    cp_async_commit();
    const uint32_t sk = ring + (t % kStages) * Cf::kStageBytes, sv = sk + Cf::kTileBytes;
    const int key0 = t * kKT;

    float s[kKT / 8][4];
#pragma unroll
    for (int j = 0; j < kKT / 8; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
    for (int kk = 0; kk < kD / 16; ++kk) {
#pragma unroll
      for (int jp = 0; jp < kKT / 16; ++jp) {  // pairs of 8-key blocks
        const int r = jp * 16 + (lane & 7) + (lane >> 4) * 8;
        uint32_t b0, b1, b2, b3;
        ldsm_x4(sk + tile_at<kCh>(r, kk * 2 + ((lane >> 3) & 1)), b0, b1, b2, b3);
        mma16816<kBf16>(s[2 * jp], qf[kk], b0, b1);
        mma16816<kBf16>(s[2 * jp + 1], qf[kk], b2, b3);
      }
    }
    if constexpr (kBias) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t sb = sv + Cf::kTileBytes + (warp * 16 + (lane >> 2) + 8 * h) * kKT * 4 + (lane & 3) * 8;
        const uint32_t swz = (lane >> 2 & 3) * 32;
#pragma unroll
        for (int j = 0; j < kKT / 8; ++j) {
          float x, y;
          asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(x), "=f"(y) : "r"(sb + ((j * 32) ^ swz)) : "memory");
          f2unpack(ffma2(f2pack(s[j][2 * h], s[j][2 * h + 1]), f2pack(p.scale, p.scale), f2pack(x, y)), s[j][2 * h],
                   s[j][2 * h + 1]);
        }
      }
    }
    if (mg || key0 + kKT > len) {
#pragma unroll
      for (int j = 0; j < kKT / 8; ++j) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int key = key0 + j * 8 + (lane & 3) * 2 + e;
          if (key >= len || (mg && mg[key] == 0)) s[j][e] = s[j][2 + e] = -INFINITY;
        }
      }
    }
    st.template softmax<kKT, kBf16>(s, to_log2);
    // O += P V, P rounded to the operands' type
#pragma unroll
    for (int kk = 0; kk < kKT / 16; ++kk) {
      uint32_t pa[4];
      pa[0] = pack2<kBf16>(s[2 * kk][0], s[2 * kk][1]);
      pa[1] = pack2<kBf16>(s[2 * kk][2], s[2 * kk][3]);
      pa[2] = pack2<kBf16>(s[2 * kk + 1][0], s[2 * kk + 1][1]);
      pa[3] = pack2<kBf16>(s[2 * kk + 1][2], s[2 * kk + 1][3]);
#pragma unroll
      for (int jp = 0; jp < kD / 16; ++jp) {  // pairs of 8-wide column blocks
        const int r = kk * 16 + (lane & 15);
        uint32_t b0, b1, b2, b3;
        ldsm_x4_t(sv + tile_at<kCh>(r, jp * 2 + (lane >> 4)), b0, b1, b2, b3);
        mma16816<kBf16>(st.acc[2 * jp], pa, b0, b1);
        mma16816<kBf16>(st.acc[2 * jp + 1], pa, b2, b3);
      }
    }
  }

  // Partial results into shared memory (over the ring, which nothing reads
  // or fills any more).
  cp_async_wait<0>();
  __syncthreads();
  float* part = reinterpret_cast<float*>(smem + Cf::kQBytes);
  const int r_lo = warp * 16 + (lane >> 2);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float l = st.l[h];
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if ((lane & 3) == 0) ml[r_lo + 8 * h] = make_float2(st.m[h], l);
    float* dst = part + (r_lo + 8 * h) * Cf::kPitch + (lane & 3) * 2;
#pragma unroll
    for (int j = 0; j < kD / 8; ++j)
      *reinterpret_cast<float2*>(dst + j * 8) = make_float2(st.acc[j][2 * h], st.acc[j][2 * h + 1]);
  }
  join_cluster<kBf16, kD, Cf::kRows, kThreads>(p, part, ml, row0, b, kvh, split, splits, to_log2);
}

// Up to 16 rows of a key head: K and V are read once and little is done with
// them, so what counts is that loads never pause.  One warp fetches 128-key
// tiles by TMA into a ring; four compute, each on 32 keys of every tile with a
// running maximum of its own, and are added up at the end.
template <bool kBf16, int kD, bool kBias>
__global__ void __launch_bounds__(FewCfg<kD>::kThreads)
    cross_few_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                     const __grid_constant__ CrossParams p, const KvShare share, int row_tiles, int splits, float* ws) {
  using Cf = FewCfg<kD>;
  constexpr int kCh = kD / 8, kStages = Cf::kStages, kTile = Cf::kTileBytes, kHalves = kD == 128 ? 2 : 1;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ uint64_t bars[2 * kStages];
  __shared__ float2 ml[Cf::kWarps * Cf::kRows];
  __shared__ float wgt[Cf::kWarps * Cf::kRows];
  __shared__ int abort_flag_s;
  uint64_t* full = bars;
  uint64_t* empty = bars + kStages;
  volatile int* abort_flag = &abort_flag_s;
  const uint32_t ring = smem_u32(smem), sq = ring + Cf::kRing;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int split = blockIdx.x % splits, item = blockIdx.x / splits;
  const int rt = item % row_tiles, bh = item / row_tiles;
  const int kvh = bh % p.kv_heads, b = bh / p.kv_heads;
  const int row0 = rt * Cf::kRows;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], Cf::kWarps);
    }
    const bool aligned = (ring & 1023u) == 0;  // the swizzled layouts need it
    abort_flag_s = aligned ? 0 : 1;
    if (!aligned) atomicCAS(&g_dev_error, 0u, static_cast<unsigned>(kErrTmaWait));
    fence_barrier_init();
  }
  const int len = cross_len(p, b);
  const int n_tiles = (len + Cf::kKT - 1) / Cf::kKT;
  const int t0 = static_cast<int>(static_cast<int64_t>(n_tiles) * split / splits);
  const int t1 = static_cast<int>(static_cast<int64_t>(n_tiles) * (split + 1) / splits);
  __syncthreads();
  const bool run = *abort_flag == 0;
  // with a bias the scores are in natural units (its lowest finite values
  // would overflow in base 2), without one they stay unscaled dot products
  const float to_log2 = kBias ? kLog2e : p.scale_log2;

  if (warp == Cf::kWarps) {
    int issued = 0;
    for (int t = t0; run && t < t1; ++t, ++issued) {
      const int st = (t - t0) % kStages;
      if (!mbar_wait_warp(&empty[st], (((t - t0) / kStages) & 1) ^ 1, kErrStageFree, abort_flag)) break;
      if (elect_one()) {
        uint8_t* dst = smem + st * 2 * kTile;
        mbar_arrive_expect_tx(&full[st], 2 * kTile);
        for (int h = 0; h < kHalves; ++h) {
          tma_load_4d(dst + h * (kTile / 2), &tk, &full[st], h * 64, t * Cf::kKT, kvh * share.kh, b * share.kb);
          tma_load_4d(dst + kTile + h * (kTile / 2), &tv, &full[st], h * 64, t * Cf::kKT, kvh * share.vh, b * share.vb);
        }
      }
      __syncwarp();
    }
    // The last copies are seen in, also where a wait gave up: this shared
    // memory may be another CTA's as soon as this one ends.
    for (int i = max(0, issued - kStages); i < issued; ++i)
      mbar_wait_warp(&full[i % kStages], (i / kStages) & 1, kErrTmaWait, nullptr);
  } else {
    // byte offset of piece c of row r in a tile as the copies lay it: for
    // D = 128 two halves of 128-byte rows
    auto at = [](int r, int c) {
      return kD == 128 ? (c >> 3) * (kTile / 2) + tile_at<8>(r, c & 7) : tile_at<kD == 128 ? 8 : kCh>(r, c);
    };
    // the queries, by this warp alone: each warp writes the same values
    for (int i = lane; i < Cf::kRows * kCh; i += 32) {
      const int r = i / kCh, c = i % kCh, row = row0 + r;
      const bool ok = row < p.rows && c * 8 < p.head_dim;
      const int q = ok ? row / p.group : 0, h = ok ? row - q * p.group : 0;
      uint4 w = make_uint4(0, 0, 0, 0);
      if (ok) w = *reinterpret_cast<const uint4*>(p.q + b * p.qb + q * p.qs + (kvh * p.group + h) * p.qh + c * 8);
      asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(sq + tile_at<kCh>(r, c)), "r"(w.x), "r"(w.y),
                   "r"(w.z), "r"(w.w)
                   : "memory");
    }
    __syncwarp();
    uint32_t qf[kD / 16][4];
#pragma unroll
    for (int kk = 0; kk < kD / 16; ++kk)
      ldsm_x4(sq + tile_at<kCh>(lane & 15, kk * 2 + (lane >> 4)), qf[kk][0], qf[kk][1], qf[kk][2], qf[kk][3]);
    const uint8_t* mg = p.key_mask ? p.key_mask + b * p.mask_stride : nullptr;
    const float* brow[2] = {nullptr, nullptr};
    if (kBias) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = min(row0 + (lane >> 2) + 8 * h, p.rows - 1);
        brow[h] = p.bias + b * p.bb + (kvh * p.group + r % p.group) * p.bh + (r / p.group) * p.bs;
      }
    }
    RowState<kD> rs;
    rs.clear();
    for (int t = t0; run && t < t1; ++t) {
      const int st = (t - t0) % kStages;
      const int key0 = t * Cf::kKT + warp * 32;
      const uint32_t on = __ballot_sync(0xffffffffu, key0 + lane < len && (!mg || mg[key0 + lane] != 0));
      float bias[kBias ? 4 : 1][4];
      if (kBias) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = key0 + j * 8 + (lane & 3) * 2 + (e & 1);
            bias[kBias ? j : 0][e] = key < len ? __ldg(brow[e >> 1] + key) : 0.f;
          }
        }
      }
      if (!mbar_wait_warp(&full[st], ((t - t0) / kStages) & 1, kErrTmaWait, abort_flag)) break;
      const uint32_t sk = ring + st * 2 * kTile, sv = sk + kTile;
      if (on != 0) {
        if (on != 0xffffffffu) {
          // V of keys that do not count: 0 * NaN would reach the sums
          if (!(on >> lane & 1)) {
#pragma unroll
            for (int c = 0; c < kCh; ++c)
              asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(sv + at(warp * 32 + lane, c)), "r"(0)
                           : "memory");
          }
          fence_proxy_async_smem();  // before the next copy into this slot
          __syncwarp();
        }
        float s[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
        for (int kk = 0; kk < kD / 16; ++kk) {
#pragma unroll
          for (int jp = 0; jp < 2; ++jp) {  // pairs of 8-key blocks
            const int r = warp * 32 + jp * 16 + (lane & 7) + (lane >> 4) * 8;
            uint32_t b0, b1, b2, b3;
            ldsm_x4(sk + at(r, kk * 2 + ((lane >> 3) & 1)), b0, b1, b2, b3);
            mma16816<kBf16>(s[2 * jp], qf[kk], b0, b1);
            mma16816<kBf16>(s[2 * jp + 1], qf[kk], b2, b3);
          }
        }
        if (kBias) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[j][e] = fmaf(s[j][e], p.scale, bias[kBias ? j : 0][e]);
        }
        if (on != 0xffffffffu) {
          const uint32_t mine = on >> ((lane & 3) * 2);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (!(mine >> (j * 8) & 1)) s[j][0] = s[j][2] = -INFINITY;
            if (!(mine >> (j * 8 + 1) & 1)) s[j][1] = s[j][3] = -INFINITY;
          }
        }
        rs.template softmax<32, kBf16>(s, to_log2);
        // O += P V, P rounded to the operands' type
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
          uint32_t pa[4];
          pa[0] = pack2<kBf16>(s[2 * kk][0], s[2 * kk][1]);
          pa[1] = pack2<kBf16>(s[2 * kk][2], s[2 * kk][3]);
          pa[2] = pack2<kBf16>(s[2 * kk + 1][0], s[2 * kk + 1][1]);
          pa[3] = pack2<kBf16>(s[2 * kk + 1][2], s[2 * kk + 1][3]);
#pragma unroll
          for (int jp = 0; jp < kD / 16; ++jp) {  // pairs of 8-wide column blocks
            const int r = warp * 32 + kk * 16 + (lane & 15);
            uint32_t b0, b1, b2, b3;
            ldsm_x4_t(sv + at(r, jp * 2 + (lane >> 4)), b0, b1, b2, b3);
            mma16816<kBf16>(rs.acc[2 * jp], pa, b0, b1);
            mma16816<kBf16>(rs.acc[2 * jp + 1], pa, b2, b3);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
    }
    // (the ring is read by others until here, and filled no more)
    asm volatile("bar.sync 1, %0;" ::"n"(32 * Cf::kWarps) : "memory");
    float* part = reinterpret_cast<float*>(smem) + warp * Cf::kRows * Cf::kPitch;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float l = rs.l[h];
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      const int r = (lane >> 2) + 8 * h;
      if ((lane & 3) == 0) ml[warp * Cf::kRows + r] = make_float2(rs.m[h], l);
      float* dst = part + r * Cf::kPitch + (lane & 3) * 2;
#pragma unroll
      for (int j = 0; j < kD / 8; ++j)
        *reinterpret_cast<float2*>(dst + j * 8) = make_float2(rs.acc[j][2 * h], rs.acc[j][2 * h + 1]);
    }
  }
  float* part = reinterpret_cast<float*>(smem);
  join_warps<kD, Cf::kRows, Cf::kWarps, Cf::kThreads>(part, ml, wgt, to_log2);
  if (ws) {
    // to cross_join_kernel: this CTA's (max, sum) and partial rows
    __syncthreads();
    float* dst = ws + static_cast<int64_t>(blockIdx.x) * Cf::kRows * (kD + 2);
    for (int i = tid; i < Cf::kRows * kD / 4; i += Cf::kThreads)
      *reinterpret_cast<float4*>(dst + i * 4) =
          *reinterpret_cast<const float4*>(part + i / (kD / 4) * Cf::kPitch + i % (kD / 4) * 4);
    if (tid < Cf::kRows) *reinterpret_cast<float2*>(dst + Cf::kRows * kD + tid * 2) = ml[tid];
    return;
  }
  join_cluster<kBf16, kD, Cf::kRows, Cf::kThreads>(p, part, ml, row0, b, kvh, split, splits, to_log2);
}

// Adds up the partial rows that cross_few_kernel left in its workspace, a CTA
// per row: 8 groups of threads take every 8th split, then are added up in order.
template <bool kBf16, int kD>
__global__ void __launch_bounds__(kD) cross_join_kernel(const __grid_constant__ CrossParams p, int row_tiles,
                                                        int splits, const float* ws, float to_log2) {
  constexpr int kRows = FewCfg<kD>::kRows, kSlab = kRows * (kD + 2), kCh = kD / 8;
  __shared__ float top[kD / 32];
  __shared__ float part[8][kD + 1];  // and the group's sum of weights
  const int r = blockIdx.x % kRows, item = blockIdx.x / kRows, rt = item % row_tiles, bh = item / row_tiles;
  const int row = rt * kRows + r;
  if (row >= p.rows) return;
  const int tid = threadIdx.x, c = tid % kCh * 8, group = tid / kCh;
  const float* src = ws + static_cast<int64_t>(item) * splits * kSlab;
  const float* ml = src + kRows * kD + r * 2;
  float m = -INFINITY;
  for (int w = tid; w < splits; w += kD) m = fmaxf(m, ml[static_cast<int64_t>(w) * kSlab]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (tid % 32 == 0) top[tid / 32] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kD / 32; ++i) m = fmaxf(m, top[i]);
  const float base = m == -INFINITY ? 0.f : m;
  float l = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
  for (int w = group; w < splits; w += 8) {
    const int64_t at = static_cast<int64_t>(w) * kSlab;
    const float2 s = *reinterpret_cast<const float2*>(ml + at);
    const float4 x = *reinterpret_cast<const float4*>(src + at + r * kD + c);
    const float4 y = *reinterpret_cast<const float4*>(src + at + r * kD + c + 4);
    const float f = ex2((s.x - base) * to_log2);
    l = fmaf(f, s.y, l);
    const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = fmaf(f, v[e], o[e]);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) part[group][c + e] = o[e];
  if (tid % kCh == 0) part[group][kD] = l;
  __syncthreads();
  if (group == 0 && c < p.head_dim) {
    l = part[0][kD];
#pragma unroll
    for (int g = 1; g < 8; ++g) {
      l += part[g][kD];
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] += part[g][c + e];
    }
    store_row<kBf16>(p, bh / p.kv_heads, bh % p.kv_heads, row, c, o, l);
  }
}

// Few keys, many rows: the CTA keeps K and V of its key head in shared memory
// and its warps walk 16-row tiles on their own: the next tile's queries are
// copied while this one is computed, and no barrier is met in the loop.  Q is
// read and O written once, which is what bounds it.
template <int kD>
struct KeepCfg {
  static constexpr int kChunks = kD / 8;
  static constexpr int kQBytes = 16 * kD * 2;  // a warp's tile, two of them
  static int smem(int keys) { return (keys + 15) / 16 * 16 * kD * 2 * 2 + (kThreads / 32) * 2 * kQBytes; }
};

template <bool kBf16, int kD, bool kBias>
__global__ void __launch_bounds__(kThreads) cross_keep_kernel(const __grid_constant__ CrossParams p, int chunks) {
  using Cf = KeepCfg<kD>;
  constexpr int kCh = Cf::kChunks, kKW = 32, kWarps = kThreads / 32;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ uint32_t on[kMaxKeep / 32];  // bit per key that counts
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int kp = (p.sk + 15) & ~15;
  const int chunk = blockIdx.x % chunks, bh = blockIdx.x / chunks;
  const int kvh = bh % p.kv_heads, b = bh / p.kv_heads;
  const int len = cross_len(p, b);
  const uint32_t sk = smem_u32(smem), sv = sk + kp * kD * 2;
  const uint32_t sq = sv + kp * kD * 2 + warp * 2 * Cf::kQBytes;
  const uint16_t* kg = p.k + b * p.kb + kvh * p.kh;
  const uint16_t* vg = p.v + b * p.vb + kvh * p.vh;
  const uint8_t* mg = p.key_mask ? p.key_mask + b * p.mask_stride : nullptr;

  // this CTA's 16-row tiles, dealt to its warps
  const int tiles = (p.rows + 15) / 16;
  const int t0 = static_cast<int>(static_cast<int64_t>(tiles) * chunk / chunks);
  const int t1 = static_cast<int>(static_cast<int64_t>(tiles) * (chunk + 1) / chunks);
  auto load_q = [&](int t, int buf) {
    if (t < t1) {
#pragma unroll
      for (int i = 0; i < 16 * kCh / 32; ++i) {
        const int r = (lane + i * 32) / kCh, c = (lane + i * 32) % kCh, row = t * 16 + r;
        const bool ok = row < p.rows && c * 8 < p.head_dim;
        const int q = ok ? row / p.group : 0, h = ok ? row - q * p.group : 0;
        const uint16_t* src = p.q + b * p.qb + q * p.qs + (kvh * p.group + h) * p.qh + (ok ? c * 8 : 0);
        cp_async16(sq + buf * Cf::kQBytes + tile_at<kCh>(r, c), src, ok);
      }
    }
    cp_async_commit();
  };
  for (int i = tid; i < kp * kCh; i += kThreads) {
    const int r = i / kCh, c = i % kCh;
    bool ok = r < len && c * 8 < p.head_dim;
    if (mg && ok) ok = mg[r] != 0;
    const int64_t at = ok ? r : 0;
    const int cc = ok ? c * 8 : 0;
    cp_async16(sk + tile_at<kCh>(r, c), kg + at * p.ks + cc, ok);
    cp_async16(sv + tile_at<kCh>(r, c), vg + at * p.vs + cc, ok);
  }
  load_q(t0 + warp, 0);
  for (int w = warp; w < (kp + 31) / 32; w += kWarps) {
    const int key = w * 32 + lane;
    const uint32_t bits = __ballot_sync(0xffffffffu, key < len && (!mg || mg[key] != 0));
    if (lane == 0) on[w] = bits;
  }
  cp_async_wait<0>();
  __syncthreads();

  const float to_log2 = kBias ? kLog2e : p.scale_log2;
  int buf = 0;
  for (int t = t0 + warp; t < t1; t += kWarps, buf ^= 1) {
    load_q(t + kWarps, buf ^ 1);
    cp_async_wait<1>();
    __syncwarp();
    const uint32_t mine = sq + buf * Cf::kQBytes;
    uint32_t qf[kD / 16][4];
#pragma unroll
    for (int kk = 0; kk < kD / 16; ++kk)
      ldsm_x4(mine + tile_at<kCh>(lane & 15, kk * 2 + (lane >> 4)), qf[kk][0], qf[kk][1], qf[kk][2], qf[kk][3]);
    const float* brow[2] = {nullptr, nullptr};
    if (kBias) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = min(t * 16 + (lane >> 2) + 8 * h, p.rows - 1);
        brow[h] = p.bias + b * p.bb + (kvh * p.group + r % p.group) * p.bh + (r / p.group) * p.bs;
      }
    }
    RowState<kD> st;
    st.clear();
    for (int k0 = 0; k0 < len; k0 += kKW) {
      const int n = min(kKW, (len - k0 + 15) & ~15);  // keys of the chunk, a multiple of 16
      float s[kKW / 8][4];
#pragma unroll
      for (int jp = 0; jp < kKW / 16; ++jp) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[2 * jp][e] = s[2 * jp + 1][e] = 0.f;
        if (jp * 16 < n) {
#pragma unroll
          for (int kk = 0; kk < kD / 16; ++kk) {
            const int r = k0 + jp * 16 + (lane & 7) + (lane >> 4) * 8;
            uint32_t b0, b1, b2, b3;
            ldsm_x4(sk + tile_at<kCh>(r, kk * 2 + ((lane >> 3) & 1)), b0, b1, b2, b3);
            mma16816<kBf16>(s[2 * jp], qf[kk], b0, b1);
            mma16816<kBf16>(s[2 * jp + 1], qf[kk], b2, b3);
          }
        }
      }
      const uint32_t bits = on[k0 / 32];
#pragma unroll
      for (int j = 0; j < kKW / 8; ++j) {
        if (kBias && j * 8 < n) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = k0 + j * 8 + (lane & 3) * 2 + (e & 1);
            s[j][e] = fmaf(s[j][e], p.scale, key < len ? __ldg(brow[e >> 1] + key) : 0.f);
          }
        }
      }
      if (bits != ~0u) {
        const uint32_t mine_on = bits >> ((lane & 3) * 2);
#pragma unroll
        for (int j = 0; j < kKW / 8; ++j) {
          if (!(mine_on >> (j * 8) & 1)) s[j][0] = s[j][2] = -INFINITY;
          if (!(mine_on >> (j * 8 + 1) & 1)) s[j][1] = s[j][3] = -INFINITY;
        }
      }
      st.template softmax<kKW, kBf16>(s, to_log2);
      // O += P V, P rounded to the operands' type
#pragma unroll
      for (int kk = 0; kk < kKW / 16; ++kk) {
        if (kk * 16 < n) {
          uint32_t pa[4];
          pa[0] = pack2<kBf16>(s[2 * kk][0], s[2 * kk][1]);
          pa[1] = pack2<kBf16>(s[2 * kk][2], s[2 * kk][3]);
          pa[2] = pack2<kBf16>(s[2 * kk + 1][0], s[2 * kk + 1][1]);
          pa[3] = pack2<kBf16>(s[2 * kk + 1][2], s[2 * kk + 1][3]);
#pragma unroll
          for (int jp = 0; jp < kD / 16; ++jp) {
            const int r = k0 + kk * 16 + (lane & 15);
            uint32_t b0, b1, b2, b3;
            ldsm_x4_t(sv + tile_at<kCh>(r, jp * 2 + (lane >> 4)), b0, b1, b2, b3);
            mma16816<kBf16>(st.acc[2 * jp], pa, b0, b1);
            mma16816<kBf16>(st.acc[2 * jp + 1], pa, b2, b3);
          }
        }
      }
    }
    // O over the tile's queries in shared memory, then rows in 16-byte pieces
    __syncwarp();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float l = st.l[h];
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // no key: zeros; NaN stays NaN
      const int r = (lane >> 2) + 8 * h;
#pragma unroll
      for (int j = 0; j < kD / 8; ++j) {
        const uint32_t w = pack2<kBf16>(st.acc[j][2 * h] * inv, st.acc[j][2 * h + 1] * inv);
        asm volatile("st.shared.b32 [%0], %1;" ::"r"(mine + tile_at<kCh>(r, j) + (lane & 3) * 4), "r"(w) : "memory");
      }
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 16 * kCh / 32; ++i) {
      const int r = (lane + i * 32) / kCh, c = (lane + i * 32) % kCh, row = t * 16 + r;
      if (row < p.rows && c * 8 < p.head_dim) {
        uint4 w;
        asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                     : "r"(mine + tile_at<kCh>(r, c))
                     : "memory");
        const int q = row / p.group, h = row - q * p.group;
        *reinterpret_cast<uint4*>(p.o + b * p.ob + q * p.os + (kvh * p.group + h) * p.oh + c * 8) = w;
      }
    }
    __syncwarp();  // the buffer's next queries may come
  }
}

// Sets a kernel's shared memory limit, once per device.
int allow_smem(const void* kernel, int bytes, bool wide_cluster, std::atomic<uint64_t>& ready) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return kErrCuda;
  if (dev >= 64 || !(ready.load() >> dev & 1)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess ||
        (wide_cluster &&
         cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)) {
      cudaGetLastError();
      return kErrCuda;
    }
    if (dev < 64) ready.fetch_or(1ull << dev);
  }
  return kOk;
}

template <class... A>
int launch_split(void (*kernel)(A...), int64_t items, int splits, int threads, int smem, cudaStream_t st,
                 bool cluster, const A&... args) {
  if (items * splits > 0x7fffffffLL) return kErrShape;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(static_cast<unsigned>(items * splits));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  if (cluster && splits > 1) {
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = splits;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
  }
  count_launches(1);
  if (cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess) return kOk;
  cudaGetLastError();  // the next call's own check must not see it
  return kErrLaunch;
}

template <bool kBf16, int kD, bool kBias>
int launch_few(const CrossParams& p, cudaStream_t st) {
  using Cf = FewCfg<kD>;
  static std::atomic<uint64_t> ready{0};
  const auto kernel = cross_few_kernel<kBf16, kD, kBias>;
  if (int rc = allow_smem(reinterpret_cast<const void*>(kernel), Cf::kSmem, true, ready)) return rc;
  CUtensorMap mk, mv;
  KvShare share;
  if (!make_kv_maps(p, kBf16 ? kBF16 : kF16, Cf::kKT, &mk, &mv, &share)) return kErrTma;
  const int row_tiles = (p.rows + Cf::kRows - 1) / Cf::kRows;
  const int64_t items = static_cast<int64_t>(row_tiles) * p.kv_heads * p.batch;
  static ClusterTable clusters;
  const int key_tiles = (p.sk + Cf::kKT - 1) / Cf::kKT;
  // Few items over long states: a cluster of 16 CTAs for each leaves SMs idle
  // (and only 7 such clusters fit where a CTA takes most of an SM).  From 16 MB
  // of K and V on the keys are split over all SMs, and a second launch adds the
  // parts up out of a workspace: 8 items, 235 MB: 48 -> 45 us; 4 items, 134 MB:
  // 35 -> 31; 1 item, 34 MB: 28 -> 14, 17 MB: 17 -> 12.
  const int64_t slots = static_cast<int64_t>(200 * 1024 / Cf::kSmem) * num_sms();
  const int64_t kv_bytes = 4ll * p.sk * p.head_dim * p.kv_heads * p.batch;
  if (items <= slots / 3 && kv_bytes >= (16ll << 20)) {
    const int splits = static_cast<int>(std::min<int64_t>(slots / items, key_tiles / 4));
    float* ws = nullptr;
    const size_t bytes = static_cast<size_t>(items) * splits * Cf::kRows * (kD + 2) * 4;
    if (splits > 1 && pool_alloc(reinterpret_cast<void**>(&ws), bytes, st) == cudaSuccess) {
      int rc = launch_split(kernel, items, splits, Cf::kThreads, Cf::kSmem, st, false, mk, mv, p, share, row_tiles,
                            splits, ws);
      if (!rc) {
        count_launches(1);
        cross_join_kernel<kBf16, kD><<<static_cast<unsigned>(items * Cf::kRows), kD, 0, st>>>(
            p, row_tiles, splits, ws, kBias ? kLog2e : p.scale_log2);
        if (cudaGetLastError() != cudaSuccess) rc = kErrLaunch;
      }
      cudaFreeAsync(ws, st);
      return rc;
    }
    cudaGetLastError();
  }
  const int splits = cluster_splits(kernel, Cf::kThreads, Cf::kSmem, items, key_tiles, 2, 16, clusters);
  return launch_split(kernel, items, splits, Cf::kThreads, Cf::kSmem, st, true, mk, mv, p, share, row_tiles, splits,
                      static_cast<float*>(nullptr));
}

template <bool kBf16, int kD, bool kBias>
int launch_rows_any(const CrossParams& p, cudaStream_t st) {
  using Cf = RowsCfg<kD, kBias>;
  static std::atomic<uint64_t> ready{0};
  const auto kernel = cross_rows_kernel<kBf16, kD, kBias>;
  if (int rc = allow_smem(reinterpret_cast<const void*>(kernel), Cf::kSmem, true, ready)) return rc;
  const int row_tiles = static_cast<int>((static_cast<int64_t>(p.rows) + Cf::kRows - 1) / Cf::kRows);
  const int64_t items = static_cast<int64_t>(row_tiles) * p.kv_heads * p.batch;
  static ClusterTable clusters;
  const int splits = cluster_splits(kernel, kThreads, Cf::kSmem, items, (p.sk + Cf::kKT - 1) / Cf::kKT, 8, 16, clusters);
  const bool wide = p.bias && (reinterpret_cast<uintptr_t>(p.bias) & 15) == 0 && p.sk % 4 == 0 && p.bb % 4 == 0 &&
                    p.bh % 4 == 0 && p.bs % 4 == 0;
  return launch_split(kernel, items, splits, kThreads, Cf::kSmem, st, true, p, row_tiles, splits, wide ? 4 : 1);
}

template <bool kBf16, int kD, bool kBias>
int launch_keep(const CrossParams& p, cudaStream_t st) {
  const auto kernel = cross_keep_kernel<kBf16, kD, kBias>;
  static std::atomic<uint64_t> ready{0};
  if (int rc = allow_smem(reinterpret_cast<const void*>(kernel), 200 * 1024, false, ready)) return rc;
  static const int regs = [&] {
    cudaFuncAttributes fa;
    if (cudaFuncGetAttributes(&fa, kernel) == cudaSuccess) return fa.numRegs;
    cudaGetLastError();  // the launch's own check must not see it
    return 255;
  }();
  const int smem = KeepCfg<kD>::smem(p.sk);
  // as many CTAs as the SMs hold at once, each with a share of the rows (one
  // more per SM than fits makes a second wave: 36 -> 50 us for image to text)
  const int64_t bh = static_cast<int64_t>(p.kv_heads) * p.batch;
  const int per_sm = std::max(1, std::min(65536 / ((regs + 7) / 8 * 8 * kThreads), 224 * 1024 / (smem + 1024)));
  const int tiles = (p.rows + 15) / 16;
  int64_t chunks = std::max<int64_t>(1, static_cast<int64_t>(per_sm) * num_sms() / bh);
  chunks = std::min<int64_t>(chunks, (tiles + kThreads / 32 - 1) / (kThreads / 32));
  if (bh * chunks > 0x7fffffffLL) return kErrShape;
  count_launches(1);
  kernel<<<static_cast<unsigned>(bh * chunks), kThreads, smem, st>>>(p, static_cast<int>(chunks));
  return cudaGetLastError() == cudaSuccess ? kOk : kErrLaunch;
}

template <bool kBf16, int kD>
int launch_rows(const CrossParams& p, cudaStream_t st) {
  if (p.rows > 64 && p.sk <= kMaxKeep && KeepCfg<kD>::smem(p.sk) <= 100 * 1024)
    return p.bias ? launch_keep<kBf16, kD, true>(p, st) : launch_keep<kBf16, kD, false>(p, st);
  if (p.rows <= 16 && cross_kv_maps(p))
    return p.bias ? launch_few<kBf16, kD, true>(p, st) : launch_few<kBf16, kD, false>(p, st);
  return p.bias ? launch_rows_any<kBf16, kD, true>(p, st) : launch_rows_any<kBf16, kD, false>(p, st);
}

}  // namespace

int launch_cross_mma(const CrossParams& p, int dtype, cudaStream_t st) {
  const bool bf = dtype == kBF16;
  if (p.head_dim <= 32) return bf ? launch_rows<true, 32>(p, st) : launch_rows<false, 32>(p, st);
  if (p.head_dim <= 64) return bf ? launch_rows<true, 64>(p, st) : launch_rows<false, 64>(p, st);
  return bf ? launch_rows<true, 128>(p, st) : launch_rows<false, 128>(p, st);
}

}  // namespace s3

using namespace s3;

namespace {

// A first call sets kernels' attributes and makes the pool; while another or
// this thread captures in the strict mode such calls end the capture.
struct RelaxedCapture {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  RelaxedCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
  ~RelaxedCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
};

}  // namespace

extern "C" int sam3cu_cross_attention(const struct sam3cu_cross_attention_args* a, void* stream) {
  if (!a) return SAM3CU_EINVAL;
  if (a->dtype != SAM3CU_BF16 && a->dtype != SAM3CU_F16) return SAM3CU_EDTYPE;
  if (a->batch < 0 || a->sq < 0 || a->sk < 0 || a->q_heads < 0 || a->kv_heads < 1 || a->head_dim < 1)
    return SAM3CU_EINVAL;
  if (a->q_heads % a->kv_heads) return SAM3CU_EINVAL;
  if (!(a->scale >= 0.f) || std::isinf(a->scale * kLog2e)) return SAM3CU_EINVAL;
  if (a->head_dim % 8 || a->head_dim > 128) return SAM3CU_ESHAPE;
  if (a->batch == 0 || a->sq == 0 || a->q_heads == 0) return SAM3CU_OK;
  const int group = a->q_heads / a->kv_heads;
  if (a->sk > 0x7fffff00) return SAM3CU_ESHAPE;
  if (group > 128 || static_cast<int64_t>(a->sq) * group > 0x7fffff00LL) return SAM3CU_ESHAPE;
  if (!a->q || !a->o || (a->sk > 0 && (!a->k || !a->v))) return SAM3CU_EINVAL;
  CrossParams p;
  memset(&p, 0, sizeof(p));
  const int64_t* from[4] = {a->q_strides, a->k_strides, a->v_strides, a->o_strides};
  int64_t* to[4][3] = {{&p.qb, &p.qs, &p.qh}, {&p.kb, &p.ks, &p.kh}, {&p.vb, &p.vs, &p.vh}, {&p.ob, &p.os, &p.oh}};
  const void* base[4] = {a->q, a->k, a->v, a->o};
  for (int t = 0; t < 4; ++t) {
    const int extent[3] = {a->batch, t == 0 || t == 3 ? a->sq : a->sk, t == 0 || t == 3 ? a->q_heads : a->kv_heads};
    if (reinterpret_cast<uintptr_t>(base[t]) & 15) return SAM3CU_ESHAPE;
    for (int i = 0; i < 3; ++i) {
      if (from[t][i] < 0) return SAM3CU_EINVAL;
      if (extent[i] <= 1) continue;  // the stride of a single element says nothing
      if (from[t][i] % 8) return SAM3CU_ESHAPE;
      if (t == 3 && from[t][i] == 0) return SAM3CU_EINVAL;  // every output element has a place of its own
      *to[t][i] = from[t][i];
    }
  }
  p.q = static_cast<const uint16_t*>(a->q);
  p.k = static_cast<const uint16_t*>(a->k);
  p.v = static_cast<const uint16_t*>(a->v);
  p.o = static_cast<uint16_t*>(a->o);
  p.batch = a->batch;
  p.sq = a->sq;
  p.sk = a->sk;
  p.kv_heads = a->kv_heads;
  p.group = group;
  p.head_dim = a->head_dim;
  p.rows = a->sq * group;
  p.scale = a->scale > 0.f ? a->scale : 1.f / sqrtf(static_cast<float>(a->head_dim));
  p.scale_log2 = p.scale * kLog2e;
  if (a->k_lens) {
    if (reinterpret_cast<uintptr_t>(a->k_lens) & 3) return SAM3CU_EINVAL;
    p.k_lens = a->k_lens;
  }
  if (a->key_mask) {
    if (a->mask_stride < 0) return SAM3CU_EINVAL;
    p.key_mask = a->key_mask;
    p.mask_stride = a->mask_stride;
  }
  if (a->bias) {
    if (reinterpret_cast<uintptr_t>(a->bias) & 3) return SAM3CU_EINVAL;
    for (int i = 0; i < 3; ++i)
      if (a->bias_strides[i] < 0) return SAM3CU_EINVAL;
    p.bias = a->bias;
    p.bb = a->bias_strides[0];
    p.bh = a->bias_strides[1];
    p.bs = a->bias_strides[2];
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const RelaxedCapture relaxed;
  // Which kernel: tcgen05 for many rows, except over few keys where heads are
  // small or the whole call is (4 x 8 heads x 5184 queries, D = 32: 77 keys 17
  // us kept in shared memory, 23 us on tcgen05, 128 keys 21 and 22, 256 keys 36
  // and 31; D = 64, 77 keys: 28 and 26, 128 keys: 34 and 25; 8 heads x 300
  // queries, D = 64, 77 keys: 5.3 and 6.9, 128 keys 6.2 and 6.9).
  const bool small = p.sk <= 128 && (p.head_dim <= 32 || static_cast<int64_t>(p.rows) * p.kv_heads * p.batch <=
                                                             128ll * num_sms());
  if (p.rows > 64 && !small && cross_tc_takes(p)) {
    const int rc = launch_cross_tc(p, a->dtype, st);
    if (rc != kCrossTcSpills) return rc;
  }
  return launch_cross_mma(p, a->dtype, st);
}
