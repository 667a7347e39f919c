// rotary.cu - rotary positions and per-head norms of queries and keys.
//
//   rope_pos       (u, w) -> a (u cos - w sin, u sin + w cos) per pair of a
//                  head, the angle 2 pi p f_i formed from the token's
//                  position p and the pair's frequency f_i
//   qk_norm_rope   RMS norm or LayerNorm over each head, then the rotation
//
// Both read and write every element once and do a few operations on it, so
// HBM bounds them; what they must not do is let anything else cost more than
// the data.  p f_i is formed and reduced in 64 bits (f_i in revolutions, so
// the reduction is a subtraction of the nearest integer), cosine and sine in
// F32 of the remainder: once per token and pair, into a shared-memory table
// of the CTA's tokens that all their heads then read.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <cstring>

#include "../../include/sam3cu.h"
#include "sam3cu_internal.h"

using namespace s3;

namespace {

constexpr int kWarps = 8;   // per CTA
constexpr int kThreads = 32 * kWarps;
constexpr int kMaxTokens = 32;  // of a CTA (rotary_vec)
constexpr int kMaxDim = 2 * SAM3CU_ROPE_MAX_PAIRS;

enum : int { kNormNone = 0, kNormRms = SAM3CU_NORM_RMS, kNormLayer = SAM3CU_NORM_LAYER };

struct View {
  const void* x;
  void* y;
  int64_t xb, xs, xh, yb, ys, yh;
  const float* gamma;
  const float* beta;
};

struct Params {
  View v[2];           // q, k
  int q_heads, heads;  // heads of q, of q and k together
  int slices;          // rotary_any: warps that share a token's heads,
  int per_slice;       //   and the heads of one
  int block_tokens;    // rotary_vec: tokens of a CTA
  int64_t tokens;      // batch * seq
  int seq, head_dim;
  const int64_t* positions;
  int64_t pos_stride, start;
  float eps;
  sam3cu_rope_freqs f;
};

template <int T>
__device__ __forceinline__ float ld1(const void* p, int64_t i) {
  if (T == kF32) return static_cast<const float*>(p)[i];
  if (T == kBF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}
template <int T>
__device__ __forceinline__ void st1(void* p, int64_t i, float v) {
  if (T == kF32) static_cast<float*>(p)[i] = v;
  else if (T == kBF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

// Eight elements as loaded: one 16-byte word, or two for F32.
template <int T>
struct Raw8 {
  uint4 w[T == kF32 ? 2 : 1];
};
template <int T>
__device__ __forceinline__ Raw8<T> ld8(const void* p, int64_t i) {
  Raw8<T> r;
  const uint4* s = reinterpret_cast<const uint4*>(static_cast<const char*>(p) + i * (T == kF32 ? 4 : 2));
  r.w[0] = s[0];
  if constexpr (T == kF32) r.w[1] = s[1];
  return r;
}
template <int T>
__device__ __forceinline__ void unpack8(const Raw8<T>& r, float* f) {
  if constexpr (T == kF32) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      f[4 * k] = __uint_as_float(r.w[k].x);
      f[4 * k + 1] = __uint_as_float(r.w[k].y);
      f[4 * k + 2] = __uint_as_float(r.w[k].z);
      f[4 * k + 3] = __uint_as_float(r.w[k].w);
    }
  } else {
    const uint32_t w[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float2 v;
      if (T == kBF16) v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[k]));
      else v = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
      f[2 * k] = v.x;
      f[2 * k + 1] = v.y;
    }
  }
}
template <int T>
__device__ __forceinline__ void st8(void* p, int64_t i, const float* f) {
  uint4* d = reinterpret_cast<uint4*>(static_cast<char*>(p) + i * (T == kF32 ? 4 : 2));
  if constexpr (T == kF32) {
    d[0] = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    d[1] = make_uint4(__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7]));
  } else {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (T == kBF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * k], f[2 * k + 1]);
        w[k] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __half2 h = __floats2half2_rn(f[2 * k], f[2 * k + 1]);
        w[k] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    d[0] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// The warp's place: token and the heads [h0, h1) of q and k together.
struct Place {
  int b, s, h0, h1;
};
__device__ __forceinline__ bool place_of(const Params& p, int warp, Place& at) {
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
  if (item >= p.tokens * p.slices) return false;
  int64_t token = item;
  int slice = 0;
  if (p.slices > 1) {
    token = item / p.slices;
    slice = static_cast<int>(item - token * p.slices);
  }
  at.b = static_cast<int>(token / p.seq);
  at.s = static_cast<int>(token - static_cast<int64_t>(at.b) * p.seq);
  at.h0 = slice * p.per_slice;
  at.h1 = min(p.heads, at.h0 + p.per_slice);
  return true;
}

// amplitude * (cos, sin) of pair i at a position: the product in 64 bits,
// whole revolutions dropped, the rest (at most half a revolution) in F32.
__device__ __forceinline__ float2 turn(const Params& p, double pos, int i) {
  const double t = pos * p.f.turns[i];
  float s, c;
  sincospif(static_cast<float>(2.0 * (t - rint(t))), &s, &c);
  return make_float2(c * p.f.amplitude, s * p.f.amplitude);
}

__device__ __forceinline__ double position_of(const Params& p, const Place& at) {
  return static_cast<double>(p.positions ? p.positions[at.b * p.pos_stride + at.s] : p.start + at.s);
}

// Heads whose dimensions are multiples of 16 and whose rows start on 16
// bytes.  A lane holds 16 elements of a head: in the interleaved layout 16
// consecutive ones, in the half layout 8 from either half, so both elements
// of a pair are always in one lane and a head takes head_dim / 16 lanes (the
// next power of two, kG, for the reductions).  The CTA's (token, head) pairs
// are dealt to its lane groups in order, so no lane idles however many heads
// there are; a group has two heads' loads in flight.
template <int T, int kNorm, bool kRot, int kG>
__global__ void __launch_bounds__(kThreads, kNorm == kNormLayer ? 2 : 3) rotary_vec(const __grid_constant__ Params p) {
  constexpr int kGroups = kThreads / kG;
  constexpr int kES = T == kF32 ? 4 : 2;
  constexpr int kU = 2;
  // cos and sin of pairs 8 slot + 2 jj, + 1 at [token][jj][slot]: the lanes
  // of a head read consecutive words
  extern __shared__ float4 table[];
  __shared__ int64_t offs[4][kMaxTokens];  // a token's row in q's x, q's y, k's x, k's y
  const int tid = threadIdx.x;
  const int64_t token0 = static_cast<int64_t>(blockIdx.x) * p.block_tokens;
  const int n_tok = static_cast<int>(min(static_cast<int64_t>(p.block_tokens), p.tokens - token0));
  const int rslots = kRot ? p.f.n_pairs / 8 : 0;  // slots that are rotated
  const int slot = tid % kG, group = tid / kG;
  const bool turned = kRot && slot < rslots;
  const bool half = kRot && p.f.layout == SAM3CU_ROPE_HALF;
  const int e0 = (half && turned) ? 8 * slot : 16 * slot;
  const int e1 = (half && turned) ? p.f.n_pairs + 8 * slot : 16 * slot + 8;
  const bool have = slot * 16 < p.head_dim;

  for (int i = tid; i < n_tok; i += kThreads) {
    const int64_t token = token0 + i;
    const int64_t b = token / p.seq, s = token - b * p.seq;
    offs[0][i] = b * p.v[0].xb + s * p.v[0].xs;
    offs[1][i] = b * p.v[0].yb + s * p.v[0].ys;
    offs[2][i] = b * p.v[1].xb + s * p.v[1].xs;
    offs[3][i] = b * p.v[1].yb + s * p.v[1].ys;
  }
  if constexpr (kRot) {
    for (int i = tid; i < n_tok * rslots * 4; i += kThreads) {
      const int per = rslots * 4, tok = i / per, at = i - tok * per;
      const int jj = at / rslots, sl = at - jj * rslots;
      const int64_t token = token0 + tok;
      const int64_t b = token / p.seq, s = token - b * p.seq;
      const double pos = static_cast<double>(p.positions ? p.positions[b * p.pos_stride + s] : p.start + s);
      const float2 c0 = turn(p, pos, 8 * sl + 2 * jj), c1 = turn(p, pos, 8 * sl + 2 * jj + 1);
      table[i] = make_float4(c0.x, c0.y, c1.x, c1.y);
    }
  }
  __syncthreads();

#pragma unroll 1
  for (int part = 0; part < 2; ++part) {
    const int heads = part ? p.heads - p.q_heads : p.q_heads;
    const View& v = p.v[part];
    // without a norm, what is not rotated need not move where it already is
    const bool mine = have && !(kNorm == kNormNone && v.x == v.y && !turned);
    const char* x = static_cast<const char*>(v.x);
    char* y = static_cast<char*>(v.y);
    float g[kNorm ? 16 : 1], bt[kNorm == kNormLayer ? 16 : 1];
    if (kNorm && have && heads > 0) {
#pragma unroll
      for (int k = 0; k < 16; k += 4) {
        const int e = k < 8 ? e0 + k : e1 + k - 8;
        float4 w = v.gamma ? __ldg(reinterpret_cast<const float4*>(v.gamma + e)) : make_float4(1.f, 1.f, 1.f, 1.f);
        g[kNorm ? k : 0] = w.x;
        g[kNorm ? k + 1 : 0] = w.y;
        g[kNorm ? k + 2 : 0] = w.z;
        g[kNorm ? k + 3 : 0] = w.w;
        if (kNorm == kNormLayer) {
          w = v.beta ? __ldg(reinterpret_cast<const float4*>(v.beta + e)) : make_float4(0.f, 0.f, 0.f, 0.f);
          bt[kNorm == kNormLayer ? k : 0] = w.x;
          bt[kNorm == kNormLayer ? k + 1 : 0] = w.y;
          bt[kNorm == kNormLayer ? k + 2 : 0] = w.z;
          bt[kNorm == kNormLayer ? k + 3 : 0] = w.w;
        }
      }
    }
    const int units = n_tok * heads;
    int tok = heads ? group / heads : 0, head = heads ? group - tok * heads : 0;
    const int step_t = heads ? kGroups / heads : 0, step_h = heads ? kGroups - step_t * heads : 0;
    // (all lanes of a warp stay in the loop while one has a unit: shuffles)
    for (int w0 = (tid / 32) * (32 / kG); w0 < units; w0 += kU * kGroups) {
      Raw8<T> ra[kU], rb[kU];
      int tk[kU], hd[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        tk[u] = tok;
        hd[u] = head;
        if (mine && tok < n_tok) {
          const char* src = x + (offs[2 * part][tok] + head * v.xh) * kES;
          ra[u] = ld8<T>(src, e0);
          rb[u] = ld8<T>(src, e1);
        }
        tok += step_t;
        head += step_h;
        if (head >= heads) {
          head -= heads;
          ++tok;
        }
      }
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const bool live = mine && tk[u] < n_tok;
        float f[16];
        if (live) {
          unpack8<T>(ra[u], f);
          unpack8<T>(rb[u], f + 8);
        } else {
#pragma unroll
          for (int k = 0; k < 16; ++k) f[k] = 0.f;
        }
        if (kNorm) {
          const float n = 1.f / static_cast<float>(p.head_dim);
          if (kNorm == kNormLayer) {
            float sum = 0.f;
#pragma unroll
            for (int k = 0; k < 16; ++k) sum += f[k];
#pragma unroll
            for (int o = kG / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            const float mean = live ? sum * n : 0.f;
#pragma unroll
            for (int k = 0; k < 16; ++k) f[k] -= mean;
          }
          float sq = 0.f;
#pragma unroll
          for (int k = 0; k < 16; ++k) sq = fmaf(f[k], f[k], sq);
#pragma unroll
          for (int o = kG / 2; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
          const float inv = 1.f / sqrtf(fmaf(sq, n, p.eps));
          if (live) {
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              if (kNorm == kNormLayer) f[k] = fmaf(f[k] * inv, g[kNorm ? k : 0], bt[kNorm == kNormLayer ? k : 0]);
              else f[k] = f[k] * inv * g[kNorm ? k : 0];
            }
            if (kNorm == kNormRms && v.beta) {  // uncommon: read as it is used
#pragma unroll
              for (int k = 0; k < 16; ++k) f[k] += __ldg(v.beta + (k < 8 ? e0 + k : e1 + k - 8));
            }
          }
        }
        if (live) {
          if (turned) {
            const float4* cs = table + tk[u] * rslots * 4 + slot;
#pragma unroll
            for (int jj = 0; jj < 4; ++jj) {
              const float4 c = cs[jj * rslots];
              if (half) {
                const float a0 = f[2 * jj], b0 = f[8 + 2 * jj], a1 = f[2 * jj + 1], b1 = f[9 + 2 * jj];
                f[2 * jj] = a0 * c.x - b0 * c.y;
                f[8 + 2 * jj] = a0 * c.y + b0 * c.x;
                f[2 * jj + 1] = a1 * c.z - b1 * c.w;
                f[9 + 2 * jj] = a1 * c.w + b1 * c.z;
              } else {
                const float a0 = f[4 * jj], b0 = f[4 * jj + 1], a1 = f[4 * jj + 2], b1 = f[4 * jj + 3];
                f[4 * jj] = a0 * c.x - b0 * c.y;
                f[4 * jj + 1] = a0 * c.y + b0 * c.x;
                f[4 * jj + 2] = a1 * c.z - b1 * c.w;
                f[4 * jj + 3] = a1 * c.w + b1 * c.z;
              }
            }
          }
          char* dst = y + (offs[2 * part + 1][tk[u]] + hd[u] * v.yh) * kES;
          st8<T>(dst, e0, f);
          st8<T>(dst, e1, f + 8);
        }
      }
    }
  }
}

// Any head_dim, rotated part, alignment and stride: a lane holds the pairs
// lane, lane + 32, ... of a head (kP of them at most) and, behind them, the
// elements that are not rotated.
template <int T, int kNorm, int kP>
__global__ void __launch_bounds__(kWarps * 32) rotary_any(const __grid_constant__ Params p, int rot) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Place at;
  if (!place_of(p, warp, at)) return;
  const int pairs = rot / 2, rest = p.head_dim - rot;
  const bool half = p.f.layout == SAM3CU_ROPE_HALF;
  float2 cs[kP];
  if (rot) {
    const double pos = position_of(p, at);
#pragma unroll
    for (int k = 0; k < kP; ++k)
      if (lane + 32 * k < pairs) cs[k] = turn(p, pos, lane + 32 * k);
  }
#pragma unroll 2
  for (int hh = at.h0; hh < at.h1; ++hh) {
    const int part = hh >= p.q_heads;
    const View& v = p.v[part];
    const int64_t h = hh - (part ? p.q_heads : 0);
    const int64_t xo = at.b * v.xb + at.s * v.xs + h * v.xh, yo = at.b * v.yb + at.s * v.ys + h * v.yh;
    float a[kP], b[kP], c[2 * kP];
#pragma unroll
    for (int k = 0; k < kP; ++k) {
      const int i = lane + 32 * k;
      a[k] = b[k] = 0.f;
      if (i < pairs) {
        a[k] = ld1<T>(v.x, xo + (half ? i : 2 * i));
        b[k] = ld1<T>(v.x, xo + (half ? pairs + i : 2 * i + 1));
      }
    }
#pragma unroll
    for (int k = 0; k < 2 * kP; ++k) {
      const int i = lane + 32 * k;
      c[k] = i < rest ? ld1<T>(v.x, xo + rot + i) : 0.f;
    }
    if (kNorm) {
      const float n = static_cast<float>(p.head_dim);
      float sum = 0.f, mean = 0.f, sq = 0.f;
      if (kNorm == kNormLayer) {
#pragma unroll
        for (int k = 0; k < kP; ++k) sum += (a[k] + b[k]) + (c[2 * k] + c[2 * k + 1]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        mean = sum / n;
      }
#pragma unroll
      for (int k = 0; k < kP; ++k) {
        if (lane + 32 * k < pairs) {
          a[k] -= mean;
          b[k] -= mean;
          sq += a[k] * a[k] + b[k] * b[k];
        }
      }
#pragma unroll
      for (int k = 0; k < 2 * kP; ++k) {
        if (lane + 32 * k < rest) {
          c[k] -= mean;
          sq = fmaf(c[k], c[k], sq);
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
      const float inv = 1.f / sqrtf(sq / n + p.eps);
      auto scaled = [&](float f, int e) {
        return fmaf(f * inv, v.gamma ? __ldg(v.gamma + e) : 1.f, v.beta ? __ldg(v.beta + e) : 0.f);
      };
#pragma unroll
      for (int k = 0; k < kP; ++k) {
        const int i = lane + 32 * k;
        if (i < pairs) {
          a[k] = scaled(a[k], half ? i : 2 * i);
          b[k] = scaled(b[k], half ? pairs + i : 2 * i + 1);
        }
      }
#pragma unroll
      for (int k = 0; k < 2 * kP; ++k)
        if (lane + 32 * k < rest) c[k] = scaled(c[k], rot + lane + 32 * k);
    }
#pragma unroll
    for (int k = 0; k < kP; ++k) {
      const int i = lane + 32 * k;
      if (i < pairs) {
        st1<T>(v.y, yo + (half ? i : 2 * i), a[k] * cs[k].x - b[k] * cs[k].y);
        st1<T>(v.y, yo + (half ? pairs + i : 2 * i + 1), a[k] * cs[k].y + b[k] * cs[k].x);
      }
    }
    if (kNorm || v.x != v.y) {
#pragma unroll
      for (int k = 0; k < 2 * kP; ++k)
        if (lane + 32 * k < rest) st1<T>(v.y, yo + rot + lane + 32 * k, c[k]);
    }
  }
}

template <int T, int kNorm>
int launch_typed(Params& p, int rot, bool vec, cudaStream_t st) {
  count_launches(1);
  if (vec) {
    const int lanes = p.head_dim / 16;
    const int g = lanes <= 1 ? 1 : lanes <= 2 ? 2 : lanes <= 4 ? 4 : lanes <= 8 ? 8 : 16;
    // Tokens of a CTA: as many as leave two CTAs to an SM, up to 32 (the
    // table's and the gammas' cost is then spread over the most heads).
    int bt = kMaxTokens;
    while (bt > 1 && (p.tokens + bt - 1) / bt < 2 * num_sms()) bt /= 2;
    p.block_tokens = bt;
    const int64_t blocks = (p.tokens + bt - 1) / bt;
    if (blocks > 0x7fffffffLL) return SAM3CU_ESHAPE;
    const dim3 grid(static_cast<unsigned>(blocks));
    const size_t smem = static_cast<size_t>(bt) * (rot / 16) * 64;
#define S3_ROT(G)                                                            \
  case G:                                                                    \
    if (rot) rotary_vec<T, kNorm, true, G><<<grid, kThreads, smem, st>>>(p); \
    else rotary_vec<T, kNorm, false, G><<<grid, kThreads, 0, st>>>(p);       \
    break
    switch (g) {
      S3_ROT(1);
      S3_ROT(2);
      S3_ROT(4);
      S3_ROT(8);
      S3_ROT(16);
    }
#undef S3_ROT
  } else {
    // few tokens: more warps to a token, so that the call fills the SMs with
    // about eight warps each
    const int64_t want = static_cast<int64_t>(num_sms()) * 8;
    int64_t slices = (want + p.tokens - 1) / p.tokens;
    if (slices > p.heads) slices = p.heads;
    p.per_slice = (p.heads + static_cast<int>(slices) - 1) / static_cast<int>(slices);
    p.slices = (p.heads + p.per_slice - 1) / p.per_slice;
    const int64_t blocks = (p.tokens * p.slices + kWarps - 1) / kWarps;
    if (blocks > 0x7fffffffLL) return SAM3CU_ESHAPE;
    const dim3 grid(static_cast<unsigned>(blocks));
    if (p.head_dim <= 64) rotary_any<T, kNorm, 1><<<grid, kThreads, 0, st>>>(p, rot);
    else if (p.head_dim <= 128) rotary_any<T, kNorm, 2><<<grid, kThreads, 0, st>>>(p, rot);
    else rotary_any<T, kNorm, 4><<<grid, kThreads, 0, st>>>(p, rot);
  }
  return cudaGetLastError() == cudaSuccess ? SAM3CU_OK : SAM3CU_ELAUNCH;
}

template <int T>
int launch_norm(Params& p, int norm, int rot, bool vec, cudaStream_t st) {
  if (norm == kNormRms) return launch_typed<T, kNormRms>(p, rot, vec, st);
  if (norm == kNormLayer) return launch_typed<T, kNormLayer>(p, rot, vec, st);
  return launch_typed<T, kNormNone>(p, rot, vec, st);
}

// Checks a view and copies it; *vec is cleared where its rows do not start
// on 16 bytes.
int take_view(const sam3cu_head_view* h, int dtype, int batch, int seq, View* v, bool* vec) {
  memset(v, 0, sizeof(*v));
  if (!h || h->heads == 0) return SAM3CU_OK;
  if (h->heads < 0) return SAM3CU_EINVAL;
  if (batch == 0 || seq == 0) return SAM3CU_OK;
  if (!h->x || !h->y) return SAM3CU_EINVAL;
  const int es = dtype == kF32 ? 4 : 2, unit = 16 / es;
  const int extent[3] = {batch, seq, h->heads};
  int64_t xs[3], ys[3];
  for (int i = 0; i < 3; ++i) {
    if (h->x_strides[i] < 0 || h->y_strides[i] < 0) return SAM3CU_EINVAL;
    xs[i] = extent[i] > 1 ? h->x_strides[i] : 0;  // the stride of a single element says nothing
    ys[i] = extent[i] > 1 ? h->y_strides[i] : 0;
    if (extent[i] > 1 && ys[i] == 0) return SAM3CU_EINVAL;  // every output element has a place of its own
    if (xs[i] % unit || ys[i] % unit) *vec = false;
  }
  const uintptr_t px = reinterpret_cast<uintptr_t>(h->x), py = reinterpret_cast<uintptr_t>(h->y);
  if (px % es || py % es) return SAM3CU_EINVAL;
  if ((px | py) & 15) *vec = false;
  if ((reinterpret_cast<uintptr_t>(h->gamma) | reinterpret_cast<uintptr_t>(h->beta)) & 15) *vec = false;
  if (h->x == h->y && memcmp(xs, ys, sizeof(xs))) return SAM3CU_EINVAL;
  if ((reinterpret_cast<uintptr_t>(h->gamma) | reinterpret_cast<uintptr_t>(h->beta)) & 3) return SAM3CU_EINVAL;
  *v = View{h->x, h->y, xs[0], xs[1], xs[2], ys[0], ys[1], ys[2], h->gamma, h->beta};
  return SAM3CU_OK;
}

int rotary_common(const sam3cu_head_view* q, const sam3cu_head_view* k, int dtype, int batch, int seq, int head_dim,
                  int norm, float eps, const int64_t* positions, int64_t pos_stride, int64_t start,
                  const sam3cu_rope_freqs* freqs, void* stream) {
  if (!q || batch < 0 || seq < 0 || head_dim < 1 || pos_stride < 0) return SAM3CU_EINVAL;
  if (dtype != SAM3CU_F32 && dtype != SAM3CU_F16 && dtype != SAM3CU_BF16) return SAM3CU_EDTYPE;
  if (head_dim > kMaxDim) return SAM3CU_ESHAPE;
  if (norm && !(eps >= 0.f)) return SAM3CU_EINVAL;
  int rot = 0;
  if (freqs) {
    if (freqs->n_pairs < 1 || freqs->n_pairs > SAM3CU_ROPE_MAX_PAIRS) return SAM3CU_EINVAL;
    if (freqs->layout != SAM3CU_ROPE_HALF && freqs->layout != SAM3CU_ROPE_INTERLEAVED) return SAM3CU_EINVAL;
    rot = 2 * freqs->n_pairs;
    if (rot > head_dim) return SAM3CU_ESHAPE;
    if (reinterpret_cast<uintptr_t>(positions) & 7) return SAM3CU_EINVAL;
  }
  Params p;
  bool vec = head_dim % 16 == 0 && rot % 16 == 0;
  int rc = take_view(q, dtype, batch, seq, &p.v[0], &vec);
  if (!rc) rc = take_view(k, dtype, batch, seq, &p.v[1], &vec);
  if (rc) return rc;
  p.q_heads = q->heads;
  const int64_t heads = static_cast<int64_t>(q->heads) + (k ? k->heads : 0);
  if (heads > (1 << 24)) return SAM3CU_ESHAPE;
  p.heads = static_cast<int>(heads);
  p.tokens = static_cast<int64_t>(batch) * seq;
  if (p.tokens == 0 || p.heads == 0) return SAM3CU_OK;
  p.seq = seq;
  p.head_dim = head_dim;
  p.positions = positions;
  p.pos_stride = pos_stride;
  p.start = start;
  p.eps = eps;
  if (freqs) p.f = *freqs;
  else memset(&p.f, 0, sizeof(p.f));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == SAM3CU_F32) return launch_norm<kF32>(p, norm, rot, vec, st);
  if (dtype == SAM3CU_F16) return launch_norm<kF16>(p, norm, rot, vec, st);
  return launch_norm<kBF16>(p, norm, rot, vec, st);
}

}  // namespace

extern "C" {

int sam3cu_rope_freqs_init(const struct sam3cu_rope_config* c, struct sam3cu_rope_freqs* out) {
  if (!c || !out) return SAM3CU_EINVAL;
  if (c->rot_dim < 2 || c->rot_dim % 2 || c->rot_dim > kMaxDim) return SAM3CU_ESHAPE;
  if (c->layout != SAM3CU_ROPE_HALF && c->layout != SAM3CU_ROPE_INTERLEAVED) return SAM3CU_EINVAL;
  if (c->scaling < SAM3CU_ROPE_SCALE_NONE || c->scaling > SAM3CU_ROPE_SCALE_BANDS) return SAM3CU_EINVAL;
  // negated comparisons, so that a NaN is refused too
  if (!(c->theta > 1.0) || std::isinf(c->theta)) return SAM3CU_EINVAL;
  if (!(c->amplitude >= 0.0) || std::isinf(c->amplitude)) return SAM3CU_EINVAL;
  const bool yarn = c->scaling == SAM3CU_ROPE_SCALE_YARN, bands = c->scaling == SAM3CU_ROPE_SCALE_BANDS;
  if (c->scaling != SAM3CU_ROPE_SCALE_NONE && (!(c->factor >= 1.0) || std::isinf(c->factor))) return SAM3CU_EINVAL;
  if ((yarn || bands) && (!(c->trained_len > 0.0) || std::isinf(c->trained_len))) return SAM3CU_EINVAL;
  if (yarn && (!(c->beta_slow > 0.0) || !(c->beta_fast > c->beta_slow) || std::isinf(c->beta_fast)))
    return SAM3CU_EINVAL;
  if (bands && (!(c->low_freq > 0.0) || !(c->high_freq > c->low_freq) || std::isinf(c->high_freq)))
    return SAM3CU_EINVAL;
  const double two_pi = 6.283185307179586476925;
  const int rot = c->rot_dim;
  double theta = c->theta;
  if (c->scaling == SAM3CU_ROPE_SCALE_NTK && rot > 2) theta *= std::pow(c->factor, rot / (rot - 2.0));
  memset(out, 0, sizeof(*out));
  out->n_pairs = rot / 2;
  out->layout = c->layout;
  double amplitude = 1.0, ramp_lo = 0.0, ramp_hi = 0.0;
  if (yarn) {
    // the (fractional) pair index whose angle makes n turns over trained_len
    auto index = [&](double n) { return rot * std::log(c->trained_len / (n * two_pi)) / (2.0 * std::log(theta)); };
    ramp_lo = std::fmax(std::floor(index(c->beta_fast)), 0.0);
    ramp_hi = std::fmin(std::ceil(index(c->beta_slow)), rot - 1.0);
    amplitude = 0.1 * std::log(c->factor) + 1.0;
  }
  for (int i = 0; i < rot / 2; ++i) {
    const double w = std::pow(theta, -2.0 * i / rot);  // radians per position
    double f = w;
    if (c->scaling == SAM3CU_ROPE_SCALE_LINEAR) {
      f = w / c->factor;
    } else if (yarn) {
      const double t = std::fmin(std::fmax((i - ramp_lo) / std::fmax(ramp_hi - ramp_lo, 0.001), 0.0), 1.0);
      f = w / c->factor * t + w * (1.0 - t);
    } else if (bands) {
      const double n = c->trained_len * w / two_pi;  // turns over trained_len
      const double t = std::fmin(std::fmax((n - c->low_freq) / (c->high_freq - c->low_freq), 0.0), 1.0);
      f = (1.0 - t) * w / c->factor + t * w;
    }
    out->turns[i] = f / two_pi;
  }
  out->amplitude = static_cast<float>(c->amplitude > 0.0 ? c->amplitude : amplitude);
  return SAM3CU_OK;
}

int sam3cu_rope_pos(const struct sam3cu_head_view* q, const struct sam3cu_head_view* k, int dtype, int batch, int seq,
                    int head_dim, const int64_t* positions, int64_t pos_stride, int64_t start,
                    const struct sam3cu_rope_freqs* freqs, void* stream) {
  if (!freqs) return SAM3CU_EINVAL;
  return rotary_common(q, k, dtype, batch, seq, head_dim, kNormNone, 0.f, positions, pos_stride, start, freqs, stream);
}

int sam3cu_qk_norm_rope(const struct sam3cu_head_view* q, const struct sam3cu_head_view* k, int dtype, int batch,
                        int seq, int head_dim, int norm, float eps, const int64_t* positions, int64_t pos_stride,
                        int64_t start, const struct sam3cu_rope_freqs* freqs, void* stream) {
  if (norm != SAM3CU_NORM_RMS && norm != SAM3CU_NORM_LAYER) return SAM3CU_EINVAL;
  return rotary_common(q, k, dtype, batch, seq, head_dim, norm, eps, positions, pos_stride, start, freqs, stream);
}

}  // extern "C"
