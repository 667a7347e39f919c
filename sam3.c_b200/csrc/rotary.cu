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
// F32 of the remainder: once per token and pair, for all of its heads.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <cstring>

#include "../../include/sam3cu.h"
#include "attention_math.cuh"
#include "sam3cu_internal.h"

using namespace s3;

namespace {

constexpr int kWarps = 8;   // per CTA
constexpr int kThreads = 32 * kWarps;
// rotary_vec: CTAs per SM it is compiled for, and heads of a lane under way.
// Measured (us: 8 x 5184 tokens x 32 heads of 64 bf16 / LayerNorm, 16 x 5184 x
// 20 heads / f16, 6185 tokens x 24 heads of 128): 3 CTAs, 4 heads 60.1 / 78.7 /
// 16.0; 4, 4: 65.1 / 80.3 / 15.5; 5, 4: 75.0 / 115 / 17.7; 3 CTAs with one head
// ahead in registers 81.1 / 98.0 / 21.5.
constexpr int kVecCtas = 3, kAhead = 4;
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
  int slices;          // warps or lane groups that share a token's heads,
  int per_slice;       //   and the heads of one
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

// The 16 elements of a lane as loaded: 16-byte pieces of kP elements.
template <int T>
struct Raw {
  static constexpr int kP = T == kF32 ? 4 : 8;
  static constexpr int kN = 16 / kP;
  uint4 w[kN];
};
// Elements 2k, 2k + 1 of a lane as a packed operand.
template <int T>
__device__ __forceinline__ uint64_t pair_of(const Raw<T>& r, int k) {
  const uint4& q = r.w[2 * k / Raw<T>::kP];
  if constexpr (T == kF32) {
    return k & 1 ? f2pack(__uint_as_float(q.z), __uint_as_float(q.w))
                 : f2pack(__uint_as_float(q.x), __uint_as_float(q.y));
  } else {
    const uint32_t w = (k & 3) == 0 ? q.x : (k & 3) == 1 ? q.y : (k & 3) == 2 ? q.z : q.w;
    float2 v;
    if (T == kBF16) v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
    else v = __half22float2(*reinterpret_cast<const __half2*>(&w));
    return f2pack(v.x, v.y);
  }
}
template <int T>
__device__ __forceinline__ void st_piece(void* p, int64_t i, const uint64_t* h) {
  float f[8];
#pragma unroll
  for (int k = 0; k < Raw<T>::kP / 2; ++k) f2unpack(h[k], f[2 * k], f[2 * k + 1]);
  uint4 w;
  if constexpr (T == kF32) {
    w = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  } else {
    w = make_uint4(pack2(f[0], f[1], T == kBF16), pack2(f[2], f[3], T == kBF16), pack2(f[4], f[5], T == kBF16),
                   pack2(f[6], f[7], T == kBF16));
  }
  *reinterpret_cast<uint4*>(static_cast<char*>(p) + i * (T == kF32 ? 4 : 2)) = w;
}

// Element of the head that piece i (of kp elements) of lane `slot` starts at,
// where the pieces are spread over the `slots` lanes of a head.
__host__ __device__ constexpr int spread_piece(int kp, int slots, int slot, int i) {
  return kp * slot + i * kp * slots;
}
// A group has as many lanes as the next power of two; those behind the head's
// hold no piece of it.  Their offsets are those of the first lanes' next
// pieces, so they must not store what the lanes of a group share.
__host__ __device__ constexpr bool holds_piece(int slots, int slot) { return slot < slots; }
// Whether the lanes that store pieces store each element of a head once.
constexpr bool one_writer_each(int kp) {
  for (int slots = 1; slots <= kMaxDim / 16; ++slots) {
    int lanes = 1;
    while (lanes < slots) lanes *= 2;
    int writers[2 * kMaxDim] = {};
    for (int slot = 0; slot < lanes; ++slot)
      for (int e = 0; holds_piece(slots, slot) && e < 16; ++e) ++writers[spread_piece(kp, slots, slot, e / kp) + e % kp];
    for (int e = 0; e < 2 * kMaxDim; ++e)
      if (writers[e] != (e < 16 * slots)) return false;
  }
  return true;
}
static_assert(one_writer_each(Raw<kF32>::kP) && one_writer_each(Raw<kBF16>::kP), "two lanes store one element");

// Heads of a lane under way: 32 bytes each, 64 for F32.
template <int T, int kRot>
constexpr int ring_depth() {
  return (T == kF32 ? kAhead / 2 : kAhead) / (kRot == 2 ? 2 : 1);  // the exchange takes shared memory too
}
template <int T, int kRot>
constexpr size_t ring_bytes() {
  return static_cast<size_t>(ring_depth<T, kRot>()) * Raw<T>::kN * 16 * kThreads;
}

// token = b * seq + s
__device__ __forceinline__ void split_token(const Params& p, int64_t token, int64_t& b, int64_t& s) {
  if (p.tokens <= 0x7fffffff) {  // the 64-bit division is several times dearer
    const uint32_t t = static_cast<uint32_t>(token), n = static_cast<uint32_t>(p.seq);
    b = t / n;
    s = t - static_cast<uint32_t>(b) * n;
  } else {
    b = token / p.seq;
    s = token - b * p.seq;
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
  int64_t b, s;
  split_token(p, token, b, s);
  at.b = static_cast<int>(b);
  at.s = static_cast<int>(s);
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
// bytes.  A lane holds 16 elements of a head in 16-byte pieces, chosen so that
// both elements of a pair are in one lane and the lanes of a head access
// consecutive pieces (whole 32-byte sectors): half of its pieces from either
// half of the rotated part in the half layout, pieces spread over the head in
// the interleaved one.  head_dim / 16 lanes (kG, the next power of two) are a
// group; a group takes the heads of one token (or, where there are few
// tokens, a slice of them) one after the other, with the cosines and sines of
// its lanes' pairs in registers and the next heads' copies under way (cp.async
// into places of the lane's own, which costs no registers).
//
// kRot 2: the half layout with halves that are not multiples of 8 elements.  A
// pair's elements are then in different lanes, which exchange the (normalised)
// head through shared memory; the pieces lie as in the interleaved layout.
template <int T, int kNorm, int kRot, int kG>
__global__ void __launch_bounds__(kThreads, kRot == 2 ? 2 : kVecCtas) rotary_vec(const __grid_constant__ Params p) {
  using R = Raw<T>;
  constexpr int kES = T == kF32 ? 4 : 2;
  constexpr int kDepth = ring_depth<T, kRot>();
  __shared__ __align__(16) float affine[kNorm ? 2 : 1][2][kNorm ? 16 * kG : 1];  // gamma, beta of q and k
  const int tid = threadIdx.x;
  const int slot = tid % kG;
  const int slots = p.head_dim / 16;              // lanes of a head
  const int rslots = kRot ? p.f.n_pairs / 8 : 0;  // half layout: those that rotate
  const bool half = kRot == 1 && p.f.layout == SAM3CU_ROPE_HALF;
  int off[R::kN];  // elements of the head that the lane's pieces start at
  bool turned = false;
#pragma unroll
  for (int i = 0; i < R::kN; ++i) {
    if (half && slot < rslots) {
      off[i] = R::kP * slot + (i % (R::kN / 2)) * R::kP * rslots + (i >= R::kN / 2 ? p.f.n_pairs : 0);
    } else if (half) {  // behind the rotated part
      off[i] = 16 * rslots + R::kP * (slot - rslots) + i * R::kP * (slots - rslots);
    } else {
      off[i] = spread_piece(R::kP, slots, slot, i);
    }
    turned = turned || (kRot && off[i] < 2 * p.f.n_pairs);
  }

  // the group's token and heads
  const int64_t item = static_cast<int64_t>(blockIdx.x) * (kThreads / kG) + tid / kG;
  const int64_t token = p.slices > 1 ? item / p.slices : item;
  const int slice = p.slices > 1 ? static_cast<int>(item - token * p.slices) : 0;
  const bool have = holds_piece(slots, slot) && token < p.tokens;
  const int h0 = slice * p.per_slice;
  const int h1 = min(p.heads, h0 + p.per_slice);
  int64_t b, s;
  split_token(p, have ? token : 0, b, s);
  const char* xq = static_cast<const char*>(p.v[0].x) + (b * p.v[0].xb + s * p.v[0].xs) * kES;
  const char* xk = static_cast<const char*>(p.v[1].x) + (b * p.v[1].xb + s * p.v[1].xs - p.q_heads * p.v[1].xh) * kES;
  char* yq = static_cast<char*>(p.v[0].y) + (b * p.v[0].yb + s * p.v[0].ys) * kES;
  char* yk = static_cast<char*>(p.v[1].y) + (b * p.v[1].yb + s * p.v[1].ys - p.q_heads * p.v[1].yh) * kES;
  // without a norm, what is not rotated need not move where it already is
  const bool mq = have && (kNorm != kNormNone || p.v[0].x != p.v[0].y || turned);
  const bool mk = have && (kNorm != kNormNone || p.v[1].x != p.v[1].y || turned);

  // The lane's pieces of a head (zeros where it has none) into its places of
  // the ring; nobody else reads them, so no barrier is needed.
  extern __shared__ uint4 ring[];  // [kDepth][pieces][kThreads]
  const uint32_t mine_s = smem_u32(ring) + tid * 16;
  auto issue = [&](int i) {
    const int h = h0 + i;
    const bool k = h >= p.q_heads;
    const bool on = h < h1 && (k ? mk : mq);
    const char* x = on ? (k ? xk : xq) + h * (k ? p.v[1].xh : p.v[0].xh) * kES : static_cast<const char*>(p.v[0].x);
    const uint32_t dst = mine_s + static_cast<uint32_t>(i % kDepth) * (R::kN * kThreads * 16);
#pragma unroll
    for (int n = 0; n < R::kN; ++n)
      cp_async16(dst + n * (kThreads * 16), x + (on ? off[n] * kES : 0), on);
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kDepth - 1; ++i) issue(i);

  if constexpr (kNorm != kNormNone) {
    for (int i = tid; i < 4 * 16 * kG; i += kThreads) {
      const int e = i % (16 * kG), which = i / (16 * kG);
      const View& v = p.v[which >> 1];
      const float* src = which & 1 ? v.beta : v.gamma;
      affine[which >> 1][which & 1][e] = src && e < p.head_dim ? src[e] : (which & 1 ? 0.f : 1.f);
    }
    __syncthreads();
  }
  // kRot 1: (cos, cos) and (sin, sin) of the lane's pairs 2 jj, 2 jj + 1.
  // kRot 2: cos, and the factor of the partner, of its elements 2 jj, 2 jj + 1.
  constexpr int kCs = kRot == 2 ? 8 : 4;
  uint64_t cc[kRot ? kCs : 1], ss[kRot ? kCs : 1];
  // a pair or element of the lane that turns (in the half layout: all or none)
  uint32_t turns = 0;
  if constexpr (kRot != 0) {
    if (have && turned) {
      const double pos =
          static_cast<double>(p.positions ? p.positions[b * p.pos_stride + s] : p.start + s);
#pragma unroll
      for (int jj = 0; jj < kCs; ++jj) {
        // element of the lane: of its low pieces, or of all
        const int e = (half || kRot == 2) ? 2 * jj : 4 * jj;
        const int at = off[e / R::kP] + e % R::kP;
        float2 c[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          c[i] = make_float2(1.f, 0.f);
          const int el = kRot == 2 ? at + i : 0;
          const int pair = kRot == 2 ? (el >= p.f.n_pairs ? el - p.f.n_pairs : el) : (half ? at : at / 2) + i;
          if (pair < p.f.n_pairs) {
            c[i] = turn(p, pos, pair);
            if (kRot == 2 && el < p.f.n_pairs) c[i].y = -c[i].y;
            turns |= 1u << (2 * jj + i);
          }
        }
        cc[jj] = f2pack(c[0].x, c[1].x);
        ss[jj] = f2pack(c[0].y, c[1].y);
      }
    }
  }

  auto process = [&](const Raw<T>& raw, int h) {
    const bool k = h >= p.q_heads;
    uint64_t h2[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) h2[i] = pair_of<T>(raw, i);
    if constexpr (kNorm != kNormNone) {
      const float n = 1.f / static_cast<float>(p.head_dim);
      if constexpr (kNorm == kNormLayer) {
        float a, c;
        f2unpack(fadd2(fadd2(fadd2(h2[0], h2[1]), fadd2(h2[2], h2[3])),
                       fadd2(fadd2(h2[4], h2[5]), fadd2(h2[6], h2[7]))),
                 a, c);
        float sum = a + c;
#pragma unroll
        for (int o = kG / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const float mean = holds_piece(slots, slot) ? -sum * n : 0.f;
        const uint64_t m2 = f2pack(mean, mean);
#pragma unroll
        for (int i = 0; i < 8; ++i) h2[i] = fadd2(h2[i], m2);
      }
      uint64_t q2[2] = {f2pack(0.f, 0.f), f2pack(0.f, 0.f)};
#pragma unroll
      for (int i = 0; i < 8; ++i) q2[i & 1] = ffma2(h2[i], h2[i], q2[i & 1]);
      float a, c;
      f2unpack(fadd2(q2[0], q2[1]), a, c);
      float sq = a + c;
#pragma unroll
      for (int o = kG / 2; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
      const float inv = rsqrtf(fmaf(sq, n, p.eps));
      const uint64_t i2 = f2pack(inv, inv);
      if (holds_piece(slots, slot)) {
        const float(&af)[2][kNorm ? 16 * kG : 1] = affine[kNorm && k ? 1 : 0];
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const int e = kNorm ? off[2 * i / R::kP] + 2 * i % R::kP : 0;
          const float4 g = *reinterpret_cast<const float4*>(&af[0][e]);
          const float4 t = *reinterpret_cast<const float4*>(&af[1][e]);
          h2[i] = ffma2(fmul2(h2[i], i2), f2pack(g.x, g.y), f2pack(t.x, t.y));
          h2[i + 1] = ffma2(fmul2(h2[i + 1], i2), f2pack(g.z, g.w), f2pack(t.z, t.w));
        }
      }
    }
    if constexpr (kRot == 2) {
      // one word of padding after eight, so that lanes and groups spread over
      // the banks
      constexpr int kPitch = kG * 18 + 1;
      __shared__ float heads[kThreads / kG][kPitch];
      float* mine_h = heads[tid / kG];
      float f[16];
      __syncwarp();  // the last head has been read
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        f2unpack(h2[i], f[2 * i], f[2 * i + 1]);
        const int e = off[2 * i / R::kP] + 2 * i % R::kP;
        if (holds_piece(slots, slot)) {
          mine_h[e + (e >> 3)] = f[2 * i];
          mine_h[e + 1 + (e >> 3)] = f[2 * i + 1];
        }
      }
      __syncwarp();
      if (turns) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float c[2], sn[2];
          f2unpack(cc[i], c[0], c[1]);
          f2unpack(ss[i], sn[0], sn[1]);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            if (turns >> (2 * i + j) & 1) {
              const int e = off[2 * i / R::kP] + 2 * i % R::kP + j;
              const int o = e < p.f.n_pairs ? e + p.f.n_pairs : e - p.f.n_pairs;
              f[2 * i + j] = f[2 * i + j] * c[j] + mine_h[o + (o >> 3)] * sn[j];
            }
          }
          h2[i] = f2pack(f[2 * i], f[2 * i + 1]);
        }
      }
    } else if constexpr (kRot == 1) {
      if (half) {
        if (turned) {
#pragma unroll
          for (int jj = 0; jj < 4; ++jj) {
            const uint64_t a2 = h2[jj], b2 = h2[4 + jj];
            h2[jj] = ffma2(b2, fneg2(ss[jj]), fmul2(a2, cc[jj]));
            h2[4 + jj] = ffma2(a2, ss[jj], fmul2(b2, cc[jj]));
          }
        }
      } else if (turns) {
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) {
          float co[2], si[2];
          f2unpack(cc[jj], co[0], co[1]);
          f2unpack(ss[jj], si[0], si[1]);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float a, c;
            f2unpack(h2[2 * jj + i], a, c);
            const uint64_t r = f2pack(a * co[i] - c * si[i], a * si[i] + c * co[i]);
            if (turns >> (2 * jj + i) & 1) h2[2 * jj + i] = r;
          }
        }
      }
    }
    if (h < h1 && (k ? mk : mq)) {
      char* y = (k ? yk : yq) + h * (k ? p.v[1].yh : p.v[0].yh) * kES;
#pragma unroll
      for (int i = 0; i < R::kN; ++i) st_piece<T>(y, off[i], h2 + i * R::kP / 2);
    }
  };
  // (every lane of a warp makes the same number of turns: shuffles)
#pragma unroll 1
  for (int i = 0; i < p.per_slice; ++i) {
    issue(i + kDepth - 1);  // into the place read last
    cp_async_wait<kDepth - 1>();
    Raw<T> raw;
#pragma unroll
    for (int n = 0; n < R::kN; ++n) raw.w[n] = ring[(i % kDepth * R::kN + n) * kThreads + tid];
    process(raw, h0 + i);
  }
}

// Any head_dim, alignment and stride: a lane holds the pairs
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
      const float inv = rsqrtf(sq / n + p.eps);
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

// At most `slices` (>= 1) slices of a token's heads.
void set_slices(Params& p, int64_t slices) {
  if (slices > p.heads) slices = p.heads;
  p.per_slice = (p.heads + static_cast<int>(slices) - 1) / static_cast<int>(slices);
  p.slices = (p.heads + p.per_slice - 1) / p.per_slice;
}

template <int T, int kNorm>
int launch_typed(Params& p, int rot, bool vec, cudaStream_t st) {
  count_launches(1);
  if (vec) {
    const int lanes = p.head_dim / 16;
    const int g = lanes <= 1 ? 1 : lanes <= 2 ? 2 : lanes <= 4 ? 4 : lanes <= 8 ? 8 : 16;
    // Lane groups that share a token's heads (they repeat its cosines): as
    // many as one wave of CTAs has room for.  Beyond a wave one, but two below two
    // waves where 16 heads are left to each: the last CTAs end sooner.  One and
    // two at 1.05 / 1.25 / 1.5 / 1.75 / 1.95 waves, bf16: 32 heads of 64 49 / 52 /
    // 62 / 71 / 79 and 44 / 50 / 61 / 69 / 76 us; 48 + 16 heads of 128 89 / 103 /
    // 122 / 137 / 153 and 86 / 97 / 115 / 133 / 146; with an RMS norm two are
    // better by up to 13% too, but worse by 2 - 10% for 32 heads of 64 and by 2 -
    // 6% at 1.95 waves of heads of 128.  Past two waves: 82944 tokens x 20 heads
    // with LayerNorm, 2.9 waves, 79 with one and 90 with two.
    const bool exchange = rot % 16 && p.f.layout == SAM3CU_ROPE_HALF;
    const int per_block = kThreads / g;
    const int64_t alone = (p.tokens + per_block - 1) / per_block;
    const int64_t wave = static_cast<int64_t>(exchange ? 4 : kVecCtas) * num_sms();  // (two waves of the exchange)
    set_slices(p, alone <= wave ? wave / alone : (alone < 2 * wave && p.heads >= 32 ? 2 : 1));
    const int64_t blocks = (p.tokens * p.slices + per_block - 1) / per_block;
    if (blocks > 0x7fffffffLL) return SAM3CU_ESHAPE;
    const dim3 grid(static_cast<unsigned>(blocks));
#define S3_ROT(G)                                                                               \
  case G:                                                                                       \
    if (!rot) rotary_vec<T, kNorm, 0, G><<<grid, kThreads, ring_bytes<T, 0>(), st>>>(p);           \
    else if (!exchange) rotary_vec<T, kNorm, 1, G><<<grid, kThreads, ring_bytes<T, 1>(), st>>>(p); \
    else rotary_vec<T, kNorm, 2, G><<<grid, kThreads, ring_bytes<T, 2>(), st>>>(p);                \
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
    set_slices(p, (want + p.tokens - 1) / p.tokens);
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
  bool vec = head_dim % 16 == 0;
  int rc = take_view(q, dtype, batch, seq, &p.v[0], &vec);
  if (!rc) rc = take_view(k, dtype, batch, seq, &p.v[1], &vec);
  if (rc) return rc;
  p.q_heads = q->heads;
  const int64_t heads = static_cast<int64_t>(q->heads) + (k ? k->heads : 0);
  if (heads > (1 << 24)) return SAM3CU_ESHAPE;
  p.heads = static_cast<int>(heads);
  p.tokens = static_cast<int64_t>(batch) * seq;
  if (p.tokens == 0 || p.heads == 0) return SAM3CU_OK;
  if (freqs && !positions && start > INT64_MAX - (seq - 1)) return SAM3CU_EINVAL;
  if (q->heads == 0) p.v[0] = p.v[1];  // where lanes without a head point must be memory too
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
  if (!(c->amplitude >= 0.0) || std::isinf(static_cast<float>(c->amplitude))) return SAM3CU_EINVAL;
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
  if (std::isinf(theta)) return SAM3CU_EINVAL;
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
