// attention_math.cuh - the softmax arithmetic of the tcgen05 attention
// kernels: packed f32x2 operations, exponentials, row maxima, 16-bit packing
// and the warp-wide bounded wait.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "sm100_ptx.cuh"

namespace s3 {

__device__ __forceinline__ uint32_t pack2(float a, float b, bool bf) {
  if (bf) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two f32 lanes in one 64-bit register for the packed f32x2 operations.
__device__ __forceinline__ uint64_t f2pack(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void f2unpack(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t ffma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t fadd2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t fmul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t fneg2(uint64_t a) { return a ^ 0x8000000080000000ull; }
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Maximum of 32 values.
__device__ __forceinline__ float max32(const float* v) {
  float m[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
  for (int c = 4; c < 28; c += 8) {
#pragma unroll
    for (int k = 0; k < 4; ++k) m[k] = max3(m[k], v[c + 2 * k], v[c + 2 * k + 1]);
  }
  return fmaxf(max3(max3(m[0], m[1], m[2]), m[3], v[28]), max3(v[29], v[30], v[31]));
}

// Maximum of 64 values: four chains of three-input max.
__device__ __forceinline__ float max64(const float* v) {
  float m[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
  for (int c = 4; c < 64; c += 8) {
#pragma unroll
    for (int k = 0; k < 4; ++k) m[k] = max3(m[k], v[c + 2 * k], v[c + 2 * k + 1]);
  }
  return fmaxf(max3(m[0], m[1], m[2]), m[3]);
}

// Maximum of 128 values: eight independent chains of three-input max
// (the softmax is latency-bound, so short chains matter).
__device__ __forceinline__ float max128(const float* v) {
  float m[8] = {v[0], v[1], v[2], v[3], v[64], v[65], v[66], v[67]};
#pragma unroll
  for (int c = 4; c < 64; c += 8) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      m[k] = max3(m[k], v[c + 2 * k], v[c + 2 * k + 1]);
      m[4 + k] = max3(m[4 + k], v[64 + c + 2 * k], v[64 + c + 2 * k + 1]);
    }
  }
  return fmaxf(fmaxf(max3(m[0], m[1], m[2]), m[3]), fmaxf(max3(m[4], m[5], m[6]), m[7]));
}

// Bounded wait by lane 0, verdict broadcast to the warp.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, unsigned err, volatile int* abort_flag,
                                          int lane) {
  int ok = 0;
  if (lane == 0) ok = mbar_wait(bar, parity, err, abort_flag) ? 1 : 0;
  return __shfl_sync(0xffffffffu, ok, 0) != 0;
}

}  // namespace s3
