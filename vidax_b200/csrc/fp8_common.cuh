// e4m3 blocks with float32 scales: the arithmetic the 8-bit kernels share.
//
// A block b (128 consecutive features of one row, or 128 x 128 weights) with
// largest magnitude a stands for q * s with
//   s = a / 448,   q = e4m3(x * (448 / a))          (round to nearest even)
// 448 is e4m3's largest value, so the block's largest element uses the whole
// range and nothing saturates. `a` is at least kAmaxFloor: an all-zero block
// gets q = 0 and a small scale instead of 0 / 0 (448 / a and a / 448 are both
// normal float32 numbers there). A NaN in a block stays a NaN in its place
// (fmaxf ignores it, the conversion keeps it); an infinity makes s infinite
// and every value of its block stands for NaN.
#pragma once

#include "sm100_common.cuh"

namespace vx {
namespace fp8 {

constexpr int kBlock = 128;                      // features (and weight rows) per scale
constexpr float kMax = 448.f;                    // largest e4m3 value
constexpr float kAmaxFloor = 7.888609052210118e-31f;  // 2^-100

// Four floats -> four e4m3 bytes, the first in the low byte.
__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(lo) : "f"(a), "f"(b));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(hi) : "f"(c), "f"(d));
  return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
}

// The block's scale and the factor its elements are multiplied with.
__device__ __forceinline__ float block_scale(float amax, float& inv) {
  const float a = fmaxf(amax, kAmaxFloor);
  inv = __fdiv_rn(kMax, a);
  return a * (1.f / kMax);
}

__device__ __forceinline__ float amax8(const float (&f)[8]) {
  float m = fmaxf(fabsf(f[0]), fabsf(f[1]));
#pragma unroll
  for (int i = 2; i < 8; ++i) m = fmaxf(m, fabsf(f[i]));
  return m;
}

// Largest value over each half-warp (16 lanes x 8 elements = one block of a row).
__device__ __forceinline__ float half_warp_max(float m) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}

__device__ __forceinline__ uint2 quantize8(const float (&f)[8], float inv) {
  return make_uint2(pack_e4m3x4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv),
                    pack_e4m3x4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv));
}

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// Eight consecutive elements at `p`, of which the first `n` exist (0 for the
// rest). kVec: `p` is 16-byte aligned (8 bf16) / 32-byte aligned (8 float).
template <bool kVec>
__device__ __forceinline__ void load8(const float* p, int n, float (&f)[8]) {
  if (kVec && n >= 8) {
    const float4 a = reinterpret_cast<const float4*>(p)[0];
    const float4 b = reinterpret_cast<const float4*>(p)[1];
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = i < n ? p[i] : 0.f;
  }
}
template <bool kVec>
__device__ __forceinline__ void load8(const __nv_bfloat16* p, int n, float (&f)[8]) {
  if (kVec && n >= 8) {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      f[2 * k] = __uint_as_float(w[k] << 16);
      f[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = i < n ? __bfloat162float(p[i]) : 0.f;
  }
}

template <bool kVec>
__device__ __forceinline__ void store8(float* p, int n, const float (&f)[8]) {
  if (kVec && n >= 8) {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = f[i];
  }
}
template <bool kVec>
__device__ __forceinline__ void store8(__nv_bfloat16* p, int n, const float (&f)[8]) {
  if (kVec && n >= 8) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]),
                                              pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = __float2bfloat16(f[i]);
  }
}
// Eight e4m3 bytes; kVec: `p` 8-byte aligned.
template <bool kVec>
__device__ __forceinline__ void store8_e4m3(uint8_t* p, int n, uint2 q) {
  if (kVec && n >= 8) {
    *reinterpret_cast<uint2*>(p) = q;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = static_cast<uint8_t>((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
  }
}

}  // namespace fp8
}  // namespace vx
