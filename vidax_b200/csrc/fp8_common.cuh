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

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

__device__ __forceinline__ float amax4(float a, float b, float c, float d) {
  return fmaxf(fmaxf(fabsf(a), fabsf(b)), fmaxf(fabsf(c), fabsf(d)));
}
template <int kLanes>
__device__ __forceinline__ float lanes_max(float m) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}

// A warp's 256 consecutive features of a row, eight per lane. kVec (rows of
// 8 k features on 16-byte boundaries): lane l holds features 8 l .. 8 l + 7,
// moved as vectors; a half-warp then holds one block of 128. Otherwise lane l
// holds features l, l + 32, ..., so that a warp's element accesses are
// neighbours; elements 0-3 and 4-7 of all lanes are the two blocks.
template <bool kVec>
__device__ __forceinline__ int feature(int lane, int i) {
  return kVec ? lane * 8 + i : i * 32 + lane;
}

// The lane's eight elements as they lie in memory (`row` points at the chunk,
// of which the first `n` features exist; the others read 0).
template <typename T, bool kVec>
struct Raw;
template <>
struct Raw<float, true> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* row, int lane, int n) {
    a = b = make_float4(0.f, 0.f, 0.f, 0.f);
    if (lane * 8 < n) {
      a = reinterpret_cast<const float4*>(row)[2 * lane];
      b = reinterpret_cast<const float4*>(row)[2 * lane + 1];
    }
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
};
template <>
struct Raw<__nv_bfloat16, true> {
  uint4 a;
  __device__ __forceinline__ void load(const __nv_bfloat16* row, int lane, int n) {
    a = make_uint4(0u, 0u, 0u, 0u);
    if (lane * 8 < n) a = reinterpret_cast<const uint4*>(row)[lane];
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      f[2 * k] = __uint_as_float(w[k] << 16);
      f[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
    }
  }
};
template <>
struct Raw<float, false> {
  float v[8];
  __device__ __forceinline__ void load(const float* row, int lane, int n) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] = 0.f;
      if (i * 32 + lane < n) v[i] = row[i * 32 + lane];
    }
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = v[i];
  }
};
template <>
struct Raw<__nv_bfloat16, false> {
  uint16_t v[8];
  __device__ __forceinline__ void load(const __nv_bfloat16* row, int lane, int n) {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] = 0;
      if (i * 32 + lane < n) v[i] = p[i * 32 + lane];
    }
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(static_cast<uint32_t>(v[i]) << 16);
  }
};

template <bool kVec>
__device__ __forceinline__ void store_chunk(float* row, int lane, int n, const float (&f)[8]) {
  if constexpr (kVec) {
    if (lane * 8 < n) {
      reinterpret_cast<float4*>(row)[2 * lane] = make_float4(f[0], f[1], f[2], f[3]);
      reinterpret_cast<float4*>(row)[2 * lane + 1] = make_float4(f[4], f[5], f[6], f[7]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i * 32 + lane < n) row[i * 32 + lane] = f[i];
  }
}
template <bool kVec>
__device__ __forceinline__ void store_chunk(__nv_bfloat16* row, int lane, int n, const float (&f)[8]) {
  if constexpr (kVec) {
    if (lane * 8 < n)
      reinterpret_cast<uint4*>(row)[lane] =
          make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                     pack_bf16x2(f[6], f[7]));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i * 32 + lane < n) row[i * 32 + lane] = __float2bfloat16(f[i]);
  }
}

// Quantises and stores the chunk (features past the end must be 0); `scale`
// points at the scale of its first block, the second is `bs` floats on.
template <bool kVec>
__device__ __forceinline__ void quantize_chunk(uint8_t* row, float* scale, long long bs, int lane,
                                               int n, const float (&f)[8]) {
  const float lo = amax4(f[0], f[1], f[2], f[3]), hi = amax4(f[4], f[5], f[6], f[7]);
  float inv;
  if constexpr (kVec) {
    const float s = block_scale(lanes_max<16>(fmaxf(lo, hi)), inv);
    if (lane * 8 < n) {
      reinterpret_cast<uint2*>(row)[lane] =
          make_uint2(pack_e4m3x4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv),
                     pack_e4m3x4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv));
      if ((lane & 15) == 0) scale[(lane >> 4) * bs] = s;
    }
  } else {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const float s = block_scale(lanes_max<32>(half ? hi : lo), inv);
      const uint32_t q = pack_e4m3x4(f[4 * half] * inv, f[4 * half + 1] * inv,
                                     f[4 * half + 2] * inv, f[4 * half + 3] * inv);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = (4 * half + i) * 32 + lane;
        if (c < n) row[c] = static_cast<uint8_t>(q >> (8 * i));
      }
      if (lane == 0 && half * kBlock < n) scale[half * bs] = s;
    }
  }
}

}  // namespace fp8
}  // namespace vx
