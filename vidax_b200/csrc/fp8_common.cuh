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

// A warp's 256 consecutive features of a row: lane l holds features 8 l ..
// 8 l + 7, so a half-warp holds one block of 128. kVec: rows of 8 k features
// on 16-byte boundaries. Any other row (odd widths or strides) is read through
// the aligned 16-byte pieces that its bytes lie in, shifted into place: a row
// starts at another offset each time, but the same for all lanes. A piece that
// holds one of the row's bytes lies in the same page, so the up to 15 bytes of
// it before the first row or behind the last cannot fault.

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
// Words w[q ..] of the pieces, q = 0..3.
template <int N>
__device__ __forceinline__ void shift_words(uint32_t (&w)[N], uint32_t q) {
#pragma unroll
  for (int i = 0; i + 2 < N; ++i) w[i] = q & 2u ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i + 1 < N; ++i) w[i] = q & 1u ? w[i + 1] : w[i];
}
__device__ __forceinline__ void put4(uint32_t* w, const uint4& v) {
  w[0] = v.x;
  w[1] = v.y;
  w[2] = v.z;
  w[3] = v.w;
}
// 0 for the elements past the first `have`.
__device__ __forceinline__ void cut8(float (&f)[8], int have) {
  if (have < 8) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i >= have) f[i] = 0.f;
  }
}
// The 16-byte piece `k` after the one that holds `p`, if bytes [16 k, ...) of
// it are wanted (`bytes` from p on).
__device__ __forceinline__ uint4 piece(const void* p, int k, int bytes) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p);
  uint4 v = make_uint4(0u, 0u, 0u, 0u);
  if (bytes > 0 && static_cast<int>(at & 15u) + bytes > 16 * k)
    v = reinterpret_cast<const uint4*>(at & ~static_cast<uintptr_t>(15))[k];
  return v;
}
template <>
struct Raw<float, false> {
  uint4 a, b, c;
  uint32_t q;
  int have;
  __device__ __forceinline__ void load(const float* row, int lane, int n) {
    const float* p = row + lane * 8;
    have = n - lane * 8;
    const int bytes = min(have, 8) * 4;
    q = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p) & 15u) >> 2;
    a = piece(p, 0, bytes);
    b = piece(p, 1, bytes);
    c = piece(p, 2, bytes);
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    uint32_t w[12];
    put4(w, a);
    put4(w + 4, b);
    put4(w + 8, c);
    shift_words(w, q);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(w[i]);
    cut8(f, have);
  }
};
template <>
struct Raw<__nv_bfloat16, false> {
  uint4 a, b;
  uint32_t at;
  int have;
  __device__ __forceinline__ void load(const __nv_bfloat16* row, int lane, int n) {
    const __nv_bfloat16* p = row + lane * 8;
    have = n - lane * 8;
    const int bytes = min(have, 8) * 2;
    at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p) & 15u);
    a = piece(p, 0, bytes);
    b = piece(p, 1, bytes);
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    uint32_t w[8];
    put4(w, a);
    put4(w + 4, b);
    shift_words(w, at >> 2);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t v = __funnelshift_r(w[i], w[i + 1], (at & 2u) * 8u);
      f[2 * i] = __uint_as_float(v << 16);
      f[2 * i + 1] = __uint_as_float(v & 0xffff0000u);
    }
    cut8(f, have);
  }
};

__device__ __forceinline__ void store8(float* p, const float (&f)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&f)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]),
                                            pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
}

// Stores the chunk. Rows off the 16-byte boundaries (`on16` false) leave
// element by element, neighbours by neighbouring lanes, through `turn` (the
// warp's own 256 elements of shared memory).
template <bool kVec, typename T>
__device__ __forceinline__ void store_chunk(T* row, int lane, int n, const float (&f)[8], bool on16,
                                            void* turn) {
  if (kVec || (on16 && n >= 256)) {
    if (lane * 8 < n) store8(row + lane * 8, f);
    return;
  }
  T* t = static_cast<T*>(turn);
  __syncwarp();
  store8(t + lane * 8, f);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i * 32 + lane < n) row[i * 32 + lane] = t[i * 32 + lane];
}

// Largest magnitude of the lane's block (a half-warp's chunk of 128 features).
__device__ __forceinline__ float block_amax(const float (&f)[8]) {
  return lanes_max<16>(fmaxf(amax4(f[0], f[1], f[2], f[3]), amax4(f[4], f[5], f[6], f[7])));
}

// The lane's eight features times `inv`, as e4m3 at their place in the chunk
// (of which `n` features exist). `on8`: the row lies on an 8-byte boundary.
template <bool kVec>
__device__ __forceinline__ void store_e4m3(uint8_t* row, int lane, int n, const float (&f)[8],
                                           float inv, bool on8) {
  const int have = n - lane * 8;
  if (have <= 0) return;
  const uint2 q = make_uint2(pack_e4m3x4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv),
                             pack_e4m3x4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv));
  uint8_t* o = row + lane * 8;
  if (kVec || (on8 && have >= 8)) {
    *reinterpret_cast<uint2*>(o) = q;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < have) o[i] = static_cast<uint8_t>((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
  }
}

// Quantises and stores the chunk (features past the end must be 0); `scale`
// points at the scale of its first block, the second is `bs` floats on.
template <bool kVec>
__device__ __forceinline__ void quantize_chunk(uint8_t* row, float* scale, long long bs, int lane,
                                               int n, const float (&f)[8], bool on8) {
  float inv;
  const float s = block_scale(block_amax(f), inv);
  store_e4m3<kVec>(row, lane, n, f, inv, on8);
  if ((lane & 15) == 0 && lane * 8 < n) scale[(lane >> 4) * bs] = s;
}

}  // namespace fp8
}  // namespace vx
