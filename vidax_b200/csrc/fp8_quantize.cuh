// Quantisation of a matrix to e4m3 with a float32 scale per block.
//
// quantize_rows_kernel: blocks of 128 features of one row (activations). A
//   half-warp holds a block, eight features per lane, so its largest
//   magnitude is four shuffles away and the row is read once. A half-warp
//   takes the same 128 features of kRows rows: their loads are all in flight
//   together, and their scales -- neighbours in memory when the scales of one
//   block of features lie side by side -- leave as one 16-byte store.
// quantize_tiles_kernel: 128 x 128 blocks (weights), one block per CTA.
//
// Both are bound by HBM: 2 or 4 bytes read, 1 + 4/128 written per element.
#pragma once

#include "fp8_common.cuh"

namespace vx {
namespace fp8 {

struct QuantizeParams {
  const void* src;
  uint8_t* dst;
  float* scale;
  long long src_stride, dst_stride;      // elements between rows
  long long scale_rs, scale_bs;          // elements between row blocks / feature blocks
  long long rows;
  int dim;
  int blocks;        // ceil(dim / 128)
  unsigned items;    // row groups * blocks
  int vec_scale;     // four rows' scales may leave as one 16-byte store
};

constexpr int kRows = 4;

template <typename T, bool kVec>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const __grid_constant__ QuantizeParams p) {
  const unsigned item = blockIdx.x * 16u + (threadIdx.x >> 4);
  // Half-warps past the end still take part in their warp's shuffles.
  const bool live = item < p.items;
  const unsigned grp = live ? item / p.blocks : 0u;
  const int blk = live ? static_cast<int>(item - grp * p.blocks) : 0;
  const int l = threadIdx.x & 15;
  const int c = blk * kBlock + l * 8;
  const int n = live ? p.dim - c : 0;
  const long long r0 = static_cast<long long>(grp) * kRows;
  float f[kRows][8];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int have = r0 + i < p.rows ? n : 0;
    load8<kVec>(static_cast<const T*>(p.src) + (have > 0 ? (r0 + i) * p.src_stride + c : 0), have,
                f[i]);
  }
  float s[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    float inv;
    s[i] = block_scale(half_warp_max(amax8(f[i])), inv);
    if (r0 + i < p.rows && n > 0)
      store8_e4m3<kVec>(p.dst + (r0 + i) * p.dst_stride + c, n, quantize8(f[i], inv));
  }
  if (live && l == 0) {
    float* out = p.scale + static_cast<long long>(blk) * p.scale_bs + r0 * p.scale_rs;
    if (p.vec_scale && r0 + kRows <= p.rows) {
      *reinterpret_cast<float4*>(out) = make_float4(s[0], s[1], s[2], s[3]);
    } else {
#pragma unroll
      for (int i = 0; i < kRows; ++i)
        if (r0 + i < p.rows) out[i * p.scale_rs] = s[i];
    }
  }
}

template <typename T, bool kVec>
__global__ void __launch_bounds__(256) quantize_tiles_kernel(const __grid_constant__ QuantizeParams p) {
  __shared__ float part[8];
  const long long grp = blockIdx.x / p.blocks;
  const int blk = static_cast<int>(blockIdx.x - grp * p.blocks);
  const int c = blk * kBlock + (threadIdx.x & 15) * 8;
  const int n = p.dim - c;
  const long long r0 = grp * kBlock + (threadIdx.x >> 4);
  float f[8][8];
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int have = r0 + 16 * i < p.rows ? n : 0;
    load8<kVec>(static_cast<const T*>(p.src) + (have > 0 ? (r0 + 16 * i) * p.src_stride + c : 0),
                have, f[i]);
    m = fmaxf(m, amax8(f[i]));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, part[i]);
  float inv;
  const float s = block_scale(m, inv);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (r0 + 16 * i < p.rows && n > 0)
      store8_e4m3<kVec>(p.dst + (r0 + 16 * i) * p.dst_stride + c, n, quantize8(f[i], inv));
  if (threadIdx.x == 0) p.scale[grp * p.scale_rs + static_cast<long long>(blk) * p.scale_bs] = s;
}

}  // namespace fp8
}  // namespace vx
