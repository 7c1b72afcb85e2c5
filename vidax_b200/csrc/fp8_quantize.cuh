// Quantisation of a matrix to e4m3 with a float32 scale per block.
//
// quantize_rows_kernel: blocks of 128 features of one row (activations). A
//   warp takes 256 features (two blocks) of kRows rows: a block's largest
//   magnitude is a few shuffles away, the row is read once, and the rows'
//   loads are all in flight together.
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
  int chunks;        // of 256 features (rows kernel) or 128 (tiles kernel) per row
  unsigned items;    // row groups * chunks
  int on8;           // the output's rows lie on 8-byte boundaries
};

constexpr int kRows = 4;

template <typename T, bool kVec>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const __grid_constant__ QuantizeParams p) {
  const unsigned item = blockIdx.x * 8u + (threadIdx.x >> 5);
  if (item >= p.items) return;
  const unsigned grp = item / p.chunks;
  const int c0 = static_cast<int>(item - grp * p.chunks) * 2 * kBlock;
  const int lane = threadIdx.x & 31;
  const int n = p.dim - c0;
  const long long r0 = static_cast<long long>(grp) * kRows;
  const int rows = static_cast<int>(min(static_cast<long long>(kRows), p.rows - r0));
  Raw<T, kVec> raw[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i)  // rows past the end: the last one again, not stored
    raw[i].load(static_cast<const T*>(p.src) + (r0 + min(i, rows - 1)) * p.src_stride + c0, lane, n);
  float f[kRows][8];
  // Lane i of a half-warp divides for row i % 4 and stores its scale; the rows
  // then take the factor from that lane.
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    raw[i].get(f[i]);
    const float a = block_amax(f[i]);
    if ((lane & (kRows - 1)) == i) m = a;
  }
  float inv;
  const float s = block_scale(m, inv);
  const int row = lane & 15, half = lane >> 4;
  if (row < rows && half * kBlock < n)
    p.scale[(r0 + row) * p.scale_rs + (c0 / kBlock + half) * p.scale_bs] = s;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const float v = __shfl_sync(0xffffffffu, inv, (lane & 16) + i);
    store_e4m3<kVec>(p.dst + (r0 + i) * p.dst_stride + c0, lane, i < rows ? n : 0, f[i], v,
                     p.on8 != 0);
  }
}

template <typename T>
__global__ void __launch_bounds__(256) quantize_tiles_kernel(const __grid_constant__ QuantizeParams p) {
  __shared__ float part[8];
  const long long grp = blockIdx.x / p.chunks;
  const int blk = static_cast<int>(blockIdx.x - grp * p.chunks);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c0 = blk * kBlock;
  // warp w: rows w, w + 8, ...; lane l: features l, l + 32, l + 64, l + 96
  float f[16][4];
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const long long r = grp * kBlock + warp + 8 * i;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = c0 + 32 * j + lane;
      f[i][j] = 0.f;
      if (r < p.rows && c < p.dim) f[i][j] = to_float(static_cast<const T*>(p.src)[r * p.src_stride + c]);
    }
    m = fmaxf(m, amax4(f[i][0], f[i][1], f[i][2], f[i][3]));
  }
  m = lanes_max<32>(m);
  if (lane == 0) part[warp] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, part[i]);
  float inv;
  const float s = block_scale(m, inv);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const long long r = grp * kBlock + warp + 8 * i;
    const uint32_t q = pack_e4m3x4(f[i][0] * inv, f[i][1] * inv, f[i][2] * inv, f[i][3] * inv);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = c0 + 32 * j + lane;
      if (r < p.rows && c < p.dim) p.dst[r * p.dst_stride + c] = static_cast<uint8_t>(q >> (8 * j));
    }
  }
  if (threadIdx.x == 0) p.scale[grp * p.scale_rs + blk * p.scale_bs] = s;
}

}  // namespace fp8
}  // namespace vx
