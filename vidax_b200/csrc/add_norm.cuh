// Residual addition, RMSNorm or LayerNorm, modulation and the output's
// rounding (bf16, or e4m3 with a scale per 128 features) in one pass over the
// residual stream.
//
//   h = x + y * gate[batch]                 stored in the stream's type; the
//                                           norm is that of the stored value
//   m = 0 (RMS) or mean(h) (layer)
//   n = (h - m) / sqrt(mean((h - m)^2) + eps) * w + b
//   o = n * (1 + scale[batch]) + shift[batch]
//
// HBM-bound: the row is read once and stays in registers between its
// statistics and its output (W warps per row, NV vectors of eight features
// per lane), so a float32 stream costs 4 + 2 bytes read and 4 + 1 written per
// element. The separate gated addition and norm read it twice (16 bytes with
// a bf16 output). The layer norm's variance is the mean of (h - m)^2 from
// those registers, not E[h^2] - m^2, which loses digits when |m| is large.
// A vector's features lie side by side in a lane, so a half-warp holds one
// block of the e4m3 output and its largest magnitude is four shuffles away.
// NV = 0 serves rows too wide for the registers: it reads the stored sum
// again for each statistic and for the output.
#pragma once

#include "fp8_common.cuh"

namespace vx {
namespace fp8 {

struct AddNormParams {
  const void* x;
  void* sum;                  // NULL: the sum is not stored (no y)
  const __nv_bfloat16* y;     // NULL: no addition
  const float* gate;          // (batches, dim) or NULL
  const float* w;             // (dim) or NULL
  const float* b;             // (dim) or NULL
  const float* scale;         // (batches, dim) or NULL
  const float* shift;         // (batches, dim) or NULL
  void* out;                  // bf16, or e4m3 when out_scale is given
  float* out_scale;
  long long x_stride, sum_stride, y_stride, out_stride;     // elements between rows
  long long gate_stride, scale_stride, shift_stride;        // floats between batch items
  long long out_scale_rs, out_scale_bs;
  long long rows;
  long long rows_per_batch;
  int dim;
  int layer;                  // 1: LayerNorm, 0: RMSNorm
  float eps;
};

template <int W>
__device__ __forceinline__ float row_sum(float v, float* part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (W == 1) return v;
  // The W warps of a row are neighbours; the whole CTA takes part in the
  // barriers (rows past the end too), so `part` may be used again after the
  // second one.
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) part[warp] = v;
  __syncthreads();
  v = 0.f;
#pragma unroll
  for (int i = 0; i < W; ++i) v += part[(warp / W) * W + i];
  __syncthreads();
  return v;
}

template <typename T>
__device__ __forceinline__ float stored(float v);
template <>
__device__ __forceinline__ float stored<float>(float v) { return v; }
template <>
__device__ __forceinline__ float stored<__nv_bfloat16>(float v) {
  return __bfloat162float(__float2bfloat16(v));
}

// One row's addresses.
template <typename T>
struct AddNormRow {
  const T* x;
  T* sum;
  const __nv_bfloat16* y;
  const float *gate, *scale, *shift;
  long long row;
};

// h of features [c, c + 8), of which `n` exist; stores the sum.
template <typename T, bool kVec>
__device__ __forceinline__ void add8(const AddNormParams& p, const AddNormRow<T>& r, int c, int n,
                                     float (&h)[8]) {
  load8<kVec>(r.x + (n > 0 ? c : 0), n, h);
  if (p.y == nullptr) return;
  float y[8];
  load8<kVec>(r.y + (n > 0 ? c : 0), n, y);
  if (r.gate != nullptr) {
    float g[8];
    load8<kVec>(r.gate + (n > 0 ? c : 0), n, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = stored<T>(fmaf(y[i], g[i], h[i]));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = stored<T>(h[i] + y[i]);
  }
  if (n > 0) store8<kVec>(r.sum + c, n, h);
}

// Normalises, modulates, rounds and stores features [c, c + 8).
template <typename T, bool kVec>
__device__ __forceinline__ void out8(const AddNormParams& p, const AddNormRow<T>& r, int c, int n,
                                     float mean, float rstd, float (&h)[8]) {
  const int cc = n > 0 ? c : 0;
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = (h[i] - mean) * rstd;
  if (p.w != nullptr) {
    load8<kVec>(p.w + cc, n, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] *= v[i];
  }
  if (p.b != nullptr) {
    load8<kVec>(p.b + cc, n, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] += v[i];
  }
  if (r.scale != nullptr) {
    load8<kVec>(r.scale + cc, n, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] *= 1.f + v[i];
  }
  if (r.shift != nullptr) {
    load8<kVec>(r.shift + cc, n, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] += v[i];
  }
  if (p.out_scale == nullptr) {
    if (n > 0) store8<kVec>(static_cast<__nv_bfloat16*>(p.out) + r.row * p.out_stride + c, n, h);
    return;
  }
  if (n < 8) {  // features past the row's end are not 0 any more
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i >= n) h[i] = 0.f;
  }
  float inv;
  const float s = block_scale(half_warp_max(amax8(h)), inv);
  if (n > 0) {
    store8_e4m3<kVec>(static_cast<uint8_t*>(p.out) + r.row * p.out_stride + c, n, quantize8(h, inv));
    if ((threadIdx.x & 15) == 0)
      p.out_scale[r.row * p.out_scale_rs + static_cast<long long>(c / kBlock) * p.out_scale_bs] = s;
  }
}

template <typename T, int W, int NV, bool kVec>
__global__ void __launch_bounds__(256) add_norm_kernel(const __grid_constant__ AddNormParams p) {
  __shared__ float part[8];
  const int lane_in_row = threadIdx.x & (32 * W - 1);
  long long row = static_cast<long long>(blockIdx.x) * (8 / W) + (threadIdx.x / (32 * W));
  // Rows past the end work on nothing but stay for the barriers and shuffles.
  const int dim = row < p.rows ? p.dim : 0;
  if (row >= p.rows) row = p.rows - 1;
  const long long bi = row / p.rows_per_batch;
  AddNormRow<T> r;
  r.x = static_cast<const T*>(p.x) + row * p.x_stride;
  r.sum = p.sum != nullptr ? static_cast<T*>(p.sum) + row * p.sum_stride : nullptr;
  r.y = p.y != nullptr ? p.y + row * p.y_stride : nullptr;
  r.gate = p.gate != nullptr ? p.gate + bi * p.gate_stride : nullptr;
  r.scale = p.scale != nullptr ? p.scale + bi * p.scale_stride : nullptr;
  r.shift = p.shift != nullptr ? p.shift + bi * p.shift_stride : nullptr;
  r.row = row;
  const float inv_n = 1.f / static_cast<float>(p.dim);
  constexpr int kStep = 32 * W * 8;
  if constexpr (NV > 0) {
    float h[NV][8];
    float s = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = v * kStep + lane_in_row * 8;
      add8<T, kVec>(p, r, c, dim - c, h[v]);
    }
    float mean = 0.f;
    if (p.layer) {
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) s += h[v][i];
      mean = row_sum<W>(s, part) * inv_n;
      s = 0.f;
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int n = dim - (v * kStep + lane_in_row * 8);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = i < n ? h[v][i] - mean : 0.f;
        s = fmaf(d, d, s);
      }
    }
    const float rstd = 1.f / sqrtf(row_sum<W>(s, part) * inv_n + p.eps);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = v * kStep + lane_in_row * 8;
      out8<T, kVec>(p, r, c, dim - c, mean, rstd, h[v]);
    }
  } else {
    float h[8];
    float s = 0.f, s2 = 0.f;
    for (int c0 = 0; c0 < p.dim; c0 += kStep) {
      const int c = c0 + lane_in_row * 8;
      add8<T, kVec>(p, r, c, dim - c, h);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s += h[i];
        s2 = fmaf(h[i], h[i], s2);
      }
    }
    const T* src = p.y != nullptr ? r.sum : r.x;
    float mean = 0.f;
    if (p.layer) {
      mean = row_sum<W>(s, part) * inv_n;
      s2 = 0.f;
      for (int c0 = 0; c0 < p.dim; c0 += kStep) {
        const int c = c0 + lane_in_row * 8;
        load8<kVec>(src + (dim > c ? c : 0), dim - c, h);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float d = i < dim - c ? h[i] - mean : 0.f;
          s2 = fmaf(d, d, s2);
        }
      }
    }
    const float rstd = 1.f / sqrtf(row_sum<W>(s2, part) * inv_n + p.eps);
    for (int c0 = 0; c0 < p.dim; c0 += kStep) {
      const int c = c0 + lane_in_row * 8;
      load8<kVec>(src + (dim > c ? c : 0), dim - c, h);
      out8<T, kVec>(p, r, c, dim - c, mean, rstd, h);
    }
  }
}

}  // namespace fp8
}  // namespace vx
