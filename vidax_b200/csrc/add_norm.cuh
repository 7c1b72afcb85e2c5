// Residual addition, RMSNorm or LayerNorm, modulation and the output's
// rounding (bf16, or e4m3 with a scale per 128 features) in one pass over the
// residual stream.
//
//   h = x + y * gate[batch]                 stored in the stream's type; the
//                                           norm is that of the stored value
//   m = 0 (RMS) or mean(h) (layer)
//   o = (h - m) / sqrt(mean((h - m)^2) + eps) * A + B
//   A = w (1 + scale[batch]),  B = b (1 + scale[batch]) + shift[batch]
//
// HBM-bound: the row is read once and stays in registers between its
// statistics and its output (W warps per row, NV chunks of eight features per
// lane), so a float32 stream costs 4 + 2 bytes read and 4 + 1 written per
// element; a gated addition and a norm apart read it twice (16 bytes with a
// bf16 output). The layer norm's variance is the mean of (h - m)^2 from those
// registers, not E[h^2] - m^2, which loses digits when |m| is large.
//
// All of a row's loads are issued before anything is stored: a store between
// them would order them (the stream may be updated in place), and the kernel
// ran at 44 % of the measured copy bandwidth that way. For the same reason A,
// B and the gate lie in shared memory, made once per CTA and batch item; a CTA
// takes a run of neighbouring rows.
//
// add_norm_wide_kernel serves rows too wide for that (dim > 16384): it reads
// the stored sum again for each statistic and for the output.
#pragma once

#include "fp8_common.cuh"

namespace vx {
namespace fp8 {

struct AddNormParams {
  const void* x;
  void* sum;                  // with y
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
  long long rows_per_cta;
  int dim;
  int layer;                  // 1: LayerNorm, 0: RMSNorm
  float eps;
  int sum_on16, out_on16;     // rows of the sum / output on 16-byte (e4m3: 8-byte) boundaries
  int cap;                    // dim rounded up to 256
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

__device__ __forceinline__ float stored(float v, float) { return v; }
__device__ __forceinline__ float stored(float v, __nv_bfloat16) {
  return __bfloat162float(__float2bfloat16(v));
}

// A and B of feature c of batch item bi.
__device__ __forceinline__ void affine(const AddNormParams& p, long long bi, int c, float& a,
                                       float& b) {
  a = p.w != nullptr ? p.w[c] : 1.f;
  b = p.b != nullptr ? p.b[c] : 0.f;
  if (p.scale != nullptr) {
    const float s = 1.f + p.scale[bi * p.scale_stride + c];
    a *= s;
    b *= s;
  }
  if (p.shift != nullptr) b += p.shift[bi * p.shift_stride + c];
}

// The lane's eight values of a chunk of floats in shared memory.
__device__ __forceinline__ void smem8(const float* chunk, int lane, float (&f)[8]) {
  const float4 a = reinterpret_cast<const float4*>(chunk)[2 * lane];
  const float4 b = reinterpret_cast<const float4*>(chunk)[2 * lane + 1];
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
  f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}

template <bool kVec>
__device__ __forceinline__ void store_out(const AddNormParams& p, long long row, int c0, int lane,
                                          int n, const float (&o)[8], void* turn) {
  if (p.out_scale == nullptr)
    store_chunk<kVec>(static_cast<__nv_bfloat16*>(p.out) + row * p.out_stride + c0, lane, n, o,
                      p.out_on16 != 0, turn);
  else
    quantize_chunk<kVec>(static_cast<uint8_t*>(p.out) + row * p.out_stride + c0,
                         p.out_scale + row * p.out_scale_rs + (c0 / kBlock) * p.out_scale_bs,
                         p.out_scale_bs, lane, n, o, p.out_on16 != 0);
}

template <typename T, int W, int NV, bool kVec>
__global__ void __launch_bounds__(256) add_norm_kernel(const __grid_constant__ AddNormParams p) {
  __shared__ float part[8];
  __shared__ float4 turn_smem[kVec ? 1 : 8 * 64];
  extern __shared__ float4 norm_smem[];
  float* const sa = reinterpret_cast<float*>(norm_smem);
  float* const sb = sa + p.cap;
  float* const sg = sb + p.cap;  // with y only
  void* const turn = turn_smem + (kVec ? 0 : (threadIdx.x >> 5) * 64);
  // Narrow rows: the next row's loads start before this one's statistics.
  constexpr bool kAhead = NV <= 2;
  const int lane = threadIdx.x & 31;
  const int chunk0 = ((threadIdx.x >> 5) & (W - 1)) * 256;  // + 256 W v
  const float inv_n = 1.f / static_cast<float>(p.dim);
  const long long last = min(p.rows, (blockIdx.x + 1LL) * p.rows_per_cta);
  for (long long row0 = blockIdx.x * p.rows_per_cta; row0 < last;) {
    const long long bi = row0 / p.rows_per_batch;
    const long long end = min(last, (bi + 1) * p.rows_per_batch);
    for (int c = threadIdx.x; c < p.cap; c += 256) {  // past the row's end: 0
      float a = 0.f, b = 0.f, g = 0.f;
      if (c < p.dim) {
        affine(p, bi, c, a, b);
        g = p.gate != nullptr ? p.gate[bi * p.gate_stride + c] : 1.f;
      }
      sa[c] = a;
      sb[c] = b;
      if (p.y != nullptr) sg[c] = g;
    }
    __syncthreads();
    // Rows past the segment's end work on its last row and store nothing, but
    // stay for the barriers and shuffles.
    Raw<T, kVec> rx[NV];
    Raw<__nv_bfloat16, kVec> ry[NV];
    auto load_row = [&](long long r0) {
      const long long row = min(r0 + threadIdx.x / (32 * W), end - 1);
      const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int c0 = chunk0 + 256 * W * v;
        rx[v].load(x + c0, lane, p.dim - c0);
      }
      if (p.y != nullptr) {
        const __nv_bfloat16* y = p.y + row * p.y_stride;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          const int c0 = chunk0 + 256 * W * v;
          ry[v].load(y + c0, lane, p.dim - c0);
        }
      }
    };
    if (kAhead) load_row(row0);
    for (; row0 < end; row0 += 8 / W) {
      const long long mine = row0 + threadIdx.x / (32 * W);
      const bool live = mine < end;
      const long long row = live ? mine : end - 1;
      if (!kAhead) load_row(row0);
      float h[NV][8];
#pragma unroll
      for (int v = 0; v < NV; ++v) rx[v].get(h[v]);
      if (p.y != nullptr) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          const int c0 = chunk0 + 256 * W * v;
          if (c0 >= p.dim) break;  // the warp's remaining chunks lie past the row's end
          float yv[8], g[8];
          ry[v].get(yv);
          smem8(sg + c0, lane, g);
#pragma unroll
          for (int i = 0; i < 8; ++i) h[v][i] = stored(fmaf(yv[i], g[i], h[v][i]), T());
        }
      }
      // In place, the next rows are other rows: their loads may pass the stores.
      if (kAhead && row0 + 8 / W < end) load_row(row0 + 8 / W);
      if (p.y != nullptr) {
        // In place is fine: each lane writes only the features it has read itself.
        T* sum = static_cast<T*>(p.sum) + row * p.sum_stride;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          const int c0 = chunk0 + 256 * W * v;
          store_chunk<kVec>(sum + c0, lane, live ? p.dim - c0 : 0, h[v], p.sum_on16 != 0, turn);
        }
      }
      float mean = 0.f, s = 0.f;
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
        const int n = p.dim - (chunk0 + 256 * W * v) - lane * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          h[v][i] -= mean;
          const float d = i < n ? h[v][i] : 0.f;
          s = fmaf(d, d, s);
        }
      }
      const float rstd = 1.f / sqrtf(row_sum<W>(s, part) * inv_n + p.eps);
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int c0 = chunk0 + 256 * W * v;
        if (c0 >= p.dim) break;
        float a[8], b[8];
        smem8(sa + c0, lane, a);
        smem8(sb + c0, lane, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[v][i] = fmaf(h[v][i] * rstd, a[i], b[i]);
        store_out<kVec>(p, row, c0, lane, live ? p.dim - c0 : 0, h[v], turn);
      }
    }
    row0 = end;
    __syncthreads();  // A, B and the gate are read before the next batch item's are written
  }
}

template <typename T, bool kVec>
__global__ void __launch_bounds__(256) add_norm_wide_kernel(const __grid_constant__ AddNormParams p) {
  __shared__ float part[8];
  __shared__ float4 turn_smem[8 * 64];
  void* const turn = turn_smem + (threadIdx.x >> 5) * 64;
  const int lane = threadIdx.x & 31;
  const int chunk0 = (threadIdx.x >> 5) * 256;
  const long long row = blockIdx.x;
  const long long bi = row / p.rows_per_batch;
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
  const float inv_n = 1.f / static_cast<float>(p.dim);
  float s = 0.f, s2 = 0.f, mean = 0.f;
  for (int c0 = chunk0; c0 < p.dim; c0 += 2048) {
    const int n = p.dim - c0;
    Raw<T, kVec> rx;
    float h[8];
    rx.load(x + c0, lane, n);
    rx.get(h);
    if (p.y != nullptr) {
      Raw<__nv_bfloat16, kVec> ry;
      Raw<float, kVec> rg;
      float y[8], g[8];
      ry.load(p.y + row * p.y_stride + c0, lane, n);
      ry.get(y);
      if (p.gate != nullptr) {
        rg.load(p.gate + bi * p.gate_stride + c0, lane, n);
        rg.get(g);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        h[i] = stored(p.gate != nullptr ? fmaf(y[i], g[i], h[i]) : h[i] + y[i], T());
      store_chunk<kVec>(static_cast<T*>(p.sum) + row * p.sum_stride + c0, lane, n, h,
                        p.sum_on16 != 0, turn);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      s += h[i];
      s2 = fmaf(h[i], h[i], s2);
    }
  }
  // read again below, in rows off the boundaries by other lanes of the warp
  __syncwarp();
  const T* src = p.y != nullptr ? static_cast<const T*>(p.sum) + row * p.sum_stride : x;
  if (p.layer) {
    mean = row_sum<8>(s, part) * inv_n;
    s2 = 0.f;
    for (int c0 = chunk0; c0 < p.dim; c0 += 2048) {
      const int n = p.dim - c0;
      Raw<T, kVec> rx;
      float h[8];
      rx.load(src + c0, lane, n);
      rx.get(h);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = lane * 8 + i < n ? h[i] - mean : 0.f;
        s2 = fmaf(d, d, s2);
      }
    }
  }
  const float rstd = 1.f / sqrtf(row_sum<8>(s2, part) * inv_n + p.eps);
  for (int c0 = chunk0; c0 < p.dim; c0 += 2048) {
    const int n = p.dim - c0;
    Raw<T, kVec> rx;
    float h[8];
    rx.load(src + c0, lane, n);
    rx.get(h);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = lane * 8 + i;
      float a = 0.f, b = 0.f;
      if (c < n) affine(p, bi, c0 + c, a, b);
      h[i] = fmaf((h[i] - mean) * rstd, a, b);
    }
    store_out<kVec>(p, row, c0, lane, n, h, turn);
  }
}

}  // namespace fp8
}  // namespace vx
