// The e4m3 matrix product for a few rows (one token up to 16): see
// fp8_linear.cuh for the formula.
//
// Bound by the weights' bytes, so by how many loads are in flight: a 128-row
// tile of the other kernel leaves most SMs idle and walks the features one
// block after the other. Here a CTA takes 16 output features and its warps
// share the input features, up to four blocks at once, straight from global
// memory into the fragments of mma.sync (m16n8k32: the weights are the 16
// rows, eight tokens the columns; no shared memory, TMEM or barriers on the
// way). The order of the features inside a block is free as long as both
// operands agree on it, so a lane loads 16 consecutive bytes and feeds them to
// two MMAs. The warps' sums meet in shared memory and are added in the order
// of the warps: the result does not depend on timing.
//
// Eight tokens, weights from HBM, in us (floor by bytes / this / the better of
// the 128-row tiles): 1536 -> 1536 0.4 / 2.6 / 5.5, 1536 -> 9216 2.2 / 6.1 /
// 9.0, 8960 -> 1536 2.1 / 6.9 / 17.3, 5120 -> 13824 11 / 17 / 25. Sixteen: 3.0 /
// 5.6, 6.7 / 8.8, 8.6 / 17.2 and 20 / 24; 13824 -> 5120 is even at 25. Beyond,
// the MMAs per load show.
//
// The e4m3 output needs the largest magnitude of 128 features: the eight CTAs
// that hold them form a cluster and read it from one another's shared memory.
// That costs some 3 us (1536 -> 8960 with GELU: one token 8.0 against 9.7 with
// the tiles, sixteen 12.2 against 9.4, so past eight tokens the tiles take
// outputs with many CTAs; 8960 -> 1536 stays ahead, 8.6 against 22.6).
#pragma once

#include <type_traits>

#include "fp8_linear.cuh"

namespace vx {
namespace fp8 {

constexpr int kFewCols = 16;     // output features per CTA
constexpr int kFewMost = 16;     // rows

struct FewParams {
  const uint8_t* x;
  const uint8_t* w;
  long long x_stride, w_stride;
  int k;
  LinearParams l;
};

__device__ __forceinline__ void mma_e4m3_16832(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                               uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes at feature k0 of a row; those at k and after are 0 (what lies there
// may be anything, a NaN times 0 too, and in the last row behind the tensor: the
// 16 bytes are aligned, so the row's own ones are in the same page).
__device__ __forceinline__ uint4 few_load(const uint8_t* row, int k0, int k) {
  uint4 v = make_uint4(0u, 0u, 0u, 0u);
  if (k0 < k) {
    v = *reinterpret_cast<const uint4*>(row + k0);
    const int have = k - k0;
    if (have < 16) {
      uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int h = have - 4 * i;
        w[i] = h >= 4 ? w[i] : h <= 0 ? 0u : w[i] & (0xffffffffu >> (32 - 8 * h));
      }
    }
  }
  return v;
}

template <int kWarps, int kNT, int kOut>
__global__ void __launch_bounds__(kWarps * 32, (kNT == 1 ? 24 : 16) / kWarps)
    linear_few_kernel(const __grid_constant__ FewParams p) {
  constexpr int kTok = 8 * kNT;
  __shared__ float part[kWarps][kTok][kFewCols + 1];
  __shared__ float amax_s[kTok];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int col0 = blockIdx.x * kFewCols;
  // rows past the end read the last one; their sums are not stored
  const uint8_t* w0 = p.w + static_cast<long long>(min(col0 + g, p.l.n - 1)) * p.w_stride;
  const uint8_t* w1 = p.w + static_cast<long long>(min(col0 + g + 8, p.l.n - 1)) * p.w_stride;
  const uint8_t* xr[kNT];
  const float* xs[kNT][2];
#pragma unroll
  for (int j = 0; j < kNT; ++j) {
    xr[j] = p.x + static_cast<long long>(min(8 * j + g, p.l.m - 1)) * p.x_stride;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      xs[j][i] = p.l.xs + static_cast<long long>(min(8 * j + 2 * t + i, p.l.m - 1)) * p.l.xs_rs;
  }
  const float* ws = p.l.ws + static_cast<long long>(min(col0, p.l.n - 1) / kBlock) * p.l.ws_rs;
  float acc[kNT][4] = {};
  // kBlocks blocks from kb on, kWarps apart; kTail: the block that may be short
  auto blocks = [&](int kb, auto count, auto tail) {
    constexpr int kBlocks = decltype(count)::value;
    constexpr bool kTail = decltype(tail)::value;
    uint4 a[kBlocks][2][2], b[kBlocks][kNT][2];
    float sw[kBlocks], sx[kBlocks][kNT][2];
    auto load = [&](const uint8_t* row, int k0) {
      return kTail ? few_load(row, k0, p.k) : *reinterpret_cast<const uint4*>(row + k0);
    };
#pragma unroll
    for (int u = 0; u < kBlocks; ++u) {
      const int kk = kb + u * kWarps, k0 = kk * kBlock + t * 16;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        a[u][c][0] = load(w0, k0 + 64 * c);
        a[u][c][1] = load(w1, k0 + 64 * c);
#pragma unroll
        for (int j = 0; j < kNT; ++j) b[u][j][c] = load(xr[j], k0 + 64 * c);
      }
      sw[u] = ws[kk * p.l.ws_bs];
#pragma unroll
      for (int j = 0; j < kNT; ++j) {
        sx[u][j][0] = xs[j][0][kk * p.l.xs_bs];
        sx[u][j][1] = xs[j][1][kk * p.l.xs_bs];
      }
    }
#pragma unroll
    for (int u = 0; u < kBlocks; ++u)
#pragma unroll
      for (int j = 0; j < kNT; ++j) {
        float s[4] = {};
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          mma_e4m3_16832(s, a[u][c][0].x, a[u][c][1].x, a[u][c][0].y, a[u][c][1].y, b[u][j][c].x,
                         b[u][j][c].y);
          mma_e4m3_16832(s, a[u][c][0].z, a[u][c][1].z, a[u][c][0].w, a[u][c][1].w, b[u][j][c].z,
                         b[u][j][c].w);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          acc[j][i] = fmaf(s[i], sx[u][j][i & 1] * sw[u], acc[j][i]);
      }
  };
  const int full = p.k / kBlock;
  int kb = warp;
  if constexpr (kNT == 1) {  // (16 tokens' operands of four blocks do not fit the registers)
    for (; kb + 3 * kWarps < full; kb += 4 * kWarps)
      blocks(kb, std::integral_constant<int, 4>(), std::false_type());
  }
  for (; kb + kWarps < full; kb += 2 * kWarps)
    blocks(kb, std::integral_constant<int, 2>(), std::false_type());
  for (; kb < full; kb += kWarps) blocks(kb, std::integral_constant<int, 1>(), std::false_type());
  if (kb < p.l.kblocks) blocks(kb, std::integral_constant<int, 1>(), std::true_type());
#pragma unroll
  for (int j = 0; j < kNT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) part[warp][8 * j + 2 * t + (i & 1)][g + 8 * (i >> 1)] = acc[j][i];
  __syncthreads();
  constexpr int kVals = kTok * kFewCols;
  constexpr int kThreads = kWarps * 32;
  constexpr int kPer = (kVals + kThreads - 1) / kThreads;
  float y[kPer];
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    const int v = threadIdx.x + q * kThreads;
    const int row = v / kFewCols, c = v % kFewCols;
    y[q] = 0.f;
    if (v < kVals && row < p.l.m && col0 + c < p.l.n) {
      float s = p.l.bias != nullptr ? p.l.bias[col0 + c] : 0.f;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) s += part[i][row][c];
      if (p.l.act == kActGeluTanh) {
        float one = 0.f;
        gelu_tanh2(s, one);
      }
      y[q] = s;
    }
  }
  float inv[kPer];
  if constexpr (kOut == kOutE4m3) {
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
      // 16 lanes hold a row's 16 features
      const int v = threadIdx.x + q * kThreads;
      const float m = lanes_max<16>(fabsf(y[q]));
      if (v < kVals && v % kFewCols == 0) amax_s[v / kFewCols] = m;
    }
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
      const int v = threadIdx.x + q * kThreads;
      const int row = min(v / kFewCols, kTok - 1);
      const uint32_t at = smem_u32(&amax_s[row]);
      float m = 0.f;
#pragma unroll
      for (int r = 0; r < kBlock / kFewCols; ++r) {
        uint32_t peer;
        float other;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(at), "r"(r));
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(other) : "r"(peer) : "memory");
        m = fmaxf(m, other);
      }
      const float s = block_scale(m, inv[q]);
      if (v < kVals && row < p.l.m && v % kFewCols == 0 && col0 % kBlock == 0 && col0 < p.l.n)
        p.l.out_scale[row * p.l.os_rs + static_cast<long long>(col0 / kBlock) * p.l.os_bs] = s;
    }
    // a CTA's shared memory stays until all have read it
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
  }
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    const int v = threadIdx.x + q * kThreads;
    const int row = v / kFewCols, c = v % kFewCols;
    if (v < kVals && row < p.l.m && col0 + c < p.l.n) {
      const long long at = row * p.l.out_stride + col0 + c;
      if constexpr (kOut == kOutBf16)
        static_cast<__nv_bfloat16*>(p.l.out)[at] = __float2bfloat16(y[q]);
      else if constexpr (kOut == kOutFloat) static_cast<float*>(p.l.out)[at] = y[q];
      else
        static_cast<uint8_t*>(p.l.out)[at] =
            static_cast<uint8_t>(pack_e4m3x4(y[q] * inv[q], 0.f, 0.f, 0.f));
    }
  }
}

}  // namespace fp8
}  // namespace vx
