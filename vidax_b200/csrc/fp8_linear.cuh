// Matrix product of e4m3 activations and weights with a float32 scale for
// each 128 features (activations: per row; weights: per 128 output features):
//
//   y[m, n] = act( sum_b xs[m, b] ws[n / 128, b] * S_b[m, n]  +  bias[n] )
//   S_b[m, n] = sum over the 128 features k of block b of xq[m, k] wq[n, k]
//
// S_b is an exact-input tensor-core product (tcgen05 kind::f8f6f4, float32
// accumulator in TMEM); the scales differ from block to block, so each S_b
// leaves TMEM and is added to a float32 sum in registers. The tensor core
// works on the next block meanwhile: TMEM holds two products of a 256-wide
// tile, four of the narrower ones.
//
// CTA roles: two or four warpgroups each add up their share of the tile's
// columns (thread = row); of the last warpgroup, the first warp feeds shared
// memory by TMA, the second and the fourth issue the MMAs, the third fetches
// the scales (cp.async, any strides) up to 16 blocks ahead: read from global
// memory where they are used, their latency cost a third of the time of a long
// sum. CTAs are persistent: each strides over the output tiles, and the roles'
// barrier phases run on across tiles, so the next tile's loads and products
// start while the last one is rounded and stored. A finished tile leaves
// through shared memory by TMA (full 128-byte lines, edges clipped by the
// tensor map); an output that TMA cannot address leaves it row by row, and so
// do the last columns of rows that do not end on a 16-byte boundary, where the
// tensor map clips at the next one and up to 15 bytes behind the row would be
// written.
//
// What bounds it, measured on 9472 x 8960 -> 2048 (171-188 us, 1930 TFLOP/s, a
// plain e4m3 product of the library 131 us): the power cap (1000 W, at 1425 of
// 1965 MHz). Of the time, adding the scaled products is some 30 us and reading
// them from TMEM 10. A block takes 920 cycles, 512 of them MMAs; the rest is
// the way from one to the next use of a TMEM buffer (MMA, commit, a look at
// the barrier of 110 cycles, the read, the hand-back). Taking cycles out of
// that way lowers the clock instead of the time by now. Pairs of CTAs on one
// 256 x 256 tile (cta_group::2), which load a third less, ran as fast within
// 2 %; two CTAs per SM with half of TMEM each, or two sets of warpgroups on
// tiles in turn, were 25 to 60 % slower.
//
// If a wait runs out of its limit, it raises the abort flag, and with the flag
// up the other waits for loads, scales and row maxima give up soon. The loads
// stop there; the issuers and the adding warps still walk all of their blocks,
// in step with one another (lin_wait_product says why that always ends). Then
// the loads in flight are waited for (with a limit), and the CTA ends with the
// code in the status word and an output that is not valid.
#pragma once

#include <type_traits>

#include "fp8_common.cuh"

namespace vx {
namespace fp8 {

enum : int { kOutBf16 = 0, kOutFloat = 1, kOutE4m3 = 2 };
enum : int { kActNone = 0, kActGeluTanh = 1 };

struct LinearParams {
  const float* xs;
  long long xs_rs, xs_bs;       // elements between rows / feature blocks
  const float* ws;
  long long ws_rs, ws_bs;       // elements between row blocks / feature blocks
  const float* bias;            // (n) or NULL
  void* out;
  long long out_stride;         // elements between rows
  float* out_scale;             // e4m3 output only
  long long os_rs, os_bs;
  int m, n, kblocks;
  int tiles_m, tiles_n, tiles;
  int act;
  int tma_out;                  // the output goes through tm_o: 1 all of it,
                                // 2 but the boxes that a row ends in
  int* status;
  // the self-test's form only: the wait limit, and the role (LinDrop) that
  // falls silent at its block `drop_at`
  long long limit;
  int drop, drop_at;
};
enum LinDrop : int { kDropNone = 0, kDropLoads, kDropScales, kDropSums, kNumDrops };

constexpr int kLinRows = 128;          // activation rows per CTA
constexpr int kGroupM = 8;             // row tiles that share a pass over the weights
constexpr int kScaleGroups = 4;        // groups of scales in shared memory,
constexpr int kGroupBlocks = 4;        // of this many blocks each
constexpr int kScaleSlots = kScaleGroups * kGroupBlocks;
constexpr int kScaleFloats = 132;      // 128 rows, the warpgroups' weight scales

template <int kBN>
struct LinDims {
  // Warpgroups that add: four for the widest tile (64 columns each), whose two
  // block products in TMEM leave the reader the shortest time; four warps per
  // SM quarter keep TMEM reads and additions going at once.
  static constexpr int kSumWG = kBN == 256 ? 4 : 2;
  static constexpr int kCols = kBN / kSumWG;
  static constexpr int kThreads = 128 * (kSumWG + 1);
  // Registers: the feeding warpgroup gives some of the launch's share up to
  // the adding ones (640 threads: 96 each, 32 + 4 * 112 = 5 * 96; 384
  // threads: 168 each, 56 + 2 * 224 = 3 * 168).
  static constexpr int kFeedRegs = kSumWG == 4 ? 32 : 56;
  static constexpr int kSumRegs = kSumWG == 4 ? 112 : 224;
  static constexpr uint32_t kABytes = kLinRows * kBlock;
  static constexpr uint32_t kBBytes = kBN * kBlock;
  static constexpr uint32_t kStageBytes = kABytes + kBBytes;
  static constexpr uint32_t kStoreBytes = kSumWG * 4 * 4096;   // 32 rows x 128 bytes per warp
  static constexpr uint32_t kBiasBytes = kSumWG * 4 * kCols * 4;
  static constexpr uint32_t kAmaxBytes = 2 * kSumWG * 512;     // 2 tiles x 128 rows
  static constexpr uint32_t kRest =
      kStoreBytes + kScaleSlots * kScaleFloats * 4 + kBiasBytes + kAmaxBytes + 512;
  static constexpr int kFit = (232448 - 1024 - kRest) / kStageBytes;
  static constexpr int kStages = kFit < 8 ? kFit : 8;
  static constexpr int kBufs = 512 / kBN < 4 ? 512 / kBN : 4;  // block products in TMEM
  // kLinDone serves the sums too: a stage comes round again only after they
  // have read the products that came between.
  static_assert(kStages > kBufs, "stages");
  static constexpr uint32_t kStore = kStages * kStageBytes;
  static constexpr uint32_t kScales = kStore + kStoreBytes;
  static constexpr uint32_t kBias = kScales + kScaleSlots * kScaleFloats * 4;
  static constexpr uint32_t kAmax = kBias + kBiasBytes;
  static constexpr uint32_t kCtl = kAmax + kAmaxBytes;
  static constexpr uint32_t kSmemBytes = kCtl + 512 + 1024;    // + alignment
  static_assert(kSmemBytes <= 232448, "exceeds the 227 KB of shared memory per CTA");
};

// control block: barriers, then the TMEM address, the abort flag and the
// number of blocks loaded
enum : int {
  kLinFull = 0,        // stages: operands landed
  kLinDone = 8,        // stages: their MMAs are done (the stage is free, the product complete)
  kLinAmax = 24,       // every warpgroup's largest magnitudes are written
  kLinScaleFull = 28,  // 4: a group's scales landed
  kLinScaleEmpty = 32, // 4: read by every adding warp
  kLinBars = 36,
};

// Position in a ring of N barriers and the phase parity of its current round.
template <int N>
struct Ring {
  int i = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() {
    if (++i == N) {
      i = 0;
      phase ^= 1u;
    }
  }
};

// True in one lane of the (converged) warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok));
  return ok != 0;
}
// 2-D tiled load (no multicast) into this CTA's shared memory.
__device__ __forceinline__ void lin_load(uint32_t dst, const CUtensorMap* tm, uint32_t bar, int x,
                                         int y, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes"
      ".L2::cache_hint [%0], [%1, {%2, %3}], [%4], %5;" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(tm)), "r"(x), "r"(y), "r"(bar), "l"(policy)
      : "memory");
}

__device__ __forceinline__ void lin_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// kind::f8f6f4 instruction descriptor: e4m3 operands (format 0), K-major,
// float32 accumulator.
__host__ __device__ constexpr uint32_t idesc_e4m3_f32(int M, int N) {
  return (1u << 4) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {  // a NaN if either is one
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
// x / (1 + exp(-2 u)) = 0.5 x (1 + tanh u), u = sqrt(2 / pi) (x + 0.044715 x^3).
// Two elements share one reciprocal, 1/a = b / (a b): the special-function
// unit bounds this step. So that the product of the denominators stays finite,
// x counts as -7.5 where it is less: the denominator is 2^60.7 there and the
// value within 2^-57 of the function's, which goes to 0. The exponent's bound
// keeps a NaN out of its neighbour's reciprocal.
__device__ __forceinline__ void gelu_tanh2(float& x, float& y) {
  constexpr float kA = -2.f * 0.7978845608028654f * 1.4426950408889634f;
  const uint64_t v = f2_pack(max_nan(x, -7.5f), max_nan(y, -7.5f));
  const uint64_t t = f2_mul(
      v, f2_fma(f2_mul(v, v), f2_pack(kA * 0.044715f, kA * 0.044715f), f2_pack(kA, kA)));
  float t0, t1, a, b;
  f2_unpack(t, t0, t1);
  f2_unpack(f2_add(f2_pack(ex2_approx(fminf(t0, 61.f)), ex2_approx(fminf(t1, 61.f))),
                   f2_pack(1.f, 1.f)),
            a, b);
  const float r = rcp_approx(a * b);
  f2_unpack(f2_mul(v, f2_pack(r * b, r * a)), x, y);
}

__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src),
               "r"(there ? 4 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void lin_store(const CUtensorMap* tm, uint32_t src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(tm)),
               "r"(x), "r"(y), "r"(src)
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c,
                                             uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c),
               "r"(d)
               : "memory");
}

// 16 bytes of output: bf16 x 8, float x 4, e4m3 x 16 (already scaled by inv).
template <int kOut>
__device__ __forceinline__ void lin_pack16(const float* v, float inv, uint32_t (&q)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (kOut == kOutBf16) q[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
    else if constexpr (kOut == kOutFloat) q[i] = __float_as_uint(v[i]);
    else
      q[i] = pack_e4m3x4(v[4 * i] * inv, v[4 * i + 1] * inv, v[4 * i + 2] * inv, v[4 * i + 3] * inv);
  }
}

// Hand-over of a TMEM buffer from the sums to an MMA issuer over a named
// barrier: a look at one in shared memory takes 110 cycles while the tensor
// core reads its operands (9472 x 8960 -> 2048: 196 us with an mbarrier, 171
// so; 4680 x 1536 -> 4608: 47.6 and 44.6). A named barrier counts arrivals, not
// who arrived, and has no limit; see lin_wait_product.
template <int kThreads>
__device__ __forceinline__ void lin_buffer_arrive(int buf) {
  asm volatile("bar.arrive %0, %1;" ::"r"(buf + 1), "n"(kThreads) : "memory");
}
template <int kThreads>
__device__ __forceinline__ void lin_buffer_sync(int buf) {
  asm volatile("bar.sync %0, %1;" ::"r"(buf + 1), "n"(kThreads) : "memory");
}

// An adding warp's wait for a block's product. It does not give up with the
// abort flag, because the warp arrives for the block at a named barrier next:
// a warp that ran ahead would arrive twice in one generation, and an issuer
// later wait for an arrival that nobody has left to make. It needs not to. An
// issuer commits for every block, whether its wait for the load was met or gave
// up, after it has taken the hand-over of the block kBufs before in the same
// buffer. So, by induction over the blocks, every product's barrier completes
// and every hand-over comes: block i's product needs the hand-over of block
// i - kBufs, waits that give up and the MMAs' own completion (before which a
// CTA could not end anyway, since they read its memory); the hand-over of block
// i needs every adding warp to have seen product i and waits that give up. And
// an arrival made after product i is seen is one for that block's generation.
// The first wait to run out takes one limit, after which the flag is up; four
// is longer than any of this can take.
__device__ __forceinline__ void lin_wait_product(uint32_t bar, uint32_t parity, volatile int* abort_flag,
                                                 int* status, long long limit) {
  if (mbar_try_wait(bar, parity)) return;
  const long long t0 = clock64();
  for (uint32_t it = 1; !mbar_try_wait(bar, parity); ++it) {
    if ((it & 255u) == 0u && clock64() - t0 > 4 * limit) {
      *abort_flag = 1;
      atomicOr(status, kDevTimeoutSoftmax);
      return;
    }
  }
}

// Output tile -> (row tile, column tile): kGroupM row tiles run down before
// the column advances, so the CTAs at work at one time share both operands
// through L2.
__device__ __forceinline__ void lin_tile(const LinearParams& p, int t, int& tm, int& tn) {
  const int per = kGroupM * p.tiles_n;
  const int g = t / per;
  const int r = t - g * per;
  const int gm = min(kGroupM, p.tiles_m - g * kGroupM);
  tn = r / gm;
  tm = g * kGroupM + (r - tn * gm);
}

// kTest: the form of the self-test (a role falls silent, short wait limit).
template <int kBN, int kOut, bool kTest = false>
__global__ void __launch_bounds__(LinDims<kBN>::kThreads, 1)
    linear_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                  const __grid_constant__ CUtensorMap tm_o, const __grid_constant__ LinearParams p) {
  using Dm = LinDims<kBN>;
  constexpr int S = Dm::kStages, kBufs = Dm::kBufs;
  constexpr int kCols = Dm::kCols;  // columns of a warpgroup
  constexpr int kFeed = 4 * Dm::kSumWG;  // first feeding warp
  extern __shared__ uint8_t smem_dyn[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t sbase = smem_u32(smem);
  auto bar = [&](int i) -> uint32_t { return sbase + Dm::kCtl + 8u * i; };
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + Dm::kCtl + 8 * kLinBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + Dm::kCtl + 8 * kLinBars + 4);
  volatile long long* loaded = reinterpret_cast<volatile long long*>(smem + Dm::kCtl + 8 * kLinBars + 8);
  const long long limit = kTest ? p.limit : kWaitLimitCycles;
  // The shuffle tells the compiler that the warp index is the same in all lanes.
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const int unit0 = blockIdx.x, unit_step = gridDim.x;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(bar(kLinFull + i), 1);
      mbar_init(bar(kLinDone + i), 1);
    }
    for (int i = 0; i < kScaleGroups; ++i) {
      mbar_init(bar(kLinScaleFull + i), 32);
      mbar_init(bar(kLinScaleEmpty + i), kFeed);
    }
    mbar_init(bar(kLinAmax), 32 * kFeed);
    *abort_flag = 0;
    *loaded = 0;
    fence_barrier_init();
  }
  if (warp == kFeed + 1) {
    tmem_alloc(sbase + Dm::kCtl + 8 * kLinBars, 512);
    tmem_relinquish();
  }
  if (warp == kFeed && lane == 0) {
    tma_prefetch_desc(&tm_x);
    tma_prefetch_desc(&tm_w);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);

  if (warp >= kFeed) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Dm::kFeedRegs));
    if (warp == kFeed) {
      // ------------------------------------------------------------ producer
      const uint64_t policy = l2_policy_evict_last();
      const bool issuer = elect_one();
      Ring<S> st;
      long long n = 0;  // blocks loaded
      bool ok = true;
      for (int t = unit0; t < p.tiles && ok; t += unit_step) {
        int tm, tn;
        lin_tile(p, t, tm, tn);
        const int row = tm * kLinRows, col = tn * kBN;
        for (int kb = 0; kb < p.kblocks; ++kb, st.next()) {
          ok = mbar_wait(bar(kLinDone + st.i), st.phase ^ 1u, abort_flag, p.status, kDevTimeoutLoad, limit);
          // After an abort a stage's MMAs may be done without its load: the
          // barrier is armed again only when the load before has landed.
          ok = ok && mbar_wait(bar(kLinFull + st.i), st.phase ^ 1u, abort_flag, p.status, kDevTimeoutLoad,
                               limit);
          if (kTest && p.drop == kDropLoads && n >= p.drop_at) ok = false;
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          ++n;
          const uint32_t dst = sbase + st.i * Dm::kStageBytes;
          if (issuer) {
            mbar_expect_tx(bar(kLinFull + st.i), Dm::kStageBytes);
            lin_load(dst, &tm_x, bar(kLinFull + st.i), kb * kBlock, row, policy);
            lin_load(dst + Dm::kABytes, &tm_w, bar(kLinFull + st.i), kb * kBlock, col, policy);
          }
        }
      }
      if (lane == 0) *loaded = n;
    } else if (warp == kFeed + 1 || warp == kFeed + 3) {
      // ------------------------------------------------------------ MMA issuers
      // Two warps take the blocks in turn, so that one's waits and issues overlap
      // the other's. Blocks are independent (each starts a product), so tiles do
      // not matter here. The whole warp walks the loop and one lane issues:
      // addresses and descriptors then stay in uniform registers.
      constexpr uint32_t kIdesc = idesc_e4m3_f32(kLinRows, kBN);
      const uint64_t desc0 = sdesc_sw128(sbase, 16, 1024);
      const bool issuer = elect_one();
      const int first = warp == kFeed + 3 ? 1 : 0;
      const int tiles = unit0 < p.tiles ? (p.tiles - 1 - unit0) / unit_step + 1 : 0;
      const long long steps = static_cast<long long>(tiles) * p.kblocks;
      Ring<S> st;
      Ring<kBufs> ac;
      if (first) {
        st.next();
        ac.next();
      }
      // steps, and then once more for each buffer, so that every arrival of the
      // sums at the named barriers is met
      for (long long i = first; i < steps + kBufs; i += 2) {
        if (i >= kBufs && i - kBufs < steps)  // the product before in this buffer has been read
          lin_buffer_sync<Dm::kSumWG * 128 + 32>(ac.i);
        if (i < steps) {
          // Only after that: an issuer sees every other block, and with an odd
          // number of stages the stage's last round was the other issuer's. A
          // wait tells odd rounds from even ones only, so a look while that
          // round's load (block i - kStages) is under way would pass. Once block
          // i - kBufs has been added, so has the one before it in this stage
          // (kBufs < kStages).
          mbar_wait(bar(kLinFull + st.i), st.phase, abort_flag, p.status, kDevTimeoutMma, limit);
          tc_fence_after();
          const uint64_t da = desc0 + static_cast<uint32_t>(st.i * (Dm::kStageBytes >> 4));
          const uint64_t db = da + (Dm::kABytes >> 4);
          const uint32_t acc = tmem + ac.i * kBN;
          if (issuer) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)  // 32 features per MMA
              lin_mma(acc, da + 2 * kk, db + 2 * kk, kIdesc, kk > 0 ? 1u : 0u);
            tc_commit(bar(kLinDone + st.i));
          }
        }
        __syncwarp();  // the named barrier wants the warp together
        st.next();
        st.next();
        ac.next();
        ac.next();
      }
    } else if (warp == kFeed + 2) {
      // ------------------------------------------------------------ scales
      Ring<kScaleGroups> sg;
      for (int t = unit0; t < p.tiles; t += unit_step) {
        int tm, tn;
        lin_tile(p, t, tm, tn);
        const int row = tm * kLinRows + lane;
        const int col = tn * kBN + (lane & (Dm::kSumWG - 1)) * kCols;
        const float* xs[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          xs[i] = p.xs + (row + 32 * i < p.m ? (row + 32 * i) * p.xs_rs : 0);
        const float* ws = p.ws + (col < p.n ? static_cast<long long>(col / kBlock) * p.ws_rs : 0);
        for (int kb0 = 0; kb0 < p.kblocks; kb0 += kGroupBlocks, sg.next()) {
          if (kTest && p.drop == kDropScales && kb0 >= p.drop_at) {
            t = p.tiles;  // no more tiles either
            break;
          }
          mbar_wait(bar(kLinScaleEmpty + sg.i), sg.phase ^ 1u, abort_flag, p.status, kDevTimeoutLoad, limit);
          const int n = min(kGroupBlocks, p.kblocks - kb0);
          uint32_t dst = sbase + Dm::kScales + sg.i * (kGroupBlocks * kScaleFloats * 4) + lane * 4;
          for (int kb = kb0; kb < kb0 + n; ++kb, dst += kScaleFloats * 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              cp_async4(dst + 128 * i, xs[i] + kb * p.xs_bs, row + 32 * i < p.m);
            if (lane < Dm::kSumWG) cp_async4(dst + 512, ws + kb * p.ws_bs, col < p.n);
          }
          cp_async_arrive(bar(kLinScaleFull + sg.i));
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Dm::kSumRegs));
    // ------------------------------------------------------------ sums and output
    const int wg = warp >> 2;
    const int r_warp = (warp & 3) * 32;
    const int r_in = r_warp + lane;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(r_warp) << 16) + wg * kCols;
    const float* scale_s = reinterpret_cast<const float*>(smem + Dm::kScales);
    float* bias_s = reinterpret_cast<float*>(smem + Dm::kBias) + warp * kCols;
    float* amax_s = reinterpret_cast<float*>(smem + Dm::kAmax);
    Ring<S> st;
    Ring<kBufs> ac;
    Ring<kScaleGroups> sg;
    uint32_t tile_parity = 0;
    // The bias goes in first. Through shared memory: every lane needs every
    // column's; a lane fetches its share a tile ahead.
    auto fetch_bias = [&](int t, float (&v)[kCols / 32]) {
      int tm = 0, tn = 0;
      if (t < p.tiles) lin_tile(p, t, tm, tn);
#pragma unroll
      for (int i = 0; i < kCols / 32; ++i) {
        const int c = tn * kBN + wg * kCols + lane + 32 * i;
        v[i] = p.bias != nullptr && c < p.n ? p.bias[c] : 0.f;
      }
    };
    float bias[kCols / 32];
    fetch_bias(unit0, bias);
    for (int t = unit0; t < p.tiles; t += unit_step, tile_parity ^= 1u) {
      int tm, tn;
      lin_tile(p, t, tm, tn);
      const int row = tm * kLinRows + r_in;
      const int col = tn * kBN + wg * kCols;
      const bool live = row < p.m;
      const int have = p.n - col;  // columns of this warpgroup that exist
      float acc[kCols];
      __syncwarp();
#pragma unroll
      for (int i = 0; i < kCols / 32; ++i) bias_s[lane + 32 * i] = bias[i];
      __syncwarp();
#pragma unroll
      for (int j = 0; j < kCols; j += 4) {
        const float4 b = *reinterpret_cast<const float4*>(bias_s + j);
        acc[j] = b.x;
        acc[j + 1] = b.y;
        acc[j + 2] = b.z;
        acc[j + 3] = b.w;
      }
      fetch_bias(t + unit_step, bias);
      for (int kb0 = 0; kb0 < p.kblocks; kb0 += kGroupBlocks, sg.next()) {
        mbar_wait(bar(kLinScaleFull + sg.i), sg.phase, abort_flag, p.status, kDevTimeoutSoftmax, limit);
        const volatile float* sp = scale_s + sg.i * (kGroupBlocks * kScaleFloats);
        float sc[kGroupBlocks];  // (of blocks past the last one: not used)
#pragma unroll
        for (int g = 0; g < kGroupBlocks; ++g)
          sc[g] = sp[g * kScaleFloats + r_in] * sp[g * kScaleFloats + 128 + wg];
        __syncwarp();
        const bool silent = kTest && p.drop == kDropSums && warp == 0 && kb0 >= p.drop_at;
        if (lane == 0 && !silent) mbar_arrive(bar(kLinScaleEmpty + sg.i));
#pragma unroll
        for (int g = 0; g < kGroupBlocks; ++g) {
          if (kb0 + g >= p.kblocks) break;
          lin_wait_product(bar(kLinDone + st.i), st.phase, abort_flag, p.status, limit);
          __syncwarp();
          tc_fence_after();
          const uint32_t tm_acc = t_lane + ac.i * kBN;
          const uint64_t sc2 = f2_pack(sc[g], sc[g]);
#pragma unroll
          for (int c = 0; c < kCols; c += 32) {
            uint32_t r[32];
            tmem_ld32(tm_acc + c, r);
            tmem_wait_ld(r);
            if (c + 32 == kCols) {  // read out: the buffer may take the next product
              tc_fence_before();
              lin_buffer_arrive<Dm::kSumWG * 128 + 32>(ac.i);
            }
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              const uint64_t v = f2_fma(f2_pack(__uint_as_float(r[j]), __uint_as_float(r[j + 1])),
                                        sc2, f2_pack(acc[c + j], acc[c + j + 1]));
              f2_unpack(v, acc[c + j], acc[c + j + 1]);
            }
          }
          st.next();
          ac.next();
        }
      }
      // ---- activation, rounding, store
      if (p.act == kActGeluTanh) {
#pragma unroll
        for (int j = 0; j < kCols; j += 2) gelu_tanh2(acc[j], acc[j + 1]);
      }
      float inv = 1.f;
      if constexpr (kOut == kOutE4m3) {
        float am = 0.f;
#pragma unroll
        for (int j = 0; j < kCols; ++j) am = fmaxf(am, fabsf(acc[j]));
        if constexpr (kCols < kBlock) {  // the block's other columns are the next warpgroup's
          // Two copies by tile parity: a copy is written again only after the
          // next tile's barrier, which every reader of this one has passed.
          volatile float* mine = amax_s + tile_parity * (128 * Dm::kSumWG);
          mine[wg * 128 + r_in] = am;
          const bool silent = kTest && p.drop == kDropSums && warp == 0 && p.kblocks > p.drop_at;
          if (!silent) mbar_arrive(bar(kLinAmax));
          mbar_wait(bar(kLinAmax), tile_parity, abort_flag, p.status, kDevTimeoutSoftmax, limit);
          am = fmaxf(am, mine[(wg ^ 1) * 128 + r_in]);
        }
        const float s = block_scale(am, inv);
        if (live && have > 0 && col % kBlock == 0)
          p.out_scale[row * p.os_rs + static_cast<long long>(col / kBlock) * p.os_bs] = s;
      }
      constexpr int kElem = kOut == kOutBf16 ? 2 : kOut == kOutFloat ? 4 : 1;
      // 32 rows x kWide bytes at a time, 16-byte pieces swizzled as the tensor
      // map says, so that lanes (rows) hit different banks
      constexpr int kWide = kCols * kElem < 128 ? kCols * kElem : 128;
      constexpr int kWideCols = kWide / kElem;
      uint8_t* const buf = smem + Dm::kStore + warp * 4096;
      const uint32_t mine = smem_u32(buf) + lane * kWide;
      auto swizzle = [](int r) { return kWide == 128 ? r & 7 : kWide == 64 ? (r >> 1) & 3 : 0; };
#pragma unroll
      for (int c = 0; c < kCols; c += kWideCols) {
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kWide / 16; ++i) {
          uint32_t q[4];
          lin_pack16<kOut>(acc + c + i * (16 / kElem), inv, q);
          st_shared_v4(mine + ((i ^ swizzle(lane)) << 4), q[0], q[1], q[2], q[3]);
        }
        if (p.tma_out == 1 || (p.tma_out == 2 && (c + kWideCols <= have || c >= have))) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0 && c < have && row < p.m) lin_store(&tm_o, smem_u32(buf), col + c, row);
        } else {  // off the 16-byte boundaries: neighbours by neighbouring lanes
          __syncwarp();
          const int rows = min(32, p.m - (row - lane)), cols = min(kWideCols, have - c);
          using Word = std::conditional_t<kElem == 4, uint32_t,
                                          std::conditional_t<kElem == 2, uint16_t, uint8_t>>;
          Word* out = static_cast<Word*>(p.out) + (row - lane) * p.out_stride + col + c;
          for (int r = 0; r < rows; ++r, out += p.out_stride) {
#pragma unroll
            for (int e = lane; e < kWideCols; e += 32) {
              const int at = e * kElem;
              if (e < cols)
                out[e] = *reinterpret_cast<const Word*>(buf + r * kWide +
                                                        (((at >> 4) ^ swizzle(r)) << 4) + (at & 15));
            }
          }
        }
      }
    }
    // the staged output has been read before the memory goes
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();  // every role has left; all products have been seen
  tc_fence_after();
  if (warp == kFeed + 1) tmem_dealloc(tmem, 512);
  if (warp == kFeed && *abort_flag) {  // the stages' last loads land before the memory goes
    const long long n = *loaded;
    for (long long i = n > S ? n - S : 0; i < n; ++i)
      mbar_wait_drain(bar(kLinFull + static_cast<int>(i % S)), static_cast<uint32_t>(i / S) & 1u, p.status);
  }
}

}  // namespace fp8
}  // namespace vx
