// The 8-bit entry points of include/vidax_cuda.h: argument checks, the choice
// of a kernel variant by sizes and alignment, launches. Nothing here allocates
// device memory, and no call leaves state for the next one.
#include "vidax_cuda.h"
#include "vx_internal.h"

#include <algorithm>
#include <climits>
#include <cmath>
#include <map>
#include <mutex>
#include <utility>

#include "add_norm.cuh"
#include "fp8_linear.cuh"
#include "fp8_linear_few.cuh"
#include "fp8_quantize.cuh"

namespace {

using namespace vx::fp8;

template <typename... A>
int fail(int code, const char* fmt, A... a) {
  return vx_internal_failf(code, fmt, a...);
}
int fail(int code, const char* msg) { return vx_internal_fail(code, msg); }

// Features that the kernels' 32-bit feature indices can step past the end of: a
// step is up to 2048 of them.
constexpr int32_t kMostFeatures = INT_MAX - 4095;

bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int launched(const char* what) {
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? VX_OK : vx_internal_cuda_fail(e, what);
}

int type_size(int32_t t) { return t == VX_TYPE_FLOAT ? 4 : t == VX_TYPE_BF16 ? 2 : 1; }

// Rows of `dim` elements, `stride` apart, that do not overlap.
int check_rows(const char* name, const void* p, int64_t stride, int64_t rows, int32_t dim,
               int elem) {
  if (p == nullptr) return fail(VX_EINVAL, "%s is NULL", name);
  if (!aligned(p, elem)) return fail(VX_EINVAL, "%s is not aligned to its element", name);
  if (stride < 0 || (rows > 1 && stride < dim))
    return fail(VX_EINVAL, "%s row stride %lld is below the row's %d elements", name,
                (long long)stride, dim);
  return VX_OK;
}

int check_scale(const char* name, const void* p, const int64_t (&st)[2]) {
  if (p == nullptr) return fail(VX_EINVAL, "%s is NULL", name);
  if (!aligned(p, 4)) return fail(VX_EINVAL, "%s is not aligned to its element", name);
  if (st[0] < 0 || st[1] < 0) return fail(VX_EINVAL, "%s has a negative stride", name);
  return VX_OK;
}

// Memory that a call touches: rows of `width` bytes, `stride` bytes apart.
struct Rows {
  uintptr_t p;
  int64_t stride, rows, width;
  Rows(const void* ptr, int64_t n, int64_t elems_between, int64_t elems, int64_t elem)
      : p(reinterpret_cast<uintptr_t>(ptr)), stride(elems_between * elem), rows(n), width(elems * elem) {
    if (rows == 1 || stride == 0) rows = 1, stride = width;  // (vectors may repeat)
  }
  bool same(const Rows& o) const { return p == o.p && rows == o.rows && (rows == 1 || stride == o.stride); }
  uintptr_t end() const { return p + (rows - 1) * stride + width; }
  // Whether a byte of one is a byte of the other.
  bool meets(const Rows& o) const {
    if (end() <= o.p || o.end() <= p) return false;
    if (rows > 1 && stride == o.stride) {  // columns of one buffer, side by side
      const int64_t d = static_cast<int64_t>(o.p - p) % stride, at = d < 0 ? d + stride : d;
      if (at >= width && at + o.width <= stride) return false;
    }
    const Rows& a = rows < o.rows ? o : *this;
    const Rows& b = rows < o.rows ? *this : o;  // the fewer rows
    for (int64_t i = 0; i < b.rows; ++i) {
      // the last row of `a` that begins before this row's end
      const int64_t from = static_cast<int64_t>(b.p - a.p) + i * b.stride, to = from + b.width;
      if (to <= 0) continue;
      if (std::min((to - 1) / a.stride, a.rows - 1) * a.stride + a.width > from) return true;
    }
    return false;
  }
};

// Rows of 8 k elements on 16-byte boundaries (8-byte ones of 1-byte elements).
bool vec8(const void* p, int64_t stride, int elem) {
  const int64_t bytes = std::min(8 * elem, 16);
  return aligned(p, bytes) && stride * elem % bytes == 0;
}

// ------------------------------------------------------------------ add_norm

std::mutex g_norm_mu;
std::map<std::pair<const void*, int>, int> g_norm_ctas;

template <typename T, int W, int NV, bool kVec>
int launch_norm(AddNormParams& p, int dev, int sms, cudaStream_t s) {
  const void* fn = reinterpret_cast<const void*>(&add_norm_kernel<T, W, NV, kVec>);
  constexpr size_t kMost = 3u * 256 * W * NV * sizeof(float);
  p.cap = (p.dim + 255) / 256 * 256;
  const size_t smem = (p.y != nullptr ? 3u : 2u) * p.cap * sizeof(float);
  int rc = vx_internal_prepare_kernel(fn, dev, kMost);
  if (rc != VX_OK) return rc;
  int per_sm;  // by registers and threads
  {
    std::lock_guard<std::mutex> lk(g_norm_mu);
    int& n = g_norm_ctas[{fn, dev}];
    if (n == 0) {
      cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, fn, 256, 0);
      if (e != cudaSuccess) return vx_internal_cuda_fail(e, "cudaOccupancyMaxActiveBlocksPerMultiprocessor");
      n = std::max(n, 1);
    }
    per_sm = n;
  }
  // and by the 228 KB of shared memory, 1 KB of which each CTA holds besides
  // its own (and 8 KB where rows lie off the boundaries)
  per_sm = std::max(1, std::min<int>(per_sm, 228 * 1024 / (smem + 1024 + (kVec ? 64 : 8256))));
  constexpr int kPer = 8 / W;  // rows at a time
  const long long groups = (p.rows + kPer - 1) / kPer;
  const long long ctas = std::min<long long>(groups, static_cast<long long>(sms) * per_sm);
  p.rows_per_cta = (groups + ctas - 1) / ctas * kPer;
  const long long grid = (p.rows + p.rows_per_cta - 1) / p.rows_per_cta;
  add_norm_kernel<T, W, NV, kVec><<<static_cast<unsigned>(grid), 256, smem, s>>>(p);
  return VX_OK;
}

template <typename T, bool kVec>
int launch_add_norm(AddNormParams& p, int dev, int sms, cudaStream_t s) {
  // Warps per row: one while the row fits a lane's registers, more for wide
  // rows, and more where there are too few rows to fill the GPU with one warp
  // each (a row's latency then counts, not its bandwidth).
  const int vecs = (p.dim + 255) / 256;
  const bool few = p.rows < 4LL * sms;
  // Rows off the 16-byte boundaries hold their pieces (up to 12 registers per
  // eight features) and the features at once.
  const int most1 = kVec ? 6 : 4;
  if (vecs <= 1) return launch_norm<T, 1, 1, kVec>(p, dev, sms, s);
  if (!few && vecs <= most1) {
    if (vecs <= 2) return launch_norm<T, 1, 2, kVec>(p, dev, sms, s);
    if (vecs <= 4) return launch_norm<T, 1, 4, kVec>(p, dev, sms, s);
    if constexpr (kVec) return launch_norm<T, 1, 6, kVec>(p, dev, sms, s);
  }
  // (5 or 6 chunks: two warps with three each against four of which some hold
  // two, rows of 1027, 1283 and 1533 features in us, bf16 stream: 700 rows 7.0 /
  // 7.8, 7.4 / 8.6, 7.8 / 8.6; 4678 rows 18.0 / 21.7, 19.7 / 23.4, 20.5 / 24.2;
  // 32760 rows 118 / 133, 128 / 145, 134 / 149)
  if constexpr (!kVec) {
    if (!few && vecs > 4 && vecs <= 6) return launch_norm<T, 2, 3, kVec>(p, dev, sms, s);
  }
  if (vecs <= 4) return launch_norm<T, 4, 1, kVec>(p, dev, sms, s);
  if (vecs <= 8) return launch_norm<T, 4, 2, kVec>(p, dev, sms, s);
  if (vecs <= 12) return launch_norm<T, 4, 3, kVec>(p, dev, sms, s);
  if (vecs <= 16) return launch_norm<T, 4, 4, kVec>(p, dev, sms, s);
  if (vecs <= 20) return launch_norm<T, 4, 5, kVec>(p, dev, sms, s);
  if (vecs <= 32) return launch_norm<T, 8, 4, kVec>(p, dev, sms, s);
  if (vecs <= 40) return launch_norm<T, 8, 5, kVec>(p, dev, sms, s);
  if (vecs <= 56) return launch_norm<T, 8, 7, kVec>(p, dev, sms, s);
  if (vecs <= 64) return launch_norm<T, 8, 8, kVec>(p, dev, sms, s);
  add_norm_wide_kernel<T, kVec><<<static_cast<unsigned>(p.rows), 256, 0, s>>>(p);
  return VX_OK;
}

// ------------------------------------------------------------------ linear

struct LinVariant {
  int bn;
  const void* fn[3];  // by output type
  uint32_t smem;
  int threads;
  int cols;           // columns of one warpgroup
  double block, tile; // time model: cycles per block of 128 features, per tile besides
};

template <int kBN>
LinVariant variant(double block, double tile) {
  return {kBN,
          {reinterpret_cast<const void*>(&linear_kernel<kBN, kOutBf16>),
           reinterpret_cast<const void*>(&linear_kernel<kBN, kOutFloat>),
           // a 128-column block of the e4m3 output lies in one tile
           kBN >= kBlock ? reinterpret_cast<const void*>(
                               &linear_kernel<(kBN >= kBlock ? kBN : kBlock), kOutE4m3>)
                         : nullptr},
          LinDims<kBN>::kSmemBytes,
          LinDims<kBN>::kThreads,
          LinDims<kBN>::kCols,
          block,
          tile};
}

// Measured: 9472 x 8960 -> 2048 takes 922 / 566 / 425 cycles per block, and a
// tile's start and output 2500 / 2000 / 2000 besides. With GELU and an e4m3
// output a tile's end is longer, by about as much for every column, so the same
// model serves. Its choice against the best of the tiles, 16 products of 64 to
// 32760 rows: with GELU and e4m3 within 2 % (4680 x 1536 -> 8960: 95 us, the
// 128-column tile 110), with a bf16 output within 3 % from 1500 rows on and within 7 %
// (0.4 us) below.
const LinVariant kVariants[] = {variant<256>(922, 2500), variant<128>(566, 2000),
                                variant<64>(425, 2000)};
constexpr int kNumVariants = sizeof(kVariants) / sizeof(kVariants[0]);

// The tile whose waves over the SMs take least by the time model: narrow ones
// where wide ones would leave SMs idle.
int pick_variant(const vx_linear_fp8_args* a, int sms) {
  int best = 0;
  double best_t = 0;
  for (int i = 0; i < kNumVariants; ++i) {
    const LinVariant& v = kVariants[i];
    if (a->out_type == VX_TYPE_E4M3 && v.fn[kOutE4m3] == nullptr) continue;
    const long long tiles =
        ((a->m - 1LL) / kLinRows + 1) * ((a->n - 1LL) / v.bn + 1);
    const double t =
        static_cast<double>((tiles - 1) / sms + 1) * ((a->k - 1) / kBlock + 1) * v.block +
        static_cast<double>((tiles - 1) / sms + 1) * v.tile;
    if (i == 0 || t < best_t) best_t = t, best = i;
  }
  return best;
}

template <int kWarps, int kNT>
const void* few_kernel(int out) {
  return out == kOutBf16  ? reinterpret_cast<const void*>(&linear_few_kernel<kWarps, kNT, kOutBf16>)
         : out == kOutFloat ? reinterpret_cast<const void*>(&linear_few_kernel<kWarps, kNT, kOutFloat>)
                            : reinterpret_cast<const void*>(&linear_few_kernel<kWarps, kNT, kOutE4m3>);
}

// Warps share the input features: more of them where few CTAs would leave too
// few loads in flight.
bool few_wide(int n, int kblocks, int sms) {
  return (n - 1) / kFewCols + 1 < 2LL * sms && kblocks > 8;
}

int launch_few(const FewParams& p, int out, int sms, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  long long ctas = (p.l.n - 1) / kFewCols + 1;
  const bool wide = few_wide(p.l.n, p.l.kblocks, sms);
  const void* fn = p.l.m <= 8 ? (wide ? few_kernel<16, 1>(out) : few_kernel<8, 1>(out))
                              : (wide ? few_kernel<16, 2>(out) : few_kernel<8, 2>(out));
  cudaLaunchAttribute at[1];
  if (out == kOutE4m3) {  // the CTAs of one block of 128 output features
    constexpr int kPeers = kBlock / kFewCols;
    ctas = (ctas + kPeers - 1) / kPeers * kPeers;
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = kPeers;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
  }
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(wide ? 512 : 256);
  cfg.stream = stream;
  void* args[1] = {const_cast<FewParams*>(&p)};
  cudaError_t e = cudaLaunchKernelExC(&cfg, fn, args);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return vx_internal_cuda_fail(e, "linear_fp8 launch");
  }
  return VX_OK;
}

}  // namespace

extern "C" int vx_quantize_fp8(const vx_quantize_fp8_args* a, vx_stream_t stream) {
  if (a == nullptr) return fail(VX_EINVAL, "args is NULL");
  if (a->rows < 0 || a->dim < 1)
    return fail(VX_EINVAL, "bad sizes (rows %lld, dim %d)", (long long)a->rows, a->dim);
  if (a->src_type != VX_TYPE_FLOAT && a->src_type != VX_TYPE_BF16)
    return fail(VX_EUNSUPPORTED, "src_type %d (float and bf16 are built)", a->src_type);
  if (a->block_rows != 1 && a->block_rows != kBlock)
    return fail(VX_EUNSUPPORTED, "block_rows %d (1 and 128 are built)", a->block_rows);
  if (a->rows == 0) return VX_OK;
  const int elem = type_size(a->src_type);
  int rc;
  if ((rc = check_rows("src", a->src, a->src_stride, a->rows, a->dim, elem)) != VX_OK) return rc;
  if ((rc = check_rows("dst", a->dst, a->dst_stride, a->rows, a->dim, 1)) != VX_OK) return rc;
  if ((rc = check_scale("scale", a->scale, a->scale_stride)) != VX_OK) return rc;
  QuantizeParams p{};
  p.src = a->src;
  p.dst = static_cast<uint8_t*>(a->dst);
  p.scale = a->scale;
  p.src_stride = a->src_stride;
  p.dst_stride = a->dst_stride;
  p.scale_rs = a->scale_stride[0];
  p.scale_bs = a->scale_stride[1];
  p.rows = a->rows;
  p.dim = a->dim;
  const bool by_row = a->block_rows == 1;
  const int per = by_row ? kRows : kBlock;
  p.chunks = (a->dim - 1) / (by_row ? 2 * kBlock : kBlock) + 1;
  const long long items = ((a->rows - 1) / per + 1) * p.chunks;
  if (a->rows > INT_MAX || items > INT_MAX) return fail(VX_EUNSUPPORTED, "too many blocks");
  p.items = static_cast<unsigned>(items);
  const bool vec =
      a->dim % 8 == 0 && vec8(p.src, p.src_stride, elem) && vec8(p.dst, p.dst_stride, 1);
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  p.on8 = vec8(p.dst, p.dst_stride, 1);
  const unsigned grid = by_row ? (p.items + 7) / 8 : p.items;
  if (a->src_type == VX_TYPE_FLOAT) {
    if (!by_row) quantize_tiles_kernel<float><<<grid, 256, 0, s>>>(p);
    else if (vec) quantize_rows_kernel<float, true><<<grid, 256, 0, s>>>(p);
    else quantize_rows_kernel<float, false><<<grid, 256, 0, s>>>(p);
  } else {
    if (!by_row) quantize_tiles_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(p);
    else if (vec) quantize_rows_kernel<__nv_bfloat16, true><<<grid, 256, 0, s>>>(p);
    else quantize_rows_kernel<__nv_bfloat16, false><<<grid, 256, 0, s>>>(p);
  }
  return launched("quantize_fp8 launch");
}

extern "C" int vx_add_norm(const vx_add_norm_args* a, vx_stream_t stream) {
  if (a == nullptr) return fail(VX_EINVAL, "args is NULL");
  if (a->rows < 0 || a->dim < 1 || a->rows_per_batch < 1 || a->rows % a->rows_per_batch != 0)
    return fail(VX_EINVAL, "bad sizes (rows %lld, dim %d, rows_per_batch %lld)", (long long)a->rows,
                a->dim, (long long)a->rows_per_batch);
  if (a->x_type != VX_TYPE_FLOAT && a->x_type != VX_TYPE_BF16)
    return fail(VX_EUNSUPPORTED, "x_type %d (float and bf16 are built)", a->x_type);
  if (a->out_type != VX_TYPE_BF16 && a->out_type != VX_TYPE_E4M3)
    return fail(VX_EUNSUPPORTED, "out_type %d (bf16 and e4m3 are built)", a->out_type);
  if (a->norm != VX_NORM_RMS && a->norm != VX_NORM_LAYER)
    return fail(VX_EUNSUPPORTED, "norm %d", a->norm);
  if (!(a->eps >= 0.f) || !std::isfinite(a->eps))
    return fail(VX_EINVAL, "eps must be finite and >= 0 (got %g)", (double)a->eps);
  if (a->y == nullptr && a->gate != nullptr) return fail(VX_EINVAL, "gate without y");
  if (a->rows == 0) return VX_OK;
  const int xe = type_size(a->x_type), oe = type_size(a->out_type);
  int rc;
  if ((rc = check_rows("x", a->x, a->x_stride, a->rows, a->dim, xe)) != VX_OK) return rc;
  if ((rc = check_rows("out", a->out, a->out_stride, a->rows, a->dim, oe)) != VX_OK) return rc;
  bool vec = a->dim % 8 == 0 && vec8(a->x, a->x_stride, xe) && vec8(a->out, a->out_stride, oe);
  if (a->y != nullptr) {
    if ((rc = check_rows("y", a->y, a->y_stride, a->rows, a->dim, 2)) != VX_OK) return rc;
    if ((rc = check_rows("sum", a->sum, a->sum_stride, a->rows, a->dim, xe)) != VX_OK) return rc;
    vec = vec && vec8(a->y, a->y_stride, 2) && vec8(a->sum, a->sum_stride, xe);
  }
  const float* vs[5] = {a->gate, a->scale, a->shift, a->weight, a->bias};
  const int64_t vst[5] = {a->gate_stride, a->scale_stride, a->shift_stride, 0, 0};
  const char* names[5] = {"gate", "scale", "shift", "weight", "bias"};
  for (int i = 0; i < 5; ++i) {
    if (vs[i] == nullptr) continue;
    if (!aligned(vs[i], 4)) return fail(VX_EINVAL, "%s is not aligned to its element", names[i]);
    if (vst[i] < 0) return fail(VX_EINVAL, "%s has a negative stride", names[i]);
    if (a->dim > 16384) vec = vec && vec8(vs[i], vst[i], 4);  // the others go through shared memory
  }
  if (a->rows > INT_MAX || a->dim > kMostFeatures)
    return fail(VX_EUNSUPPORTED, "too many rows or features (%lld x %d)", (long long)a->rows, a->dim);
  // What is written while other rows are still read lies apart from them. In
  // place (the sum's rows are x's own) each lane has read what it writes.
  const Rows x_rows(a->x, a->rows, a->x_stride, a->dim, xe);
  const Rows y_rows(a->y, a->rows, a->y_stride, a->dim, 2);
  const Rows sum_rows(a->sum, a->rows, a->sum_stride, a->dim, xe);
  const Rows out_rows(a->out, a->rows, a->out_stride, a->dim, oe);
  const bool in_place = a->y != nullptr && sum_rows.same(x_rows);
  if (out_rows.meets(x_rows) ||
      (a->y != nullptr && (out_rows.meets(y_rows) || out_rows.meets(sum_rows))))
    return fail(VX_EINVAL, "out must lie apart from x, y and sum");
  if (a->y != nullptr && !in_place && sum_rows.meets(x_rows))
    return fail(VX_EINVAL, "sum must be x itself or lie apart from x");
  if (a->y != nullptr && !(in_place && y_rows.same(sum_rows) && xe == 2) && sum_rows.meets(y_rows))
    return fail(VX_EINVAL, "sum must lie apart from y");
  for (int i = 0; i < 5; ++i) {
    if (vs[i] == nullptr) continue;
    const Rows v(vs[i], i < 3 ? a->rows / a->rows_per_batch : 1, vst[i], a->dim, 4);
    if (out_rows.meets(v) || (a->y != nullptr && sum_rows.meets(v)))
      return fail(VX_EINVAL, "sum and out must lie apart from %s", names[i]);
  }
  if (a->out_type == VX_TYPE_E4M3 &&
      (rc = check_scale("out_scale", a->out_scale, a->out_scale_stride)) != VX_OK)
    return rc;
  int dev, sms;
  if ((rc = vx_internal_device(&dev, &sms)) != VX_OK) return rc;
  AddNormParams p{};
  p.x = a->x;
  p.sum = a->y != nullptr ? a->sum : nullptr;
  p.y = static_cast<const __nv_bfloat16*>(a->y);
  p.gate = a->gate;
  p.w = a->weight;
  p.b = a->bias;
  p.scale = a->scale;
  p.shift = a->shift;
  p.out = a->out;
  p.out_scale = a->out_type == VX_TYPE_E4M3 ? a->out_scale : nullptr;
  p.x_stride = a->x_stride;
  p.sum_stride = a->sum_stride;
  p.y_stride = a->y_stride;
  p.out_stride = a->out_stride;
  p.gate_stride = a->gate_stride;
  p.scale_stride = a->scale_stride;
  p.shift_stride = a->shift_stride;
  p.out_scale_rs = a->out_scale_stride[0];
  p.out_scale_bs = a->out_scale_stride[1];
  p.rows = a->rows;
  p.rows_per_batch = a->rows_per_batch;
  p.dim = a->dim;
  p.layer = a->norm == VX_NORM_LAYER;
  p.eps = a->eps;
  p.sum_on16 = a->y != nullptr && vec8(a->sum, a->sum_stride, xe);
  p.out_on16 = vec8(a->out, a->out_stride, oe);
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (a->x_type == VX_TYPE_FLOAT)
    rc = vec ? launch_add_norm<float, true>(p, dev, sms, s) : launch_add_norm<float, false>(p, dev, sms, s);
  else
    rc = vec ? launch_add_norm<__nv_bfloat16, true>(p, dev, sms, s)
             : launch_add_norm<__nv_bfloat16, false>(p, dev, sms, s);
  if (rc != VX_OK) return rc;
  return launched("add_norm launch");
}

namespace {

// The self-test of the wide kernel's waits: the role that falls silent, at
// which of its blocks, and the wait limit.
struct LinTest {
  int drop, after;
  long long limit;
};

int linear_call(const vx_linear_fp8_args* a, const LinTest* test, vx_stream_t stream) {
  if (a == nullptr) return fail(VX_EINVAL, "args is NULL");
  if (a->m < 0 || a->n < 1 || a->k < 1)
    return fail(VX_EINVAL, "bad sizes (m %d, n %d, k %d)", a->m, a->n, a->k);
  if (a->n > kMostFeatures || a->k > kMostFeatures)
    return fail(VX_EUNSUPPORTED, "too many features (n %d, k %d)", a->n, a->k);
  const int out_idx = a->out_type == VX_TYPE_BF16    ? kOutBf16
                      : a->out_type == VX_TYPE_FLOAT ? kOutFloat
                      : a->out_type == VX_TYPE_E4M3  ? kOutE4m3
                                                     : -1;
  if (out_idx < 0) return fail(VX_EUNSUPPORTED, "out_type %d", a->out_type);
  if (a->activation != VX_ACT_NONE && a->activation != VX_ACT_GELU_TANH)
    return fail(VX_EUNSUPPORTED, "activation %d", a->activation);
  if (a->variant < 0 || a->variant > kNumVariants + 1) return fail(VX_EINVAL, "variant %d", a->variant);
  bool few = a->variant == kNumVariants + 1;
  if (few && a->m > kFewMost)
    return fail(VX_EUNSUPPORTED, "this variant takes up to %d rows", kFewMost);
  if (!few && a->variant > 0 && kVariants[a->variant - 1].fn[out_idx] == nullptr)
    return fail(VX_EUNSUPPORTED, "this variant has no e4m3 output");
  if (a->m == 0) return VX_OK;
  int rc;
  if ((rc = check_rows("x", a->x, a->x_stride, a->m, a->k, 1)) != VX_OK) return rc;
  if ((rc = check_rows("w", a->w, a->w_stride, a->n, a->k, 1)) != VX_OK) return rc;
  if ((rc = check_rows("out", a->out, a->out_stride, a->m, a->n, type_size(a->out_type))) != VX_OK)
    return rc;
  if (!aligned(a->x, 16) || !aligned(a->w, 16) || a->x_stride % 16 != 0 || a->w_stride % 16 != 0)
    return fail(VX_EINVAL, "x and w must start, and their rows must lie, on 16-byte boundaries");
  if ((rc = check_scale("x_scale", a->x_scale, a->x_scale_stride)) != VX_OK) return rc;
  if ((rc = check_scale("w_scale", a->w_scale, a->w_scale_stride)) != VX_OK) return rc;
  if (out_idx == kOutE4m3 &&
      (rc = check_scale("out_scale", a->out_scale, a->out_scale_stride)) != VX_OK)
    return rc;
  if (a->bias != nullptr && !aligned(a->bias, 4))
    return fail(VX_EINVAL, "bias is not aligned to its element");
  int dev, sms;
  if ((rc = vx_internal_device(&dev, &sms)) != VX_OK) return rc;
  LinearParams p{};
  p.xs = a->x_scale;
  p.xs_rs = a->x_scale_stride[0];
  p.xs_bs = a->x_scale_stride[1];
  p.ws = a->w_scale;
  p.ws_rs = a->w_scale_stride[0];
  p.ws_bs = a->w_scale_stride[1];
  p.bias = a->bias;
  p.out = a->out;
  p.out_stride = a->out_stride;
  p.out_scale = a->out_scale;
  p.os_rs = a->out_scale_stride[0];
  p.os_bs = a->out_scale_stride[1];
  p.m = a->m;
  p.n = a->n;
  p.kblocks = (a->k - 1) / kBlock + 1;
  p.act = a->activation;
  // One row needs no stride; the kernels want one that is a multiple of 16.
  const uint64_t xst = a->m > 1 ? a->x_stride : (static_cast<uint64_t>(a->k) + 15) / 16 * 16;
  const uint64_t wst = a->n > 1 ? a->w_stride : (static_cast<uint64_t>(a->k) + 15) / 16 * 16;
  if (a->variant == 0 && test == nullptr)  // (measured: fp8_linear_few.cuh)
    few = a->m <= kFewMost &&
          (out_idx != kOutE4m3 || a->m <= 8 || few_wide(a->n, p.kblocks, sms));
  if (few) {
    FewParams f{static_cast<const uint8_t*>(a->x), static_cast<const uint8_t*>(a->w),
                static_cast<long long>(xst), static_cast<long long>(wst), a->k, p};
    return launch_few(f, out_idx, sms, reinterpret_cast<cudaStream_t>(stream));
  }

  // (the self-test: four adding warpgroups with two TMEM buffers, row maxima
  // between warpgroups; or two with four buffers)
  const LinVariant& v = kVariants[test != nullptr      ? (out_idx == kOutE4m3 ? 0 : kNumVariants - 1)
                                  : a->variant > 0     ? a->variant - 1
                                                       : pick_variant(a, sms)];
  const void* fn = v.fn[out_idx];
  if (test != nullptr) {
    fn = out_idx == kOutE4m3 ? reinterpret_cast<const void*>(&linear_kernel<256, kOutE4m3, true>)
                             : reinterpret_cast<const void*>(&linear_kernel<64, kOutBf16, true>);
    p.limit = test->limit;
    p.drop = test->drop;
    p.drop_at = test->after;
  }
  p.tiles_m = (a->m - 1) / kLinRows + 1;
  p.tiles_n = (a->n - 1) / v.bn + 1;
  const long long tiles = static_cast<long long>(p.tiles_m) * p.tiles_n;
  if (tiles > INT_MAX / 2 || static_cast<long long>(kGroupM) * p.tiles_n > INT_MAX)
    return fail(VX_EUNSUPPORTED, "too many output tiles (%lld)", tiles);
  p.tiles = static_cast<int>(tiles);
  const int oe = type_size(a->out_type);
  p.tma_out = !aligned(a->out, 16) || a->out_stride * oe % 16 != 0 ? 0
              : static_cast<int64_t>(a->n) * oe % 16 == 0              ? 1
                                                                       : 2;
  if ((rc = vx_internal_status_word(&p.status)) != VX_OK) return rc;

  CUtensorMap tx, tw, to;
  if ((rc = vx_internal_byte_tmap(&tx, a->x, a->k, a->m, xst, 128, kLinRows)) != VX_OK) return rc;
  if ((rc = vx_internal_byte_tmap(&tw, a->w, a->k, a->n, wst, 128, v.bn)) != VX_OK) return rc;
  to = tx;  // not used without tma_out
  if (p.tma_out) {
    const uint64_t row = static_cast<uint64_t>(a->n) * oe;
    const uint64_t ost = a->m > 1 ? static_cast<uint64_t>(a->out_stride) * oe : (row + 15) / 16 * 16;
    if ((rc = vx_internal_byte_tmap(&to, a->out, row, a->m, ost, std::min(128, v.cols * oe), 32,
                                    oe)) != VX_OK)
      return rc;
  }
  if ((rc = vx_internal_prepare_kernel(fn, dev, v.smem)) != VX_OK) return rc;
  void* args[4] = {&tx, &tw, &to, &p};
  cudaError_t e = cudaLaunchKernel(fn, dim3(static_cast<unsigned>(std::min(p.tiles, sms))),
                                   dim3(v.threads), args, v.smem, reinterpret_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) {
    cudaGetLastError();
    return vx_internal_cuda_fail(e, "linear_fp8 launch");
  }
  return VX_OK;
}

}  // namespace

extern "C" int vx_linear_fp8(const vx_linear_fp8_args* a, vx_stream_t stream) {
  return linear_call(a, nullptr, stream);
}

extern "C" int vx_selftest_linear_fp8(const vx_linear_fp8_args* a, int32_t role, int32_t after,
                                      int64_t limit_cycles, vx_stream_t stream) {
  if (a == nullptr) return fail(VX_EINVAL, "args is NULL");
  if (role < 0 || role >= kNumDrops || after < 0)
    return fail(VX_EINVAL, "role must be in [0, %d) and after >= 0", (int)kNumDrops);
  if (limit_cycles <= 0 || limit_cycles > 4000000000LL)
    return fail(VX_EINVAL, "limit_cycles must be in (0, 4e9]");
  if (a->variant != 0 || (a->out_type != VX_TYPE_E4M3 && a->out_type != VX_TYPE_BF16))
    return fail(VX_EUNSUPPORTED, "the self-test takes variant 0 and an e4m3 or bf16 output");
  const LinTest test{role, after, limit_cycles};
  return linear_call(a, &test, stream);
}
