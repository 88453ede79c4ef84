// The linear layer y = act(x w^T + b) + residual and its gradients: operand preparation, the few-row
// kernel, and the choice between them and the tiled products (gemm.hpp).
#include <algorithm>
#include <cmath>

#include "linear.hpp"

namespace qvh {

// ---- plan -------------------------------------------------------------------------------------

// The estimate below is fitted to products from 128 x 128 x 64 to 10,000 x 768 x 4,608 with every tile and
// split (bf16, both operands by rows): it picked the fastest or one within 15% of it. Both sides of
// typical choices, in us: 1,024 x 1,024 x 4,096 as 64-tiles in one piece 37.2, in four 25.0, as 128-tiles in
// one 47.1; 2,048^3 as 128-tiles 29.5, 256-tiles 51.0; 8,192 x 2,048 x 768 as 256-tiles 35.5, 128-tiles
// 37.1, 64-tiles 51.2; 1,024 x 4,096 x 16,384 as 256-tiles in four pieces 131, 128-tiles in one 181.
GemmPlan gemm_plan(uint64_t m, uint64_t n, uint64_t k, Kind kind, uint32_t batches, bool symmetric) {
  struct Cost {
    uint64_t bm, bn, threads, together;  // tile, its work-group, and how many of those a CU holds
    double alone, shared, end;  // us per step: one work-group on a CU, each of several; prologue and epilogue
  };
  constexpr Cost kCosts[6][3] = {
      {{64, 64, 256, 4, 0.45, 0.22, 2.0}, {128, 128, 256, 2, 0.70, 0.53, 4.0}, {256, 256, 512, 1, 1.75, 1.75, 8.0}},
      {{64, 64, 256, 3, 0.40, 0.20, 2.0}, {128, 128, 512, 2, 0.55, 0.45, 4.0}, {}},
      {{64, 64, 256, 3, 0.50, 0.35, 2.0}, {128, 128, 512, 1, 0.95, 0.95, 4.0}, {256, 128, 512, 1, 1.80, 1.80, 6.0}},
      {{64, 64, 256, 3, 0.70, 0.52, 2.0}, {128, 128, 256, 2, 2.10, 2.00, 4.0}, {}},
      {{64, 64, 256, 4, 0.56, 0.35, 2.0}, {128, 128, 256, 2, 1.05, 0.75, 4.0}, {}},
      {{64, 64, 256, 3, 0.90, 0.62, 2.0}, {128, 128, 256, 2, 2.40, 2.10, 4.0}, {}}};
  constexpr uint32_t kSplits[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64};
  constexpr double kCus = 256.0;
  GemmPlan best;
  double least = -1.0;
  const uint64_t steps = ceil_div(k, kind == Kind::kPlane1 || kind == Kind::kNarrow ? 64 : 32);
  for (int t = 0; t < 3; ++t) {
    const Cost& c = kCosts[static_cast<int>(kind)][t];
    if (c.bm == 0 || (symmetric && c.bm != c.bn)) continue;
    const uint64_t tm = ceil_div(m, c.bm), tn = ceil_div(n, c.bn);
    const uint64_t tiles = (symmetric ? tm * (tm + 1) / 2 : tm * tn) * batches;
    for (const uint32_t splits : kSplits) {
      if (splits > 1 && steps < 2 * splits) break;
      // P X of an orthogonalisation is split as shallow 128-tiles only (launch_gemm): where the others would gain by it,
      // 64-tiles in one piece are faster still (300,000 shapes, none of them split otherwise without this line).
      if (kind == Kind::kPlane2 && !symmetric && splits > 1 && (t == 0 || tiles * splits <= 256)) continue;
      // What one launch has room for: the tiles, or the pieces that are joined.
      if (tiles / batches * splits * c.threads >= kGridThreads || (splits > 1 && m * ceil_div(n, 8) >= kGridThreads)) break;
      const double groups = static_cast<double>(tiles) * splits;
      const double per_cu = std::ceil(groups / kCus);
      const double rounds = std::ceil(per_cu / static_cast<double>(c.together));
      const double at_once = std::ceil(per_cu / std::max(rounds, 1.0));
      const double step = std::max(c.alone, c.shared * at_once);
      double us = rounds * (std::ceil(static_cast<double>(steps) / splits) * step + c.end + 0.5 * at_once);
      // The partial sums go out and come back, through the last-level cache, in a launch of their own.
      if (splits > 1) us += 5.5 + 0.1 * splits + static_cast<double>(splits) * batches * m * n * 8.0 / 7e6;
      if (least < 0.0 || us < least) {
        least = us;
        best.tile = t;
        best.splits = splits;
      }
    }
  }
  if (least < 0.0) {
    best.tile = -1;
    best.us = HUGE_VAL;
    return best;
  }
  best.us = least;
  if (best.splits > 1) best.partial_bytes = static_cast<size_t>(best.splits) * batches * m * (ceil_div(n, 8) * 8) * 4;
  return best;
}

namespace {

constexpr uint64_t kMaxRows = uint64_t{1} << 31, kMaxStride = uint64_t{1} << 22;
constexpr uint32_t kMaxWidth = 1u << 20;
constexpr uint64_t kSumRows = 512;  // rows whose column sums one work-group makes
constexpr int kPlanes = 3;         // bf16 parts of an fp32 value
constexpr char kTooLarge[] = "the matrix product is too large";

// ---- operand preparation ----------------------------------------------------------------------

struct PrepareArgs {
  const void* src = nullptr;
  uint64_t rows = 0, stride = 0;
  uint32_t cols = 0;
  void* dst = nullptr;  // [planes][rows][ld], ld = cols rounded up to 8, zeros behind the columns
  uint64_t ld = 0, plane = 0;
  uint32_t blocks = 0;
};

/// The three bf16 parts of an fp32 value, each the rounding of what the ones before it leave: their sum is
/// the value, and the products of parts that the pairs leave out are below 2^-24 of the product (with parts
/// cut off instead of rounded 2^-21, all of one sign). A first part that would round up to infinity is cut
/// off. Of an infinity or NaN the first part is all.
__device__ __forceinline__ void split3(float x, bhalf_t (&out)[3]) {
  out[0] = static_cast<bhalf_t>(x);
  const bool finite = fabsf(x) < __builtin_huge_valf();
  if (finite && fabsf(static_cast<float>(out[0])) == __builtin_huge_valf()) {
    out[0] = __builtin_bit_cast(bhalf_t, static_cast<uint16_t>(__float_as_uint(x) >> 16));
  }
  const float r1 = finite ? x - static_cast<float>(out[0]) : 0.0f;
  out[1] = static_cast<bhalf_t>(r1);
  out[2] = static_cast<bhalf_t>(r1 - static_cast<float>(out[1]));
}

template <class T>
__device__ __forceinline__ void store_prepared(void* dst, uint64_t at, uint64_t plane, const float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    Pack<bhalf_t, 8> part[3];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      bhalf_t s[3];
      split3(v[i], s);
      part[0].v[i] = s[0];
      part[1].v[i] = s[1];
      part[2].v[i] = s[2];
    }
#pragma unroll
    for (int p = 0; p < 3; ++p) *reinterpret_cast<Pack<bhalf_t, 8>*>(static_cast<bhalf_t*>(dst) + p * plane + at) = part[p];
  } else {
    store_floats<T, 8>(static_cast<T*>(dst) + at, v);
  }
}

/// Copies up to two matrices into rows that the tiled product can read: aligned, padded with zeros, fp32 in
/// its three parts. Bound by memory: 10,000 x 768 and 768 x 768 fp32 83 MB in 14 us.
template <class T>
__device__ __forceinline__ void prepare_rows(uint32_t block, uint32_t thread, const PrepareArgs& a, const PrepareArgs& b) {
  const bool second = block >= a.blocks;
  const PrepareArgs& p = second ? b : a;
  const uint32_t per_row = static_cast<uint32_t>(p.ld / 8);
  const auto [r, chunk] = row_and_chunk(second ? block - a.blocks : block, per_row, thread);
  if (r >= p.rows) return;
  const uint32_t c = chunk * 8;
  float v[8];
  load8(static_cast<const T*>(p.src) + r * p.stride + c, v, p.cols - c);
  store_prepared<T>(p.dst, r * p.ld + c, p.plane, v);
}

template <class T>
__global__ void __launch_bounds__(256) prepare_kernel(PrepareArgs a, PrepareArgs b) {
  prepare_rows<T>(blockIdx.x, threadIdx.x, a, b);
}

/// dz = grad * act'(z) (stored if asked for) and its column sums over this work-group's rows. A thread
/// has eight columns; LY threads share them, each taking every LY-th row. Bound by memory: 16,384 x
/// 4,096 bf16 with GELU 403 MB in 82 us, 4.9 TB/s. dz is written for 16-bit results in their type, since it feeds the
/// matrix unit, which takes no wider ones: a rounding of each term by 2^-9 (bf16; 2^-12 in fp16, 2^-25 absolute below
/// 2^-14), no larger than the one that the gradient came with; 2.3e-3 of a bf16 gradient's size altogether, 1.7e-3 without
/// it. A second part for the rest would double both products.
struct SlopeArgs {
  const void* grad;
  const void* pre;
  uint64_t rows, ld_grad, ld_pre;
  uint32_t cols;
  int act;
  void* dz;  // as PrepareArgs::dst, or null
  int plain;  // dz in its own type, also where that is fp32
  uint64_t ld, plane;
  float* sums;  // [work-group][cols rounded up to 8], or null
  void* total;  // the sums themselves, where one work-group has all rows, or null
  uint32_t rows_each, across, blocks;
};

/// Work-groups past the slope's make the copies of x and w.
template <class T, int LX, int LY, bool STREAM>
__global__ void __launch_bounds__(LX* LY) slope_kernel(SlopeArgs a, PrepareArgs copy_a, PrepareArgs copy_b) {
  constexpr uint32_t kRows = LY, kCols = LX * 8, kParts = LX * LY / 256;
  __shared__ float s_sum[kRows][kCols + 4];
  if (blockIdx.x >= a.blocks) {
    const uint32_t block = (blockIdx.x - a.blocks) * kParts + threadIdx.x / 256;
    if (block < copy_a.blocks + copy_b.blocks) prepare_rows<T>(block, threadIdx.x % 256, copy_a, copy_b);
    return;
  }
  const uint32_t group = blockIdx.x / a.across, across = blockIdx.x - group * a.across;
  const uint32_t lane = threadIdx.x % LX, part = threadIdx.x / LX;
  const uint32_t c = across * kCols + lane * 8;
  const uint64_t r0 = static_cast<uint64_t>(group) * a.rows_each;
  const uint64_t r1 = r0 + a.rows_each < a.rows ? r0 + a.rows_each : a.rows;
  float sum[8] = {};
  if (c < a.cols) {
    const uint32_t left = a.cols - c;
#pragma unroll 2
    for (uint64_t r = r0 + part; r < r1; r += kRows) {
      float g[8];
      load8<STREAM>(static_cast<const T*>(a.grad) + r * a.ld_grad + c, g, left);
      if (a.act != QVH_ACT_NONE) {
        float z[8];
        load8<STREAM>(static_cast<const T*>(a.pre) + r * a.ld_pre + c, z, left);
        if (a.act == QVH_ACT_RELU) {
#pragma unroll
          for (int i = 0; i < 8; ++i) g[i] *= activate_slope<sizeof(T) == 4>(z[i], QVH_ACT_RELU);
        } else if (a.act == QVH_ACT_GELU) {
#pragma unroll
          for (int i = 0; i < 8; ++i) g[i] *= activate_slope<sizeof(T) == 4>(z[i], QVH_ACT_GELU);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) g[i] *= activate_slope<sizeof(T) == 4>(z[i], QVH_ACT_SILU);
        }
      }
      if (a.dz) {
        if (sizeof(T) == 4 && a.plain) {
          store8(static_cast<T*>(a.dz) + r * a.ld + c, g, 8);  // zeros behind the last column
        } else {
          store_prepared<T>(a.dz, r * a.ld + c, a.plane, g);
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[i] += g[i];
    }
  }
  if (!a.sums && !a.total) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) s_sum[part][lane * 8 + i] = sum[i];
  __syncthreads();
  const uint32_t ld = (a.cols + 7) / 8 * 8;
  const uint32_t col = across * kCols + threadIdx.x;
  if (threadIdx.x < kCols && col < ld) {
    float eight[8] = {};
    for (uint32_t p = 0; p < kRows; p += 8) {
#pragma unroll
      for (uint32_t u = 0; u < 8; ++u) eight[u] += s_sum[p + u][threadIdx.x];
    }
    const float t = sum8(eight);
    if (a.sums) {
      a.sums[static_cast<uint64_t>(group) * ld + col] = t;
    } else if (col < a.cols) {
      static_cast<T*>(a.total)[col] = static_cast<T>(t);
    }
  }
}

/// Adds the work-groups' column sums, where no launch of a product does.
template <class T>
__global__ void __launch_bounds__(256) column_sum_kernel(ColumnSums a, T* __restrict__ out) {
  add_columns(a, blockIdx.x, out);
}

// ---- few rows ---------------------------------------------------------------------------------
//
// Small products in one launch, whatever their rows' alignment: every work-group reads 16 rows of the weight
// and up to 64 of x straight into the fragments of the matrix unit, its eight waves taking every eighth step
// of k, and adds the waves' sums in LDS. One row of x: the weight is the traffic. Many: the loads, of 64
// bytes from each of 16 rows, are what takes the time, 0.4 us a step for 16 rows of x and 1.1 for 64
// (loading four steps ahead changes nothing), so that long k is better split and joined.

constexpr int kFewWaves = 8;

template <class T>
__device__ __forceinline__ void load_k(const T* row, uint32_t k, uint32_t depth, typename Frag<T>::type& f) {
  constexpr int kEach = Frag<T>::kEach;
  if (k + kEach <= depth) {
    f = reinterpret_cast<const Loose<T, kEach>*>(row + k)->v;
  } else {
#pragma unroll
    for (int e = 0; e < kEach; ++e) f[e] = k + e < depth ? row[k + e] : static_cast<T>(0.0f);
  }
}

__device__ __forceinline__ f32x4_t mfma16(Frag<half_t>::x8 a, Frag<half_t>::x8 b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4_t mfma16(Frag<bhalf_t>::x8 a, Frag<bhalf_t>::x8 b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4_t mfma16(f32x4_t a, f32x4_t b, f32x4_t c) {
#pragma unroll
  for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
  return c;
}

template <class T, int MT>
__global__ void __launch_bounds__(kFewWaves * 64) few_rows_kernel(const T* __restrict__ x, uint64_t ldx,
                                                                  const T* __restrict__ w, uint64_t ldw, uint32_t m,
                                                                  uint32_t n, uint32_t k,
                                                                  LinearEpilogue<T> epi) {
  using F = typename Frag<T>::type;
  constexpr uint32_t kEach = Frag<T>::kEach;  // k per lane and step
  constexpr uint32_t kDepth = kEach * 4;
  __shared__ float s_sum[kFewWaves][16 * MT][17];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, h = lane >> 4;
  const uint32_t n0 = blockIdx.x * 16, m0 = blockIdx.y * (16 * MT);
  const T* wr = w + static_cast<uint64_t>(n0 + i < n ? n0 + i : n - 1) * ldw;
  const T* xr[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) xr[t] = x + static_cast<uint64_t>(m0 + 16 * t + i < m ? m0 + 16 * t + i : m - 1) * ldx;
  f32x4_t acc[MT] = {};
  for (uint32_t k0 = wave * kDepth; k0 < k; k0 += kFewWaves * kDepth) {
    F fw, fx[MT];
    load_k<T>(wr, k0 + h * kEach, k, fw);
#pragma unroll
    for (int t = 0; t < MT; ++t) load_k<T>(xr[t], k0 + h * kEach, k, fx[t]);
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = mfma16(fw, fx[t], acc[t]);
  }
  // Lane (i, h) holds rows 4 h .. + 3 of w against row i of x.
#pragma unroll
  for (int t = 0; t < MT; ++t) {
#pragma unroll
    for (int r = 0; r < 4; ++r) s_sum[wave][16 * t + i][4 * h + r] = acc[t][r];
  }
  __syncthreads();
  for (uint32_t o = threadIdx.x; o < 256 * MT; o += kFewWaves * 64) {
    const uint32_t row = o / 16, col = o % 16;
    float sum = 0.0f;
#pragma unroll
    for (int v = 0; v < kFewWaves; ++v) sum += s_sum[v][row][col];
    if (m0 + row < m && n0 + col < n) epi.one(m0 + row, n0 + col, sum);
  }
}

// ---- host side --------------------------------------------------------------------------------

/// How the tiled products can read a matrix: 16 bytes at a time, four, or only a copy of it.
enum class Fit { kWide, kDwords, kNot };

Fit fit_of(const void* p, uint64_t stride, uint64_t cols, size_t elem) {
  const auto whole = [&](uint64_t bytes) {
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && stride * elem % bytes == 0 && cols * elem % bytes == 0;
  };
  return whole(16) ? Fit::kWide : whole(4) ? Fit::kDwords : Fit::kNot;
}

struct Space {
  size_t at = 0;
  char* base = nullptr;
  void* take(size_t bytes) {
    void* p = base ? base + at : nullptr;
    at += (bytes + 255) / 256 * 256;
    return p;
  }
};

/// A matrix as an operand of a tiled product: itself, or a copy to be made.
struct Prepared {
  GemmOperand op;
  PrepareArgs job;
  bool copy = false;
};

struct Matrix {
  const void* p;
  uint64_t rows, stride;
  uint32_t cols;
};

Prepared as_it_is(const Matrix& x) {
  Prepared p;
  p.op.base = x.p;
  p.op.ld = x.stride;
  return p;
}

/// Aligned rows, zeros behind the last column; fp32 in its three parts.
Prepared copy_of(const Matrix& x, int dtype, Space& ws) {
  Prepared p;
  p.copy = true;
  p.job.src = x.p;
  p.job.rows = x.rows;
  p.job.stride = x.stride;
  p.job.cols = x.cols;
  p.job.ld = ceil_div(x.cols, 8) * 8;
  p.job.plane = p.job.ld * x.rows;
  p.job.dst = ws.take(p.job.plane * (dtype == QVH_FP32 ? kPlanes : 1) * 2);
  const uint64_t blocks = ceil_div(p.job.ld / 8 * x.rows, 256);
  QVH_REQUIRE(blocks * 256 < kGridThreads, kTooLarge);
  p.job.blocks = static_cast<uint32_t>(blocks);
  p.op.base = p.job.dst;
  p.op.ld = p.job.ld;
  p.op.plane = p.job.plane;
  return p;
}

/// us of a launch that copies `elements`.
double copy_us(int dtype, double elements) { return 6.0 + elements * (dtype == QVH_FP32 ? 10.0 : 4.0) / 3.5e6; }

/// The kind that reads both operands as they are; for 16-bit types only where both fit.
Kind direct_kind(int dtype, Fit a, Fit b) {
  const bool wide = a == Fit::kWide && b == Fit::kWide;
  if (dtype == QVH_FP32) return wide ? Kind::kFloat : Kind::kFloatNarrow;
  return wide ? Kind::kPlane1 : Kind::kNarrow;
}

Kind copied_kind(int dtype) { return dtype == QVH_FP32 ? Kind::kPlane3 : Kind::kPlane1; }

void launch_prepare(int dtype, const Prepared& a, const Prepared& b, hipStream_t s) {
  const PrepareArgs none;
  const PrepareArgs& first = a.copy ? a.job : b.copy ? b.job : none;
  const PrepareArgs& second = a.copy && b.copy ? b.job : none;
  const uint64_t blocks = static_cast<uint64_t>(first.blocks) + second.blocks;
  if (blocks == 0) return;
  QVH_REQUIRE(blocks * 256 < kGridThreads, kTooLarge);
  with_dtype(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    hipLaunchKernelGGL((prepare_kernel<T>), dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, first, second);
  });
  QVH_HIP(hipGetLastError());
}

void run_product(Form form, Kind kind, int dtype, GemmArgs g, const void* bias, const void* residual, uint64_t ld_residual,
                 void* out, uint64_t ld_out, void* keep, uint64_t ld_keep, int act, const GemmPlan& plan, void* partial,
                 hipStream_t s, const ColumnSums& columns = {}, void* column_out = nullptr) {
  with_dtype(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    LinearEpilogue<T> e;
    e.columns = columns;
    e.column_out = static_cast<T*>(column_out);
    e.bias = static_cast<const T*>(bias);
    e.residual = static_cast<const T*>(residual);
    e.out = static_cast<T*>(out);
    e.keep = static_cast<T*>(keep);
    e.ld_residual = ld_residual;
    e.ld_out = ld_out;
    e.ld_keep = ld_keep;
    e.act = act;
    if constexpr (std::is_same_v<T, float>) {
      gemm_fp32(form, kind, g, e, plan, partial, s);
    } else if constexpr (std::is_same_v<T, half_t>) {
      gemm_fp16(form, kind, g, e, plan, partial, s);
    } else {
      gemm_bf16(form, kind, g, e, plan, partial, s);
    }
  });
}

void check_shape(const std::string& w, uint64_t m, uint32_t k, uint32_t n, int dtype, int act) {
  require_dtype(w.c_str(), dtype);
  QVH_REQUIRE(act >= QVH_ACT_NONE && act <= QVH_ACT_SILU, w + ": unknown activation");
  QVH_REQUIRE(m < kMaxRows, w + ": m must be below 2^31");
  QVH_REQUIRE(k <= kMaxWidth && n <= kMaxWidth, w + ": k and n must be at most 2^20");
}

void check_matrix(const std::string& w, const char* name, const void* p, uint64_t rows, uint64_t cols, uint64_t stride,
                  size_t elem) {
  QVH_REQUIRE(p != nullptr || rows == 0 || cols == 0, w + ": " + name + " is null");
  QVH_REQUIRE(reinterpret_cast<uintptr_t>(p) % elem == 0, w + ": " + name + " is not aligned to its element type");
  QVH_REQUIRE((stride >= cols || rows <= 1) && stride <= kMaxStride, w + ": " + name + "'s stride must be in [row length, 2^22]");
}

/// us of the few-row kernel, fitted to 204 products from 1 x 64 x 64 to 3,721 x 2,019 x 65, bf16 and fp32. Taken
/// where it promises to beat the tiled products, it was the slower by more than 12% in 10 of them (by rows of x
/// alone, up to 64, in far more: 13% slower than the better one on average, against 2%). Both sides, few rows
/// first: 64 x 512 x 1,024 4.5 and 4.9, 64 x 4,096 x 1,024 19.8 and 9.0, 614 x 96 x 74 2.7 and 3.9.
double few_us(uint64_t m, uint32_t k, uint32_t n, int dtype) {
  const uint64_t groups = ceil_div(m, 64) * ceil_div(n, 16);
  double step = m <= 16 ? 0.42 : m <= 32 ? 0.64 : 1.07;
  if (dtype != QVH_FP32 && k % 2 != 0) step *= 3.2;  // rows that begin inside a dword
  return 2.0 + static_cast<double>(ceil_div(groups, 256)) * (0.3 + static_cast<double>(ceil_div(k, dtype == QVH_FP32 ? 128 : 256)) * step);
}

struct LinearRun {
  bool few = false;
  Kind kind = Kind::kPlane1;
  Prepared x, w;
  GemmPlan plan;
  void* partial = nullptr;
  size_t bytes = 0;
};

// fp32: the fp32 matrix instructions read the operands as they are; the bf16 ones, sixteen times as fast, need
// copies in three parts and then six products. Both sides, copies included, in us: 512^3 12 and 22, 1,024^3 28
// and 41, 2,048^3 140 and 112, 10,000 x 768 x 768 114 and 92. 16-bit rows that are whole dwords but not whole
// 16-byte pieces, read as they are and copied: 1,003 x 98 x 384 5.2 and 8.1, 2,048^2 x 2,046 39 and 45.
LinearRun plan_linear(const qvh_linear_args& a, void* ws) {
  LinearRun r;
  if (a.m == 0 || a.n == 0) return r;
  Space sp;
  sp.base = static_cast<char*>(ws);
  const size_t e = dtype_size(a.dtype);
  const Matrix x{a.x, a.m, a.x_stride, a.k}, w{a.weight, a.n, a.weight_stride, a.k};
  const Fit fx = fit_of(a.x, a.x_stride, a.k, e), fw = fit_of(a.weight, a.weight_stride, a.k, e);
  const bool all = a.dtype == QVH_FP32;  // copies are made of everything, in parts
  const bool copy_x = all || fx != Fit::kWide, copy_w = all || fw != Fit::kWide;
  const double elements = (copy_x ? static_cast<double>(a.m) * a.k : 0.0) + (copy_w ? static_cast<double>(a.n) * a.k : 0.0);
  r.kind = copied_kind(a.dtype);
  r.plan = gemm_plan(a.m, a.n, a.k, r.kind, 1, false);
  bool copies = copy_x || copy_w;
  if (copies && (all || (fx != Fit::kNot && fw != Fit::kNot))) {
    const Kind direct = direct_kind(a.dtype, fx, fw);
    const GemmPlan p = gemm_plan(a.m, a.n, a.k, direct, 1, false);
    if (p.us < r.plan.us + copy_us(a.dtype, elements)) {
      copies = false;
      r.kind = direct;
      r.plan = p;
    }
  }
  r.few = ceil_div(a.m, 64) <= 65535 && few_us(a.m, a.k, a.n, a.dtype) < r.plan.us + (copies ? copy_us(a.dtype, elements) : 0.0);
  if (r.few) return r;
  QVH_REQUIRE(r.plan.tile >= 0, kTooLarge);
  r.x = copies && copy_x ? copy_of(x, a.dtype, sp) : as_it_is(x);
  r.w = copies && copy_w ? copy_of(w, a.dtype, sp) : as_it_is(w);
  r.partial = sp.take(r.plan.partial_bytes);
  r.bytes = sp.at;
  return r;
}

void check_linear(const char* who, const qvh_linear_args* a) {
  const std::string w(who);
  QVH_REQUIRE(a != nullptr, w + ": null arguments");
  check_shape(w, a->m, a->k, a->n, a->dtype, a->activation);
  const size_t e = dtype_size(a->dtype);
  check_matrix(w, "x", a->x, a->m, a->k, a->x_stride, e);
  check_matrix(w, "weight", a->weight, a->n, a->k, a->weight_stride, e);
  check_matrix(w, "out", a->out, a->m, a->n, a->out_stride, e);
  if (a->residual) check_matrix(w, "residual", a->residual, a->m, a->n, a->residual_stride, e);
  if (a->preactivation) check_matrix(w, "preactivation", a->preactivation, a->m, a->n, a->preactivation_stride, e);
  QVH_REQUIRE(reinterpret_cast<uintptr_t>(a->bias) % e == 0, w + ": bias is not aligned to its element type");
}

template <class T>
void launch_few(const qvh_linear_args& a, hipStream_t s) {
  LinearEpilogue<T> e;
  e.bias = static_cast<const T*>(a.bias);
  e.residual = static_cast<const T*>(a.residual);
  e.out = static_cast<T*>(a.out);
  e.keep = static_cast<T*>(a.preactivation);
  e.ld_residual = a.residual_stride;
  e.ld_out = a.out_stride;
  e.ld_keep = a.preactivation_stride;
  e.act = a.activation;
  const auto go = [&](auto tiles) {
    hipLaunchKernelGGL((few_rows_kernel<T, decltype(tiles)::value>), dim3(static_cast<unsigned>(ceil_div(a.n, 16)), static_cast<unsigned>(ceil_div(a.m, 64))),
                       dim3(kFewWaves * 64), 0, s, static_cast<const T*>(a.x), a.x_stride,
                       static_cast<const T*>(a.weight), a.weight_stride, static_cast<uint32_t>(a.m), a.n, a.k, e);
  };
  if (a.m <= 16) {
    go(std::integral_constant<int, 1>{});
  } else if (a.m <= 32) {
    go(std::integral_constant<int, 2>{});
  } else {
    go(std::integral_constant<int, 4>{});
  }
  QVH_HIP(hipGetLastError());
}

struct GradRun {
  bool slope = false;  // dz is written or summed
  bool one = false;    // by work-groups that have all rows
  SlopeArgs job{};
  uint32_t sum_parts = 0;
  GemmOperand dz;
  Prepared x, w;
  Kind kind_x = Kind::kPlane1, kind_w = Kind::kPlane1;
  GemmPlan plan_x, plan_w;
  void *partial_x = nullptr, *partial_w = nullptr;
  size_t bytes = 0;
};

GradRun plan_grad(const qvh_linear_grad_args& a, void* ws) {
  GradRun r;
  if (a.n == 0 || (a.m == 0 && a.k == 0)) return r;
  const size_t e = dtype_size(a.dtype);
  Space sp;
  sp.base = static_cast<char*>(ws);
  const bool of_x = a.grad_x && a.k > 0, of_w = a.grad_weight && a.k > 0;
  const bool fp32 = a.dtype == QVH_FP32;
  const Matrix x{a.x, a.m, a.x_stride, a.k}, w{a.weight, a.n, a.weight_stride, a.k};
  const Fit fx = fit_of(a.x, a.x_stride, a.k, e), fw = fit_of(a.weight, a.weight_stride, a.k, e);

  // fp32: both products on fp32 instructions, or both on parts. dz is grad itself where there is no
  // activation and the products can read it.
  bool parts = false;
  if (fp32 && (of_x || of_w)) {
    double direct = 0.0, split = copy_us(a.dtype, static_cast<double>(a.m) * a.n);
    if (of_x) {
      direct += gemm_plan(a.m, a.k, a.n, direct_kind(a.dtype, Fit::kWide, fw), 1, false).us;
      split += gemm_plan(a.m, a.k, a.n, Kind::kPlane3, 1, false).us + static_cast<double>(a.n) * a.k * 10.0 / 3.5e6;
    }
    if (of_w) {
      direct += gemm_plan(a.n, a.k, a.m, direct_kind(a.dtype, Fit::kWide, fx), 1, false).us;
      split += gemm_plan(a.n, a.k, a.m, Kind::kPlane3, 1, false).us + static_cast<double>(a.m) * a.k * 10.0 / 3.5e6;
    }
    parts = split < direct;
  }
  Fit fz = fit_of(a.grad, a.grad_stride, a.n, e);
  const bool as_is = a.activation == QVH_ACT_NONE && !parts && (fz == Fit::kWide || (fp32 && fz == Fit::kDwords));
  const bool writes = (of_x || of_w) && !as_is;
  r.slope = writes || a.grad_bias;
  if (r.slope) {
    SlopeArgs& j = r.job;
    j.grad = a.grad;
    j.pre = a.preactivation;
    j.rows = a.m;
    j.ld_grad = a.grad_stride;
    j.ld_pre = a.preactivation_stride;
    j.cols = a.n;
    j.act = a.activation;
    j.ld = ceil_div(a.n, 8) * 8;
    j.plane = j.ld * a.m;
    j.plain = !parts;
    if (writes) j.dz = sp.take(j.plane * (parts ? kPlanes * 2 : e));
    // A work-group with all rows of 64 columns saves the launch that adds up the parts; its threads (256, or 1,024)
    // then walk down up to four rows each. Otherwise 256 columns, rows spread over about a thousand
    // work-groups, at least 16 rows each. (All of linear_grad, bf16: 90 x 1,024 x 80 16.7 us against 21.2.)
    r.one = a.grad_bias && a.m <= kSumRows;
    j.across = static_cast<uint32_t>(ceil_div(a.n, r.one ? 64 : 256));
    j.rows_each = r.one ? static_cast<uint32_t>(std::max<uint64_t>(a.m, 1))
                        : static_cast<uint32_t>(std::max<uint64_t>(16, ceil_div(ceil_div(a.m, 8), ceil_div(1024, j.across)) * 8));
    r.sum_parts = r.one ? 1 : static_cast<uint32_t>(ceil_div(a.m, j.rows_each));
    j.blocks = r.sum_parts * j.across;
    if (r.one) {
      j.total = a.grad_bias;
    } else if (a.grad_bias) {
      j.sums = static_cast<float*>(sp.take(static_cast<size_t>(r.sum_parts) * j.ld * 4));
    }
  }
  if (writes) {
    r.dz.base = r.job.dz;
    r.dz.ld = r.job.ld;
    r.dz.plane = r.job.plane;
    fz = Fit::kWide;
  } else {
    r.dz.base = a.grad;
    r.dz.ld = a.grad_stride;
  }
  const auto product = [&](const Matrix& other, Fit fit, uint64_t m, uint64_t depth, Prepared& prepared, Kind& kind,
                           GemmPlan& plan, void*& partial) {
    if (parts) {
      kind = Kind::kPlane3;
      plan = gemm_plan(m, a.k, depth, kind, 1, false);
      prepared = copy_of(other, a.dtype, sp);
    } else if (fp32 || (fit == Fit::kWide && fz == Fit::kWide)) {
      kind = direct_kind(a.dtype, fz, fit);
      plan = gemm_plan(m, a.k, depth, kind, 1, false);
      prepared = as_it_is(other);
    } else {  // 16-bit: dz is wide by now
      kind = Kind::kPlane1;
      plan = gemm_plan(m, a.k, depth, kind, 1, false);
      prepared = as_it_is(other);
      const GemmPlan narrow = gemm_plan(m, a.k, depth, Kind::kNarrow, 1, false);
      if (fit == Fit::kDwords && narrow.us < plan.us + copy_us(a.dtype, static_cast<double>(other.rows) * other.cols)) {
        kind = Kind::kNarrow;
        plan = narrow;
      } else {
        prepared = copy_of(other, a.dtype, sp);
      }
    }
    QVH_REQUIRE(plan.tile >= 0, kTooLarge);
    partial = sp.take(plan.partial_bytes);
  };
  if (of_x) product(w, fw, a.m, a.n, r.w, r.kind_x, r.plan_x, r.partial_x);
  if (of_w) product(x, fx, a.n, a.m, r.x, r.kind_w, r.plan_w, r.partial_w);
  r.bytes = sp.at;
  return r;
}

void check_grad(const char* who, const qvh_linear_grad_args* a) {
  const std::string w(who);
  QVH_REQUIRE(a != nullptr, w + ": null arguments");
  check_shape(w, a->m, a->k, a->n, a->dtype, a->activation);
  const size_t e = dtype_size(a->dtype);
  check_matrix(w, "grad", a->grad, a->m, a->n, a->grad_stride, e);
  if (a->activation != QVH_ACT_NONE) {
    QVH_REQUIRE(a->preactivation != nullptr || a->m == 0 || a->n == 0, w + ": an activation's gradient needs the pre-activation");
    check_matrix(w, "preactivation", a->preactivation, a->m, a->n, a->preactivation_stride, e);
  }
  if (a->grad_x) {
    check_matrix(w, "weight", a->weight, a->n, a->k, a->weight_stride, e);
    check_matrix(w, "grad_x", a->grad_x, a->m, a->k, a->grad_x_stride, e);
  }
  if (a->grad_weight) {
    check_matrix(w, "x", a->x, a->m, a->k, a->x_stride, e);
    check_matrix(w, "grad_weight", a->grad_weight, a->n, a->k, a->grad_weight_stride, e);
  }
  QVH_REQUIRE(reinterpret_cast<uintptr_t>(a->grad_bias) % e == 0, w + ": grad_bias is not aligned to its element type");
}

}  // namespace
}  // namespace qvh

extern "C" {

qvh_status qvh_linear_workspace(const qvh_linear_args* args, uint64_t* bytes) {
  return qvh::guarded([&] {
    QVH_REQUIRE(bytes != nullptr, "qvh_linear_workspace: null output");
    qvh::check_linear("qvh_linear_workspace", args);
    *bytes = qvh::plan_linear(*args, nullptr).bytes;
  });
}

qvh_status qvh_linear_device(const qvh_linear_args* args, void* d_workspace, uint64_t workspace_bytes, void* stream) {
  return qvh::guarded([&] {
    using namespace qvh;
    check_linear("qvh_linear_device", args);
    const qvh_linear_args& a = *args;
    if (a.m == 0 || a.n == 0) return;
    const LinearRun r = plan_linear(a, d_workspace);
    check_workspace("qvh_linear_device", d_workspace, workspace_bytes, r.bytes);
    const DeviceScope device;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (r.few) {
      with_dtype(a.dtype, [&](auto* t) { launch_few<std::remove_pointer_t<decltype(t)>>(a, s); });
      return;
    }
    launch_prepare(a.dtype, r.x, r.w, s);
    GemmArgs g;
    g.a = r.x.op;
    g.b = r.w.op;
    g.m = static_cast<uint32_t>(a.m);
    g.n = a.n;
    g.k = a.k;
    run_product(Form::kRowsRows, r.kind, a.dtype, g, a.bias, a.residual, a.residual_stride, a.out, a.out_stride, a.preactivation,
                a.preactivation_stride, a.activation, r.plan, r.partial, s);
  });
}

qvh_status qvh_linear_grad_workspace(const qvh_linear_grad_args* args, uint64_t* bytes) {
  return qvh::guarded([&] {
    QVH_REQUIRE(bytes != nullptr, "qvh_linear_grad_workspace: null output");
    qvh::check_grad("qvh_linear_grad_workspace", args);
    *bytes = qvh::plan_grad(*args, nullptr).bytes;
  });
}

qvh_status qvh_linear_grad_device(const qvh_linear_grad_args* args, void* d_workspace, uint64_t workspace_bytes,
                                  void* stream) {
  return qvh::guarded([&] {
    using namespace qvh;
    check_grad("qvh_linear_grad_device", args);
    const qvh_linear_grad_args& a = *args;
    const GradRun r = plan_grad(a, d_workspace);
    check_workspace("qvh_linear_grad_device", d_workspace, workspace_bytes, r.bytes);
    const DeviceScope device;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const bool products = a.k > 0 && (a.grad_x || a.grad_weight);
    if (r.slope && r.job.blocks > 0) {
      const PrepareArgs none;
      const PrepareArgs& first = r.x.copy ? r.x.job : r.w.copy ? r.w.job : none;
      const PrepareArgs& second = r.x.copy && r.w.copy ? r.w.job : none;
      const uint64_t copies = static_cast<uint64_t>(first.blocks) + second.blocks;
      QVH_REQUIRE((r.job.blocks + copies) * 256 < kGridThreads, kTooLarge);
      with_dtype(a.dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const bool tall = r.one && a.m > 128;
        // What the L2s cannot hold is read past them, so that more of dz is still there for the products (linear_grad of
        // 16,384 x 1,024 x 4,096 bf16 351 and 340 us; 4,096 x 512 x 1,024, 8 MB, 38.7 and 39.9).
        const bool stream = a.m * a.n * sizeof(T) >= kStreamed;
        const auto kernel = tall     ? slope_kernel<T, 8, 128, false>
                            : r.one  ? slope_kernel<T, 8, 32, false>
                            : stream ? slope_kernel<T, 32, 8, true>
                                     : slope_kernel<T, 32, 8, false>;
        const uint64_t groups = r.job.blocks + ceil_div(copies, tall ? 4 : 1);
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(groups)), dim3(tall ? 1024 : 256), 0, s, r.job, first, second);
      });
      QVH_HIP(hipGetLastError());
    } else if (products) {
      launch_prepare(a.dtype, r.x, r.w, s);
    }
    // The parts are added by the launch that joins the weight gradient's splits, or by one of their own.
    ColumnSums columns;
    if (a.grad_bias && a.n > 0 && !r.one) {
      columns.parts = r.job.sums;
      columns.count = r.sum_parts;
      columns.cols = a.n;
    }
    const bool joined = products && a.grad_weight && r.plan_w.splits > 1;
    if (columns.cols > 0 && !joined) {
      with_dtype(a.dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        hipLaunchKernelGGL((column_sum_kernel<T>), dim3(static_cast<unsigned>(ceil_div(a.n, 64))), dim3(256), 0, s, columns,
                           static_cast<T*>(a.grad_bias));
      });
      QVH_HIP(hipGetLastError());
      columns = ColumnSums{};
    }
    if (!products) return;
    GemmArgs g;
    g.a = r.dz;
    if (a.grad_x && a.m > 0) {
      g.b = r.w.op;
      g.m = static_cast<uint32_t>(a.m);
      g.n = a.k;
      g.k = a.n;
      run_product(Form::kRowsK, r.kind_x, a.dtype, g, nullptr, nullptr, 0, a.grad_x, a.grad_x_stride, nullptr, 0, QVH_ACT_NONE,
                  r.plan_x, r.partial_x, s);
    }
    if (a.grad_weight && a.n > 0) {
      g.b = r.x.op;
      g.m = a.n;
      g.n = a.k;
      g.k = static_cast<uint32_t>(a.m);
      run_product(Form::kKK, r.kind_w, a.dtype, g, nullptr, nullptr, 0, a.grad_weight, a.grad_weight_stride, nullptr, 0, QVH_ACT_NONE,
                  r.plan_w, r.partial_w, s, columns, a.grad_bias);
    }
  });
}

}  // extern "C"
