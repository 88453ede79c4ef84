// Orthogonalising an update by Newton-Schulz products.
//
// X = G / |G|_F, then per step S = X X^T, P = a + b S + c S S, X <- P X (from the right, S = X^T X and
// X <- X P, where there are more rows than columns): every singular value s goes through
// s (a + b s^2 + c s^4). Three products a step; the polynomial is the second one's epilogue.
//
// Precision. A rounding of X early on is amplified by as much as the step lifts small singular values
// (up to a factor `a` each), so 16-bit iterates would leave errors of a percent. Every matrix is kept as
// two fp16 parts, high + low, of 22 bits together, and a product runs over (high, low), (low, high) and
// (high, high). The parts hold the value times 2^12: nothing here exceeds 15 (the coefficients are
// checked for that), and the low part of values around 1/1000 stays a normal number.
#include <algorithm>
#include <cmath>

#include "gemm.hpp"

namespace qvh {
namespace {

constexpr uint32_t kMaxSide = 65536;
constexpr float kScale = 4096.0f;
constexpr uint32_t kNormParts = 64;

template <class T>
__global__ void __launch_bounds__(256) norm_kernel(const T* __restrict__ g, uint64_t count, double* __restrict__ parts) {
  __shared__ double s_sum[4];
  const T* x = g + blockIdx.y * count;
  double sum = 0.0;
  for (uint64_t i = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x; i < count; i += kNormParts * 256) {
    const double v = static_cast<double>(static_cast<float>(x[i]));
    sum += v * v;
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 64);
  if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) parts[blockIdx.y * kNormParts + blockIdx.x] = ((s_sum[0] + s_sum[1]) + s_sum[2]) + s_sum[3];
}

/// high + low = v in fp16.
__device__ __forceinline__ void split2(float v, half_t& high, half_t& low) {
  high = static_cast<half_t>(v);
  low = static_cast<half_t>(v - static_cast<float>(high));
}

__device__ __forceinline__ void store_parts(half_t* p, uint64_t plane, const float (&v)[8]) {
  Pack<half_t, 8> high, low;
#pragma unroll
  for (int i = 0; i < 8; ++i) split2(v[i], high.v[i], low.v[i]);
  *reinterpret_cast<Pack<half_t, 8>*>(p) = high;
  *reinterpret_cast<Pack<half_t, 8>*>(p + plane) = low;
}

/// X = G / |G|_F in parts, rows padded with zeros to ld.
template <class T>
__global__ void __launch_bounds__(256) start_kernel(const T* __restrict__ g, uint32_t m, uint32_t n,
                                                    const double* __restrict__ parts, half_t* __restrict__ x,
                                                    uint64_t ld, uint64_t plane) {
  __shared__ double s_factor;
  if (threadIdx.x < 64) {
    double sum = parts[blockIdx.y * kNormParts + threadIdx.x];
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 64);
    // 2^12 / norm; nothing for a zero matrix, NaN where something is not finite.
    if (threadIdx.x == 0) {
      s_factor = sum == 0.0 ? 0.0f : !(sum < __builtin_huge_val()) ? __builtin_nan("") : kScale / sqrt(sum);
    }
  }
  __syncthreads();
  const double factor = s_factor;  // past fp32's range for an update near its smallest numbers
  const uint64_t i = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x;
  const uint32_t per_row = static_cast<uint32_t>(ld / 8);
  const uint64_t r = i / per_row;
  if (r >= m) return;
  const uint32_t c = static_cast<uint32_t>(i - r * per_row) * 8;
  float v[8];
  load8(g + (static_cast<uint64_t>(blockIdx.y) * m + r) * n + c, v, n - c, false);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = c + e < n ? static_cast<float>(v[e] * factor) : 0.0f;
  store_parts(x + blockIdx.y * 2 * plane + r * ld + c, plane, v);
}

/// Parts of scale * acc, or of a + b S + c scale * acc with S's parts given; zeros behind the last column.
struct PartsEpilogue {
  half_t* out;
  const half_t* s;  // null: no polynomial
  uint64_t ld, plane;
  float scale, a, b;
  __device__ __forceinline__ void operator()(uint32_t z, uint32_t m, uint32_t n, uint32_t left, float (&v)[8]) const {
    const uint64_t at = z * 2 * plane + m * ld + n;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= scale;
    if (s) {
      const Pack<half_t, 8> high = *reinterpret_cast<const Pack<half_t, 8>*>(s + at);
      const Pack<half_t, 8> low = *reinterpret_cast<const Pack<half_t, 8>*>(s + at + plane);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = fmaf(b, static_cast<float>(high.v[i]) + static_cast<float>(low.v[i]), v[i]);
        if (m == n + i) v[i] += a;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = static_cast<uint32_t>(i) < left ? v[i] : 0.0f;
    store_parts(out + at, plane, v);
  }
};

/// The last product: X itself, in the caller's type.
template <class T>
struct ResultEpilogue {
  T* out;
  uint64_t ld, batch;
  float scale;
  int vec;
  __device__ __forceinline__ void operator()(uint32_t z, uint32_t m, uint32_t n, uint32_t left, float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= scale;
    store8(out + z * batch + m * ld + n, v, left, vec);
  }
};

/// No steps: X as it starts.
template <class T>
__global__ void __launch_bounds__(256) parts_to_result_kernel(const half_t* __restrict__ x, uint64_t ld, uint64_t plane,
                                                              uint32_t m, uint32_t n, T* __restrict__ out) {
  const uint64_t i = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= static_cast<uint64_t>(m) * n) return;
  const half_t* p = x + blockIdx.y * 2 * plane + i / n * ld + i % n;
  out[static_cast<uint64_t>(blockIdx.y) * m * n + i] =
      static_cast<T>((static_cast<float>(p[0]) + static_cast<float>(p[plane])) / kScale);
}

struct OrthoLayout {
  uint32_t side;               // the smaller of m and n
  uint64_t ldx, lds;           // rounded up to 8
  uint64_t plane_x, plane_s;   // elements of a part
  size_t norm, x[2], s, p, partial, total;
  GemmPlan gram, square, update;
};

OrthoLayout ortho_layout(uint64_t batch, uint32_t m, uint32_t n) {
  OrthoLayout l{};
  const auto round = [](size_t b) { return (b + 255) / 256 * 256; };
  l.side = std::min(m, n);
  l.ldx = ceil_div(n, 8) * 8;
  l.lds = ceil_div(l.side, 8) * 8;
  l.plane_x = l.ldx * m;
  l.plane_s = l.lds * l.side;
  const uint32_t b = static_cast<uint32_t>(batch);
  l.gram = gemm_plan(l.side, l.side, std::max(m, n), 3, b);
  l.square = gemm_plan(l.side, l.side, l.side, 3, b);
  l.update = gemm_plan(m, n, l.side, 3, b);
  size_t at = round(batch * kNormParts * 8);
  for (size_t& x : l.x) {
    x = at;
    at += round(batch * 2 * l.plane_x * 2);
  }
  l.s = at;
  at += round(batch * 2 * l.plane_s * 2);
  l.p = at;
  at += round(batch * 2 * l.plane_s * 2);
  l.partial = at;
  l.total = at + round(std::max({l.gram.partial_bytes, l.square.partial_bytes, l.update.partial_bytes}));
  return l;
}

/// Whether no step can push a singular value of [0, 1] past 3.5 or the polynomial past 15.
bool bounded(uint32_t steps, double a, double b, double c) {
  double top = 1.0;
  for (uint32_t i = 0; i < steps; ++i) {
    double next = 0.0;
    for (int j = 0; j <= 4096; ++j) {
      const double s = top * j / 4096, p = a + b * s * s + c * s * s * s * s;
      if (!(std::fabs(p) <= 15.0) || !(std::fabs(b) * s * s <= 200.0)) return false;
      next = std::max(next, std::fabs(s * p));
    }
    if (!(next <= 3.5)) return false;
    if (next <= top) return true;  // never leaves [0, top] from here on
    top = next;
  }
  return true;
}

void check_ortho(const char* who, uint64_t batch, uint32_t m, uint32_t n) {
  const std::string w(who);
  QVH_REQUIRE(m <= kMaxSide && n <= kMaxSide, w + ": m and n must be at most 65536");
  QVH_REQUIRE(batch <= 65535, w + ": at most 65535 matrices");
}

GemmArgs product(const half_t* a, uint64_t lda, uint64_t plane_a, const half_t* b, uint64_t ldb, uint64_t plane_b,
                 uint32_t m, uint32_t n, uint32_t k, uint64_t batch) {
  GemmArgs g;
  g.a.base = a;
  g.a.ld = lda;
  g.a.plane = plane_a;
  g.a.batch = 2 * plane_a;
  g.b.base = b;
  g.b.ld = ldb;
  g.b.plane = plane_b;
  g.b.batch = 2 * plane_b;
  g.m = m;
  g.n = n;
  g.k = k;
  g.batches = static_cast<uint32_t>(batch);
  g.pairs = 3;
  g.pa = 0x010;  // (high, low), (low, high), (high, high)
  g.pb = 0x001;
  return g;
}

template <class T>
void orthogonalize(const T* update, uint64_t batch, uint32_t m, uint32_t n, uint32_t steps, float a, float b, float c,
                   T* out, char* ws, hipStream_t s) {
  const OrthoLayout l = ortho_layout(batch, m, n);
  double* norm = reinterpret_cast<double*>(ws + l.norm);
  half_t* x[2] = {reinterpret_cast<half_t*>(ws + l.x[0]), reinterpret_cast<half_t*>(ws + l.x[1])};
  half_t* gram = reinterpret_cast<half_t*>(ws + l.s);
  half_t* poly = reinterpret_cast<half_t*>(ws + l.p);
  void* partial = ws + l.partial;
  const unsigned nb = static_cast<unsigned>(batch);
  hipLaunchKernelGGL((norm_kernel<T>), dim3(kNormParts, nb), dim3(256), 0, s, update, static_cast<uint64_t>(m) * n, norm);
  QVH_HIP(hipGetLastError());
  hipLaunchKernelGGL((start_kernel<T>), dim3(static_cast<unsigned>(ceil_div(l.ldx / 8 * m, 256)), nb), dim3(256), 0, s,
                     update, m, n, norm, x[0], l.ldx, l.plane_x);
  QVH_HIP(hipGetLastError());
  if (steps == 0) {
    hipLaunchKernelGGL((parts_to_result_kernel<T>), dim3(static_cast<unsigned>(ceil_div(static_cast<uint64_t>(m) * n, 256)), nb),
                       dim3(256), 0, s, x[0], l.ldx, l.plane_x, m, n, out);
    QVH_HIP(hipGetLastError());
    return;
  }
  const bool tall = m > n;
  for (uint32_t i = 0; i < steps; ++i) {
    const half_t* cur = x[i & 1];
    half_t* next = x[(i + 1) & 1];
    const GemmArgs g1 = product(cur, l.ldx, l.plane_x, cur, l.ldx, l.plane_x, l.side, l.side, std::max(m, n), batch);
    const PartsEpilogue e1{gram, nullptr, l.lds, l.plane_s, 1.0f / kScale, 0.0f, 0.0f};
    if (tall) {
      launch_gemm<half_t, true, true>(g1, e1, l.gram, partial, s);
    } else {
      launch_gemm<half_t, false, false>(g1, e1, l.gram, partial, s);
    }
    const GemmArgs g2 = product(gram, l.lds, l.plane_s, gram, l.lds, l.plane_s, l.side, l.side, l.side, batch);
    const PartsEpilogue e2{poly, gram, l.lds, l.plane_s, c / kScale, a * kScale, b};
    launch_gemm<half_t, false, false>(g2, e2, l.square, partial, s);
    // P is symmetric: it may be read by rows on either side.
    const GemmArgs g3 = tall ? product(cur, l.ldx, l.plane_x, poly, l.lds, l.plane_s, m, n, l.side, batch)
                             : product(poly, l.lds, l.plane_s, cur, l.ldx, l.plane_x, m, n, l.side, batch);
    const auto third = [&](const auto& e) {
      if (tall) {
        launch_gemm<half_t, false, false>(g3, e, l.update, partial, s);
      } else {
        launch_gemm<half_t, false, true>(g3, e, l.update, partial, s);
      }
    };
    if (i + 1 < steps) {
      third(PartsEpilogue{next, nullptr, l.ldx, l.plane_x, 1.0f / kScale, 0.0f, 0.0f});
    } else {
      const int vec = reinterpret_cast<uintptr_t>(out) % 16 == 0 && n * sizeof(T) % 16 == 0;
      third(ResultEpilogue<T>{out, n, static_cast<uint64_t>(m) * n, 1.0f / (kScale * kScale), vec});
    }
  }
}

}  // namespace
}  // namespace qvh

extern "C" {

qvh_status qvh_orthogonalize_workspace(uint64_t batch, uint32_t m, uint32_t n, uint64_t* bytes) {
  return qvh::guarded([&] {
    using namespace qvh;
    QVH_REQUIRE(bytes != nullptr, "qvh_orthogonalize_workspace: null output");
    check_ortho("qvh_orthogonalize_workspace", batch, m, n);
    *bytes = batch == 0 || m == 0 || n == 0 ? 0 : ortho_layout(batch, m, n).total;
  });
}

qvh_status qvh_orthogonalize_device(const void* d_update, uint64_t batch, uint32_t m, uint32_t n, int dtype,
                                    uint32_t steps, float a, float b, float c, void* d_out, void* d_workspace,
                                    uint64_t workspace_bytes, void* stream) {
  return qvh::guarded([&] {
    using namespace qvh;
    const std::string w("qvh_orthogonalize_device");
    require_dtype(w.c_str(), dtype);
    check_ortho(w.c_str(), batch, m, n);
    QVH_REQUIRE(bounded(steps, a, b, c), w + ": these coefficients let singular values grow without bound");
    if (batch == 0 || m == 0 || n == 0) return;
    QVH_REQUIRE(d_update && d_out, w + ": null buffer");
    QVH_REQUIRE(reinterpret_cast<uintptr_t>(d_update) % dtype_size(dtype) == 0 &&
                    reinterpret_cast<uintptr_t>(d_out) % dtype_size(dtype) == 0,
                w + ": a buffer is not aligned to its element type");
    QVH_REQUIRE(d_workspace != nullptr && workspace_bytes >= ortho_layout(batch, m, n).total, w + ": the workspace is too small");
    QVH_REQUIRE(reinterpret_cast<uintptr_t>(d_workspace) % 16 == 0, w + ": the workspace must be 16-byte aligned");
    current_device();
    with_dtype(dtype, [&](auto* t) {
      using T = std::remove_pointer_t<decltype(t)>;
      orthogonalize<T>(static_cast<const T*>(d_update), batch, m, n, steps, a, b, c, static_cast<T*>(d_out),
                       static_cast<char*>(d_workspace), static_cast<hipStream_t>(stream));
    });
  });
}

}  // extern "C"
