// Orthogonalising an update by Newton-Schulz products.
//
// X = G / |G|_F, then per step S = X X^T, P = a + b S + c S S, X <- P X (from the right, S = X^T X and
// X <- X P, where there are more rows than columns): every singular value s goes through
// s (a + b s^2 + c s^4). Three products a step; the polynomial is the second one's epilogue.
//
// Precision. A rounding of X early on is amplified by as much as the step lifts small singular values
// (up to a factor `a` each), so 16-bit iterates would leave errors of a percent. Every matrix is kept as
// two fp16 parts, high + low, of 22 bits together; a product is high x low + low x high + high x high. The
// parts hold the value times 2^12: nothing here exceeds 15 (the coefficients are checked for that), and the low
// part of values around 1/1000 stays a normal number. fp32 products of the same matrices would run on
// instructions sixteen times as slow, three bf16 parts take twice the products.
//
// 4,096 x 1,024 bf16, five steps, 354 to 372 us: per step S 24 us and 5 to join its three parts of k, S S 15 in one piece, P X 29
// (1,024 x 1,024 results of two parts are a third of a chip's tiles; the matrix instructions of P X are busy 34% of
// the time). Since S and S S are symmetric, only their lower tiles are computed.
#include <algorithm>
#include <cmath>

#include "gemm.hpp"

namespace qvh {
namespace {

constexpr uint32_t kMaxSide = 65536;
constexpr float kScale = 4096.0f;
constexpr uint32_t kNormParts = 256;

/// Adds v over the work-group's four waves; the sum is in every thread.
__device__ __forceinline__ double block_sum(double v, double* s_sum) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
  if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = v;
  __syncthreads();
  return ((s_sum[0] + s_sum[1]) + s_sum[2]) + s_sum[3];
}

/// Sum of squares in parts, in fp64: the norm of an update with entries near either end of fp32's range. 5 us for
/// 4,096 x 1,024 bf16.
template <class T>
__global__ void __launch_bounds__(256) norm_kernel(const T* __restrict__ g, uint64_t count,
                                                   double* __restrict__ parts) {
  __shared__ double s_sum[4];
  const T* x = g + blockIdx.y * count;
  double sum = 0.0;
  for (uint64_t i = (static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x) * 8; i < count; i += kNormParts * 2048) {
    float v[8];
    load8(x + i, v, count - i < 8 ? static_cast<uint32_t>(count - i) : 8u);
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += static_cast<double>(v[e]) * v[e];
  }
  sum = block_sum(sum, s_sum);
  if (threadIdx.x == 0) parts[blockIdx.y * kNormParts + blockIdx.x] = sum;
}

/// 2^12 / norm from the sum of squares; nothing for a zero matrix, NaN where something is not finite.
__device__ __forceinline__ double start_factor(double sum) {
  return sum == 0.0 ? 0.0 : !(sum < __builtin_huge_val()) ? __builtin_nan("") : kScale / sqrt(sum);
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

/// X = G / |G|_F in parts, rows padded with zeros to ld. 4,096 x 1,024 bf16: 25 MB in 11 us.
template <class T>
__global__ void __launch_bounds__(256) start_kernel(const T* __restrict__ g, uint32_t m, uint32_t n,
                                                    const double* __restrict__ parts, half_t* __restrict__ x,
                                                    uint64_t ld, uint64_t plane) {
  __shared__ double s_sum[4];
  static_assert(kNormParts == 256, "one part per thread");
  // Past fp32's range for an update near its smallest numbers, so a double.
  const double factor = start_factor(block_sum(parts[blockIdx.y * kNormParts + threadIdx.x], s_sum));
  const auto [r, chunk] = row_and_chunk(blockIdx.x, static_cast<uint32_t>(ld / 8), threadIdx.x);
  if (r >= m) return;
  const uint32_t c = chunk * 8;
  float v[8];
  load8(g + (static_cast<uint64_t>(blockIdx.y) * m + r) * n + c, v, n - c);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = c + e < n ? static_cast<float>(v[e] * factor) : 0.0f;
  store_parts(x + blockIdx.y * 2 * plane + r * ld + c, plane, v);
}

/// Parts of scale * acc, or of a + b S + c scale * acc with S's parts given; zeros behind the last column.
struct PartsEpilogue {
  static constexpr bool kSymmetric = true;  // S and S S are
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
  __device__ __forceinline__ void operator()(uint32_t z, uint32_t m, uint32_t n, uint32_t left, float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= scale;
    store8(out + z * batch + m * ld + n, v, left);
  }
};

/// No steps: X as it starts.
template <class T>
__global__ void __launch_bounds__(256) parts_to_result_kernel(const half_t* __restrict__ x, uint64_t ld, uint64_t plane,
                                                              uint32_t m, uint32_t n, T* __restrict__ out) {
  const uint64_t count = static_cast<uint64_t>(m) * n;
  for (uint64_t i = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x; i < count; i += static_cast<uint64_t>(gridDim.x) * 256) {
    const half_t* p = x + blockIdx.y * 2 * plane + i / n * ld + i % n;
    out[blockIdx.y * count + i] = static_cast<T>((static_cast<float>(p[0]) + static_cast<float>(p[plane])) / kScale);
  }
}

// ---- small matrices: one work-group does all steps ---------------------------------------------
//
// Where X and S fit LDS (128 x 128, 64 x 512), the seventeen launches of a call would take several times
// longer than their work: 128 x 128 fp32 54 us in one launch (11 a step, by the LDS reads of its fragments and
// five barriers); 64 x 64 20; 79 x 1,220, too large for it, 95. The waves each compute 32 x 32 blocks from LDS (sixteen waves with one block of X
// each, or eight with up to five, which have the registers for it); P takes S's place, X the old
// X's, between barriers. More rows than columns: the transpose is worked on. Rows are padded to an odd
// number of 16-byte pieces, so that sixteen neighbouring rows at one k lie on different banks.

constexpr uint32_t kSmallBlocks = 40;  // 32 x 32 blocks of X
constexpr uint32_t kSmallLds = 160 * 1024;  // what a work-group may have

struct SmallShape {
  uint32_t side, depth;     // rounded up to 32
  uint32_t row_x, row_s;    // bytes
  uint32_t bytes;
};

__host__ __device__ inline SmallShape small_shape(uint32_t m, uint32_t n) {
  SmallShape s;
  s.side = ((m < n ? m : n) + 31) / 32 * 32;
  s.depth = ((m < n ? n : m) + 31) / 32 * 32;
  s.row_x = s.depth * 2 + 16;
  s.row_s = s.side * 2 + 16;
  s.bytes = 2 * s.side * (s.row_x + s.row_s);
  return s;
}

/// Waves for it: their registers hold its blocks.
inline uint32_t small_waves(const SmallShape& s) { return s.side / 32 * (s.depth / 32) <= 16 ? 16 : 8; }

/// Whether a matrix is done by one work-group.
inline bool is_small(uint32_t m, uint32_t n) {
  if (std::max(m, n) > 2048) return false;
  const SmallShape s = small_shape(m, n);
  return s.bytes <= kSmallLds - 1024 && s.side / 32 * (s.depth / 32) <= kSmallBlocks;
}

/// BLOCKS: of X per wave.
template <class T, int WAVES, int BLOCKS>
__global__ void __launch_bounds__(WAVES * 64) ortho_small_kernel(const T* __restrict__ update, uint32_t m, uint32_t n,
                                                                       uint32_t steps, float a, float b, float c,
                                                                       T* __restrict__ out) {
  using X8 = Frag<half_t>::x8;
  using X4 = Frag<half_t>::x4;
  extern __shared__ __attribute__((aligned(16))) char s_dyn[];
  __shared__ double s_sum[WAVES];
  const SmallShape sh = small_shape(m, n);
  const bool tall = m > n;
  const uint32_t lane = threadIdx.x & 63, j32 = lane & 31, h = lane >> 5;
  const uint32_t wave = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6)));
  char* const x = s_dyn;                                // high part, low part
  char* const s = s_dyn + 2 * sh.side * sh.row_x;
  const uint32_t plane_x = sh.side * sh.row_x, plane_s = sh.side * sh.row_s;
  const uint32_t count = m * n;
  const T* g = update + static_cast<uint64_t>(blockIdx.x) * count;
  T* o = out + static_cast<uint64_t>(blockIdx.x) * count;

  // f(index, value) for this thread's elements of the update, in the order they lie, four vectors loaded at once.
  constexpr uint32_t kVec = 16 / sizeof(T), kThreads = WAVES * 64;
  const auto each = [&](auto&& f) {
    const uint32_t vectors = count / kVec;
    for (uint32_t i0 = threadIdx.x; i0 < vectors; i0 += 4 * kThreads) {
      float v[4][kVec];
#pragma unroll
      for (uint32_t u = 0; u < 4; ++u) {
        if (i0 + u * kThreads < vectors) load_floats<T, kVec>(g + (i0 + u * kThreads) * kVec, v[u]);
      }
#pragma unroll
      for (uint32_t u = 0; u < 4; ++u) {
        if (i0 + u * kThreads < vectors) f((i0 + u * kThreads) * kVec, v[u], kVec);
      }
    }
    const uint32_t left = count % kVec;
    if (threadIdx.x < left) {
      float v[kVec];
      v[0] = static_cast<float>(g[count - left + threadIdx.x]);
      f(count - left + threadIdx.x, v, 1u);
    }
  };
  double sum = 0.0;
  each([&](uint32_t, const float (&v)[kVec], uint32_t valid) {
#pragma unroll
    for (uint32_t e = 0; e < kVec; ++e) {
      if (e < valid) sum = fma(static_cast<double>(v[e]), static_cast<double>(v[e]), sum);
    }
  });
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 64);
  if (lane == 0) s_sum[wave] = sum;
  for (uint32_t i = threadIdx.x; i < sh.bytes / 16; i += WAVES * 64) {
    *reinterpret_cast<f32x4_t*>(s_dyn + i * 16) = f32x4_t{};
  }
  __syncthreads();
  sum = 0.0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) sum += s_sum[w];
  const double factor = start_factor(sum);
  each([&](uint32_t i, const float (&v)[kVec], uint32_t valid) {
    uint32_t r = i / n, q = i - r * n;
#pragma unroll
    for (uint32_t e = 0; e < kVec; ++e) {
      if (e < valid) {
        half_t high, low;
        split2(static_cast<float>(v[e] * factor), high, low);
        char* at = x + (tall ? q * sh.row_x + r * 2 : r * sh.row_x + q * 2);
        *reinterpret_cast<half_t*>(at) = high;
        *reinterpret_cast<half_t*>(at + plane_x) = low;
      }
      if (++q == n) {
        q = 0;
        ++r;
      }
    }
  });
  __syncthreads();

  // 8 k of one row; rows by k.
  const auto rows = [&](const char* base, uint32_t stride, uint32_t row0, uint32_t kk) {
    return *reinterpret_cast<const X8*>(base + (row0 + j32) * stride + (kk * 16 + 8 * h) * 2);
  };
  const auto by_k = [&](const char* base, uint32_t stride, uint32_t col0, uint32_t kk) {
    X4 part[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const uint32_t p = lane & 15, k = kk * 16 + 8 * h + 4 * q + (p >> 2);
      const char* at = base + k * stride + (col0 + 16 * (lane >> 4 & 1) + 4 * (p & 3)) * 2;
      part[q] = __builtin_bit_cast(X4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(at)));
    }
    return __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7);
  };
  // A block of a product over 16-deep slices `from` .. `to` - 1, an even number of them: the small terms by
  // themselves, so that the matrix instructions wait less for one another, and two slices' fragments
  // fetched at a time.
  const auto product_of = [](uint32_t from, uint32_t to, auto&& a_at, auto&& b_at) {
    f32x16_t small{}, large{};
    for (uint32_t kk = from; kk < to; kk += 2) {
      X8 ah[2], al[2], bh[2], bl[2];
#pragma unroll
      for (uint32_t u = 0; u < 2; ++u) {
        ah[u] = a_at(0, kk + u);
        bl[u] = b_at(1, kk + u);
        al[u] = a_at(1, kk + u);
        bh[u] = b_at(0, kk + u);
      }
#pragma unroll
      for (uint32_t u = 0; u < 2; ++u) {
        small = Frag<half_t>::mfma(ah[u], bl[u], small);
        large = Frag<half_t>::mfma(ah[u], bh[u], large);
        small = Frag<half_t>::mfma(al[u], bh[u], small);
      }
    }
    return large + small;
  };

  // Block v of a product, transposed: lane j32 holds a row of what is stored, four neighbouring columns at a
  // time, so that the stores are of 8 bytes (as rows of the block itself they would be of two).
  const auto put = [&](char* base, uint32_t stride, uint32_t plane, uint32_t bi, uint32_t bj, const f32x16_t& v) {
    char* at = base + (bj * 32 + j32) * stride + (bi * 32 + 4 * h) * 2;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      Pack<half_t, 4> high, low;
#pragma unroll
      for (int e = 0; e < 4; ++e) split2(v[4 * q + e], high.v[e], low.v[e]);
      *reinterpret_cast<Pack<half_t, 4>*>(at + q * 16) = high;
      *reinterpret_cast<Pack<half_t, 4>*>(at + q * 16 + plane) = low;
    }
  };

  const uint32_t sb = sh.side / 32, db = sh.depth / 32;
  // Waves to a block of S: a KB of its place each. Adding up their parts takes 1.5 us a step, 32 k less for a wave
  // save 0.15 (32 x 1,100 bf16: 78 us a call with one wave, 58 with five; 64 x 256: 37 with one, 43 with four).
  f32x4_t* const s_part = reinterpret_cast<f32x4_t*>(s);
  const uint32_t most = sb == 1 ? 5 : WAVES / (sb * sb) < 4 ? WAVES / (sb * sb) : 4;
  const uint32_t ways = db - db / (most > 0 ? most : 1) >= 12 ? most : 1;
  // Addresses that follow from the wave's number are computed where they are used: kept over all steps, those
  // of five blocks took 250 registers more than there are.
  const auto fresh = [](uint32_t w) {
    asm volatile("" : "+s"(w));
    return w;
  };
  for (uint32_t step = 0; step < steps; ++step) {
    // S = X X^T. All blocks: the waves that its symmetry would save have nothing else to do. Where there are
    // several waves to a block and k is long, each takes a part of it; the first adds the parts up, four rows
    // at a time, which lie in S's place until then.
    const auto x_rows = [&](uint32_t row0) {
      return [&, row0](uint32_t p, uint32_t kk) { return rows(x + p * plane_x, sh.row_x, row0, kk); };
    };
    if (ways > 1) {
      const uint32_t t = fresh(wave) / ways, way = fresh(wave) % ways;
      const uint32_t bi = t / sb, bj = t % sb, pairs = sh.depth / 32;
      f32x16_t acc{};
      if (t < sb * sb) {
        acc = product_of(pairs * way / ways * 2, pairs * (way + 1) / ways * 2, x_rows(bi * 32), x_rows(bj * 32));
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        f32x4_t part;
#pragma unroll
        for (int e = 0; e < 4; ++e) part[e] = acc[4 * q + e];
        if (t < sb * sb) s_part[wave * 64 + lane] = part;
        __syncthreads();
        if (t < sb * sb && way == 0) {
          for (uint32_t v = 1; v < ways; ++v) part += s_part[(wave + v) * 64 + lane];
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[4 * q + e] = part[e];
        }
        __syncthreads();
      }
      if (t < sb * sb && way == 0) put(s, sh.row_s, plane_s, bi, bj, acc * (1.0f / kScale));
    } else {
#pragma unroll
      for (int u = 0; u < BLOCKS; ++u) {
        const uint32_t t = fresh(wave) + static_cast<uint32_t>(u) * WAVES;
        if (t < sb * sb) {
          const uint32_t bi = t / sb, bj = t % sb;
          const f32x16_t acc = product_of(0, sh.depth / 16, x_rows(bi * 32), x_rows(bj * 32));
          put(s, sh.row_s, plane_s, bi, bj, acc * (1.0f / kScale));
        }
      }
    }
    __syncthreads();
    // P = a + b S + c S S in S's place.
    f32x16_t kept[BLOCKS];
#pragma unroll
    for (int u = 0; u < BLOCKS; ++u) {
      const uint32_t t = fresh(wave) + static_cast<uint32_t>(u) * WAVES;
      if (t < sb * sb) {
        const uint32_t bi = t / sb, bj = t % sb;
        f32x16_t acc = product_of(
            0, sh.side / 16, [&](uint32_t p, uint32_t kk) { return rows(s + p * plane_s, sh.row_s, bi * 32, kk); },
            [&](uint32_t p, uint32_t kk) { return rows(s + p * plane_s, sh.row_s, bj * 32, kk); });
        const char* at = s + (bj * 32 + j32) * sh.row_s + (bi * 32 + 4 * h) * 2;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const Pack<half_t, 4> high = *reinterpret_cast<const Pack<half_t, 4>*>(at + q * 16);
          const Pack<half_t, 4> low = *reinterpret_cast<const Pack<half_t, 4>*>(at + q * 16 + plane_s);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float sv = static_cast<float>(high.v[e]) + static_cast<float>(low.v[e]);
            const bool diagonal = bi == bj && static_cast<uint32_t>(8 * q + e) + 4 * h == j32;
            acc[4 * q + e] = fmaf(b, sv, acc[4 * q + e] * (c / kScale)) + (diagonal ? a * kScale : 0.0f);
          }
        }
        kept[u] = acc;
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < BLOCKS; ++u) {
      const uint32_t t = fresh(wave) + static_cast<uint32_t>(u) * WAVES;
      if (t < sb * sb) put(s, sh.row_s, plane_s, t / sb, t % sb, kept[u]);
    }
    __syncthreads();
    // P X in X's place, computed as its transpose (P is symmetric); the last one is the result.
#pragma unroll
    for (int u = 0; u < BLOCKS; ++u) {
      const uint32_t t = fresh(wave) + static_cast<uint32_t>(u) * WAVES;
      if (t < sb * db) {
        const uint32_t bi = t / sb, bj = t % sb;  // columns of X, rows of P
        kept[u] = product_of(
            0, sh.side / 16, [&](uint32_t p, uint32_t kk) { return by_k(x + p * plane_x, sh.row_x, bi * 32, kk); },
            [&](uint32_t p, uint32_t kk) { return rows(s + p * plane_s, sh.row_s, bj * 32, kk); });
      }
    }
    const bool last = step + 1 == steps;
    if (!last) __syncthreads();
#pragma unroll
    for (int u = 0; u < BLOCKS; ++u) {
      const uint32_t t = fresh(wave) + static_cast<uint32_t>(u) * WAVES;
      if (t < sb * db) {
        const uint32_t bi = t / sb, bj = t % sb;
        if (!last) {
          kept[u] *= 1.0f / kScale;
          put(x, sh.row_x, plane_x, bi, bj, kept[u]);
        } else {
          const uint32_t row = bj * 32 + j32;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const uint32_t col = bi * 32 + static_cast<uint32_t>(8 * (r / 4) + r % 4) + 4 * h;
            if (row < (tall ? n : m) && col < (tall ? m : n)) {
              o[tall ? col * n + row : row * n + col] = static_cast<T>(kept[u][r] * (1.0f / (kScale * kScale)));
            }
          }
        }
      }
    }
    __syncthreads();
  }
  if (steps == 0) {
    for (uint32_t i = threadIdx.x; i < count; i += WAVES * 64) {
      const uint32_t r = i / n, q = i - r * n;
      const char* at = x + (tall ? q * sh.row_x + r * 2 : r * sh.row_x + q * 2);
      o[i] = static_cast<T>((static_cast<float>(*reinterpret_cast<const half_t*>(at)) +
                             static_cast<float>(*reinterpret_cast<const half_t*>(at + plane_x))) /
                            kScale);
    }
  }
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
  if (is_small(m, n)) return l;  // needs nothing
  const auto round = [](size_t b) { return (b + 255) / 256 * 256; };
  l.side = std::min(m, n);
  l.ldx = ceil_div(n, 8) * 8;
  l.lds = ceil_div(l.side, 8) * 8;
  l.plane_x = l.ldx * m;
  l.plane_s = l.lds * l.side;
  const uint32_t b = static_cast<uint32_t>(batch);
  l.gram = gemm_plan(l.side, l.side, std::max(m, n), Kind::kPlane2, b, true);
  l.square = gemm_plan(l.side, l.side, l.side, Kind::kPlane2, b, true);
  l.update = gemm_plan(m, n, l.side, Kind::kPlane2, b, false);
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

/// Whether no step can push a singular value of [0, 1] past 3.5 or the polynomial past 15. On [0, top] both
/// are largest at an end or where their derivative is zero, which for q = s^2 is a quadratic's or a
/// line's zero.
bool bounded(uint32_t steps, double a, double b, double c) {
  double top = 1.0;
  for (uint32_t i = 0; i < steps; ++i) {
    double next = 0.0;
    bool small = true;
    const auto at = [&](double q) {
      if (!(q > 0.0)) q = 0.0;
      if (q > top * top) return;
      const double p = a + b * q + c * q * q;
      small = small && std::fabs(p) <= 15.0;
      next = std::max(next, std::fabs(std::sqrt(q) * p));
    };
    at(0.0);
    at(top * top);
    if (c != 0.0) at(-b / (2.0 * c));
    const double root = 9.0 * b * b - 20.0 * a * c;  // of a + 3 b q + 5 c q^2
    if (c != 0.0 && root >= 0.0) {
      at((-3.0 * b + std::sqrt(root)) / (10.0 * c));
      at((-3.0 * b - std::sqrt(root)) / (10.0 * c));
    } else if (c == 0.0 && b != 0.0) {
      at(-a / (3.0 * b));
    }
    if (!small || !(next <= 3.5)) return false;  // NaN coefficients among them
    if (next <= top) return true;                // stays in [0, top] from here on
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
  return g;
}

template <class T>
void orthogonalize(const T* update, uint64_t batch, uint32_t m, uint32_t n, uint32_t steps, float a, float b, float c,
                   T* out, char* ws, hipStream_t s) {
  if (is_small(m, n)) {
    const SmallShape sh = small_shape(m, n);
    const auto go = [&](auto waves, auto blocks) {
      constexpr int W = decltype(waves)::value;
      const auto kernel = ortho_small_kernel<T, W, decltype(blocks)::value>;
      static const hipError_t allowed = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                            hipFuncAttributeMaxDynamicSharedMemorySize, kSmallLds - 1024);
      QVH_HIP(allowed);
      hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(batch)), dim3(W * 64), sh.bytes, s, update, m, n, steps,
                         a, b, c, out);
    };
    if (small_waves(sh) == 16) {  // side <= depth, so S has no more blocks than X
      go(std::integral_constant<int, 16>{}, std::integral_constant<int, 1>{});
    } else {
      go(std::integral_constant<int, 8>{}, std::integral_constant<int, 5>{});
    }
    QVH_HIP(hipGetLastError());
    return;
  }
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
    hipLaunchKernelGGL((parts_to_result_kernel<T>), dim3(static_cast<unsigned>(std::min<uint64_t>(ceil_div(static_cast<uint64_t>(m) * n, 256), 1u << 20)), nb),
                       dim3(256), 0, s, x[0], l.ldx, l.plane_x, m, n, out);
    QVH_HIP(hipGetLastError());
    return;
  }
  const bool tall = m > n;
  for (uint32_t i = 0; i < steps; ++i) {
    const half_t* cur = x[i & 1];
    half_t* next = x[(i + 1) & 1];
    GemmArgs g1 = product(cur, l.ldx, l.plane_x, cur, l.ldx, l.plane_x, l.side, l.side, std::max(m, n), batch);
    g1.symmetric = 1;
    const PartsEpilogue e1{gram, nullptr, l.lds, l.plane_s, 1.0f / kScale, 0.0f, 0.0f};
    if (tall) {
      launch_gemm<half_t, Kind::kPlane2, true, true>(g1, e1, l.gram, partial, s);
    } else {
      launch_gemm<half_t, Kind::kPlane2, false, false>(g1, e1, l.gram, partial, s);
    }
    GemmArgs g2 = product(gram, l.lds, l.plane_s, gram, l.lds, l.plane_s, l.side, l.side, l.side, batch);
    g2.symmetric = 1;
    const PartsEpilogue e2{poly, gram, l.lds, l.plane_s, c / kScale, a * kScale, b};
    launch_gemm<half_t, Kind::kPlane2, false, false>(g2, e2, l.square, partial, s);
    // P is symmetric: it may be read by rows on either side.
    const GemmArgs g3 = tall ? product(cur, l.ldx, l.plane_x, poly, l.lds, l.plane_s, m, n, l.side, batch)
                             : product(poly, l.lds, l.plane_s, cur, l.ldx, l.plane_x, m, n, l.side, batch);
    const auto third = [&](const auto& e) {
      if (tall) {
        launch_gemm<half_t, Kind::kPlane2, false, false>(g3, e, l.update, partial, s);
      } else {
        launch_gemm<half_t, Kind::kPlane2, false, true>(g3, e, l.update, partial, s);
      }
    };
    if (i + 1 < steps) {
      third(PartsEpilogue{next, nullptr, l.ldx, l.plane_x, 1.0f / kScale, 0.0f, 0.0f});
    } else {
      third(ResultEpilogue<T>{out, n, static_cast<uint64_t>(m) * n, 1.0f / (kScale * kScale)});
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
    const size_t need = ortho_layout(batch, m, n).total;
    QVH_REQUIRE(need == 0 || (d_workspace != nullptr && workspace_bytes >= need), w + ": the workspace is too small");
    QVH_REQUIRE(reinterpret_cast<uintptr_t>(d_workspace) % 16 == 0, w + ": the workspace must be 16-byte aligned");
    const DeviceScope device;
    with_dtype(dtype, [&](auto* t) {
      using T = std::remove_pointer_t<decltype(t)>;
      orthogonalize<T>(static_cast<const T*>(d_update), batch, m, n, steps, a, b, c, static_cast<T*>(d_out),
                       static_cast<char*>(d_workspace), static_cast<hipStream_t>(stream));
    });
  });
}

}  // extern "C"
