// Matrix product of the encoder operators on the matrix unit: C[m][n] = sum_k A(m, k) B(n, k), accumulated in
// fp32, with an epilogue.
//
// Operands. Each is stored either by rows ([row][k], k contiguous) or by k ([k][row], row contiguous): a
// layer's forward pass reads both by rows, its input gradient the weight by k, its weight gradient both by
// k, so no pass ever transposes a matrix in memory. Elements are of 16 bits, or fp32 for the fp32
// instructions. Operands of more than 16 bits may also come as a sum of two or three 16-bit planes; a step then
// holds all of them, and every fragment that was read from LDS enters two or three of the three or six
// products that count.
//
// A work-group takes a BM x BN tile in steps of 64 or 32 k. The steps go from memory straight into LDS
// (16 bytes per lane where the rows are aligned so, 4 otherwise; no registers), the next one or two while the
// present one is multiplied; LDS holds each row's (or each k's) 16-byte pieces permuted so that the
// fragments of the matrix unit are read without bank conflicts, and because such loads fill LDS in lane order
// the permutation is in the addresses that the lanes load from. Nothing is read outside the operands: rows
// and k past the end are clamped to the last one, the results of clamped rows are not stored, and elements past
// the last k are replaced by zeros in registers, in the last step only.
//
// Work-groups go to the XCDs in runs of neighbouring tiles, so that an L2 reads an operand about once: 16,384 x
// 1,024 x 4,096 bf16 fetches 203 MB, of operands of 42 of which every XCD needs the weight's 8.
//
// What bounds it. Large products, by the matrix unit and the clock under load: 8,192^3 bf16 about 1,200 TFLOP/s, its
// instructions busy 63% of the time at 1.7 GHz (the installed library: 1,500). A layer of 16,384 x 1,024 x 4,096 with GELU and the
// kept pre-activation, by its 16 steps' start and the 268 MB that its epilogue writes at the end of every tile:
// 171 us, 800 TFLOP/s, the main loop alone 115. Small products, by the latency of a step (0.4 to 0.7 us) and a
// launch. Tried without gain: five or more steps ahead, loads spread over several slices, prefetches into the L2,
// wave priorities, tiles of 256 x 256 with four waves.
#pragma once

#include "types16.hpp"

namespace qvh {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));

/// What a lane holds of one row of a 32 x 32 block: `kEach` neighbouring k, lanes 32 .. 63 the next ones.
template <class T>
struct Frag;
template <>
struct Frag<half_t> {
  typedef half_t x8 __attribute__((ext_vector_type(8)));
  typedef half_t x4 __attribute__((ext_vector_type(4)));
  typedef x8 type;
  static constexpr int kEach = 8;
  static __device__ __forceinline__ f32x16_t mfma(x8 a, x8 b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Frag<bhalf_t> {
  typedef bhalf_t x8 __attribute__((ext_vector_type(8)));
  typedef bhalf_t x4 __attribute__((ext_vector_type(4)));
  typedef x8 type;
  static constexpr int kEach = 8;
  static __device__ __forceinline__ f32x16_t mfma(x8 a, x8 b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};

template <>
struct Frag<float> {
  typedef f32x4_t type;
  static constexpr int kEach = 4;
  // The instruction takes one k per lane and half: four of them, each with the halves' k of one index.
  static __device__ __forceinline__ f32x16_t mfma(f32x4_t a, f32x4_t b, f32x16_t c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
};

/// One operand: element (row, k) of plane p at base[p * plane + row * ld + k], or [.. k * ld + row] where
/// it is stored by k. Loaded 16 bytes at a time: base and rows 16-byte aligned, the contiguous extent rounded
/// up to 16 bytes readable. Four bytes at a time: base, rows and the extent in whole dwords.
struct GemmOperand {
  const void* base = nullptr;
  uint64_t ld = 0, plane = 0, batch = 0;  // in elements
};

struct GemmArgs {
  GemmOperand a, b;
  uint32_t m = 0, n = 0, k = 0;
  uint32_t tiles_m = 0, tiles_n = 0, splits = 1, batches = 1;
  uint32_t symmetric = 0;  // the product equals its transpose (m = n): tiles above the diagonal are mirrored
  float* partial = nullptr;  // [split][batch][m][n rounded up to 8] when splits > 1
};

/// The upper tail of the normal distribution at a >= 0 for 16-bit results, and *e = exp(-z^2 / 2): e times a polynomial of
/// t = 1 / (1 + 0.316 a), the form of Abramowitz and Stegun's 7.1.26. The coefficients are the minimax fit of the
/// error times max(1, a) (Lawson's iteration): 1.7e-8, and with its fp32 evaluation 7e-8 of GELU, as erff leaves, but 2e-8
/// past a = 3, where an fp16 result is spaced by 5e-7 and less. About a fifth of erff's cost, which would take longer
/// than a short product's matrix instructions.
__device__ __forceinline__ float normal_tail(float a, float z, float* e) {
  const float t = __builtin_amdgcn_rcpf(fmaf(a, 0.316f, 1.0f));
  float p = fmaf(t, -0.134293224f, 0.533036075f);
  p = fmaf(t, p, -0.321486162f);
  p = fmaf(t, p, 0.350168908f);
  p = fmaf(t, p, 0.0659144477f);
  p = fmaf(t, p, 0.00665994266f);
  *e = __builtin_amdgcn_exp2f(z * z * -0.72134752f);
  return p * *e;
}

/// exp(-z), z from -88 on, to its last bits: two to the power z log2(e) is rounded to, times what that leaves out of z.
__device__ __forceinline__ float exp_minus(float z) {
  const float t = z * -1.44269504f, e = __builtin_amdgcn_exp2f(t);
  return fmaf(e, fmaf(t, 1.90465421e-9f, fmaf(t, -0.69314718f, -z)), e);  // ln 2 in two parts
}

/// 1 / (1 + exp(-z)), *other the same of -z. FINE: for fp32 results, to the last bits for every z (0 below -87.4, where it would be
/// less than the smallest normal number). Four instructions more than the other form, 0.8 us of the 92 of 10,000 x 768 x 768 with
/// SiLU; expf and a division would take 4. For 16-bit ones the hardware's exponential of z, whose error of |z| 2^-24 is far
/// below their rounding.
template <bool FINE>
__device__ __forceinline__ float logistic(float z, float* other) {
  const float e = FINE ? exp_minus(__builtin_amdgcn_fmed3f(z, -88.0f, 88.0f)) : __expf(-z);
  const float s = __builtin_amdgcn_rcpf(1.0f + e);
  *other = FINE ? e * s : 1.0f - s;
  return s;
}

/// FINE: for fp32 results.
template <bool FINE>
__device__ __forceinline__ float activate(float z, int act) {
  if (act == QVH_ACT_RELU) return z > 0.0f || z != z ? z : 0.0f;
  if (act == QVH_ACT_GELU) {
    if constexpr (FINE) return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
    // max(z, 0) - |z| tail(|z|), the product of +infinity and 0 kept out.
    const float a = fmaxf(-z, fminf(z, 64.0f));
    float e;
    return fmaf(-a, normal_tail(a, z, &e), fmaxf(z, 0.0f));
  }
  if (act == QVH_ACT_SILU) {
    float other;
    return z * logistic<FINE>(z, &other);
  }
  return z;
}

/// d activate / dz.
template <bool FINE>
__device__ __forceinline__ float activate_slope(float z, int act) {
  if (act == QVH_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
  if (act == QVH_ACT_GELU) {
    if constexpr (FINE) {
      return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) + z * exp_minus(fminf(0.5f * z * z, 120.0f)) * 0.39894228040143268f;
    }
    float e;
    const float tail = normal_tail(fabsf(z), z, &e);
    return fmaf(z * 0.39894228f, e, z > 0.0f ? 1.0f - tail : tail);
  }
  if (act == QVH_ACT_SILU) {
    float other;
    const float s = logistic<FINE>(z, &other);
    return s * (1.0f + z * other);
  }
  return 1.0f;
}

/// Row and eight-element piece of this thread where rows hold per_row pieces and work-groups of 256 threads take
/// them in order. The 64-bit division only where the numbers need it.
struct RowChunk {
  uint64_t row;
  uint32_t chunk;
};
__device__ __forceinline__ RowChunk row_and_chunk(uint32_t block, uint32_t per_row, uint32_t thread) {
  if (block < (1u << 24)) {
    const uint32_t i = block * 256 + thread, r = i / per_row;
    return {r, i - r * per_row};
  }
  const uint64_t i = static_cast<uint64_t>(block) * 256 + thread, r = i / per_row;
  return {r, static_cast<uint32_t>(i - r * per_row)};
}

/// Eight values as vector accesses, or those of them that the row still has one by one. STREAM: past the caches.
template <bool STREAM = false, class T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8], uint32_t left) {
  if (left >= 8) {
    if constexpr (sizeof(T) == 2) {
      store_floats<T, 8, STREAM>(p, v);
    } else {
      const float lo[4] = {v[0], v[1], v[2], v[3]}, hi[4] = {v[4], v[5], v[6], v[7]};
      store_floats<T, 4, STREAM>(p, lo);
      store_floats<T, 4, STREAM>(p + 4, hi);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (static_cast<uint32_t>(i) < left) p[i] = static_cast<T>(v[i]);
    }
  }
}

template <bool STREAM = false, class T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8], uint32_t left) {
  if (left >= 8) {
    if constexpr (sizeof(T) == 2) {
      load_floats<T, 8, STREAM>(p, v);
    } else {
      float lo[4], hi[4];
      load_floats<T, 4, STREAM>(p, lo);
      load_floats<T, 4, STREAM>(p + 4, hi);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = lo[i];
        v[4 + i] = hi[i];
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = static_cast<uint32_t>(i) < left ? static_cast<float>(p[i]) : 0.0f;
  }
}

/// Column sums of work-groups that share the rows, [part][cols rounded up to 8], to be added up.
struct ColumnSums {
  const float* parts = nullptr;
  uint32_t count = 0, cols = 0;
};

__device__ __forceinline__ float sum8(const float (&t)[8]) {
  return ((t[0] + t[1]) + (t[2] + t[3])) + ((t[4] + t[5]) + (t[6] + t[7]));
}

/// 64 columns' parts: four waves take contiguous shares of them.
template <class T>
__device__ __forceinline__ void add_columns(const ColumnSums& a, uint32_t block, T* __restrict__ out) {
  __shared__ float s_sum[4][64];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, ld = (a.cols + 7) / 8 * 8;
  const uint32_t c = block * 64 + lane, share = (a.count + 3) / 4;
  const uint32_t p0 = wave * share < a.count ? wave * share : a.count, p1 = p0 + share < a.count ? p0 + share : a.count;
  float t[8] = {};  // every eighth part each: eight loads under way, and short sums
  if (c < a.cols) {
    for (uint32_t p = p0; p < p1; p += 8) {
#pragma unroll
      for (uint32_t u = 0; u < 8; ++u) t[u] += p + u < p1 ? a.parts[static_cast<uint64_t>(p + u) * ld + c] : 0.0f;
    }
  }
  s_sum[wave][lane] = sum8(t);
  __syncthreads();
  if (wave == 0 && c < a.cols) {
    out[c] = static_cast<T>(((s_sum[0][lane] + s_sum[1][lane]) + s_sum[2][lane]) + s_sum[3][lane]);
  }
}

/// y = act(acc + bias) + residual, the sum in front of the activation kept where it is asked for.
template <class T>
struct LinearEpilogue {
  const T* bias = nullptr;
  const T* residual = nullptr;
  T* out = nullptr;
  T* keep = nullptr;
  uint64_t ld_residual = 0, ld_out = 0, ld_keep = 0;
  int act = QVH_ACT_NONE;
  // Column sums that the launch which joins a product's splits adds up besides, and where they go.
  ColumnSums columns;
  T* column_out = nullptr;

  /// The same for one element.
  __device__ __forceinline__ void one(uint32_t m, uint32_t n, float v) const {
    if (bias) v += static_cast<float>(bias[n]);
    if (keep) keep[m * ld_keep + n] = static_cast<T>(v);
    v = activate<sizeof(T) == 4>(v, act);
    if (residual) v += static_cast<float>(residual[m * ld_residual + n]);
    out[m * ld_out + n] = static_cast<T>(v);
  }

  __device__ __forceinline__ void operator()(uint32_t, uint32_t m, uint32_t n, uint32_t left, float (&v)[8]) const {
    apply<false>(m, n, left, v);
  }

  template <bool STREAM>
  __device__ __forceinline__ void apply(uint32_t m, uint32_t n, uint32_t left, float (&v)[8]) const {
    if (bias) {
      float b[8];
      load8(bias + n, b, left);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += b[i];
    }
    if (keep) store8<STREAM>(keep + m * ld_keep + n, v, left);
    if (act == QVH_ACT_RELU) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = activate<sizeof(T) == 4>(v[i], QVH_ACT_RELU);
    } else if (act == QVH_ACT_GELU) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = activate<sizeof(T) == 4>(v[i], QVH_ACT_GELU);
    } else if (act == QVH_ACT_SILU) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = activate<sizeof(T) == 4>(v[i], QVH_ACT_SILU);
    }
    if (residual) {
      float r[8];
      load8(residual + m * ld_residual + n, r, left);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += r[i];
    }
    store8<STREAM>(out + m * ld_out + n, v, left);
  }
};

/// The same for results too large for the L2s.
template <class T>
struct StreamedEpilogue {
  LinearEpilogue<T> of;
  __device__ __forceinline__ void operator()(uint32_t, uint32_t m, uint32_t n, uint32_t left, float (&v)[8]) const {
    of.template apply<true>(m, n, left, v);
  }
};

/// The partial sums of one split of k.
struct PartialEpilogue {
  float* out;
  uint64_t ld, batch;
  __device__ __forceinline__ void operator()(uint32_t z, uint32_t m, uint32_t n, uint32_t, float (&v)[8]) const {
    store8(out + z * batch + m * ld + n, v, 8);
  }
};

// ---- the kernel -------------------------------------------------------------------------------

/// The 16-byte pieces of one operand's R x D step: addresses for the loads into LDS (WIDE bytes per lane), and
/// fragments.
template <class T, bool BY_K, int R, int D, int WAVES, int WIDE>
struct Stage {
  static constexpr int kEach = Frag<T>::kEach, kElem = sizeof(T);
  static constexpr int kBytes = R * D * kElem;
  static constexpr int kLoads = kBytes / (64 * WIDE) / WAVES;
  static constexpr int kLine = (BY_K ? R : D) * kElem;  // bytes per line: a k, or a row
  static_assert(BY_K || kLine == 64 || kLine == 128, "a row is 64 or 128 bytes in LDS");
  static_assert(WIDE == 16 || WIDE == 4, "bytes that a lane loads");
  static_assert(kLoads >= 1 && kBytes % (64 * WIDE * WAVES) == 0, "every wave makes whole loads");

  /// Piece c of a line lies at c ^ flip(line). LDS serves 256 bytes at a time, sixteen pieces: by rows, those of
  /// sixteen neighbouring rows at one k fall on different banks (two rows, or four, share 256 bytes), by k
  /// those of the k that one read takes.
  static __device__ __forceinline__ uint32_t flip(uint32_t line) {
    if constexpr (BY_K) return kElem == 4 ? (line >> 2 & 1) * 8 : (line & (R / 32 - 1)) * 4;
    return kLine == 128 ? line >> 1 & 7 : line >> 2 & 3;
  }

  /// Byte offset (from the tile's first row and the step's first k) of what this lane loads in load i; the
  /// lanes fill LDS in order. `rows` and `depth`: how many of each there are from the tile's start on.
  static __device__ __forceinline__ uint32_t offset(int i, int wave, int lane, uint32_t ld, uint32_t rows, uint32_t depth) {
    const uint32_t at = static_cast<uint32_t>(((i * WAVES + wave) * 64 + lane) * WIDE);
    uint32_t line = at / kLine;
    const uint32_t lines = BY_K ? depth : rows, extent = (BY_K ? rows : depth) * kElem;
    uint32_t byte = ((at % kLine / 16) ^ flip(line)) * 16 + at % 16;
    line = line < lines ? line : lines - 1;
    const uint32_t last = (extent + WIDE - 1) / WIDE * WIDE - WIDE;  // rows that end inside it are padded to whole ones
    byte = byte < last ? byte : last;
    return line * ld * kElem + byte;
  }

  /// Fragment of rows row0 .. row0 + 31 (a multiple of 32) and slice kk of 2 kEach k.
  static __device__ __forceinline__ typename Frag<T>::type fragment(const char* lds, int row0, int kk, int lane) {
    if constexpr (BY_K && kElem == 4) {
      const int k = kk * 8 + 4 * (lane >> 5), row = row0 + (lane & 31);
      const char* at = lds + k * kLine + ((static_cast<uint32_t>(row / 4) ^ flip(static_cast<uint32_t>(k))) * 16 + row % 4 * 4);
      f32x4_t f;
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = *reinterpret_cast<const float*>(at + e * kLine);
      return f;
    } else if constexpr (BY_K) {
      typedef typename Frag<T>::x4 x4;
      x4 part[2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int p = lane & 15, j = p >> 2;
        const int k = kk * 16 + 8 * (lane >> 5) + 4 * q + j;
        const uint32_t chunk = static_cast<uint32_t>(row0 / 8 + 2 * (lane >> 4 & 1) + (p >> 1 & 1));
        const char* at = lds + k * kLine + ((chunk ^ flip(static_cast<uint32_t>(4 * q + j))) * 16 + (p & 1) * 8);
        const s16x4_t v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4_t*)(at));
        part[q] = __builtin_bit_cast(x4, v);
      }
      return __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      const int row = row0 + (lane & 31);
      return *reinterpret_cast<const typename Frag<T>::type*>(
          lds + row * kLine + (((kk * 2 + (lane >> 5)) ^ flip(static_cast<uint32_t>(lane & 31))) * 16));
    }
  }
};

/// 64 lanes x WIDE bytes from rsrc + offset into LDS at lds (wave-uniform), in lane order. Nothing waits for it
/// but s_waitcnt vmcnt. The instructions in front keep the distances that the hardware asks for between a
/// lane read or m0 and the load (the compiler does not look into the block).
template <int WIDE>
__device__ __forceinline__ void load_to_lds(uint32_t lds, uint32_t offset, u32x4_t rsrc) {
  if constexpr (WIDE == 16) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :
                 : "s"(lds), "v"(offset), "s"(rsrc)
                 : "memory");
  } else {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dword %1, %2, 0 offen lds"
                 :
                 : "s"(lds), "v"(offset), "s"(rsrc)
                 : "memory");
  }
}

__device__ __forceinline__ u32x4_t buffer_resource(const void* base) {
  const uint64_t p = reinterpret_cast<uint64_t>(base);
  u32x4_t r;
  r[0] = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(p)));
  r[1] = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(p >> 32))) & 0xFFFFu;
  r[2] = 0xFFFFFFFFu;
  r[3] = 0x00027000u;
  return r;
}

/// Elements of a fragment at or past `depth` (k counted from the fragment's step) become zero.
template <int EACH, class F>
__device__ __forceinline__ F clip(F f, int kk, int lane, uint32_t depth) {
  const int first = (kk * 2 + (lane >> 5)) * EACH;
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    if (static_cast<uint32_t>(first + e) >= depth) f[e] = 0;
  }
  return f;
}

/// Tile of a work-group, its waves, the depth of a step, the steps that LDS holds, the operands' planes, and the
/// bytes that a lane loads at a time.
template <int BM_, int BN_, int WM_, int WN_, int D_, int STAGES_, int PLANES_, int WIDE_ = 16>
struct Tile {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, D = D_, STAGES = STAGES_, PLANES = PLANES_, WIDE = WIDE_;
};

/// The pairs of planes whose products count, the smallest first. Two planes: all but low x low; three: those
/// of at least 2^-16 of the product.
template <int PLANES>
struct Pairs;
template <>
struct Pairs<1> {
  static constexpr int kCount = 1, kA[1] = {0}, kB[1] = {0};
};
template <>
struct Pairs<2> {
  static constexpr int kCount = 3, kA[3] = {1, 0, 0}, kB[3] = {0, 1, 0};
};
template <>
struct Pairs<3> {
  static constexpr int kCount = 6, kA[6] = {2, 0, 1, 1, 0, 0}, kB[6] = {0, 2, 1, 0, 1, 0};
};

/// Eight elements of plane p of an operand for this lane's row and its half of sixteen k: what Stage::fragment gives.
template <bool BY_K>
__device__ __forceinline__ Frag<bhalf_t>::x8 plane_fragment(const GemmOperand& o, uint64_t batch, int p, uint32_t row, uint32_t k, uint32_t depth) {
  const bhalf_t* base = static_cast<const bhalf_t*>(o.base) + batch * o.batch + p * o.plane;
  Frag<bhalf_t>::x8 f{};
  if constexpr (BY_K) {
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) {
      if (k + e < depth) f[e] = base[(k + e) * o.ld + row];
    }
  } else {  // rows are whole 16 bytes, with zeros behind the last element
    if (k < depth) f = *reinterpret_cast<const Frag<bhalf_t>::x8*>(base + row * o.ld + k);
  }
  return f;
}

/// A 32 x 32 block of a product of three planes, where it is NaN. An infinity meets the zeros and the opposite signs of
/// the other operand's lower planes and turns into NaN. What it should be follows from the products with an infinity or
/// NaN alone, whatever the finite ones: so from a product of classes, 1 for a finite number with its sign, 0 for zero,
/// infinities and NaN themselves. Where that is finite, finite products were too large, and their parts overflowed
/// both ways: the six products again of numbers scaled by 2^-80. A layer of 4,096 x 1,024 x 1,024 with an infinity in each
/// row: 142 us for 66 (11,800 when every element was added up by itself).
template <bool AK, bool BK>
__device__ __forceinline__ void repair_block(const GemmArgs& g, uint64_t batch, uint32_t row, uint32_t col, uint32_t begin, uint32_t end,
                                             int lane, f32x16_t& acc) {
  using x8 = Frag<bhalf_t>::x8;
  typedef uint16_t bits_t __attribute__((ext_vector_type(8)));
  row = row + (lane & 31) < g.m ? row + (lane & 31) : g.m - 1;
  col = col + (lane & 31) < g.n ? col + (lane & 31) : g.n - 1;
  const auto class_of = [](x8 f) {
    bits_t b = __builtin_bit_cast(bits_t, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint16_t size = b[e] & 0x7FFF;
      b[e] = size >= 0x7F80 || size == 0 ? b[e] : (b[e] & 0x8000) | 0x3F80;
    }
    return __builtin_bit_cast(x8, b);
  };
  f32x16_t kind{};
#pragma unroll 1
  for (uint32_t k = begin + 8 * (lane >> 5); k - 8 * (lane >> 5) < end; k += 16) {
    kind = Frag<bhalf_t>::mfma(class_of(plane_fragment<AK>(g.a, batch, 0, row, k, g.k)),
                               class_of(plane_fragment<BK>(g.b, batch, 0, col, k, g.k)), kind);
  }
  bool open = false;
#pragma unroll
  for (int r = 0; r < 16; ++r) open = open || (acc[r] != acc[r] && fabsf(kind[r]) < __builtin_huge_valf());
  f32x16_t scaled{};
  if (__builtin_amdgcn_ballot_w64(open) != 0) {
    using P = Pairs<3>;
#pragma unroll 1
    for (uint32_t k = begin + 8 * (lane >> 5); k - 8 * (lane >> 5) < end; k += 16) {
      x8 a[3], b[3];
#pragma unroll
      for (int p = 0; p < 3; ++p) {
        a[p] = plane_fragment<AK>(g.a, batch, p, row, k, g.k);
        b[p] = plane_fragment<BK>(g.b, batch, p, col, k, g.k);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          a[p][e] = static_cast<bhalf_t>(static_cast<float>(a[p][e]) * 0x1p-80f);
          b[p][e] = static_cast<bhalf_t>(static_cast<float>(b[p][e]) * 0x1p-80f);
        }
      }
#pragma unroll
      for (int q = 0; q < P::kCount; ++q) scaled = Frag<bhalf_t>::mfma(a[P::kA[q]], b[P::kB[q]], scaled);
    }
  }
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const float sum = fabsf(kind[r]) < __builtin_huge_valf() ? scaled[r] * 0x1p80f * 0x1p80f : kind[r];
    acc[r] = acc[r] != acc[r] ? sum : acc[r];
  }
}

/// Block t of the lower triangle, row by row.
__device__ __forceinline__ void lower_block(uint32_t t, uint32_t& bi, uint32_t& bj) {
  bi = static_cast<uint32_t>((sqrtf(8.0f * static_cast<float>(t) + 1.0f) - 1.0f) * 0.5f);
  while (bi * (bi + 1) / 2 > t) --bi;
  while ((bi + 1) * (bi + 2) / 2 <= t) ++bi;
  bj = t - bi * (bi + 1) / 2;
}

template <class T, bool AK, bool BK, class Shape, class Epi>
__global__ void __launch_bounds__(Shape::WM* Shape::WN * 64, Shape::BM* Shape::BN / (Shape::WM * Shape::WN) > 128 * 64 ? 1 : 2)
    gemm_kernel(GemmArgs g, Epi epi) {
  constexpr int BM = Shape::BM, BN = Shape::BN, WM = Shape::WM, WN = Shape::WN, kStep = Shape::D, kStages = Shape::STAGES;
  constexpr int kPlanes = Shape::PLANES;
  using P = Pairs<kPlanes>;
  constexpr int kWaves = WM * WN;
  using SA = Stage<T, AK, BM, kStep, kWaves, Shape::WIDE>;
  using SB = Stage<T, BK, BN, kStep, kWaves, Shape::WIDE>;
  constexpr int kStageBytes = (SA::kBytes + SB::kBytes) * kPlanes;
  constexpr int TM = BM / WM / 32, TN = BN / WN / 32;  // 32 x 32 blocks per wave
  constexpr int kSlabLd = BN / WN + 8;
  constexpr int kSlabBytes = 32 * kSlabLd * 4 * kWaves;
  constexpr int kLds = kStages * kStageBytes > kSlabBytes ? kStages * kStageBytes : kSlabBytes;
  __shared__ __attribute__((aligned(1024))) char s_mem[kLds];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;

  // Work-groups go round the XCDs in order of their number; each XCD takes a contiguous run of tiles,
  // walked in bands of eight tile rows, so that its L2 serves the rows and columns they share.
  const uint32_t per = g.symmetric ? g.tiles_m * (g.tiles_m + 1) / 2 : g.tiles_m * g.tiles_n;
  const uint32_t total = per * g.splits;
  uint32_t id = blockIdx.x;
  {
    const uint32_t x = id % 8, q = total / 8, r = total % 8;
    id = (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + id / 8;
  }
  const uint32_t split = id / per;
  const uint32_t tile = id % per;
  uint32_t tm, tn;
  if (g.symmetric) {
    lower_block(tile, tm, tn);
  } else {
    const uint32_t band = 8 * g.tiles_n, b0 = tile / band * 8;
    const uint32_t high = g.tiles_m - b0 < 8 ? g.tiles_m - b0 : 8;
    tm = b0 + tile % band % high;
    tn = tile % band / high;
  }
  const uint32_t z = blockIdx.y;

  const uint32_t row0 = tm * BM, col0 = tn * BN;
  const uint32_t rows = g.m - row0, cols = g.n - col0;
  const uint32_t whole = g.k / kStep, rest = g.k % kStep;  // the last step may be a shorter one
  const uint32_t steps = whole + (rest ? 1 : 0);
  const uint32_t first = static_cast<uint32_t>(static_cast<uint64_t>(steps) * split / g.splits);
  const uint32_t end = static_cast<uint32_t>(static_cast<uint64_t>(steps) * (split + 1) / g.splits);
  const uint32_t whole_end = end < whole ? end : whole;

  const T* const a0 = static_cast<const T*>(g.a.base) + z * g.a.batch + (AK ? uint64_t{row0} : row0 * g.a.ld);
  const T* const b0p = static_cast<const T*>(g.b.base) + z * g.b.batch + (BK ? uint64_t{col0} : col0 * g.b.ld);
  const uint32_t lda = static_cast<uint32_t>(g.a.ld), ldb = static_cast<uint32_t>(g.b.ld);
  uint32_t oa[SA::kLoads], ob[SB::kLoads];
#pragma unroll
  for (int i = 0; i < SA::kLoads; ++i) oa[i] = SA::offset(i, wave, lane, lda, rows, kStep);
#pragma unroll
  for (int i = 0; i < SB::kLoads; ++i) ob[i] = SB::offset(i, wave, lane, ldb, cols, kStep);
  const uint32_t lds0 = static_cast<uint32_t>(
      reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)(s_mem)));

  // Loads the step that begins at pa and pb into place `buf`, at the lanes' offsets.
  constexpr int kPieces = (SA::kLoads + SB::kLoads) * kPlanes;
  struct Sources {
    u32x4_t a[kPlanes], b[kPlanes];
  };
  const auto sources = [&](uint32_t step) {
    const uint64_t k0 = static_cast<uint64_t>(step) * kStep;
    const T* pa = a0 + (AK ? k0 * g.a.ld : k0);
    const T* pb = b0p + (BK ? k0 * g.b.ld : k0);
    Sources s;
#pragma unroll
    for (int p = 0; p < kPlanes; ++p) {
      s.a[p] = buffer_resource(pa + p * g.a.plane);
      s.b[p] = buffer_resource(pb + p * g.b.plane);
    }
    return s;
  };
  // In LDS: the planes of a, then those of b.
  const auto load_piece = [&](int i, const Sources& s, int buf, const uint32_t(&at_a)[SA::kLoads],
                              const uint32_t(&at_b)[SB::kLoads]) {
    const uint32_t to = lds0 + static_cast<uint32_t>(buf) * kStageBytes + (i * kWaves + wave) * (64 * Shape::WIDE);
    constexpr int kOfA = SA::kLoads * kPlanes;
    if (i < kOfA) {
      load_to_lds<Shape::WIDE>(to, at_a[i % SA::kLoads], s.a[i / SA::kLoads]);
    } else {
      load_to_lds<Shape::WIDE>(to, at_b[(i - kOfA) % SB::kLoads], s.b[(i - kOfA) / SB::kLoads]);
    }
  };
  const auto load = [&](const Sources& s, int buf, const uint32_t(&at_a)[SA::kLoads], const uint32_t(&at_b)[SB::kLoads]) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) load_piece(i, s, buf, at_a, at_b);
  };

  f32x16_t acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i) {
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x16_t{};
  }

  const int ra0 = wm * (BM / WM), rb0 = wn * (BN / WN);
  constexpr int kDepth = 2 * Frag<T>::kEach;  // k of a slice
  struct Fragments {
    typename Frag<T>::type a[kPlanes][TM], b[kPlanes][TN];
  };
  const auto fetch = [&](Fragments& f, int buf, int kk) {
    const char* la = s_mem + buf * kStageBytes;
#pragma unroll
    for (int p = 0; p < kPlanes; ++p) {
#pragma unroll
      for (int i = 0; i < TM; ++i) f.a[p][i] = SA::fragment(la + p * SA::kBytes, ra0 + 32 * i, kk, lane);
    }
#pragma unroll
    for (int p = 0; p < kPlanes; ++p) {
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        f.b[p][j] = SB::fragment(la + kPlanes * SA::kBytes + p * SB::kBytes, rb0 + 32 * j, kk, lane);
      }
    }
  };
  // Matrix instruction x of a slice.
  constexpr int kOps = TM * TN * P::kCount;
  const auto step_of = [&](const Fragments& f, int x) {
    const int i = x / TN % TM, j = x % TN, q = x / (TM * TN);
    acc[i][j] = Frag<T>::mfma(f.a[P::kA[q]][i], f.b[P::kB[q]][j], acc[i][j]);
  };
  const auto multiply = [&](const Fragments& f) {
#pragma unroll
    for (int x = 0; x < kOps; ++x) step_of(f, x);
  };

  // Fragments are fetched one slice ahead of their matrix instructions. The step's last slice is
  // in registers before its instructions start: from then on the step's place in LDS is free for the step
  // kStages on, and the next step's first slice is fetched while the last one is multiplied.
  if (first < whole_end) {
    constexpr int kSlices = kStep / kDepth;
    Fragments f[2];
#pragma unroll
    for (int i = 0; i < kStages; ++i) {
      if (first + i < whole_end) load(sources(first + i), i, oa, ob);
    }
    // All but the first step's loads may still be under way.
    if (first + kStages <= whole_end) {
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"((kStages - 1) * kPieces) : "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");  // no fetch moves up across the barrier
    fetch(f[0], 0, 0);
    int buf = 0;
    for (uint32_t s = first; s < whole_end; ++s) {
#pragma unroll
      for (int kk = 0; kk + 1 < kSlices; ++kk) {
        fetch(f[(kk + 1) & 1], buf, kk + 1);
        __builtin_amdgcn_sched_barrier(0);
        multiply(f[kk & 1]);
        __builtin_amdgcn_sched_barrier(0);
      }
      // This wave's fetches are done, and its loads of the next step have arrived.
      if (s + kStages <= whole_end) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((kStages - 2) * kPieces) : "memory");
      } else {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      }
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      const bool more = s + kStages < whole_end;
      const Sources src = sources(s + kStages);
      const int free_buf = buf;
      buf = buf + 1 == kStages ? 0 : buf + 1;
      if (s + 1 < whole_end) fetch(f[0], buf, 0);
      __builtin_amdgcn_sched_barrier(0);
      // The loads go out between the matrix instructions, which cover their issue.
#pragma unroll
      for (int x = 0; x < kOps; ++x) {
        step_of(f[(kSlices - 1) & 1], x);
        __builtin_amdgcn_sched_barrier(0);
        if (more) {
#pragma unroll
          for (int i = x * kPieces / kOps; i < (x + 1) * kPieces / kOps; ++i) load_piece(i, src, free_buf, oa, ob);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  if (rest && end == steps && first < end) {
    uint32_t ta[SA::kLoads], tb[SB::kLoads];
#pragma unroll
    for (int i = 0; i < SA::kLoads; ++i) ta[i] = SA::offset(i, wave, lane, lda, rows, rest);
#pragma unroll
    for (int i = 0; i < SB::kLoads; ++i) tb[i] = SB::offset(i, wave, lane, ldb, cols, rest);
    load(sources(whole), 0, ta, tb);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll 1
    for (int kk = 0; static_cast<uint32_t>(kk * kDepth) < rest; ++kk) {
      Fragments f;
      fetch(f, 0, kk);
#pragma unroll
      for (int p = 0; p < kPlanes; ++p) {
#pragma unroll
        for (int i = 0; i < TM; ++i) f.a[p][i] = clip<Frag<T>::kEach>(f.a[p][i], kk, lane, rest);
#pragma unroll
        for (int j = 0; j < TN; ++j) f.b[p][j] = clip<Frag<T>::kEach>(f.b[p][j], kk, lane, rest);
      }
      multiply(f);
    }
  }
  if constexpr (kPlanes == 3) {
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        float all = 0.0f;  // NaN for an infinity too
#pragma unroll
        for (int r = 0; r < 16; ++r) all = fmaf(acc[i][j][r], 0.0f, all);
        if (__builtin_amdgcn_ballot_w64(all != all) != 0) {
          const uint32_t last = end * kStep < g.k ? end * kStep : g.k;
          repair_block<AK, BK>(g, z, row0 + static_cast<uint32_t>(ra0 + 32 * i), col0 + static_cast<uint32_t>(rb0 + 32 * j),
                               first * kStep, last, lane, acc[i][j]);
        }
      }
    }
  }
  __syncthreads();

  // The accumulators of 32 rows at a time through the wave's own piece of LDS, so that a lane gets eight
  // neighbouring columns of one row: whole lines for the residual and the stores.
  float* slab = reinterpret_cast<float*>(s_mem) + wave * (32 * kSlabLd);
  constexpr int kPerRow = BN / WN / 8;      // lanes per row
  constexpr int kRowsAtOnce = 64 / kPerRow;
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int j = 0; j < TN; ++j) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        slab[(8 * (r / 4) + 4 * (lane >> 5) + r % 4) * kSlabLd + 32 * j + (lane & 31)] = acc[i][j][r];
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const uint32_t n = col0 + static_cast<uint32_t>(rb0 + lane % kPerRow * 8);
#pragma unroll
    for (int q = 0; q < 32 / kRowsAtOnce; ++q) {
      const int r = q * kRowsAtOnce + lane / kPerRow;
      const uint32_t m = row0 + static_cast<uint32_t>(ra0 + 32 * i + r);
      const f32x4_t lo = *reinterpret_cast<const f32x4_t*>(slab + r * kSlabLd + lane % kPerRow * 8);
      const f32x4_t hi = *reinterpret_cast<const f32x4_t*>(slab + r * kSlabLd + lane % kPerRow * 8 + 4);
      float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      if (m < g.m && n < g.n) epi(g.splits > 1 ? split * g.batches + z : z, m, n, g.n - n, v);
    }
    if (g.symmetric && g.splits == 1 && tm != tn) {
      // The same values at their mirrored places: a lane takes eight rows of one column.
#pragma unroll
      for (int q = 0; q < BN / WN / 16; ++q) {
        const int c = q * 16 + lane / 4, r = lane % 4 * 8;
        const uint32_t mm = col0 + static_cast<uint32_t>(rb0 + c), nn = row0 + static_cast<uint32_t>(ra0 + 32 * i + r);
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = slab[(r + e) * kSlabLd + c];
        if (mm < g.n && nn < g.m) epi(z, mm, nn, g.m - nn, v);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

/// Eight elements' partial sums, the splits in order.
__device__ __forceinline__ void add_splits(const float* p, uint32_t splits, uint64_t step, float (&v)[8]) {
  uint32_t s = 0;
  for (; s + 4 <= splits; s += 4, p += 4 * step) {  // four loads under way at a time
    float x[4][8];
#pragma unroll
    for (int u = 0; u < 4; ++u) load8(p + u * step, x[u], 8);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += x[u][e];
    }
  }
  for (; s < splits; ++s, p += step) {
    float x[8];
    load8(p, x, 8);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += x[e];
  }
}

template <class Epi>
struct HasColumns {
  static constexpr bool value = false;
};
template <class T>
struct HasColumns<LinearEpilogue<T>> {
  static constexpr bool value = true;
};

/// Whether products with this epilogue may be symmetric ones.
template <class Epi, class = void>
struct MaySymmetric : std::false_type {};
template <class Epi>
struct MaySymmetric<Epi, std::void_t<decltype(Epi::kSymmetric)>> : std::true_type {};

/// Adds the splits' partial sums and runs the epilogue. Four splits of 4,096 x 1,024: 67 MB from the last-level
/// cache and 8 out in 13 us. Work-groups from `blocks` on add column sums.
template <class Epi>
__global__ void __launch_bounds__(256) gemm_join_kernel(GemmArgs g, Epi epi, uint32_t blocks) {
  if constexpr (HasColumns<Epi>::value) {
    if (blockIdx.x >= blocks) return add_columns(epi.columns, blockIdx.x - blocks, epi.column_out);
  }
  const uint32_t ld = (g.n + 7) / 8 * 8;
  const auto [m, chunk] = row_and_chunk(blockIdx.x, ld / 8, threadIdx.x);
  if (m >= g.m) return;
  const uint32_t n = chunk * 8;
  const uint64_t batch = static_cast<uint64_t>(g.m) * ld;
  float v[8] = {};
  add_splits(g.partial + blockIdx.y * batch + m * ld + n, g.splits, batch * g.batches, v);
  epi(blockIdx.y, static_cast<uint32_t>(m), n, g.n - n, v);
}

/// The same for a symmetric product (1,024 x 1,024 in three splits 5 us), of which only the lower tiles have
/// sums: work-groups of 128 threads per 32 x 32 block of the lower triangle, which go through LDS to their
/// mirrored places.
template <class Epi>
__global__ void __launch_bounds__(128) gemm_join_symmetric_kernel(GemmArgs g, Epi epi) {
  __shared__ float s_block[32][33];
  uint32_t bi, bj;
  lower_block(blockIdx.x, bi, bj);
  const uint32_t ld = (g.n + 7) / 8 * 8;
  const uint64_t batch = static_cast<uint64_t>(g.m) * ld;
  const uint32_t r = threadIdx.x / 4, c = threadIdx.x % 4 * 8;
  const uint32_t m = bi * 32 + r, n = bj * 32 + c;
  float v[8] = {};
  if (m < g.m && n < g.n) {
    add_splits(g.partial + blockIdx.y * batch + m * static_cast<uint64_t>(ld) + n, g.splits, batch * g.batches, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) s_block[r][c + e] = v[e];
    epi(blockIdx.y, m, n, g.n - n, v);
  }
  if (bi == bj) return;
  __syncthreads();
  const uint32_t mm = bj * 32 + r, nn = bi * 32 + c;
  if (mm < g.n && nn < g.m) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = s_block[c + e][r];
    epi(blockIdx.y, mm, nn, g.m - nn, v);
  }
}

// ---- launching --------------------------------------------------------------------------------

/// Tile shape and number of splits for a product; the same for the workspace's size and for the launch.
struct GemmPlan {
  int tile = 0;  // which of the kind's shapes; -1: none whose tiles go into one launch
  uint32_t splits = 1;
  size_t partial_bytes = 0;
  double us = 0.0;  // the estimate that chose them
};

enum class Kind : int;

/// `symmetric`: m = n, and only the tiles on and below the diagonal are computed.
GemmPlan gemm_plan(uint64_t m, uint64_t n, uint64_t k, Kind kind, uint32_t batches, bool symmetric);

/// SPLIT: whether the plan may split k.
template <class T, bool AK, bool BK, class Shape, bool SPLIT = true, class Epi>
void launch_tile(GemmArgs g, const Epi& epi, hipStream_t s) {
  g.tiles_m = static_cast<uint32_t>(ceil_div(g.m, Shape::BM));
  g.tiles_n = static_cast<uint32_t>(ceil_div(g.n, Shape::BN));
  const uint64_t tiles = g.symmetric ? static_cast<uint64_t>(g.tiles_m) * (g.tiles_m + 1) / 2
                                     : static_cast<uint64_t>(g.tiles_m) * g.tiles_n;
  const dim3 grid(static_cast<unsigned>(tiles * g.splits), g.batches);  // gemm_plan: fits a launch
  if constexpr (SPLIT) {
    if (g.splits > 1) {
      const uint64_t ld = ceil_div(g.n, 8) * 8;
      const PartialEpilogue pe{g.partial, ld, ld * g.m};
      hipLaunchKernelGGL((gemm_kernel<T, AK, BK, Shape, PartialEpilogue>), grid, dim3(Shape::WM * Shape::WN * 64), 0, s, g, pe);
      QVH_HIP(hipGetLastError());
      if constexpr (MaySymmetric<Epi>::value) {
        if (g.symmetric) {
          const uint32_t side = static_cast<uint32_t>(ceil_div(g.m, 32));
          hipLaunchKernelGGL((gemm_join_symmetric_kernel<Epi>), dim3(side * (side + 1) / 2, g.batches), dim3(128), 0, s, g, epi);
          QVH_HIP(hipGetLastError());
          return;
        }
      }
      const uint32_t join = static_cast<uint32_t>(ceil_div(ld / 8 * g.m, 256));
      uint32_t more = 0;
      if constexpr (HasColumns<Epi>::value) more = static_cast<uint32_t>(ceil_div(epi.columns.cols, 64));
      hipLaunchKernelGGL((gemm_join_kernel<Epi>), dim3(join + more, g.batches), dim3(256), 0, s, g, epi, join);
      QVH_HIP(hipGetLastError());
      return;
    }
  }
  hipLaunchKernelGGL((gemm_kernel<T, AK, BK, Shape, Epi>), grid, dim3(Shape::WM * Shape::WN * 64), 0, s, g, epi);
  QVH_HIP(hipGetLastError());
}

/// How a product reads its operands, and the shapes it may take. A row of a 64-deep step is a whole 128-byte line
/// of the L2, of a 32-deep one half of it; with more than one plane only the small tiles, or one work-group on
/// a CU, have the LDS for two such steps.
enum class Kind : int {
  kPlane1 = 0,  // 16-bit operands
  kPlane2 = 1,  // two 16-bit planes
  kPlane3 = 2,  // three 16-bit planes
  kFloat = 3,   // fp32 operands on fp32 matrix instructions
  kNarrow = 4,  // 16-bit operands, loaded four bytes at a time
  kFloatNarrow = 5
};
template <Kind K>
struct Shapes;
template <>
struct Shapes<Kind::kPlane1> {
  using S0 = Tile<64, 64, 2, 2, 64, 3, 1>;
  using S1 = Tile<128, 128, 2, 2, 64, 2, 1>;
  using S2 = Tile<256, 256, 2, 4, 64, 2, 1>;
};
template <>
struct Shapes<Kind::kPlane2> {
  using S0 = Tile<64, 64, 2, 2, 64, 2, 2>;
  using S1 = Tile<128, 128, 2, 2, 32, 2, 2>;
  using S2 = void;
  using Alone = Tile<128, 128, 2, 4, 64, 2, 2>;
};
template <>
struct Shapes<Kind::kPlane3> {
  using S0 = Tile<64, 64, 2, 2, 32, 2, 3>;
  using S1 = Tile<128, 128, 2, 4, 32, 3, 3>;
  using S2 = Tile<256, 128, 4, 2, 32, 2, 3>;
};
template <>
struct Shapes<Kind::kFloat> {
  using S0 = Tile<64, 64, 2, 2, 32, 3, 1>;
  using S1 = Tile<128, 128, 2, 2, 32, 2, 1>;
  using S2 = void;
};
template <>
struct Shapes<Kind::kNarrow> {
  using S0 = Tile<64, 64, 2, 2, 64, 2, 1, 4>;
  using S1 = Tile<128, 128, 2, 2, 64, 2, 1, 4>;
  using S2 = void;
};
template <>
struct Shapes<Kind::kFloatNarrow> {
  using S0 = Tile<64, 64, 2, 2, 32, 3, 1, 4>;
  using S1 = Tile<128, 128, 2, 2, 32, 2, 1, 4>;
  using S2 = void;
};

template <class T, Kind K, bool AK, bool BK, class Epi>
void launch_gemm(GemmArgs g, const Epi& epi, const GemmPlan& plan, void* partial, hipStream_t s) {
  if (g.m == 0 || g.n == 0 || g.batches == 0) return;
  g.splits = plan.splits;
  g.partial = static_cast<float*>(partial);
  using S = Shapes<K>;
  if constexpr (!std::is_void_v<typename S::S2>) {
    if (plan.tile == 2) return launch_tile<T, AK, BK, typename S::S2>(g, epi, s);
  }
  // One operand by rows and one by k is P X (gemm_plan: neither its 64-tiles nor its deep ones are split).
  constexpr bool kSplit = K != Kind::kPlane2 || AK == BK;
  if constexpr (K == Kind::kPlane2) {
    // The deep tile where every work-group has a CU to itself; past that two shallow ones on a CU hide each
    // other's waits (orthogonalisation of 1,024 x 4,096 393 us, 364 with it; six of 678 x 1,096 451, 482).
    const uint64_t groups = ceil_div(g.m, 128) * ceil_div(g.n, 128) * g.splits * g.batches;
    if (plan.tile == 1 && groups <= 256) return launch_tile<T, AK, BK, typename S::Alone, kSplit>(g, epi, s);
  }
  if (plan.tile >= 1) return launch_tile<T, AK, BK, typename S::S1>(g, epi, s);
  launch_tile<T, AK, BK, typename S::S0, kSplit>(g, epi, s);
}

}  // namespace qvh
