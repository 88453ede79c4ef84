// Linear attention with a decay for each head, forward, backward and one token at a time.
//
//   S_t = d S_{t-1} + k_t v_t^T,  o_t = scale S_t^T q_t,  d = exp(log_decay)
//
// A pass (attention_kernel) takes the tokens in chunks of 64. Within a chunk the result is a product of masked, decayed
// scores and values; what came before it is in the state X [dk][dv], held in fp32 registers over all chunks:
//
//   o_r = sum over s <= r of d^(r-s) (q_r k_s) v_s  +  d^(r+1) X^T q_r        r, s: rows of the chunk, n of them
//   X <- d^n X + sum over s of d^(n-1-s) k_s v_s^T
//
// The gradients are three such passes. With dO the result's gradient, dq_t = scale S_t dO_t is the pass of (dO, v, k). Backwards
// in time, G_s = sum over t >= s of d^(t-s) scale q_t dO_t^T + d^(T-1-s) dS_T gives dk_s = G_s v_s, the pass of (v, dO, q), and
// dv_s = G_s^T k_s, the pass of (k, q, dO), both over the tokens from the last to the first; there the state decays
// behind a token and not ahead of it (AttentionPass::ahead), and ends as the first state's gradient.
//
// Work. A work-group of four waves has one head of one text and 64 columns of v. A wave has 16 rows of the chunk for
// the scores and the result and 16 columns of X for the update. Scores are computed transposed, K Q^T, so that a
// lane's accumulators are four neighbouring s of one row: what the next product takes as its operand, without a way through
// LDS. K, V and X's copy for the matrix unit lie in LDS, the next chunk's K, V and Q are loaded while this one is
// computed. Where there are few heads, a text is cut into segments: a first pass makes the state that each leaves by itself, a
// scan over the segments the states that they start from.
//
// Precision. 16-bit: scores and X are rounded to the type where the matrix unit takes them (for float16 behind a
// power of two, so that neither overflows or vanishes), once each, like the result. The update multiplies v by its decay and
// adds up in fp32 to its last bits: the weighed v is a sum of three bfloat16 parts (24 bits) or two float16 ones (22).
// fp32: fp32 matrix instructions throughout.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "gemm.hpp"

namespace qvh {
namespace {

constexpr uint32_t kRows = 64;   // of a chunk
constexpr uint32_t kCols = 64;   // of v, a work-group's
constexpr uint32_t kMaxHead = 256;

/// Tokens of one tensor: element strides of text, token and head; `share` heads of the call to one of its own.
struct TokenTensor {
  const void* base = nullptr;
  uint64_t batch = 0, token = 0, head = 0;
  uint32_t share = 1;
};

struct AttentionPass {
  uint64_t tokens = 0;
  uint32_t batch = 0, heads = 0, dk = 0, dv = 0;
  TokenTensor q, k, v;
  void* out = nullptr;  // [batch][token][head][dv]
  bool out_fp32 = false;
  const float* log_decay = nullptr;
  const void* lengths = nullptr;
  int index_bytes = 0;
  const float* state = nullptr;  // [text and head][..]: element (i of dk, j of dv) at i * state_dk + j * state_dv
  float* state_out = nullptr;
  uint32_t state_dk = 0, state_dv = 0;
  bool reverse = false;
  uint32_t ahead = 1;  // the state decays ahead of a token
  float kv_scale = 1.0f, near_scale = 1.0f, far_scale = 1.0f;
  // Segments of a text, and what each leaves by itself, then what it starts from: [segment][text and head][dk][dv].
  uint32_t segments = 1;
  uint64_t segment = 0;  // tokens
  float* states = nullptr;
};

typedef float f32x8_t __attribute__((ext_vector_type(8)));

/// Operands of 16 x 16 blocks: eight k of a row or column a lane.
template <class T>
struct Op;
template <>
struct Op<bhalf_t> {
  typedef bhalf_t x8 __attribute__((ext_vector_type(8)));
  typedef bhalf_t x4 __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ f32x4_t mma(x8 a, x8 b, f32x4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Op<half_t> {
  typedef half_t x8 __attribute__((ext_vector_type(8)));
  typedef half_t x4 __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ f32x4_t mma(x8 a, x8 b, f32x4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Op<float> {
  typedef f32x8_t x8;
  typedef f32x4_t x4;
  static __device__ __forceinline__ f32x4_t mma(x8 a, x8 b, f32x4_t c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
};

/// Eight elements of a row in memory, those past its end zero.
template <class T>
__device__ __forceinline__ typename Op<T>::x8 fetch8(const T* p, uint32_t left) {
  typename Op<T>::x8 v{};
  if (left >= 8) {
    if constexpr (sizeof(T) == 2) {
      v = reinterpret_cast<const Loose<T, 8>*>(p)->v;
    } else {
      const f32x4_t lo = reinterpret_cast<const Loose<T, 4>*>(p)->v, hi = reinterpret_cast<const Loose<T, 4>*>(p + 4)->v;
      v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (static_cast<uint32_t>(i) < left) v[i] = p[i];
    }
  }
  return v;
}

/// Rows row0 + 4 g .. + 3 of column col0 + (lane & 15) in LDS, g = lane / 16. 16-bit elements go through the transposing
/// read: each lane addresses four neighbours of one row.
template <class T>
__device__ __forceinline__ typename Op<T>::x4 column4(const T* s, uint32_t stride, uint32_t row0, uint32_t col0) {
  const uint32_t l = threadIdx.x & 15, g = threadIdx.x >> 4 & 3;
  if constexpr (sizeof(T) == 2) {
    const T* at = s + (row0 + 4 * g + (l >> 2)) * stride + col0 + 4 * (l & 3);
    return __builtin_bit_cast(typename Op<T>::x4,
                              __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(at)));
  } else {
    f32x4_t v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = s[(row0 + 4 * g + i) * stride + col0 + l];
    return v;
  }
}

template <class V4>
__device__ __forceinline__ auto join(V4 a, V4 b) {
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

/// Where column c of the work-group's 64 lies in LDS: the four columns 16 g + 4 j + i, i = 0 .. 3, at 16 j + 4 g + i, so that
/// a lane's accumulators of blocks j = 0 .. 3 are 16 neighbours of a result's row.
__device__ __forceinline__ uint32_t place(uint32_t c) { return 16 * (c >> 2 & 3) + 4 * (c >> 4) + (c & 3); }
__device__ __forceinline__ uint32_t column_at(uint32_t p) { return 16 * (p >> 2 & 3) + 4 * (p >> 4) + (p & 3); }

__device__ __forceinline__ uint64_t length_of(const AttentionPass& a, uint32_t text) {
  if (!a.lengths) return a.tokens;
  const int64_t n = a.index_bytes == 8 ? static_cast<const int64_t*>(a.lengths)[text] : static_cast<const int32_t*>(a.lengths)[text];
  return n < 0 ? 0 : static_cast<uint64_t>(n) < a.tokens ? static_cast<uint64_t>(n) : a.tokens;
}

/// log2 of the decay; a decay of nothing as one that no power but the zeroth survives.
__device__ __forceinline__ double log2_decay(const AttentionPass& a, uint32_t head) {
  const double g = static_cast<double>(a.log_decay[head]) * 1.4426950408889634;
  return g < -1e30 ? -1e30 : g;
}

/// d^n in two floats.
__device__ __forceinline__ void power(double log2d, uint64_t n, float* high, float* low) {
  const double f = exp2(log2d * static_cast<double>(n));
  *high = static_cast<float>(f);
  *low = static_cast<float>(f - static_cast<double>(*high));
}

/// The power of two that brings v to 2^top .. 2^(top + 1); none for zero, infinities and NaN.
__device__ __forceinline__ int lift(float v, int top, int most) {
  if (!(v > 0.0f && v < __builtin_huge_valf())) return 0;
  const int e = top - ilogbf(v);
  return e > most ? most : e < -most ? -most : e;
}

__device__ __forceinline__ bool is_finite(float v) { return fabsf(v) < __builtin_huge_valf(); }

/// Whether all eight are finite.
template <class T>
__device__ __forceinline__ bool all_finite(typename Op<T>::x8 v) {
  if constexpr (sizeof(T) == 2) {
    constexpr uint32_t kExponent = std::is_same<T, half_t>::value ? 0x7C007C00u : 0x7F807F80u;
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    const u32x4_t bits = __builtin_bit_cast(u32x4_t, v) & kExponent;
    u16x2 most{};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t two = bits[i];  // a value: a bit cast of the element itself takes the first one's bits
      most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, two));
    }
    return most[0] < (kExponent & 0xFFFF) && most[1] < (kExponent & 0xFFFF);
  } else {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fmaf(v[i], 0.0f, sum);
    return sum == 0.0f;
  }
}

/// Zeros for what is not finite.
template <class V>
__device__ __forceinline__ V only_finite(V v) {
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(V) / sizeof(v[0])); ++i) {
    if (!is_finite(static_cast<float>(v[i]))) v[i] = 0.0f;
  }
  return v;
}

template <class T, int KD>
struct AttentionShape {
  static constexpr uint32_t kStride = KD + 16 / sizeof(T);                 // of K and X in LDS: rows four banks apart
  static constexpr uint32_t kVStride = kCols + (sizeof(T) == 2 ? 16 : 4);  // of V, read by columns
};

/// One chunk's operands on their way from memory.
template <class T, int KD, bool STATES>
struct ChunkLoads {
  using X8 = typename Op<T>::x8;
  X8 k[KD / 32], v[2], q[STATES ? 1 : KD / 32];
};

/// A tensor's rows of one head of one text in chunks of 64, from the text's start or its end.
template <class T, bool WHOLE>
struct ChunkRows {
  const char* base;  // the chunk's first row in memory
  int64_t step;      // bytes from row to row
  bool reverse;
  __device__ __forceinline__ ChunkRows(const TokenTensor& t, uint32_t text, uint32_t head, uint32_t col, bool back, uint64_t length, uint64_t first)
      : step(static_cast<int64_t>(t.token * sizeof(T))), reverse(back) {
    base = static_cast<const char*>(t.base) + (text * t.batch + head / t.share * t.head + col) * sizeof(T);
    base += (back ? static_cast<int64_t>(length) - kRows - static_cast<int64_t>(first) : static_cast<int64_t>(first)) * step;
  }
  __device__ __forceinline__ void advance() { base += reverse ? -step * kRows : step * kRows; }

  /// Where this thread's elements c .. of row r lie; past everything where there are none.
  __device__ __forceinline__ uint32_t offset(uint32_t r, uint32_t c, uint32_t cols) const {
    return c < cols ? (reverse ? kRows - 1 - r : r) * static_cast<uint32_t>(step) + c * sizeof(T) : 1u << 31;
  }
  /// The rows that are there as a buffer: loads outside of it give zeros, so nothing has to ask for the text's end.
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(uint32_t rows, uint32_t cols) const {
    const char* p = base + (reverse ? (kRows - rows) * step : 0);
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(p), 0, static_cast<int>((rows - 1) * step + cols * sizeof(T)), 0x27000);
  }
  __device__ __forceinline__ uint32_t shift(uint32_t rows) const { return reverse ? (kRows - rows) * static_cast<uint32_t>(step) : 0; }

  static __device__ __forceinline__ typename Op<T>::x8 take(__amdgpu_buffer_rsrc_t b, uint32_t offset) {
    const u32x4_t lo = __builtin_amdgcn_raw_buffer_load_b128(b, static_cast<int>(offset), 0, 0);
    if constexpr (sizeof(T) == 2) {
      return __builtin_bit_cast(typename Op<T>::x8, lo);
    } else {
      const u32x4_t hi = __builtin_amdgcn_raw_buffer_load_b128(b, static_cast<int>(offset) + 16, 0, 0);
      return join(__builtin_bit_cast(f32x4_t, lo), __builtin_bit_cast(f32x4_t, hi));
    }
  }
  /// Eight elements from column c of row r, by ordinary loads, where rows are not whole pieces.
  __device__ __forceinline__ typename Op<T>::x8 take(uint32_t r, uint32_t c, uint32_t cols, uint64_t rows) const {
    const T* at = reinterpret_cast<const T*>(base + (reverse ? kRows - 1 - r : r) * step) + c;
    return fetch8(at, r < rows && c < cols ? cols - c : 0u);
  }
};

/// WHOLE: rows of q, k and v are whole pieces of eight elements, 16-byte aligned, 2^31 bytes a chunk at most.
template <class T, int KD, bool STATES, bool WHOLE>
__global__ void __launch_bounds__(256, (sizeof(T) == 2 && KD <= 128) ? 2 : 1) attention_kernel(AttentionPass a) {
  using Shape = AttentionShape<T, KD>;
  using X8 = typename Op<T>::x8;
  using X4 = typename Op<T>::x4;
  constexpr bool kHalf = std::is_same<T, half_t>::value;
  constexpr uint32_t kS = Shape::kStride, kVS = Shape::kVStride;
  constexpr int NX = KD / 16, NK = KD / 32;
  __shared__ __attribute__((aligned(16))) T s_k[kRows * kS];
  __shared__ __attribute__((aligned(16))) T s_v[kRows * kVS];
  __shared__ __attribute__((aligned(16))) T s_x[STATES ? 16 : kCols * kS];
  __shared__ __attribute__((aligned(16))) float s_unlift[kHalf ? kCols : 4];
  __shared__ uint32_t s_odd[4];

  // The column slices of one head, which read the same q and k, follow one another on one XCD.
  const uint32_t slices = (a.dv + kCols - 1) / kCols, index = blockIdx.x >> 3;
  const uint32_t segments = STATES ? a.segments - 1 : a.segments;
  const uint64_t item = static_cast<uint64_t>(index / slices) * 8 + (blockIdx.x & 7);
  const uint32_t all = a.batch * a.heads;
  if (item >= static_cast<uint64_t>(all) * segments) return;
  const uint32_t segment = static_cast<uint32_t>(item / all), bh = static_cast<uint32_t>(item % all);
  const uint32_t text = bh / a.heads, head = bh % a.heads, col0 = index % slices * kCols;
  const uint64_t first = segment * a.segment;
  const uint64_t last = segment + 1 == a.segments ? a.tokens : first + a.segment;  // tokens of the segment end here
  const uint64_t length = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(length_of(a, text))));  // below 2^31
  const uint64_t stop = length < last ? length : last;

  const uint32_t lane = threadIdx.x & 63, l = lane & 15, g = lane >> 4;
  const uint32_t w = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6)));

  // Token p of the pass, from the text's start or its end; those past the end stay where they are.
  const auto token = [&](uint64_t p) { return a.reverse && p < length ? length - 1 - p : p; };
  // This thread's pieces of a chunk.
  constexpr uint32_t kPieces = KD / 8, kKRows = 256 / kPieces;
  const uint32_t k_row = threadIdx.x / kPieces, k_col = threadIdx.x % kPieces * 8;
  const uint32_t v_row = threadIdx.x / 8, v_col = threadIdx.x % 8 * 8, q_row = 16 * w + l;
  const uint32_t v_cols = a.dv - col0;
  using Rows = ChunkRows<T, WHOLE>;
  Rows k_at(a.k, text, head, 0, a.reverse, length, first), v_at(a.v, text, head, col0, a.reverse, length, first);
  Rows q_at(STATES ? a.k : a.q, text, head, 0, a.reverse, length, first);
  const uint32_t k_off = WHOLE ? k_at.offset(k_row, k_col, a.dk) : 0, v_off = WHOLE ? v_at.offset(v_row, v_col, v_cols) : 0;
  const uint32_t q_off = WHOLE ? q_at.offset(q_row, 8 * g, a.dk) : 0;

  const double log2d = log2_decay(a, head);
  const float lg = static_cast<float>(log2d);
  const auto decay = [&](int n) { return __builtin_amdgcn_exp2f(lg * static_cast<float>(n)); };
  float whole_high, whole_low;
  power(log2d, kRows, &whole_high, &whole_low);

  // Factors of the scores, row 16 w + l against s = 16 b + 4 g + i: of the block on the diagonal, and of those before it
  // d^(16 + l - 4 g - i) d^(16 (w - b - 1)). Of v in the update, s = 16 c + 4 g + i: d^(15 - 4 g - i) d^(n - ahead - 15 - 16 c).
  const auto uniform = [](float f) { return __uint_as_float(static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(__float_as_uint(f))))); };
  float diagonal[4], before[4], within[4], far_factor = 0.0f, block_factor[4], weight_factor[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int apart = static_cast<int>(l) - static_cast<int>(4 * g + i);
    diagonal[i] = apart >= 0 ? a.near_scale * decay(apart) : 0.0f;
    before[i] = a.near_scale * decay(16 + apart);
    within[i] = decay(15 - static_cast<int>(4 * g + i));
    weight_factor[i] = uniform(a.kv_scale * decay(49 - static_cast<int>(a.ahead) - 16 * i));
    const int away = static_cast<int>(w) - i - 1;
    block_factor[i] = uniform(away >= 0 ? decay(16 * away) : 0.0f);
  }
  if constexpr (!STATES) far_factor = a.far_scale * decay(static_cast<int>(16 * w + l + a.ahead));

  // X: dk 16 n + 4 g + i, this wave's column at place 16 w + l. float16: times 2^x_lift, by columns.
  f32x4_t x[NX];
  int x_lift = 0;
  bool settled = false;  // X holds infinities or NaN, perhaps
  {
    const float* from = nullptr;
    uint64_t sk = a.dv, sv = 1;
    if (!STATES && a.segments > 1) {
      from = a.states + (static_cast<uint64_t>(segment) * all + bh) * a.dk * a.dv;
    } else if (!STATES && a.state) {
      from = a.state + static_cast<uint64_t>(bh) * a.dk * a.dv;
      sk = a.state_dk;
      sv = a.state_dv;
    }
    const uint32_t c = col0 + column_at(16 * w + l);
#pragma unroll
    for (int n = 0; n < NX; ++n) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t r = 16 * n + 4 * g + i;
        x[n][i] = from && r < a.dk && c < a.dv ? from[r * sk + c * sv] : 0.0f;
        settled = settled || !is_finite(x[n][i]);
      }
    }
    settled = __any(settled);
  }

  ChunkLoads<T, KD, STATES> next;
  const auto load = [&](uint64_t rows) {
    if constexpr (WHOLE) {
      const uint32_t n = rows < kRows ? static_cast<uint32_t>(rows) : kRows;
      const auto k_rows = k_at.buffer(n, a.dk), v_rows = v_at.buffer(n, v_cols);
      const uint32_t k0 = k_off - k_at.shift(n), v0 = v_off - v_at.shift(n);
      const uint32_t k_next = a.reverse ? -kKRows * static_cast<uint32_t>(k_at.step) : kKRows * static_cast<uint32_t>(k_at.step);
      const uint32_t v_next = a.reverse ? -32 * static_cast<uint32_t>(v_at.step) : 32 * static_cast<uint32_t>(v_at.step);
#pragma unroll
      for (int u = 0; u < KD / 32; ++u) next.k[u] = Rows::take(k_rows, k0 + u * k_next);
#pragma unroll
      for (int u = 0; u < 2; ++u) next.v[u] = Rows::take(v_rows, v0 + u * v_next);
      if constexpr (!STATES) {
        const auto q_rows = q_at.buffer(n, a.dk);
        const uint32_t q0 = q_off - q_at.shift(n);
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) next.q[kk] = Rows::take(q_rows, 32 * kk + 8 * g < a.dk ? q0 + 32 * kk * sizeof(T) : 1u << 31);
      }
    } else {
#pragma unroll
      for (int u = 0; u < KD / 32; ++u) next.k[u] = k_at.take(k_row + u * kKRows, k_col, a.dk, rows);
#pragma unroll
      for (int u = 0; u < 2; ++u) next.v[u] = v_at.take(v_row + u * 32, v_col, v_cols, rows);
      if constexpr (!STATES) {
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) next.q[kk] = q_at.take(q_row, 32 * kk + 8 * g, a.dk, rows);
      }
    }
    k_at.advance();
    v_at.advance();
    q_at.advance();
  };

  const auto left = [](uint32_t all_of_it, uint32_t from) { return all_of_it <= from ? 0u : WHOLE ? 8u : all_of_it - from; };
  const auto store_row = [&](uint64_t t, const float (&lo)[8], const float (&hi)[8]) {
    const uint32_t c = col0 + 16 * g;
    const uint64_t at = ((text * a.tokens + t) * a.heads + head) * a.dv + c;
    const auto put = [&](auto* out) {
      if (left(a.dv, c)) store8(out + at, lo, left(a.dv, c));
      if (left(a.dv, c + 8)) store8(out + at + 8, hi, left(a.dv, c + 8));
    };
    if (a.out_fp32) return put(static_cast<float*>(a.out));
    put(static_cast<T*>(a.out));
  };

  if (first < stop) load(stop - first);
  for (uint64_t c0 = first; c0 < stop; c0 += kRows) {
    const uint32_t rows = stop - c0 < kRows ? static_cast<uint32_t>(stop - c0) : kRows;
    int copy_lift = 0, x_size = 0;  // float16: of X's copy beside X, and the binary order of X's column
    if constexpr (kHalf) {
      float most = 0.0f;
#pragma unroll
      for (int n = 0; n < NX; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) most = fmaxf(most, fabsf(x[n][i]));
      }
      if (settled) {  // by what is finite, then
        most = 0.0f;
#pragma unroll
        for (int n = 0; n < NX; ++n) {
#pragma unroll
          for (int i = 0; i < 4; ++i) most = fmaxf(most, is_finite(x[n][i]) ? fabsf(x[n][i]) : 0.0f);
        }
      }
      most = fmaxf(most, __shfl_xor(most, 16, 64));
      most = fmaxf(most, __shfl_xor(most, 32, 64));
      copy_lift = lift(most, 14, 120);
      x_size = most > 0.0f && is_finite(most) ? ilogbf(most) : -120;
    }
    bool finite = true;
#pragma unroll
    for (int u = 0; u < KD / 32; ++u) finite = all_finite<T>(next.k[u]) && finite;
#pragma unroll
    for (int u = 0; u < 2; ++u) finite = all_finite<T>(next.v[u]) && finite;
    finite = !__any(!finite);
    __syncthreads();  // the last chunk's reads of LDS are done
    if (lane == 0) s_odd[w] = !finite;
    if (kHalf && !STATES && g == 0) s_unlift[16 * w + l] = ldexpf(1.0f, -(x_lift + copy_lift));
#pragma unroll
    for (int u = 0; u < KD / 32; ++u) *reinterpret_cast<X8*>(s_k + (k_row + u * kKRows) * kS + k_col) = next.k[u];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      T* at = s_v + (v_row + u * 32) * kVS;
      *reinterpret_cast<X4*>(at + place(v_col)) = __builtin_shufflevector(next.v[u], next.v[u], 0, 1, 2, 3);
      *reinterpret_cast<X4*>(at + place(v_col + 4)) = __builtin_shufflevector(next.v[u], next.v[u], 4, 5, 6, 7);
    }
    X8 qf[STATES ? 1 : NK];
    if constexpr (!STATES) {
#pragma unroll
      for (int n = 0; n < NX; ++n) {
        X4 copy;
#pragma unroll
        for (int i = 0; i < 4; ++i) copy[i] = static_cast<T>(kHalf ? ldexpf(x[n][i], copy_lift) : x[n][i]);
        *reinterpret_cast<X4*>(s_x + (16 * w + l) * kS + 16 * n + 4 * g) = copy;
      }
#pragma unroll
      for (int kk = 0; kk < NK; ++kk) qf[kk] = next.q[kk];
    }
    __syncthreads();
    // Infinities or NaN in k or v: what the plain products would spread is kept apart.
    const bool odd = __builtin_amdgcn_readfirstlane(static_cast<int>(s_odd[0] | s_odd[1] | s_odd[2] | s_odd[3])) != 0;
    if (c0 + kRows < stop) load(stop - c0 - kRows);

    if constexpr (!STATES) {
      // Scores of this wave's rows, decayed, zeros where s comes later. (All four blocks for 16 bits: the wave with the most
      // of them decides, and without branches their products follow one another closely.)
      float p[4][4];
      f32x4_t acc[4]{};
#pragma unroll
      for (uint32_t b = 0; b < 4; ++b) {
        if (sizeof(T) == 4 && b > w) continue;
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) acc[b] = Op<T>::mma(*reinterpret_cast<const X8*>(s_k + (16 * b + l) * kS + 32 * kk + 8 * g), qf[kk], acc[b]);
      }
      __builtin_amdgcn_sched_barrier(0);
      // What the state gives.
      f32x4_t o[4]{};
#pragma unroll
      for (int kk = 0; kk < NK; ++kk) {
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = Op<T>::mma(*reinterpret_cast<const X8*>(s_x + (16 * j + l) * kS + 32 * kk + 8 * g), qf[kk], o[j]);
      }
#pragma unroll
      for (uint32_t b = 0; b < 4; ++b) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float factor = b == w ? diagonal[i] : before[i] * block_factor[b];
          p[b][i] = b < w || (b == w && 4 * g + i <= l) ? acc[b][i] * factor : 0.0f;
        }
      }
      int p_lift = 0;  // float16: this row's scores and sums are 2^p_lift as large
      if constexpr (kHalf) {
        float most = 0.0f;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
#pragma unroll
          for (int i = 0; i < 4; ++i) most = fmaxf(most, fabsf(p[b][i]));
        }
        most = fmaxf(most, __shfl_xor(most, 16, 64));
        most = fmaxf(most, __shfl_xor(most, 32, 64));
        p_lift = lift(most, 13, 40);
        const float factor = ldexpf(far_factor, p_lift);
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const f32x4_t unlift = *reinterpret_cast<const f32x4_t*>(s_unlift + 16 * b + 4 * g);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            p[b][i] = ldexpf(p[b][i], p_lift);
            o[b][i] *= unlift[i] * factor;
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] *= far_factor;
      }
      __builtin_amdgcn_sched_barrier(0);
      // Scores that the mask takes away are zeros; against infinities and NaN of v they would still count. There those of v
      // are left out, and the ones that the mask lets through are added by themselves.
#pragma unroll
      for (uint32_t m = 0; m < 2; ++m) {
        if (sizeof(T) == 4 && 2 * m > w) continue;
        X8 pb;
#pragma unroll
        for (int e = 0; e < 8; ++e) pb[e] = static_cast<T>(p[2 * m + (e >> 2)][e & 3]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          X4 v0 = column4(s_v, kVS, 32 * m, 16 * j), v1 = column4(s_v, kVS, 32 * m + 16, 16 * j);
          if (odd && 2 * m >= w) v0 = only_finite(v0);
          if (odd && 2 * m + 1 >= w) v1 = only_finite(v1);
          o[j] = Op<T>::mma(join(v0, v1), pb, o[j]);
        }
      }
      if (odd) {
        float own[4];  // the scores of the block on the diagonal
#pragma unroll
        for (int i = 0; i < 4; ++i) own[i] = w == 0 ? p[0][i] : w == 1 ? p[1][i] : w == 2 ? p[2][i] : p[3][i];
#pragma unroll 1
        for (uint32_t s = 0; s < 16; ++s) {
          const uint32_t i0 = s & 3;
          const float mine = i0 == 0 ? own[0] : i0 == 1 ? own[1] : i0 == 2 ? own[2] : own[3];
          const float score = __shfl(mine, static_cast<int>(l + 16 * (s >> 2)), 64);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float value = static_cast<float>(s_v[(16 * w + s) * kVS + 16 * j + 4 * g + i]);
              if (s <= l && !is_finite(value)) o[j][i] = fmaf(score, value, o[j][i]);
            }
          }
        }
      }
      if (c0 + q_row < last) {
        float lo[8], hi[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float y0 = o[e >> 2][e & 3], y1 = o[2 + (e >> 2)][e & 3];
          lo[e] = q_row >= rows ? 0.0f : kHalf ? ldexpf(y0, -p_lift) : y0;
          hi[e] = q_row >= rows ? 0.0f : kHalf ? ldexpf(y1, -p_lift) : y1;
        }
        store_row(token(c0 + q_row), lo, hi);
      }
    }

    __builtin_amdgcn_sched_barrier(0);
    // X: this wave's columns. v times its decay in fp32, as three bfloat16 parts or two float16 ones, against k as it is.
    constexpr int kParts = sizeof(T) == 4 ? 1 : kHalf ? 2 : 3;
    X8 part[2][kParts];
    int new_lift = x_lift;
    {
      float y[2][8];
#pragma unroll
      for (uint32_t m = 0; m < 2; ++m) {
        const X8 vf = join(column4(s_v, kVS, 32 * m, 16 * w), column4(s_v, kVS, 32 * m + 16, 16 * w));
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) {
          float weight = within[e & 3] * weight_factor[2 * m + (e >> 2)];
          if (rows < kRows) {
            const int after = static_cast<int>(rows - a.ahead) - static_cast<int>(32 * m + 16 * (e >> 2) + 4 * g + (e & 3));
            weight = a.kv_scale * decay(after > 0 ? after : 0);
          }
          y[m][e] = static_cast<float>(vf[e]) * weight;
        }
      }
      if constexpr (kHalf) {
        // Behind a power of two by columns, as large as float16 and X's own size allow.
        float most = 0.0f;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
#pragma unroll
          for (int e = 0; e < 8; ++e) most = fmaxf(most, odd && !is_finite(y[m][e]) ? 0.0f : fabsf(y[m][e]));
        }
        most = fmaxf(most, __shfl_xor(most, 16, 64));
        most = fmaxf(most, __shfl_xor(most, 32, 64));
        if (most > 0.0f) {
          const int top = 14 - ilogbf(most), room = 100 - (x_size - x_lift);
          new_lift = top < room ? top : room;
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
#pragma unroll
          for (int e = 0; e < 8; ++e) y[m][e] = ldexpf(y[m][e], new_lift);
        }
      }
#pragma unroll
      for (int m = 0; m < 2; ++m) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float rest = y[m][e];
#pragma unroll
          for (int z = 0; z < kParts; ++z) {
            part[m][z][e] = static_cast<T>(rest);
            if (z + 1 < kParts) rest -= static_cast<float>(part[m][z][e]);
          }
        }
        if (odd) {  // an infinity has no lower parts
#pragma unroll
          for (int z = 1; z < kParts; ++z) part[m][z] = only_finite(part[m][z]);
        }
      }
    }
    float high = whole_high, low = whole_low;
    if (rows < kRows) power(log2d, rows, &high, &low);
    if constexpr (kHalf) {
      high = ldexpf(high, new_lift - x_lift);
      low = ldexpf(low, new_lift - x_lift);
      x_lift = new_lift;
    }
    // The decay's second float counts over many chunks; times an infinity it would be NaN.
    if (settled) {
#pragma unroll
      for (int n = 0; n < NX; ++n) x[n] *= high;
    } else {
#pragma unroll
      for (int n = 0; n < NX; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[n][i] = fmaf(x[n][i], high, x[n][i] * low);
      }
    }
    settled = settled || odd;
#pragma unroll
    for (uint32_t m = 0; m < 2; ++m) {
#pragma unroll
      for (int n0 = 0; n0 < NX; n0 += 4) {
        X8 kf[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) kf[n] = join(column4(s_k, kS, 32 * m, 16 * (n0 + n)), column4(s_k, kS, 32 * m + 16, 16 * (n0 + n)));
        if (odd && kParts > 1) {
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const X8 lower = only_finite(kf[n]);  // zeros among v's lower parts are none of v's
#pragma unroll
            for (int z = kParts - 1; z >= 0; --z) x[n0 + n] = Op<T>::mma(z ? lower : kf[n], part[m][z], x[n0 + n]);
          }
        } else {
#pragma unroll
          for (int z = kParts - 1; z >= 0; --z) {
#pragma unroll
            for (int n = 0; n < 4; ++n) x[n0 + n] = Op<T>::mma(kf[n], part[m][z], x[n0 + n]);
          }
        }
      }
    }
    if (odd && a.dk < KD) {  // rows that X does not have stay zeros
#pragma unroll
      for (int n = 0; n < NX; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[n][i] = 16 * n + 4 * g + i < a.dk ? x[n][i] : 0.0f;
      }
    }
  }

  if constexpr (!STATES) {
    // Tokens past the text's end, in chunks of their own.
    const uint64_t done = first < stop ? first + (stop - first + kRows - 1) / kRows * kRows : first;
    const float zero[8] = {};
    for (uint64_t t = done + q_row; t < last; t += kRows) store_row(t, zero, zero);
  }
  float* to = nullptr;
  uint64_t sk = a.dv, sv = 1;
  if constexpr (STATES) {
    to = a.states + (static_cast<uint64_t>(segment) * all + bh) * a.dk * a.dv;
  } else if (a.state_out && segment + 1 == a.segments) {
    to = a.state_out + static_cast<uint64_t>(bh) * a.dk * a.dv;
    sk = a.state_dk;
    sv = a.state_dv;
  }
  if (!to) return;
  asm volatile("" : "+s"(sk), "+s"(sv));  // the addresses anew: kept over the loop, they took more registers than there are
  const uint32_t c = col0 + column_at(16 * w + l);
#pragma unroll
  for (int n = 0; n < NX; ++n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t r = 16 * n + 4 * g + i;
      if (r < a.dk && c < a.dv) to[r * sk + c * sv] = kHalf ? ldexpf(x[n][i], -x_lift) : x[n][i];
    }
  }
}

/// From what each segment leaves by itself to what it starts from.
__global__ void __launch_bounds__(256) attention_scan_kernel(AttentionPass a) {
  const uint32_t all = a.batch * a.heads, bh = blockIdx.y;
  const uint32_t size = a.dk * a.dv, at = blockIdx.x * 256 + threadIdx.x;
  if (at >= size) return;
  const uint64_t length = length_of(a, bh / a.heads);
  const double log2d = log2_decay(a, bh % a.heads);
  float x = 0.0f;
  if (a.state) x = a.state[static_cast<uint64_t>(bh) * size + static_cast<uint64_t>(at / a.dv) * a.state_dk + static_cast<uint64_t>(at % a.dv) * a.state_dv];
  float* s = a.states + static_cast<uint64_t>(bh) * size + at;
  const uint64_t step = static_cast<uint64_t>(all) * size;
  float high, low;
  power(log2d, a.segment, &high, &low);
  for (uint32_t i = 0; i < a.segments; ++i) {
    const float own = i + 1 < a.segments ? s[i * step] : 0.0f;
    s[i * step] = x;
    const uint64_t from = i * a.segment, n = length > from ? length - from : 0;
    if (n < a.segment) power(log2d, n, &high, &low);
    x = is_finite(x) ? fmaf(x, high, fmaf(x, low, own)) : fmaf(x, high, own);
  }
}

/// The gradients of the heads that share one: their sum, in order.
template <class T>
__global__ void __launch_bounds__(256) attention_shared_kernel(const float* __restrict__ parts, uint64_t rows, uint32_t share,
                                                               uint32_t dim, T* __restrict__ out) {
  const uint64_t count = rows * dim;
  for (uint64_t i = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x; i < count; i += static_cast<uint64_t>(gridDim.x) * 256) {
    const float* p = parts + i / dim * share * dim + i % dim;
    float v = p[0];
    for (uint32_t h = 1; h < share; ++h) v += p[static_cast<uint64_t>(h) * dim];
    out[i] = static_cast<T>(v);
  }
}

// ---- few tokens: the recurrence itself --------------------------------------------------------

/// One head of one text and 64 columns of its state: R * 16 rows in registers, four neighbouring columns a lane, rows a
/// sixteenth of them apart. Bound by the state's bytes, read once and written once.
template <class T, int R>
__global__ void __launch_bounds__(256) attention_step_kernel(AttentionPass a) {
  __shared__ float s_o[4][64];
  const uint32_t slices = (a.dv + kCols - 1) / kCols;
  const uint32_t bh = blockIdx.x / slices, col0 = blockIdx.x % slices * kCols;
  const uint32_t text = bh / a.heads, head = bh % a.heads;
  const uint32_t row = threadIdx.x >> 4, c = col0 + (threadIdx.x & 15) * 4;
  const uint32_t lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const uint64_t length = length_of(a, text);
  const uint64_t size = static_cast<uint64_t>(a.dk) * a.dv;
  float x[R][4];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const uint32_t r = row + 16 * i;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[i][e] = 0.0f;
    if (!a.state || r >= a.dk) continue;
    const float* from = a.state + bh * size + static_cast<uint64_t>(r) * a.dv + c;
    if (c + 4 <= a.dv) {
      load_floats<float, 4>(from, x[i]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (c + e < a.dv) x[i][e] = from[e];
      }
    }
  }
  const T* q = static_cast<const T*>(a.q.base) + text * a.q.batch + head / a.q.share * a.q.head;
  const T* k = static_cast<const T*>(a.k.base) + text * a.k.batch + head / a.k.share * a.k.head;
  const T* v = static_cast<const T*>(a.v.base) + text * a.v.batch + head / a.v.share * a.v.head;
  const float d = static_cast<float>(exp2(log2_decay(a, head)));
  T* out = static_cast<T*>(a.out);
  for (uint64_t t = 0; t < a.tokens; ++t) {
    float o[4] = {};
    if (t < length) {
      float value[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) value[e] = c + e < a.dv ? static_cast<float>(v[t * a.v.token + c + e]) : 0.0f;
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const uint32_t r = row + 16 * i;
        if (r >= a.dk) continue;
        const float key = static_cast<float>(k[t * a.k.token + r]), query = static_cast<float>(q[t * a.q.token + r]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[i][e] = fmaf(key, value[e], x[i][e] * d);
          o[e] = fmaf(query, x[i][e], o[e]);
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[e] += __shfl_xor(o[e], 16, 64);
      o[e] += __shfl_xor(o[e], 32, 64);
      if (lane < 16) s_o[w][lane * 4 + e] = o[e];
    }
    __syncthreads();
    if (threadIdx.x < 64 && col0 + threadIdx.x < a.dv) {
      const uint32_t i = threadIdx.x;
      out[((text * a.tokens + t) * a.heads + head) * a.dv + col0 + i] =
          static_cast<T>(a.near_scale * ((s_o[0][i] + s_o[1][i]) + (s_o[2][i] + s_o[3][i])));
    }
    __syncthreads();
  }
  if (!a.state_out) return;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const uint32_t r = row + 16 * i;
    if (r >= a.dk) continue;
    float* to = a.state_out + bh * size + static_cast<uint64_t>(r) * a.dv + c;
    if (c + 4 <= a.dv) {
      store_floats<float, 4>(to, x[i]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (c + e < a.dv) to[e] = x[i][e];
      }
    }
  }
}

// ---- plans ------------------------------------------------------------------------------------

constexpr uint64_t kFewTokens = 8;  // the recurrence itself, up to here

template <class F>
void with_depth(uint32_t dk, F&& f) {
  if (dk <= 64) return f(std::integral_constant<int, 64>{});
  if (dk <= 128) return f(std::integral_constant<int, 128>{});
  f(std::integral_constant<int, 256>{});
}

/// Segments of a pass, as many as it takes to fill the device, of eight chunks or more.
void cut(AttentionPass& a) {
  const uint64_t slices = ceil_div(a.dv, kCols), groups = static_cast<uint64_t>(a.batch) * a.heads * slices;
  const uint64_t chunks = ceil_div(a.tokens, kRows);
  uint64_t segments = groups >= 512 || groups == 0 ? 1 : 1024 / groups;
  segments = std::max<uint64_t>(1, std::min(segments, chunks / 8));
  const uint64_t each = ceil_div(std::max<uint64_t>(chunks, 1), segments);
  a.segment = each * kRows;
  a.segments = static_cast<uint32_t>(ceil_div(std::max<uint64_t>(chunks, 1), each));
}

uint64_t state_bytes(const AttentionPass& a) {
  return a.segments > 1 ? static_cast<uint64_t>(a.segments) * a.batch * a.heads * a.dk * a.dv * sizeof(float) : 0;
}

/// Whether rows of a tensor are whole pieces (attention_kernel's WHOLE).
bool whole_rows(const TokenTensor& t, uint32_t dim, size_t size) {
  const uint64_t odd = reinterpret_cast<uintptr_t>(t.base) | t.batch * size | t.token * size | t.head * size;
  return dim % 8 == 0 && odd % 16 == 0 && (t.token + dim) * size * kRows < (uint64_t{1} << 31);
}

template <class T>
void launch_pass(const AttentionPass& a, hipStream_t s) {
  const bool whole = whole_rows(a.q, a.dk, sizeof(T)) && whole_rows(a.k, a.dk, sizeof(T)) && whole_rows(a.v, a.dv, sizeof(T));
  const auto with_rows = [&](auto&& f) { whole ? f(std::true_type{}) : f(std::false_type{}); };
  const uint64_t slices = ceil_div(a.dv, kCols), all = static_cast<uint64_t>(a.batch) * a.heads;
  with_depth(a.dk, [&](auto depth) {
    constexpr int KD = decltype(depth)::value;
    const auto grid = [&](uint64_t segments) { return dim3(static_cast<unsigned>(ceil_div(all * segments, 8) * 8 * slices)); };
    if (a.segments > 1) {
      with_rows([&](auto rows) {
        hipLaunchKernelGGL((attention_kernel<T, KD, true, decltype(rows)::value>), grid(a.segments - 1), dim3(256), 0, s, a);
        QVH_HIP(hipGetLastError());
      });
      hipLaunchKernelGGL(attention_scan_kernel, dim3(static_cast<unsigned>(ceil_div(static_cast<uint64_t>(a.dk) * a.dv, 256)), static_cast<unsigned>(all)),
                         dim3(256), 0, s, a);
      QVH_HIP(hipGetLastError());
    }
    with_rows([&](auto rows) {
      hipLaunchKernelGGL((attention_kernel<T, KD, false, decltype(rows)::value>), grid(a.segments), dim3(256), 0, s, a);
      QVH_HIP(hipGetLastError());
    });
  });
}

template <class T>
void launch_step(const AttentionPass& a, hipStream_t s) {
  const unsigned groups = static_cast<unsigned>(a.batch * a.heads * ceil_div(a.dv, kCols));
  with_depth(a.dk, [&](auto depth) {
    hipLaunchKernelGGL((attention_step_kernel<T, decltype(depth)::value / 16>), dim3(groups), dim3(256), 0, s, a);
    QVH_HIP(hipGetLastError());
  });
}

void check_tensor(const std::string& who, const char* name, const void* p, const uint64_t (&stride)[3]) {
  QVH_REQUIRE(p != nullptr, who + ": null " + name);
  for (int i = 0; i < 3; ++i) QVH_REQUIRE(stride[i] < (uint64_t{1} << 40), who + ": " + name + "'s strides must be below 2^40");
}

/// True where there is work: a token, or a state to carry over.
bool check_attention(const char* name, const qvh_attention_args& a) {
  const std::string who(name);
  require_dtype(name, a.dtype);
  QVH_REQUIRE(a.heads > 0 && a.kv_heads > 0 && a.heads % a.kv_heads == 0, who + ": heads must be a multiple of kv_heads");
  QVH_REQUIRE(a.dk > 0 && a.dk <= kMaxHead && a.dv > 0 && a.dv <= kMaxHead, who + ": dk and dv must be in [1, 256]");
  QVH_REQUIRE(a.batch < (uint64_t{1} << 31) && a.tokens < (uint64_t{1} << 31), who + ": batch and tokens must be below 2^31");
  QVH_REQUIRE(a.batch * a.heads < (uint64_t{1} << 16), who + ": batch times heads must be below 2^16");
  QVH_REQUIRE(!a.lengths || a.index_bytes == 4 || a.index_bytes == 8, who + ": lengths must be int32 or int64");
  QVH_REQUIRE(std::isfinite(a.scale), who + ": scale must be finite");
  if (a.batch == 0) return false;
  QVH_REQUIRE(a.log_decay != nullptr, who + ": null log_decay");
  if (a.tokens > 0) {
    check_tensor(who, "q", a.q, a.q_stride);
    check_tensor(who, "k", a.k, a.k_stride);
    check_tensor(who, "v", a.v, a.v_stride);
  }
  return true;
}

TokenTensor tensor_of(const void* p, const uint64_t (&stride)[3], uint32_t share) { return {p, stride[0], stride[1], stride[2], share}; }

AttentionPass forward_pass(const qvh_attention_args& in) {
  AttentionPass a;
  a.tokens = in.tokens;
  a.batch = static_cast<uint32_t>(in.batch);
  a.heads = in.heads;
  a.dk = in.dk;
  a.dv = in.dv;
  const uint32_t share = in.heads / in.kv_heads;
  a.q = tensor_of(in.q, in.q_stride, 1);
  a.k = tensor_of(in.k, in.k_stride, share);
  a.v = tensor_of(in.v, in.v_stride, share);
  a.out = in.out;
  a.log_decay = in.log_decay;
  a.lengths = in.lengths;
  a.index_bytes = in.index_bytes;
  a.state = in.state;
  a.state_out = in.state_out;
  a.state_dk = in.dv;
  a.state_dv = 1;
  a.near_scale = a.far_scale = in.scale;
  cut(a);
  return a;
}

/// The three passes of the gradients, and where their workspaces lie: the segments' states, one pass after another, and
/// shared heads' gradients by themselves.
struct GradPasses {
  AttentionPass q, k, v;
  float *parts_k = nullptr, *parts_v = nullptr;
  uint64_t bytes = 0;
};

GradPasses grad_passes(const qvh_attention_grad_args& in, void* workspace) {
  const qvh_attention_args& f = in.forward;
  GradPasses g;
  const uint32_t share = f.heads / f.kv_heads;
  AttentionPass a = forward_pass(f);
  const TokenTensor q = a.q, k = a.k, v = a.v, o = tensor_of(in.grad, in.grad_stride, 1);
  a.state_out = nullptr;
  // dq: forwards, the state transposed.
  g.q = a;
  g.q.dk = f.dv;
  g.q.dv = f.dk;
  g.q.q = o;
  g.q.k = v;
  g.q.v = k;
  g.q.out = in.grad_q;
  g.q.state_dk = 1;
  g.q.state_dv = f.dv;
  cut(g.q);
  // dv: backwards from the last state's gradient to the first one's.
  a.reverse = true;
  a.ahead = 0;
  a.state = in.grad_state;
  a.kv_scale = f.scale;
  a.far_scale = 1.0f;
  a.out_fp32 = share > 1;
  g.v = a;
  g.v.q = k;
  g.v.k = q;
  g.v.v = o;
  g.v.state_out = in.grad_first;
  cut(g.v);
  // dk: the same, transposed.
  g.k = a;
  g.k.dk = f.dv;
  g.k.dv = f.dk;
  g.k.q = v;
  g.k.k = o;
  g.k.v = q;
  g.k.state_dk = 1;
  g.k.state_dv = f.dv;
  cut(g.k);
  char* at = static_cast<char*>(workspace);
  const auto take = [&](uint64_t bytes) {
    char* p = at ? at + g.bytes : nullptr;
    g.bytes += ceil_div(bytes, 16) * 16;
    return reinterpret_cast<float*>(p);
  };
  float* states = take(std::max({state_bytes(g.q), state_bytes(g.k), state_bytes(g.v)}));
  g.q.states = g.k.states = g.v.states = states;
  const uint64_t rows = f.batch * f.tokens * f.heads;
  if (share > 1) {
    g.parts_k = take(rows * f.dk * sizeof(float));
    g.parts_v = take(rows * f.dv * sizeof(float));
    g.k.out = g.parts_k;
    g.v.out = g.parts_v;
  } else {
    g.k.out = in.grad_k;
    g.v.out = in.grad_v;
  }
  return g;
}

bool check_attention_grad(const char* name, const qvh_attention_grad_args* args) {
  const std::string who(name);
  QVH_REQUIRE(args != nullptr, who + ": null arguments");
  const bool work = check_attention(name, args->forward);
  if (work && args->forward.tokens > 0) {
    check_tensor(who, "grad", args->grad, args->grad_stride);
    QVH_REQUIRE(args->grad_q && args->grad_k && args->grad_v, who + ": null result");
  }
  return work;
}

}  // namespace
}  // namespace qvh

extern "C" {

qvh_status qvh_attention_workspace(const qvh_attention_args* args, uint64_t* bytes) {
  return qvh::guarded([&] {
    QVH_REQUIRE(bytes != nullptr, "qvh_attention_workspace: null output");
    QVH_REQUIRE(args != nullptr, "qvh_attention_workspace: null arguments");
    *bytes = 0;
    if (!qvh::check_attention("qvh_attention_workspace", *args) || args->tokens <= qvh::kFewTokens) return;
    *bytes = qvh::state_bytes(qvh::forward_pass(*args));
  });
}

qvh_status qvh_attention_device(const qvh_attention_args* args, void* d_workspace, uint64_t workspace_bytes, void* stream) {
  return qvh::guarded([&] {
    using namespace qvh;
    const char* who = "qvh_attention_device";
    QVH_REQUIRE(args != nullptr, std::string(who) + ": null arguments");
    if (!check_attention(who, *args)) return;
    QVH_REQUIRE(args->tokens == 0 || args->out != nullptr, std::string(who) + ": null result");
    AttentionPass a = forward_pass(*args);
    const bool few = a.tokens <= kFewTokens;
    check_workspace(who, d_workspace, workspace_bytes, few ? 0 : state_bytes(a));
    if (a.tokens == 0 && !a.state_out) return;
    const DeviceScope device;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    a.states = static_cast<float*>(d_workspace);
    with_dtype(args->dtype, [&](auto* t) {
      using T = std::remove_pointer_t<decltype(t)>;
      if (few) return launch_step<T>(a, s);
      launch_pass<T>(a, s);
    });
  });
}

qvh_status qvh_attention_grad_workspace(const qvh_attention_grad_args* args, uint64_t* bytes) {
  return qvh::guarded([&] {
    QVH_REQUIRE(bytes != nullptr, "qvh_attention_grad_workspace: null output");
    *bytes = 0;
    if (!qvh::check_attention_grad("qvh_attention_grad_workspace", args)) return;
    *bytes = qvh::grad_passes(*args, nullptr).bytes;
  });
}

qvh_status qvh_attention_grad_device(const qvh_attention_grad_args* args, void* d_workspace, uint64_t workspace_bytes, void* stream) {
  return qvh::guarded([&] {
    using namespace qvh;
    const char* who = "qvh_attention_grad_device";
    if (!check_attention_grad(who, args)) return;
    const GradPasses g = grad_passes(*args, d_workspace);
    check_workspace(who, d_workspace, workspace_bytes, g.bytes);
    const DeviceScope device;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const qvh_attention_args& f = args->forward;
    with_dtype(f.dtype, [&](auto* t) {
      using T = std::remove_pointer_t<decltype(t)>;
      launch_pass<T>(g.q, s);
      launch_pass<T>(g.k, s);
      launch_pass<T>(g.v, s);
      if (g.parts_k && f.tokens > 0) {
        const uint64_t rows = f.batch * f.tokens * f.kv_heads;
        const auto sum = [&](const float* parts, uint32_t dim, void* out) {
          const uint64_t groups = std::min<uint64_t>(ceil_div(rows * dim, 256), 4096);
          hipLaunchKernelGGL((attention_shared_kernel<T>), dim3(static_cast<unsigned>(groups)), dim3(256), 0, s, parts, rows,
                             f.heads / f.kv_heads, dim, static_cast<T*>(out));
          QVH_HIP(hipGetLastError());
        };
        sum(g.parts_k, f.dk, args->grad_k);
        sum(g.parts_v, f.dv, args->grad_v);
      }
    });
  });
}

}  // extern "C"
