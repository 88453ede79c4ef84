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
// What bounds it. 8 texts of 4,096 tokens, 16 heads of 128 bf16 (537 MB, 106 us at a copy's rate): 148 us a pass where every CU
// has two work-groups (512 of them), 3.6 TB/s, 195 to 202 with one (256); backwards, three passes in one launch, 470 to 520. A wave has
// 72 matrix instructions (1,150 cycles) and 360 others (1,450) a chunk and waits for the rest of its 5,700: for LDS behind the
// two barriers, for one product's result in the next. LDS moves data 35% of the time. Three work-groups a CU would need
// 168 registers a wave and keep the rest in memory (596 us a pass); eight waves with 128 columns and tokens, which load q
// and k once, took as long and left half of the CUs empty at 128 heads. fp32: 8 texts of 1,000 tokens, 12 heads of 64, 49 us and 18 for the
// segments' states: the fp32 matrix unit, which needs 22 of them. One token for each of 256 texts, 16 heads of 128: 105 us, the
// states' 537 MB at 5.1 TB/s.
//
// Registers that the compiler's report finds in scratch memory: at depth 128 13 in bf16 and 47 in fp16, 47 and 57 where rows are no
// whole pieces; at depth 256 6 and 13, 58 and 65, and 94 in fp32 there. Deep heads and such rows are the farthest from their bytes, in
// calls of 8 texts of 1,000 tokens, 12 heads: bf16 of 128 51 us (19 at a copy's rate), one element off whole pieces 76, of 100 114,
// of 256 178; fp32 of 128 161, of 256 592 (41 and 165 by its matrix unit).
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

constexpr int kWaves = 4;                // of a work-group
constexpr uint32_t kRows = 16 * kWaves;  // tokens of a chunk
constexpr uint32_t kCols = 16 * kWaves;  // of v, a work-group's
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
  bool exact = false;  // the state is a result
  bool wide = false;   // fp32
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
  /// Segments whose own state is made, of a text that is cut: the last one's too where a result follows from it.
  __host__ __device__ uint32_t parts() const { return state_out ? segments : segments - 1; }
};

/// The passes of one launch: the gradients' three, which have nothing to wait for in one another.
struct AttentionPasses {
  AttentionPass pass[3];
};

/// One of the launch's passes, where its arguments lie: a copy with a varying index would go to memory of its own.
__device__ __forceinline__ const AttentionPass& pass_of(uint32_t i) {
  typedef const __attribute__((address_space(4))) AttentionPass* Constant;
  return *(const AttentionPass*)((Constant)__builtin_amdgcn_kernarg_segment_ptr() + i);
}

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

/// Where a column of v lies in LDS: columns 32 u + 8 g + 4 t + i, i = 0 .. 3, at 16 (2 u + t) + 4 g + i, so that a lane's accumulators
/// of blocks 2 u and 2 u + 1 are eight neighbours of a result's row, and four lanes' are 32.
__device__ __forceinline__ uint32_t place(uint32_t c) { return 32 * (c >> 5) + 16 * (c >> 2 & 1) + 4 * (c >> 3 & 3) + (c & 3); }
__device__ __forceinline__ uint32_t column_at(uint32_t p) { return 32 * (p >> 5) + 8 * (p >> 2 & 3) + 4 * (p >> 4 & 1) + (p & 3); }

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
  // Zero times each: NaN for infinities and NaN.
  float sum = 0.0f;
  if constexpr (sizeof(T) == 2) {
    typedef T x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const x2 two = {v[2 * i], v[2 * i + 1]};
      if constexpr (std::is_same<T, half_t>::value) {
        sum = __builtin_amdgcn_fdot2(two, x2{}, sum, false);
      } else {
        sum = __builtin_amdgcn_fdot2_f32_bf16(two, x2{}, sum, false);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fmaf(v[i], 0.0f, sum);
  }
  return sum == 0.0f;
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

/// One chunk's operands on their way from memory.
template <class T, int KD, bool STATES>
struct ChunkLoads {
  using X8 = typename Op<T>::x8;
  X8 k[KD / 32], v[kWaves / 2], q[STATES ? 1 : KD / 32];
};

/// A tensor's rows of one head of one text, `rows` of them from token `first` of the pass on, in chunks of 64. WHOLE: a buffer that
/// holds them and no more; offsets of 32 bits run through it, forwards or back, and loads outside give zeros, so nothing has to
/// ask for the text's end. Otherwise ordinary loads, element by element where a row ends inside a piece.
template <class T, bool WHOLE>
struct ChunkRows {
  using X8 = typename Op<T>::x8;
  const char* base;  // the first row of the pass; or of the chunk
  int64_t step;      // bytes from row to row of the pass
  uint64_t left;     // rows from the chunk on
  __amdgpu_buffer_rsrc_t buffer;
  uint32_t cols;

  __device__ __forceinline__ ChunkRows(const TokenTensor& t, uint32_t text, uint32_t head, uint32_t col, uint32_t dim, bool back, uint64_t length,
                                       uint64_t first, uint64_t rows)
      : step(static_cast<int64_t>(t.token * sizeof(T))), left(rows), cols(dim - col) {
    base = static_cast<const char*>(t.base) + (text * t.batch + head / t.share * t.head + col) * sizeof(T);
    base += (back ? static_cast<int64_t>(length) - 1 - static_cast<int64_t>(first) : static_cast<int64_t>(first)) * step;
    if (back) step = -step;
    if constexpr (WHOLE) {
      const char* low = back && rows > 0 ? base + static_cast<int64_t>(rows - 1) * step : base;
      const int64_t bytes = rows > 0 ? static_cast<int64_t>(rows - 1) * (back ? -step : step) + static_cast<int64_t>(cols * sizeof(T)) : 0;
      buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(low), 0, static_cast<int>(bytes), 0x27000);
    }
  }
  /// Where column c of row r of the first chunk is; what lies in no row stays outside through all chunks (2^31 bytes at most).
  __device__ __forceinline__ uint32_t offset(uint32_t r, uint32_t c) const {
    const uint32_t s = static_cast<uint32_t>(step);
    if (c >= cols) return step < 0 ? 0xFFFFFF00u : 1u << 31;
    return (step < 0 ? -(static_cast<uint32_t>(left) - 1) * s : 0) + r * s + c * sizeof(T);
  }
  __device__ __forceinline__ X8 take(uint32_t offset) const {
    const u32x4_t lo = __builtin_amdgcn_raw_buffer_load_b128(buffer, static_cast<int>(offset), 0, 0);
    if constexpr (sizeof(T) == 2) {
      return __builtin_bit_cast(X8, lo);
    } else {
      const u32x4_t hi = __builtin_amdgcn_raw_buffer_load_b128(buffer, static_cast<int>(offset) + 16, 0, 0);
      return join(__builtin_bit_cast(f32x4_t, lo), __builtin_bit_cast(f32x4_t, hi));
    }
  }
  /// Eight elements from column c of the chunk's row r.
  __device__ __forceinline__ X8 take(uint32_t r, uint32_t c) const {
    return fetch8(reinterpret_cast<const T*>(base + r * step) + c, r < left && c < cols ? cols - c : 0u);
  }
  __device__ __forceinline__ void advance() {
    base += step * kRows;
    left = left > kRows ? left - kRows : 0;
  }
};

/// WHOLE: rows of q, k and v are whole pieces of eight elements, 16-byte aligned, and a segment spans less than 2^31 bytes.
template <class T, int KD, bool STATES, bool WHOLE>
__global__ void __launch_bounds__(256, (sizeof(T) == 2 && KD <= 128) ? 2 : 1) attention_kernel(AttentionPasses) {
  const AttentionPass& a = pass_of(blockIdx.y);
  using X8 = typename Op<T>::x8;
  using X4 = typename Op<T>::x4;
  constexpr bool kHalf = std::is_same<T, half_t>::value;
  constexpr uint32_t kKS = KD + (sizeof(T) == 2 ? 16 : 4);    // of K, read by rows and by columns
  constexpr uint32_t kS = KD + 16 / sizeof(T);                 // of X in LDS: rows four banks apart
  constexpr uint32_t kVS = kCols + (sizeof(T) == 2 ? 16 : 4);  // of V, read by columns
  constexpr int NX = KD / 16, NK = KD / 32;
  __shared__ __attribute__((aligned(16))) T s_k[kRows * kKS];
  __shared__ __attribute__((aligned(16))) T s_v[kRows * kVS];
  __shared__ __attribute__((aligned(16))) T s_x[STATES ? 16 : kCols * kS];
  __shared__ __attribute__((aligned(16))) float s_unlift[kHalf ? kCols : 4];
  __shared__ uint32_t s_odd[kWaves];

  // Neighbouring heads, whose rows are neighbours in memory, go to one XCD, and the column slices of a head, which read the same
  // q and k, follow one another on it.
  const uint32_t slices = (a.dv + kCols - 1) / kCols, index = blockIdx.x >> 3;
  const uint32_t all = a.batch * a.heads;
  const uint64_t items = static_cast<uint64_t>(all) * (STATES ? a.parts() : a.segments), share = (items + 7) / 8;
  const uint64_t item = (blockIdx.x & 7) * share + index / slices;
  if (index / slices >= share || item >= items) return;
  const uint32_t segment = static_cast<uint32_t>(item / all), bh = static_cast<uint32_t>(item % all);
  const uint32_t text = bh / a.heads, head = bh % a.heads, col0 = index % slices * kCols;
  const uint64_t first = segment * a.segment;
  const uint64_t last = segment + 1 == a.segments ? a.tokens : first + a.segment;  // the segment's tokens end here
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
  const uint64_t here = stop > first ? stop - first : 0;
  using Rows = ChunkRows<T, WHOLE>;
  Rows k_at(a.k, text, head, 0, a.dk, a.reverse, length, first, here), v_at(a.v, text, head, col0, a.dv, a.reverse, length, first, here);
  Rows q_at(STATES ? a.k : a.q, text, head, 0, a.dk, a.reverse, length, first, here);
  uint32_t k_off = k_at.offset(k_row, k_col), v_off = v_at.offset(v_row, v_col), q_off = q_at.offset(q_row, 8 * g);

  const double log2d = log2_decay(a, head);
  const float lg = static_cast<float>(log2d);
  const auto decay = [&](int n) { return __builtin_amdgcn_exp2f(lg * static_cast<float>(n)); };
  float whole_high, whole_low;
  power(log2d, kRows, &whole_high, &whole_low);

  // Factors of the scores, row 16 w + l against s = 16 b + 4 g + i: of the block on the diagonal, of the one before it
  // d^(16 + l - 4 g - i), and d^16 more of each further one. Of v in the update, s = 16 c + 4 g + i: of the last sixteen
  // rows d^(15 - 4 g - i + 1 - ahead), and again d^16 more of those before.
  const auto uniform = [](float f) { return __uint_as_float(static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(__float_as_uint(f))))); };
  float diagonal[4], before[4], within[4], far_factor = 0.0f;
  const float sixteen = uniform(decay(16));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int apart = static_cast<int>(l) - static_cast<int>(4 * g + i);
    diagonal[i] = a.near_scale * decay(apart > 0 ? apart : 0);
    before[i] = a.near_scale * decay(16 + apart);
    within[i] = a.kv_scale * decay(16 - static_cast<int>(4 * g + i + a.ahead));
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
  const auto load = [&] {
    const uint32_t k_step = static_cast<uint32_t>(k_at.step), v_step = static_cast<uint32_t>(v_at.step), q_step = static_cast<uint32_t>(q_at.step);
#pragma unroll
    for (int u = 0; u < KD / 32; ++u) next.k[u] = WHOLE ? k_at.take(k_off + u * kKRows * k_step) : k_at.take(k_row + u * kKRows, k_col);
#pragma unroll
    for (int u = 0; u < kWaves / 2; ++u) next.v[u] = WHOLE ? v_at.take(v_off + u * 32 * v_step) : v_at.take(v_row + u * 32, v_col);
    if constexpr (!STATES) {
#pragma unroll
      for (int kk = 0; kk < NK; ++kk) {
        // dk is KD but for heads of other sizes, whose last pieces may be none.
        const bool none = a.dk < KD && 32 * kk + 8 * g >= a.dk;
        if constexpr (WHOLE) {
          next.q[kk] = q_at.take(none ? (1u << 31) | q_off : q_off + 32 * kk * static_cast<uint32_t>(sizeof(T)));
        } else {
          next.q[kk] = q_at.take(q_row, 32 * kk + 8 * g);
        }
      }
    }
    if constexpr (WHOLE) {
      k_off += kRows * k_step;
      v_off += kRows * v_step;
      q_off += kRows * q_step;
    } else {
      k_at.advance();
      v_at.advance();
      q_at.advance();
    }
  };

  const auto left = [](uint32_t all_of_it, uint32_t from) { return all_of_it <= from ? 0u : WHOLE ? 8u : all_of_it - from; };
  const bool all_columns = col0 + kCols <= a.dv;
  // This lane's columns of a result's row, by eights.
  const auto store_row = [&](uint64_t t, auto&& eight) {
    const uint64_t at = ((text * a.tokens + t) * a.heads + head) * a.dv;
    const auto put = [&](auto* out) {
#pragma unroll
      for (int u = 0; u < kWaves / 2; ++u) {
        const uint32_t c = col0 + 32 * u + 8 * g;
        float v[8];
        eight(u, v);
        if (all_columns) {
          store8(out + at + c, v, 8);
        } else if (left(a.dv, c)) {
          store8(out + at + c, v, left(a.dv, c));
        }
      }
    };
    if (a.out_fp32) return put(static_cast<float*>(a.out));
    put(static_cast<T*>(a.out));
  };

  if (first < stop) load();
  for (uint64_t c0 = first; c0 < stop; c0 += kRows) {
    const uint32_t rows = stop - c0 < kRows ? static_cast<uint32_t>(stop - c0) : kRows;
    // Products of these and what the text's end asks for are made where they are used: kept over the loop they took
    // more registers than there are.
    uint32_t own_g = g, own_l = l, own_dk = a.dk;
    asm volatile("" : "+v"(own_g), "+v"(own_l), "+s"(own_dk));
#pragma unroll
    for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(within[i]), "+v"(before[i]));
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
    for (int u = 0; u < kWaves / 2; ++u) finite = all_finite<T>(next.v[u]) && finite;
    finite = !__any(!finite);
    __syncthreads();  // the last chunk's reads of LDS are done
    if (lane == 0) s_odd[w] = !finite;
    if (kHalf && !STATES && g == 0) s_unlift[16 * w + l] = ldexpf(1.0f, -(x_lift + copy_lift));
#pragma unroll
    for (int u = 0; u < KD / 32; ++u) *reinterpret_cast<X8*>(s_k + (k_row + u * kKRows) * kKS + k_col) = next.k[u];
#pragma unroll
    for (int u = 0; u < kWaves / 2; ++u) {
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
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) any |= s_odd[i];
    const bool odd = __builtin_amdgcn_readfirstlane(static_cast<int>(any)) != 0;
    if (c0 + kRows < stop) load();

    // Whole chunks of finite values have no questions to ask.
    const auto results = [&](auto slow) {
      constexpr bool kSlow = decltype(slow)::value;
      if constexpr (!STATES) {
        // Scores of this wave's rows, decayed, zeros where s comes later, two blocks at a time so that their products follow
        // one another closely.
        float p[kHalf ? kWaves : 1][4], own[4] = {};  // own: the scores of the block on the diagonal
        X8 pb[kWaves / 2];
        float away[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) away[i] = before[i];
#pragma unroll
        for (int m = kWaves / 2 - 1; m >= 0; --m) {
          f32x4_t acc[2]{};
          if (sizeof(T) == 2 || 2 * m <= static_cast<int>(w)) {
#pragma unroll
            for (int kk = 0; kk < NK; ++kk) {
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                if (sizeof(T) == 4 && 2 * m + u > static_cast<int>(w)) continue;
                acc[u] = Op<T>::mma(*reinterpret_cast<const X8*>(s_k + (32 * m + 16 * u + l) * kKS + 32 * kk + 8 * g), qf[kk], acc[u]);
              }
            }
          }
#pragma unroll
          for (int u = 1; u >= 0; --u) {
            const int b = 2 * m + u, at = static_cast<int>(w);
            float y[4];
            if (b < at) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                y[i] = acc[u][i] * away[i];
                away[i] *= sixteen;
              }
            } else if (b == at) {  // a choice, not a factor of zero: scores behind the mask may be infinite
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                y[i] = 4 * own_g + i <= own_l ? acc[u][i] * diagonal[i] : 0.0f;
                if (kSlow) own[i] = y[i];
              }
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i) y[i] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if constexpr (kHalf) {
                p[b][i] = y[i];
              } else {
                pb[m][4 * u + i] = static_cast<T>(y[i]);
              }
            }
          }
        }
        // What the state gives.
        f32x4_t o[kWaves]{};
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) {
#pragma unroll
          for (int j = 0; j < kWaves; ++j) o[j] = Op<T>::mma(*reinterpret_cast<const X8*>(s_x + (16 * j + l) * kS + 32 * kk + 8 * g), qf[kk], o[j]);
        }
        int p_lift = 0;  // float16: this row's scores and sums are 2^p_lift as large
        if constexpr (kHalf) {
          float most = 0.0f;
#pragma unroll
          for (int b = 0; b < kWaves; ++b) {
#pragma unroll
            for (int i = 0; i < 4; ++i) most = fmaxf(most, fabsf(p[b][i]));
          }
          most = fmaxf(most, __shfl_xor(most, 16, 64));
          most = fmaxf(most, __shfl_xor(most, 32, 64));
          p_lift = lift(most, 13, 40);
          const float factor = ldexpf(far_factor, p_lift);
#pragma unroll
          for (int b = 0; b < kWaves; ++b) {
            const f32x4_t unlift = *reinterpret_cast<const f32x4_t*>(s_unlift + 16 * b + 4 * g);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              pb[b >> 1][4 * (b & 1) + i] = static_cast<T>(ldexpf(p[b][i], p_lift));
              o[b][i] *= unlift[i] * factor;
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < kWaves; ++j) o[j] *= far_factor;
        }
        // Scores that the mask takes away are zeros; against infinities and NaN of v they would still count. There those of v
        // are left out, and the ones that the mask lets through are added by themselves.
#pragma unroll
        for (uint32_t m = 0; m < kWaves / 2; ++m) {
          if (sizeof(T) == 4 && 2 * m > w) continue;
#pragma unroll
          for (int j = 0; j < kWaves; ++j) {
            X4 v0 = column4(s_v, kVS, 32 * m, 16 * j), v1 = column4(s_v, kVS, 32 * m + 16, 16 * j);
            if (kSlow && odd && 2 * m >= w) v0 = only_finite(v0);
            if (kSlow && odd && 2 * m + 1 >= w) v1 = only_finite(v1);
            o[j] = Op<T>::mma(join(v0, v1), pb[m], o[j]);
          }
        }
        if (kSlow && odd) {
          if constexpr (kHalf) {
#pragma unroll
            for (int i = 0; i < 4; ++i) own[i] = ldexpf(own[i], p_lift);
          }
#pragma unroll 1
          for (uint32_t s = 0; s < 16; ++s) {
            const uint32_t i0 = s & 3;
            const float mine = i0 == 0 ? own[0] : i0 == 1 ? own[1] : i0 == 2 ? own[2] : own[3];
            const float score = __shfl(mine, static_cast<int>(l + 16 * (s >> 2)), 64);
#pragma unroll
            for (int j = 0; j < kWaves; ++j) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float value = static_cast<float>(s_v[(16 * w + s) * kVS + 16 * j + 4 * g + i]);
                if (s <= l && !is_finite(value)) o[j][i] = fmaf(score, value, o[j][i]);
              }
            }
          }
        }
        if (!kSlow || c0 + q_row < last) {
          store_row(token(c0 + q_row), [&](int u, float (&v)[8]) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float y = o[2 * u + (e >> 2)][e & 3];
              v[e] = kSlow && q_row >= rows ? 0.0f : kHalf ? ldexpf(y, -p_lift) : y;
            }
          });
        }
      }

    };
    const auto update = [&](auto slow, auto exact) {
      constexpr bool kSlow = decltype(slow)::value, kExact = decltype(exact)::value;
      // X: this wave's columns. v times its decay in fp32, as three bfloat16 parts or two float16 ones, against k as it is. Where
      // nobody asks for the state, whose copy has 8 bits or 11, two parts do, and a decay rounded to fp32.
      constexpr int kParts = sizeof(T) == 4 ? 1 : kHalf || !kExact ? 2 : 3;
      // m from the last to the first, `scale` from `within` on.
      const auto weighed = [&](int m, float (&scale)[4], float (&y)[8]) {
        const X8 vf = join(column4(s_v, kVS, 32 * m, 16 * w), column4(s_v, kVS, 32 * m + 16, 16 * w));
#pragma unroll
        for (int u = 1; u >= 0; --u) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float weight = scale[i];
            if (kSlow && rows < kRows) {
              const int after = static_cast<int>(rows - a.ahead) - static_cast<int>(32 * m + 16 * u + 4 * own_g + i);
              weight = a.kv_scale * decay(after > 0 ? after : 0);
            }
            y[4 * u + i] = static_cast<float>(vf[4 * u + i]) * weight;
            scale[i] *= sixteen;
          }
        }
      };
      float high = whole_high, low = whole_low;
      if (kSlow && rows < kRows) power(log2d, rows, &high, &low);
      if constexpr (kHalf) {
        // Behind a power of two by columns, as large as float16 and X's own size allow.
        float most = 0.0f, scale[4] = {within[0], within[1], within[2], within[3]};
#pragma unroll
        for (int m = kWaves / 2 - 1; m >= 0; --m) {
          float y[8];
          weighed(m, scale, y);
#pragma unroll
          for (int e = 0; e < 8; ++e) most = fmaxf(most, kSlow && odd && !is_finite(y[e]) ? 0.0f : fabsf(y[e]));
        }
        most = fmaxf(most, __shfl_xor(most, 16, 64));
        most = fmaxf(most, __shfl_xor(most, 32, 64));
        int new_lift = x_lift;
        if (most > 0.0f) {
          const int top = 14 - ilogbf(most), room = 100 - (x_size - x_lift);
          new_lift = top < room ? top : room;
        }
        high = ldexpf(high, new_lift - x_lift);
        low = ldexpf(low, new_lift - x_lift);
        x_lift = new_lift;
      }
      // The decay's second float counts over many chunks; times an infinity it would be NaN.
      if (!kExact || settled) {
#pragma unroll
        for (int n = 0; n < NX; ++n) x[n] *= high;
      } else {
#pragma unroll
        for (int n = 0; n < NX; ++n) {
#pragma unroll
          for (int i = 0; i < 4; ++i) x[n][i] = fmaf(x[n][i], high, x[n][i] * low);
        }
      }
      settled = settled || (kSlow && odd);
      float scale[4] = {within[0], within[1], within[2], within[3]};
#pragma unroll
      for (int m = kWaves / 2 - 1; m >= 0; --m) {
        X8 part[kParts];
        float rest[8];
        weighed(m, scale, rest);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if constexpr (kHalf) rest[e] = ldexpf(rest[e], x_lift);
#pragma unroll
          for (int z = 0; z < kParts; ++z) {
            part[z][e] = static_cast<T>(rest[e]);
            if (z + 1 < kParts) rest[e] -= static_cast<float>(part[z][e]);
          }
        }
        if (kSlow && odd) {  // an infinity has no lower parts
#pragma unroll
          for (int z = 1; z < kParts; ++z) part[z] = only_finite(part[z]);
        }
#pragma unroll
        for (int n0 = 0; n0 < NX; n0 += 4) {
          X8 kf[4];
#pragma unroll
          for (int n = 0; n < 4; ++n) kf[n] = join(column4(s_k, kKS, 32 * m, 16 * (n0 + n)), column4(s_k, kKS, 32 * m + 16, 16 * (n0 + n)));
          if (kSlow && odd && kParts > 1) {
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              const X8 lower = only_finite(kf[n]);  // zeros among v's lower parts are none of v's
#pragma unroll
              for (int z = kParts - 1; z >= 0; --z) x[n0 + n] = Op<T>::mma(z ? lower : kf[n], part[z], x[n0 + n]);
            }
          } else {
#pragma unroll
            for (int z = kParts - 1; z >= 0; --z) {
#pragma unroll
              for (int n = 0; n < 4; ++n) x[n0 + n] = Op<T>::mma(kf[n], part[z], x[n0 + n]);
            }
          }
        }
      }
      if (kSlow && odd && own_dk < KD) {  // rows that X does not have stay zeros
#pragma unroll
        for (int n = 0; n < NX; ++n) {
#pragma unroll
          for (int i = 0; i < 4; ++i) x[n][i] = 16 * n + 4 * own_g + i < own_dk ? x[n][i] : 0.0f;
        }
      }
    };
    if (odd || rows < kRows) {
      results(std::true_type{});
      update(std::true_type{}, std::true_type{});
    } else {
      results(std::false_type{});
      if (sizeof(T) == 4 || (a.exact && (STATES || a.segments == 1))) {
        update(std::false_type{}, std::true_type{});
      } else {
        update(std::false_type{}, std::false_type{});
      }
    }
  }

  if constexpr (!STATES) {
    // Tokens past the text's end, in chunks of their own.
    const uint64_t done = first < stop ? first + (stop - first + kRows - 1) / kRows * kRows : first;
    for (uint64_t t = done + q_row; t < last; t += kRows) {
      store_row(t, [](int, float (&v)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.0f;
      });
    }
  }
  float* to = nullptr;
  uint64_t sk = a.dv, sv = 1;
  if constexpr (STATES) {
    to = a.states + (static_cast<uint64_t>(segment) * all + bh) * a.dk * a.dv;
  } else if (a.state_out && a.segments == 1) {
    to = a.state_out + static_cast<uint64_t>(bh) * a.dk * a.dv;
    sk = a.state_dk;
    sv = a.state_dv;
  }
  if (!to) return;
  uint32_t dk = a.dk;
  asm volatile("" : "+s"(sk), "+s"(sv), "+s"(dk));  // the addresses anew: kept over the loop, they took more registers than there are
  const uint32_t c = col0 + column_at(16 * w + l);
#pragma unroll
  for (int n = 0; n < NX; ++n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t r = 16 * n + 4 * g + i;
      if (r < dk && c < a.dv) to[r * sk + c * sv] = kHalf ? ldexpf(x[n][i], -x_lift) : x[n][i];
    }
  }
}

/// From what each segment leaves by itself to what it starts from, and what the last one leaves.
__global__ void __launch_bounds__(256) attention_scan_kernel(AttentionPasses) {
  const AttentionPass& a = pass_of(blockIdx.z);
  const uint32_t all = a.batch * a.heads, bh = blockIdx.y;
  const uint32_t size = a.dk * a.dv, at = blockIdx.x * 256 + threadIdx.x;
  if (at >= size) return;
  const uint64_t length = length_of(a, bh / a.heads);
  const double log2d = log2_decay(a, bh % a.heads);
  float x = 0.0f;
  const uint64_t place_of_state = static_cast<uint64_t>(bh) * size + static_cast<uint64_t>(at / a.dv) * a.state_dk + static_cast<uint64_t>(at % a.dv) * a.state_dv;
  if (a.state) x = a.state[place_of_state];
  float* s = a.states + static_cast<uint64_t>(bh) * size + at;
  const uint64_t step = static_cast<uint64_t>(all) * size;
  float high, low;
  power(log2d, a.segment, &high, &low);
  for (uint32_t i = 0; i < a.segments; ++i) {
    const float own = i < a.parts() ? s[i * step] : 0.0f;
    s[i * step] = x;
    const uint64_t from = i * a.segment, n = length > from ? length - from : 0;
    if (n < a.segment) power(log2d, n, &high, &low);
    x = is_finite(x) ? fmaf(x, high, fmaf(x, low, own)) : fmaf(x, high, own);
  }
  if (a.state_out) a.state_out[place_of_state] = x;
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

/// The recurrence itself up to here, by chunks above. Both sides, us: one text, 16 heads of 64 bf16, two tokens 5.7 and 8.2, four 7.9
/// and 8.2, eight 12.5 and 8.3; 64 texts, 16 heads of 128, two 32 and 54, four 43 and 54, eight 65 and 54.
constexpr uint64_t kFewTokens = 4;

template <class F>
void with_depth(uint32_t dk, F&& f) {
  if (dk <= 64) return f(std::integral_constant<int, 64>{});
  if (dk <= 128) return f(std::integral_constant<int, 128>{});
  f(std::integral_constant<int, 256>{});
}

/// Whether launches take so many segments of `all` texts and heads.
bool fits(uint64_t all, uint64_t segments, uint64_t slices) {
  return segments == 1 || (all < (uint64_t{1} << 16) && ceil_div(all * segments, 8) * 8 * slices * 256 < kGridThreads);
}

/// Segments of a pass that is launched with `together` - 1 others like it: enough to fill the device, with work-groups of four chunks
/// or more, where there is less than a work-group for most CUs. (A CU holds two of them, or one of a deep or fp32 head.) The
/// segments' states are a third to a half of the pass again. Both sides, us, one segment and more: 8 texts of 4,096 tokens, 16
/// heads of 128 bf16 (256 work-groups) 202 and 223 in two; 4 texts, 8 heads of 256 (128) 345 and 269 in two; one of 32,768, 16
/// heads of 128 (32) 1,400 and 235 in sixteen, 247 in 32; one of 4,096, 8 heads of 64 (8) 113 and 28 in sixteen.
void cut(AttentionPass& a, uint32_t together) {
  const uint64_t groups = ceil_div(a.dv, kCols) * a.batch * a.heads * together;
  const uint64_t chunks = std::max<uint64_t>(ceil_div(a.tokens, kRows), 1);
  const uint64_t at_once = a.dk <= (a.wide ? 64u : 128u) ? 512 : 256;
  uint64_t segments = groups >= 192 || groups == 0 ? 1 : std::max<uint64_t>(1, at_once / groups);
  segments = std::max<uint64_t>(1, std::min(segments, chunks / 4));
  // Rows far apart: segments that a buffer of 2^31 bytes holds, with room for the chunks around, where that can be and the launches have
  // room for as many; else whole texts by ordinary loads.
  const uint64_t apart = std::max({a.q.token, a.k.token, a.v.token}) * 4, most = apart ? (uint64_t{1} << 31) / apart / kRows : chunks + 4;
  const uint64_t all = static_cast<uint64_t>(a.batch) * a.heads;
  if (most > 8 && fits(all, ceil_div(chunks, most - 4), ceil_div(std::max(a.dk, a.dv), kCols))) {
    segments = std::max(segments, ceil_div(chunks, most - 4));
  }
  const uint64_t each = ceil_div(chunks, segments);
  a.segment = each * kRows;
  a.segments = static_cast<uint32_t>(ceil_div(chunks, each));
}

uint64_t state_bytes(const AttentionPass& a) {
  return a.segments > 1 ? static_cast<uint64_t>(a.segments) * a.batch * a.heads * a.dk * a.dv * sizeof(float) : 0;
}

/// Whether rows of a tensor are whole pieces that lie apart, and a segment's fit a buffer (attention_kernel's WHOLE). The other way costs
/// half as much again: 8 texts of 4,096 tokens, 16 heads of 128 bf16 at whole pieces 222 us, one element further 355.
bool whole_rows(const AttentionPass& a, const TokenTensor& t, uint32_t dim, size_t size) {
  const uint64_t odd = reinterpret_cast<uintptr_t>(t.base) | t.batch * size | t.token * size | t.head * size;
  return dim % 8 == 0 && odd % 16 == 0 && t.token >= dim && (a.segment + 2 * kRows) * t.token * size < (uint64_t{1} << 31);
}

/// `count` passes of one shape: the same dk and dv (or their swap, within one depth), texts and heads. Each is cut by itself, so some
/// may be whole texts: those have no states in the workspace, and are not among the passes that make them.
template <class T>
void launch_passes(const AttentionPasses& p, uint32_t count, hipStream_t s) {
  AttentionPasses cut_ones;
  uint32_t cut_count = 0;
  bool whole = true;
  uint32_t depth = 0, segments = 1, parts = 0;
  uint64_t slices = 1, size = 0;
  for (uint32_t i = 0; i < count; ++i) {
    const AttentionPass& a = p.pass[i];
    whole = whole && whole_rows(a, a.q, a.dk, sizeof(T)) && whole_rows(a, a.k, a.dk, sizeof(T)) && whole_rows(a, a.v, a.dv, sizeof(T));
    depth = std::max(depth, a.dk);
    segments = std::max(segments, a.segments);
    if (a.segments > 1) {
      QVH_REQUIRE(a.states != nullptr, "linear attention: a text in segments without their states");
      parts = std::max(parts, a.parts());
      cut_ones.pass[cut_count++] = a;
    }
    slices = std::max(slices, ceil_div(a.dv, kCols));
    size = std::max<uint64_t>(size, static_cast<uint64_t>(a.dk) * a.dv);
  }
  const uint64_t all = static_cast<uint64_t>(p.pass[0].batch) * p.pass[0].heads;
  QVH_REQUIRE(fits(all, segments, slices), "linear attention: too many segments for one launch");
  const auto grid = [&](uint64_t each, uint32_t passes) { return dim3(static_cast<unsigned>(ceil_div(all * each, 8) * 8 * slices), passes); };
  with_depth(depth, [&](auto kd) {
    constexpr int KD = decltype(kd)::value;
    const auto go = [&](auto rows) {
      constexpr bool WHOLE = decltype(rows)::value;
      if (cut_count > 0) {
        hipLaunchKernelGGL((attention_kernel<T, KD, true, WHOLE>), grid(parts, cut_count), dim3(256), 0, s, cut_ones);
        QVH_HIP(hipGetLastError());
        hipLaunchKernelGGL(attention_scan_kernel, dim3(static_cast<unsigned>(ceil_div(size, 256)), static_cast<unsigned>(all), cut_count), dim3(256), 0,
                           s, cut_ones);
        QVH_HIP(hipGetLastError());
      }
      hipLaunchKernelGGL((attention_kernel<T, KD, false, WHOLE>), grid(segments, count), dim3(256), 0, s, p);
      QVH_HIP(hipGetLastError());
    };
    whole ? go(std::true_type{}) : go(std::false_type{});
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
  QVH_REQUIRE(a.batch * a.heads <= (uint64_t{1} << 21), who + ": batch times heads must be at most 2^21");
  QVH_REQUIRE(!a.lengths || a.index_bytes == 4 || a.index_bytes == 8, who + ": lengths must be int32 or int64");
  QVH_REQUIRE(std::isfinite(a.scale), who + ": scale must be finite");
  if (a.batch == 0) return false;
  if (a.state && a.state_out && a.state != a.state_out) {
    const uint64_t size = a.batch * a.heads * a.dk * a.dv;
    QVH_REQUIRE(a.state + size <= a.state_out || a.state_out + size <= a.state, who + ": state_out overlaps a part of state");
  }
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
  a.wide = in.dtype == QVH_FP32;
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
  a.exact = in.state_out != nullptr;
  a.state_dk = in.dv;
  a.state_dv = 1;
  a.near_scale = a.far_scale = in.scale;
  cut(a, 1);
  return a;
}

/// The three passes of the gradients, and where their workspaces lie: the segments' states and shared heads' gradients.
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
  a.exact = false;
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
  g.v.exact = in.grad_first != nullptr;
  // dk: the same, transposed.
  g.k = a;
  g.k.dk = f.dv;
  g.k.dv = f.dk;
  g.k.q = v;
  g.k.k = o;
  g.k.v = q;
  g.k.state_dk = 1;
  g.k.state_dv = f.dv;
  char* at = static_cast<char*>(workspace);
  const auto take = [&](uint64_t bytes) {
    char* p = at ? at + g.bytes : nullptr;
    g.bytes += ceil_div(bytes, 16) * 16;
    return reinterpret_cast<float*>(p);
  };
  for (AttentionPass* p : {&g.q, &g.k, &g.v}) {
    cut(*p, 3);
    const uint64_t bytes = state_bytes(*p);
    p->states = bytes > 0 ? take(bytes) : nullptr;
  }
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
      launch_passes<T>(AttentionPasses{{a, {}, {}}}, 1, s);
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
      launch_passes<T>(AttentionPasses{{g.q, g.k, g.v}}, 3, s);
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
