// The way from one block of an encoder to the next, in one pass, and its gradient:
//
//   u = y / sqrt(mean(y^2) + eps) * post        the norm behind the block
//   r = x + scale * act(gate) * u               the residual stream
//   h = r / sqrt(mean(r^2) + eps) * weight      the norm in front of the next block
//
// Backwards, with a = dh * weight, rn = r / sqrt(..), yn = y / sqrt(..), D columns:
//
//   dx = dr + (a - rn mean(a rn)) / sqrt(mean(r^2) + eps)        dweight = sum of dh rn over the rows
//   dgate = dx scale u act'(gate)                                dscale = sum of dx act(gate) u
//   du = dx scale act(gate), b = du post                         dpost = sum of du yn
//   dy = (b - yn mean(b yn)) / sqrt(mean(y^2) + eps)
//
// A row stays in registers from its load to its last store, so every matrix is read or written once, and the vectors
// are loaded once per work-group, which takes many rows. Memory bounds it: forward five matrices, backward eight.
// Rows of up to 64 pieces of 16 bytes belong to a wave or a part of one (8, 16 or 32 lanes, so that short rows leave few
// lanes idle) and need no barrier; longer ones to two, four, eight or sixteen waves. 16,384 x 1,024 bf16 with a gate and a
// scale: forward 30 us, 168 MB at 5.6 TB/s; backward 55 and 4.7 for the sums, 268 MB at 4.5; 24 x 768 forward 4.2, the launch. The columns' sums of the
// backward pass stay in registers too, over all rows of a work-group, and a second launch adds the work-groups' parts
// up in order: no atomics, the same bits each time.
//
// Backward rows past 4,096 columns do not fit: sixteen waves leave a thread 128 registers, and with a block a row, the next one, three
// vectors and three sums take more, so that parts of them lie in scratch memory, by the compiler's report 61 to 77 registers of
// 16-bit rows up to 8,192 columns and 264 to 279 past them, 100 to 180 and 457 to 639 of fp32 ones. That bounds them: 16.8 million
// elements with a gate and a scale, calls in a row, 4,096 columns bf16 63 us and fp32 110, 5,000 237 and 403, 8,192 166 and 296, 16,384
// 469 and 676. Without a block only the widest do (10 to 17, fp32 129): 27, 29, 27, 36 us and 43, 45, 46, 127. Forward rows
// fit but for fp32 past 8,192 with a gate (25): 30, 45, 35, 39 us and 61, 72, 70, 90.
#include <algorithm>

#include "gemm.hpp"

namespace qvh {
namespace {

constexpr uint32_t kMaxNorm = 16384;  // columns

struct NormArgs {
  uint64_t rows = 0;
  uint32_t dim = 0, lanes = 0;  // lanes of a row that is a part of a wave
  int act = QVH_ACT_NONE;
  float eps = 0.0f, share = 0.0f;  // 1 / dim
  const void *x = nullptr, *y = nullptr, *gate = nullptr, *weight = nullptr, *post = nullptr, *scale = nullptr;
  uint64_t x_stride = 0, y_stride = 0, gate_stride = 0;
  // forward: results; backward: x is r, and the gradients
  void *r = nullptr, *h = nullptr;
  const void *grad_h = nullptr, *grad_r = nullptr;
  uint64_t grad_h_stride = 0, grad_r_stride = 0;
  void *grad_x = nullptr, *grad_y = nullptr, *grad_gate = nullptr;
  float* parts = nullptr;  // [weight, post, scale][work-group][dim rounded up to 8]
};

/// The sum over the threads that share a row, in all of them. s: a slot per wave, not in use by other threads.
template <int W>
__device__ __forceinline__ float row_sum(float v, uint32_t lanes, float* s) {
  const auto add = [&](int stride) { v += __uint_as_float(lane_xor_u32(__float_as_uint(v), stride)); };
  add(1);
  add(2);
  add(4);
  if (W > 1 || lanes > 8) add(8);
  if (W > 1 || lanes > 16) add(16);
  if (W > 1 || lanes > 32) add(32);
  if constexpr (W > 1) {
    const uint32_t wave = threadIdx.x >> 6, first = wave / W * W;
    if ((threadIdx.x & 63) == 0) s[wave] = v;
    __syncthreads();
    v = s[first];
#pragma unroll
    for (int w = 1; w < W; ++w) v += s[first + w];
  }
  return v;
}

/// act(gate), and its slope. The logistic function in fp32's last bits for every type: memory bounds these kernels.
__device__ __forceinline__ float open_gate(float z, int act, float* slope) {
  if (act == QVH_ACT_NONE) {
    *slope = 1.0f;
    return z;
  }
  float other;
  float s = logistic<true>(z, &other);
  s = z != z ? z : s;
  if (act == QVH_ACT_SIGMOID) {
    *slope = s * other;
    return s;
  }
  *slope = s * fmaf(z, other, 1.0f);
  return z * s;
}

/// Where a thread's pieces of a row lie. The last piece of a row is moved back to end with it (vector_width); `again`
/// is how many of its elements the piece before has too, which sums over the row count once.
template <int V, int P>
struct Pieces {
  uint32_t col[P], again[P];
  bool on[P];
  __device__ __forceinline__ Pieces(uint32_t thread, uint32_t threads, uint32_t dim) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const uint32_t c = (thread + p * threads) * V;
      on[p] = c < dim;
      col[p] = c + V <= dim ? c : dim - V;
      again[p] = on[p] ? c - col[p] : 0;
    }
  }
};

template <class T, int V, int P>
__device__ __forceinline__ void load_row(const void* base, uint64_t at, const Pieces<V, P>& k, bool valid, Loose<T, V> (&out)[P]) {
  const T* p0 = static_cast<const T*>(base) + at;
#pragma unroll
  for (int p = 0; p < P; ++p) {
    out[p] = Loose<T, V>{};
    if (valid && k.on[p]) out[p] = *reinterpret_cast<const Loose<T, V>*>(p0 + k.col[p]);
  }
}

template <class T, int V, int P, class F>
__device__ __forceinline__ void store_row(void* base, uint64_t at, const Pieces<V, P>& k, bool valid, F&& value) {
  T* p0 = static_cast<T*>(base) + at;
#pragma unroll
  for (int p = 0; p < P; ++p) {
    if (!(valid && k.on[p])) continue;
    Loose<T, V> o;
#pragma unroll
    for (int i = 0; i < V; ++i) o.v[i] = static_cast<T>(value(p, i));
    *reinterpret_cast<Loose<T, V>*>(p0 + k.col[p]) = o;
  }
}

/// W waves and P pieces a thread for a row, or (W = 1) a.lanes of a wave.
template <class T, int V, int W, int P, bool BLOCK, bool GATE>
__global__ void __launch_bounds__(W == 1 ? 256 : W * 64) norm_kernel(NormArgs a) {
  __shared__ float s_sum[2][W];
  const uint32_t lanes = W == 1 ? a.lanes : W * 64;
  const uint32_t thread = threadIdx.x & (lanes - 1);
  const uint64_t per_group = W == 1 ? 256 / lanes : 1;
  const Pieces<V, P> k(thread, lanes, a.dim);
  Loose<T, V> weight[P], post[P], scale[P];
  load_row<T, V, P>(a.weight, 0, k, true, weight);
  if constexpr (BLOCK) {
    load_row<T, V, P>(a.post, 0, k, true, post);
    if (a.scale) load_row<T, V, P>(a.scale, 0, k, true, scale);
  }
  // The first row of the wave decides, so that a wave stays together.
  const uint64_t lead = blockIdx.x * per_group + (W == 1 ? (threadIdx.x & ~63u) / lanes : 0);
  const uint64_t own = W == 1 ? (threadIdx.x & 63) / lanes : 0;
  for (uint64_t row0 = lead; row0 < a.rows; row0 += gridDim.x * per_group) {
    const uint64_t row = row0 + own;
    const bool valid = row < a.rows;
    Loose<T, V> x[P], y[P], gate[P];
    load_row<T, V, P>(a.x, row * a.x_stride, k, valid, x);
    float r[P][V], sum = 0.0f;
    if constexpr (BLOCK) {
      load_row<T, V, P>(a.y, row * a.y_stride, k, valid, y);
      if constexpr (GATE) load_row<T, V, P>(a.gate, row * a.gate_stride, k, valid, gate);
#pragma unroll
      for (int p = 0; p < P; ++p) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float v = static_cast<uint32_t>(i) >= k.again[p] ? static_cast<float>(y[p].v[i]) : 0.0f;
          sum = fmaf(v, v, sum);
        }
      }
      const float inv = 1.0f / sqrtf(fmaf(row_sum<W>(sum, lanes, s_sum[0]), a.share, a.eps));
      sum = 0.0f;
#pragma unroll
      for (int p = 0; p < P; ++p) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float u = static_cast<float>(y[p].v[i]) * inv * static_cast<float>(post[p].v[i]);
          if constexpr (GATE) {
            float slope;
            u *= open_gate(static_cast<float>(gate[p].v[i]), a.act, &slope);
          }
          if (a.scale) u *= static_cast<float>(scale[p].v[i]);
          r[p][i] = static_cast<float>(x[p].v[i]) + u;
        }
      }
      store_row<T, V, P>(a.r, row * a.dim, k, valid, [&](int p, int i) { return r[p][i]; });
    } else {
#pragma unroll
      for (int p = 0; p < P; ++p) {
#pragma unroll
        for (int i = 0; i < V; ++i) r[p][i] = static_cast<float>(x[p].v[i]);
      }
    }
#pragma unroll
    for (int p = 0; p < P; ++p) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float v = static_cast<uint32_t>(i) >= k.again[p] && k.on[p] ? r[p][i] : 0.0f;
        sum = fmaf(v, v, sum);
      }
    }
    const float inv = 1.0f / sqrtf(fmaf(row_sum<W>(sum, lanes, s_sum[1]), a.share, a.eps));
    store_row<T, V, P>(a.h, row * a.dim, k, valid, [&](int p, int i) { return r[p][i] * inv * static_cast<float>(weight[p].v[i]); });
    // Without a block every row uses the same slots.
    if constexpr (W > 1 && !BLOCK) __syncthreads();
  }
}

/// The matrices' pieces of one row.
template <class T, int V, int P, bool BLOCK, bool GATE>
struct GradRow {
  Loose<T, V> r[P], dh[P], dr[P], y[BLOCK ? P : 1], gate[GATE ? P : 1];
  __device__ __forceinline__ void load(const NormArgs& a, uint64_t row, const Pieces<V, P>& k, bool valid) {
    load_row<T, V, P>(a.x, row * a.x_stride, k, valid, r);
    load_row<T, V, P>(a.grad_h, row * a.grad_h_stride, k, valid, dh);
    if (a.grad_r) load_row<T, V, P>(a.grad_r, row * a.grad_r_stride, k, valid, dr);
    if constexpr (BLOCK) load_row<T, V, P>(a.y, row * a.y_stride, k, valid, y);
    if constexpr (GATE) load_row<T, V, P>(a.gate, row * a.gate_stride, k, valid, gate);
  }
};

/// The threads of a backward work-group.
constexpr int grad_threads(int W) { return W <= 4 ? 256 : W * 64; }

/// A work-group has as many rows at a time as its waves make up; the next ones are loaded while these are computed.
template <class T, int V, int W, int P, bool BLOCK, bool GATE>
__global__ void __launch_bounds__(grad_threads(W)) norm_grad_kernel(NormArgs a) {
  constexpr int kGroup = grad_threads(W), kWaves = kGroup / 64;
  __shared__ float s_sum[4][kWaves];
  const uint32_t lanes = W == 1 ? a.lanes : W * 64;
  const uint32_t thread = threadIdx.x & (lanes - 1);
  const uint64_t per_group = kGroup / lanes;
  const Pieces<V, P> k(thread, lanes, a.dim);
  Loose<T, V> weight[P], post[P], scale[P];
  load_row<T, V, P>(a.weight, 0, k, true, weight);
  if constexpr (BLOCK) {
    load_row<T, V, P>(a.post, 0, k, true, post);
    if (a.scale) load_row<T, V, P>(a.scale, 0, k, true, scale);
  }
  float sums[BLOCK ? 3 : 1][P][V] = {};
  // The first row of the wave decides (of the work-group, where a row has several waves), so that it stays together.
  const uint64_t in_wave = W == 1 ? (threadIdx.x & 63) / lanes : threadIdx.x / lanes;
  const uint64_t step = gridDim.x * per_group;
  uint64_t row0 = blockIdx.x * per_group + (W == 1 ? (threadIdx.x & ~63u) / lanes : 0);
  GradRow<T, V, P, BLOCK, GATE> next;
  if (row0 < a.rows) next.load(a, row0 + in_wave, k, row0 + in_wave < a.rows);
  for (; row0 < a.rows; row0 += step) {
    const uint64_t row = row0 + in_wave;
    const bool valid = row < a.rows;
    const GradRow<T, V, P, BLOCK, GATE> now = next;
    if (row0 + step < a.rows) next.load(a, row + step, k, row + step < a.rows);
    float rr = 0.0f, ar = 0.0f, yy = 0.0f;
#pragma unroll
    for (int p = 0; p < P; ++p) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const bool once = static_cast<uint32_t>(i) >= k.again[p] && k.on[p];
        const float v = once ? static_cast<float>(now.r[p].v[i]) : 0.0f;
        rr = fmaf(v, v, rr);
        const float g = once ? static_cast<float>(now.dh[p].v[i]) * static_cast<float>(weight[p].v[i]) : 0.0f;
        ar = fmaf(g, v, ar);
        if constexpr (BLOCK) {
          const float w = once ? static_cast<float>(now.y[p].v[i]) : 0.0f;
          yy = fmaf(w, w, yy);
        }
      }
    }
    rr = row_sum<W>(rr, lanes, s_sum[0]);
    ar = row_sum<W>(ar, lanes, s_sum[1]);
    const float inv = 1.0f / sqrtf(fmaf(rr, a.share, a.eps));
    const float along = ar * inv * a.share;  // mean(a rn)
    float dx[P][V];
#pragma unroll
    for (int p = 0; p < P; ++p) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float rn = static_cast<float>(now.r[p].v[i]) * inv, g = static_cast<float>(now.dh[p].v[i]);
        // A row past the last adds nothing, whatever its factors (eps may be 0, and the row's norm with it).
        if (valid) sums[0][p][i] = fmaf(g, rn, sums[0][p][i]);
        dx[p][i] = inv * fmaf(-rn, along, g * static_cast<float>(weight[p].v[i]));
        if (a.grad_r) dx[p][i] += static_cast<float>(now.dr[p].v[i]);
      }
    }
    if (a.grad_x) store_row<T, V, P>(a.grad_x, row * a.dim, k, valid, [&](int p, int i) { return dx[p][i]; });
    if constexpr (BLOCK) {
      yy = row_sum<W>(yy, lanes, s_sum[2]);
      const float inv_y = 1.0f / sqrtf(fmaf(yy, a.share, a.eps));
      float by = 0.0f;
      float dgate[P][V];
#pragma unroll
      for (int p = 0; p < P; ++p) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float yn = static_cast<float>(now.y[p].v[i]) * inv_y, w = static_cast<float>(post[p].v[i]);
          const float u = yn * w;
          float du = dx[p][i], opened = 1.0f;
          if (a.scale) du *= static_cast<float>(scale[p].v[i]);
          if constexpr (GATE) {
            float slope;
            opened = open_gate(static_cast<float>(now.gate[p].v[i]), a.act, &slope);
            dgate[p][i] = du * u * slope;
            du *= opened;
          }
          if (valid) {
            sums[2][p][i] = fmaf(dx[p][i] * opened, u, sums[2][p][i]);
            sums[1][p][i] = fmaf(du, yn, sums[1][p][i]);
          }
          dx[p][i] = du * w;  // b
          if (static_cast<uint32_t>(i) >= k.again[p] && k.on[p]) by = fmaf(dx[p][i], yn, by);
        }
      }
      if constexpr (GATE) {
        if (a.grad_gate) store_row<T, V, P>(a.grad_gate, row * a.dim, k, valid, [&](int p, int i) { return dgate[p][i]; });
      }
      const float along_y = row_sum<W>(by, lanes, s_sum[3]) * a.share;
      if (a.grad_y) {
        store_row<T, V, P>(a.grad_y, row * a.dim, k, valid, [&](int p, int i) {
          return inv_y * fmaf(-(static_cast<float>(now.y[p].v[i]) * inv_y), along_y, dx[p][i]);
        });
      }
    }
  }

  // This work-group's part of the columns' sums.
  const uint64_t ld = (a.dim + 7) / 8 * 8;
  constexpr int kVectors = BLOCK ? 3 : 1;
  const auto put = [&](int which, const float (&v)[P][V]) {
    float* out = a.parts + (static_cast<uint64_t>(which) * gridDim.x + blockIdx.x) * ld;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      if (k.on[p]) store_floats<float, V <= 4 ? V : 4>(out + k.col[p], reinterpret_cast<const float(&)[V <= 4 ? V : 4]>(v[p]));
      if constexpr (V == 8) {
        if (k.on[p]) store_floats<float, 4>(out + k.col[p] + 4, reinterpret_cast<const float(&)[4]>(v[p][4]));
      }
    }
  };
  if constexpr (W * 64 == kGroup) {
#pragma unroll
    for (int which = 0; which < kVectors; ++which) put(which, sums[which]);
  } else {
    // Rows of one wave first, then of the work-group's waves.
    constexpr int kRowGroups = kWaves / W;
    __shared__ float s_col[kRowGroups][W * 64 * P * V + 4];
    const uint32_t group = threadIdx.x / (W * 64), own = threadIdx.x & (W * 64 - 1);
#pragma unroll
    for (int which = 0; which < kVectors; ++which) {
#pragma unroll
      for (int p = 0; p < P; ++p) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float v = sums[which][p][i];
          if (lanes <= 8) v += __uint_as_float(lane_xor_u32(__float_as_uint(v), 8));
          if (lanes <= 16) v += __uint_as_float(lane_xor_u32(__float_as_uint(v), 16));
          if (lanes <= 32) v += __uint_as_float(lane_xor_u32(__float_as_uint(v), 32));
          s_col[group][(p * W * 64 + own) * V + i] = v;
        }
      }
      __syncthreads();
      if (threadIdx.x < lanes) {
        float total[P][V];
#pragma unroll
        for (int p = 0; p < P; ++p) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < kRowGroups; ++w) v += s_col[w][(p * W * 64 + own) * V + i];
            total[p][i] = v;
          }
        }
        put(which, total);
      }
      __syncthreads();
    }
  }
}

struct NormSums {
  const float* parts = nullptr;
  uint32_t count = 0, dim = 0;
  void* out[3] = {};
};

/// The work-groups' parts of 64 columns of one vector, in order: sixteen waves take contiguous shares of them.
template <class T>
__global__ void __launch_bounds__(1024) norm_sums_kernel(NormSums a) {
  __shared__ float s_sum[16][64];
  T* out = static_cast<T*>(blockIdx.y == 0 ? a.out[0] : blockIdx.y == 1 ? a.out[1] : a.out[2]);
  if (!out) return;
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
  const uint64_t ld = (a.dim + 7) / 8 * 8;
  const float* parts = a.parts + static_cast<uint64_t>(blockIdx.y) * a.count * ld + c;
  const uint32_t share = (a.count + 15) / 16, p0 = wave * share, p1 = p0 + share < a.count ? p0 + share : a.count;
  float t[8] = {};
  if (c < a.dim) {
    for (uint32_t p = p0; p < p1; p += 8) {
#pragma unroll
      for (uint32_t u = 0; u < 8; ++u) t[u] += p + u < p1 ? parts[(p + u) * ld] : 0.0f;
    }
  }
  s_sum[wave][lane] = sum8(t);
  __syncthreads();
  if (wave == 0 && c < a.dim) {
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < 16; ++w) v += s_sum[w][lane];
    out[c] = static_cast<T>(v);
  }
}

/// Calls f<V, W, P>() for rows of `dim` elements of T; `lanes` are a row's threads: one piece each as long as sixteen waves reach
/// (two pieces of a wave: 16,384 x 1,024 bf16 forward 30.5 us, backward 113; one of two waves 30.0 and 59), and as few lanes
/// of a wave as hold the row (10,007 x 100 fp32 on 32 lanes 5.2 us forward and 14.1 backward, on 64 6.7 and 17.4; 100,000 x 64
/// bf16 on 8 lanes 10.1, on 64 39.9).
template <class T, class F>
void with_shape(uint32_t dim, uint32_t* lanes, F&& f) {
  constexpr int V = 16 / sizeof(T);
  using std::integral_constant;
  const auto go = [&](auto v, auto w, auto p, uint32_t n) {
    *lanes = n;
    f(v, w, p);
  };
  const integral_constant<int, V> v;
  const integral_constant<int, 1> one;
  const integral_constant<int, 2> two;
  const integral_constant<int, 4> four;
  const integral_constant<int, 8> eight;
  const integral_constant<int, 16> sixteen;
  if (dim < V) return go(one, one, one, 8u);
  const uint32_t pieces = static_cast<uint32_t>(ceil_div(dim, V));
  if (pieces <= 64) return go(v, one, one, pieces <= 8 ? 8u : pieces <= 16 ? 16u : pieces <= 32 ? 32u : 64u);
  if (pieces <= 128) return go(v, two, one, 128u);
  if (pieces <= 256) return go(v, four, one, 256u);
  if (pieces <= 512) return go(v, eight, one, 512u);
  if (pieces <= 1024) return go(v, sixteen, one, 1024u);
  if (sizeof(T) == 2 || pieces <= 2048) return go(v, sixteen, two, 1024u);
  if constexpr (sizeof(T) == 4) go(v, sixteen, four, 1024u);
}

template <class F>
void with_parts(bool block, bool gate, F&& f) {
  if (!block) return f(std::false_type{}, std::false_type{});
  if (!gate) return f(std::true_type{}, std::false_type{});
  f(std::true_type{}, std::true_type{});
}

/// Work-groups of a backward pass, two a CU or fewer: as many parts of every vector's sums. Measured where a thread has 182 registers
/// (16,384 x 1,024 bf16 with a gate: 512 of them 55 us, 768 63). fp32 rows take 122 at most and would leave room for four a CU; for
/// them more were not measured (10,007 x 100 fp32 takes 11.4 us of 6.3 by its bytes, its last round of rows less than half full).
uint32_t grad_groups(uint64_t rows, uint32_t dim, int dtype) {
  uint64_t groups = 0;
  uint32_t lanes = 0;
  with_dtype(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    with_shape<T>(dim, &lanes, [&](auto, auto w, auto) {
      constexpr int W = decltype(w)::value;
      groups = std::min<uint64_t>(ceil_div(rows, grad_threads(W) / lanes), W <= 4 ? 512 : 256);
    });
  });
  return static_cast<uint32_t>(groups);
}

uint64_t grad_bytes(uint64_t rows, uint32_t dim, int dtype, bool block) {
  return (block ? 3 : 1) * ceil_div(dim, 8) * 8 * sizeof(float) * static_cast<uint64_t>(grad_groups(rows, dim, dtype));
}

void check_shape(const char* who, uint64_t rows, uint32_t dim, int dtype, int act, float eps) {
  require_dtype(who, dtype);
  QVH_REQUIRE(dim > 0 && dim <= kMaxNorm, std::string(who) + ": dim must be in [1, 16384]");
  QVH_REQUIRE(rows < (uint64_t{1} << 31), std::string(who) + ": rows must be below 2^31");
  QVH_REQUIRE(act == QVH_ACT_NONE || act == QVH_ACT_SILU || act == QVH_ACT_SIGMOID,
              std::string(who) + ": a gate's activation must be none, silu or sigmoid");
  QVH_REQUIRE(eps >= 0.0f && eps < __builtin_huge_valf(), std::string(who) + ": eps must be finite and not negative");
}

void check_matrix(const char* who, const char* name, const void* p, uint64_t stride, uint64_t rows, uint32_t dim) {
  QVH_REQUIRE(rows == 0 || p != nullptr, std::string(who) + ": null " + name);
  QVH_REQUIRE(stride >= dim && stride <= (uint64_t{1} << 22), std::string(who) + ": " + name + "'s stride must be in [dim, 2^22]");
}

void check_forward(const qvh_block_norm_args* args) {
  const char* who = "qvh_block_norm_device";
  QVH_REQUIRE(args != nullptr, std::string(who) + ": null arguments");
  const qvh_block_norm_args& a = *args;
  check_shape(who, a.rows, a.dim, a.dtype, a.gate_activation, a.eps);
  check_matrix(who, "x", a.x, a.x_stride, a.rows, a.dim);
  QVH_REQUIRE(a.weight != nullptr, std::string(who) + ": null weight");
  QVH_REQUIRE(a.rows == 0 || a.h != nullptr, std::string(who) + ": null h");
  if (a.y) {
    check_matrix(who, "y", a.y, a.y_stride, a.rows, a.dim);
    QVH_REQUIRE(a.post_weight != nullptr, std::string(who) + ": null post_weight");
    QVH_REQUIRE(a.rows == 0 || a.r != nullptr, std::string(who) + ": null r");
    if (a.gate) check_matrix(who, "gate", a.gate, a.gate_stride, a.rows, a.dim);
  } else {
    QVH_REQUIRE(a.rows == 0 || (!a.gate && !a.post_weight && !a.scale), std::string(who) + ": a gate, post_weight and scale belong to y");
  }
}

void check_backward(const char* who, const qvh_block_norm_grad_args* args) {
  QVH_REQUIRE(args != nullptr, std::string(who) + ": null arguments");
  const qvh_block_norm_grad_args& a = *args;
  check_shape(who, a.rows, a.dim, a.dtype, a.gate_activation, a.eps);
  check_matrix(who, "grad_h", a.grad_h, a.grad_h_stride, a.rows, a.dim);
  check_matrix(who, "r", a.r, a.r_stride, a.rows, a.dim);
  if (a.grad_r) check_matrix(who, "grad_r", a.grad_r, a.grad_r_stride, a.rows, a.dim);
  QVH_REQUIRE(a.weight != nullptr, std::string(who) + ": null weight");
  if (a.y) {
    check_matrix(who, "y", a.y, a.y_stride, a.rows, a.dim);
    QVH_REQUIRE(a.post_weight != nullptr, std::string(who) + ": null post_weight");
    if (a.gate) check_matrix(who, "gate", a.gate, a.gate_stride, a.rows, a.dim);
    QVH_REQUIRE(a.gate || !a.grad_gate, std::string(who) + ": grad_gate without a gate");
    QVH_REQUIRE(a.scale || !a.grad_scale, std::string(who) + ": grad_scale without a scale");
  } else {
    QVH_REQUIRE(a.rows == 0 || (!a.gate && !a.post_weight && !a.scale && !a.grad_y && !a.grad_gate && !a.grad_post && !a.grad_scale),
                std::string(who) + ": a gate, post_weight, scale and their gradients belong to y");
  }
}

}  // namespace
}  // namespace qvh

extern "C" {

qvh_status qvh_block_norm_device(const qvh_block_norm_args* args, void* stream) {
  return qvh::guarded([&] {
    using namespace qvh;
    check_forward(args);
    const qvh_block_norm_args& in = *args;
    if (in.rows == 0) return;
    const DeviceScope device;
    NormArgs a;
    a.rows = in.rows;
    a.dim = in.dim;
    a.act = in.gate_activation;
    a.eps = in.eps;
    a.share = 1.0f / static_cast<float>(in.dim);
    a.x = in.x;
    a.x_stride = in.x_stride;
    a.y = in.y;
    a.y_stride = in.y_stride;
    a.gate = in.gate;
    a.gate_stride = in.gate_stride;
    a.weight = in.weight;
    a.post = in.post_weight;
    a.scale = in.scale;
    a.r = in.r;
    a.h = in.h;
    with_dtype(in.dtype, [&](auto* t) {
      using T = std::remove_pointer_t<decltype(t)>;
      with_shape<T>(in.dim, &a.lanes, [&](auto v, auto w, auto p) {
        constexpr int V = decltype(v)::value, W = decltype(w)::value, P = decltype(p)::value;
        with_parts(in.y != nullptr, in.gate != nullptr, [&](auto block, auto gate) {
          const uint64_t groups = ceil_div(a.rows, W == 1 ? 256 / a.lanes : 1);
          const uint64_t most = W == 16 ? 512 : 2048;
          hipLaunchKernelGGL((norm_kernel<T, V, W, P, decltype(block)::value, decltype(gate)::value>),
                             dim3(static_cast<unsigned>(std::min(groups, most))), dim3(W == 1 ? 256 : W * 64), 0,
                             static_cast<hipStream_t>(stream), a);
          QVH_HIP(hipGetLastError());
        });
      });
    });
  });
}

qvh_status qvh_block_norm_grad_workspace(uint64_t rows, uint32_t dim, int dtype, int block, uint64_t* bytes) {
  return qvh::guarded([&] {
    QVH_REQUIRE(bytes != nullptr, "qvh_block_norm_grad_workspace: null output");
    qvh::check_shape("qvh_block_norm_grad_workspace", rows, dim, dtype, QVH_ACT_NONE, 0.0f);
    *bytes = qvh::grad_bytes(rows, dim, dtype, block != 0);
  });
}

qvh_status qvh_block_norm_grad_device(const qvh_block_norm_grad_args* args, void* d_workspace, uint64_t workspace_bytes,
                                      void* stream) {
  return qvh::guarded([&] {
    using namespace qvh;
    check_backward("qvh_block_norm_grad_device", args);
    const qvh_block_norm_grad_args& in = *args;
    check_workspace("qvh_block_norm_grad_device", d_workspace, workspace_bytes, grad_bytes(in.rows, in.dim, in.dtype, in.y != nullptr));
    const DeviceScope device;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    NormArgs a;
    a.rows = in.rows;
    a.dim = in.dim;
    a.act = in.gate_activation;
    a.eps = in.eps;
    a.share = 1.0f / static_cast<float>(in.dim);
    a.x = in.r;
    a.x_stride = in.r_stride;
    a.y = in.y;
    a.y_stride = in.y_stride;
    a.gate = in.gate;
    a.gate_stride = in.gate_stride;
    a.weight = in.weight;
    a.post = in.post_weight;
    a.scale = in.scale;
    a.grad_h = in.grad_h;
    a.grad_h_stride = in.grad_h_stride;
    a.grad_r = in.grad_r;
    a.grad_r_stride = in.grad_r_stride;
    a.grad_x = in.grad_x;
    a.grad_y = in.grad_y;
    a.grad_gate = in.grad_gate;
    a.parts = static_cast<float*>(d_workspace);
    const uint32_t groups = grad_groups(in.rows, in.dim, in.dtype);
    with_dtype(in.dtype, [&](auto* t) {
      using T = std::remove_pointer_t<decltype(t)>;
      if (groups > 0) {
        with_shape<T>(in.dim, &a.lanes, [&](auto v, auto w, auto p) {
          constexpr int V = decltype(v)::value, W = decltype(w)::value, P = decltype(p)::value;
          with_parts(in.y != nullptr, in.gate != nullptr, [&](auto block, auto gate) {
            hipLaunchKernelGGL((norm_grad_kernel<T, V, W, P, decltype(block)::value, decltype(gate)::value>), dim3(groups),
                               dim3(grad_threads(W)), 0, s, a);
            QVH_HIP(hipGetLastError());
          });
        });
      }
      NormSums sums;
      sums.parts = a.parts;
      sums.count = groups;
      sums.dim = in.dim;
      sums.out[0] = in.grad_weight;
      sums.out[1] = in.grad_post;
      sums.out[2] = in.grad_scale;
      const unsigned vectors = in.grad_post || in.grad_scale ? 3u : 1u;
      if (vectors == 3 || in.grad_weight) {
        hipLaunchKernelGGL((norm_sums_kernel<T>), dim3(static_cast<unsigned>(ceil_div(in.dim, 64)), vectors), dim3(1024), 0, s, sums);
        QVH_HIP(hipGetLastError());
      }
    });
  });
}

}  // extern "C"
