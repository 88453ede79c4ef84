// The norm over all gradients of a model, and the gradients scaled down to a limit: |g| = sqrt(sum of x^2), and each
// element times min(1, max_norm / (|g| + eps)).
//
// The tensors' addresses and sizes go with the launch (up to kTable of them, so a call can be captured and needs no copy to the
// device); a work-group finds the tensor of a chunk of kChunk elements by bisection. One launch leaves a sum of squares per
// work-group in fp64, which neither the range of fp32 nor the number of elements troubles; each work-group of the
// second adds them up, all in the same order, and scales its chunks. No atomics: a call repeats bit for bit. Memory
// bounds both launches: 335 million gradients of 290 tensors, 670 MB, 400 us a call in three launches of each, the norm 153, the
// scaling, which reads them again, 245. Fourteen small tensors: 4.2 and 4.9.
#include <algorithm>
#include <cmath>
#include <iterator>
#include <utility>
#include <vector>

#include "types16.hpp"

namespace qvh {
namespace {

constexpr uint32_t kTable = 120;        // tensors of a launch: its arguments stay below 4 KB
constexpr uint32_t kChunk = 8192;       // elements: 256 threads, eight vectors of four or four of eight each
constexpr uint32_t kClipGroups = 2048;  // eight work-groups a CU

constexpr uint64_t kMostGradients = uint64_t{1} << 20;

struct ClipTable {
  const void* in[kTable];
  void* out[kTable];
  uint64_t size[kTable];
  uint32_t chunk[kTable];  // the tensor's first
  uint8_t dtype[kTable];
  uint32_t tensors = 0, chunks = 0;
};
static_assert(sizeof(ClipTable) <= 3900, "arguments of a launch");

/// The tensor of a chunk: the last one that does not start behind it.
__device__ __forceinline__ uint32_t tensor_of(const ClipTable& t, uint32_t chunk) {
  uint32_t lo = 0, hi = t.tensors;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (t.chunk[mid] <= chunk) {
      lo = mid;
    } else {
      hi = mid;
    }
  }
  return lo;
}

/// Calls f<T>(first element, how many) for a chunk.
template <bool BACK, class F>
__device__ __forceinline__ void with_chunk(const ClipTable& t, uint32_t chunk, F&& f) {
  const uint32_t i = tensor_of(t, chunk), at = chunk - t.chunk[i];
  const uint64_t chunks = (t.size[i] + kChunk - 1) / kChunk;
  const uint64_t from = (BACK ? chunks - 1 - at : at) * kChunk, left = t.size[i] - from;
  const uint32_t n = left < kChunk ? static_cast<uint32_t>(left) : kChunk;
  if (t.dtype[i] == QVH_FP32) return f(static_cast<const float*>(t.in[i]) + from, static_cast<float*>(t.out[i]) + from, n);
  if (t.dtype[i] == QVH_FP16) return f(static_cast<const half_t*>(t.in[i]) + from, static_cast<half_t*>(t.out[i]) + from, n);
  f(static_cast<const bhalf_t*>(t.in[i]) + from, static_cast<bhalf_t*>(t.out[i]) + from, n);
}

/// The sum over the work-group's four waves, in every thread.
__device__ __forceinline__ double group_sum(double v, double* s) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  return (s[0] + s[1]) + (s[2] + s[3]);
}

template <class T>
__device__ __forceinline__ double squares(const T* x, uint32_t n) {
  constexpr uint32_t V = 16 / sizeof(T), kEach = kChunk / (256 * V);
  double sum = 0.0;
  if (n == kChunk) {
    float v[kEach][V];
#pragma unroll
    for (uint32_t u = 0; u < kEach; ++u) load_floats<T, V>(x + (u * 256 + threadIdx.x) * V, v[u]);
#pragma unroll
    for (uint32_t u = 0; u < kEach; ++u) {
#pragma unroll
      for (uint32_t e = 0; e < V; ++e) sum = fma(static_cast<double>(v[u][e]), static_cast<double>(v[u][e]), sum);
    }
    return sum;
  }
  uint32_t i = threadIdx.x * V;
  for (; i + V <= n; i += 256 * V) {
    float v[V];
    load_floats<T, V>(x + i, v);
#pragma unroll
    for (uint32_t e = 0; e < V; ++e) sum = fma(static_cast<double>(v[e]), static_cast<double>(v[e]), sum);
  }
  for (; i < n; ++i) {  // of one thread, less than a vector
    const double v = static_cast<float>(x[i]);
    sum = fma(v, v, sum);
  }
  return sum;
}

__global__ void __launch_bounds__(256) clip_norm_kernel(ClipTable t, double* __restrict__ parts) {
  __shared__ double s_sum[4];
  double sum = 0.0;
  for (uint32_t c = blockIdx.x; c < t.chunks; c += gridDim.x) {
    with_chunk<false>(t, c, [&](auto* x, auto*, uint32_t n) { sum += squares(x, n); });
  }
  sum = group_sum(sum, s_sum);
  if (threadIdx.x == 0) parts[blockIdx.x] = sum;
}

template <class T, bool PAST>
__device__ __forceinline__ void scaled(const T* x, T* out, uint32_t n, float factor, int power) {
  constexpr uint32_t V = 16 / sizeof(T), kEach = kChunk / (256 * V);
  if (n == kChunk) {
    float v[kEach][V];
#pragma unroll
    for (uint32_t u = 0; u < kEach; ++u) load_floats<T, V>(x + (u * 256 + threadIdx.x) * V, v[u]);
#pragma unroll
    for (uint32_t u = 0; u < kEach; ++u) {
#pragma unroll
      for (uint32_t e = 0; e < V; ++e) v[u][e] = ldexpf(v[u][e] * factor, power);
      store_floats<T, V, PAST>(out + (u * 256 + threadIdx.x) * V, v[u]);
    }
    return;
  }
  uint32_t i = threadIdx.x * V;
  for (; i + V <= n; i += 256 * V) {
    float v[V];
    load_floats<T, V>(x + i, v);
#pragma unroll
    for (uint32_t e = 0; e < V; ++e) v[e] = ldexpf(v[e] * factor, power);
    store_floats<T, V>(out + i, v);
  }
  for (; i < n; ++i) out[i] = static_cast<T>(ldexpf(static_cast<float>(x[i]) * factor, power));
}

/// All parts added up, in every thread, the same bits in every work-group.
__device__ __forceinline__ double all_parts(const double* __restrict__ parts, uint32_t count, double* s) {
  double sum = 0.0;
  for (uint32_t i = threadIdx.x; i < count; i += 256) sum += parts[i];
  return group_sum(sum, s);
}

/// From the last gradient to the first, and each backwards: what the norm read last may still be in the last-level cache.
/// PAST: results that the L2s cannot hold are stored past them, and leave the last-level cache to the gradients: 335 million, 670
/// MB, 400 us a call, 440 without.
template <bool PAST>
__global__ void __launch_bounds__(256) clip_scale_kernel(ClipTable t, const double* __restrict__ parts, uint32_t count,
                                                         float max_norm, float eps, float* __restrict__ norm) {
  __shared__ double s_sum[4];
  const double n = sqrt(all_parts(parts, count, s_sum));
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(n);
  const double over = n + static_cast<double>(eps);
  const double ratio = over == 0.0 ? 1.0 : static_cast<double>(max_norm) / over;  // zeros stay
  // Factors near the end of fp32's range and past it, which it would round or lose, as one in [0.5, 1) and a power of two.
  int power = 0;
  const float factor = ratio >= 1.0 ? 1.0f : static_cast<float>(ratio < 0x1p-100 ? frexp(ratio, &power) : ratio);  // NaN stays
  for (uint32_t c = blockIdx.x; c < t.chunks; c += gridDim.x) {
    with_chunk<true>(t, c, [&](auto* x, auto* out, uint32_t k) {
      if (factor != 1.0f || power != 0 || x != out) scaled<std::remove_pointer_t<decltype(out)>, PAST>(x, out, k, factor, power);
    });
  }
}

/// The norm alone.
__global__ void __launch_bounds__(256) norm_result_kernel(const double* __restrict__ parts, uint32_t count, float* __restrict__ norm) {
  __shared__ double s_sum[4];
  const double n = sqrt(all_parts(parts, count, s_sum));
  if (threadIdx.x == 0) *norm = static_cast<float>(n);
}

uint64_t chunks_of(const qvh_gradient& g) { return ceil_div(g.count, kChunk); }

uint32_t groups_of(uint64_t chunks, uint64_t all) {
  return static_cast<uint32_t>(std::min<uint64_t>(chunks, ceil_div(chunks * kClipGroups, all)));
}

/// Results lie apart from one another, and from every gradient but their own.
void check_apart(const char* who, const qvh_gradient* g, uint64_t n) {
  const std::string w(who);
  typedef std::pair<uintptr_t, uintptr_t> Span;
  const auto span = [&](const void* p, uint64_t i) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    return Span(at, at + g[i].count * dtype_size(g[i].dtype));
  };
  std::vector<Span> outs;
  outs.reserve(n);
  for (uint64_t i = 0; i < n; ++i) {
    if (g[i].count) outs.push_back(span(g[i].out, i));
  }
  std::sort(outs.begin(), outs.end());
  for (size_t i = 1; i < outs.size(); ++i) QVH_REQUIRE(outs[i - 1].second <= outs[i].first, w + ": results overlap");
  for (uint64_t i = 0; i < n; ++i) {
    if (g[i].count == 0 || g[i].out == g[i].grad) continue;
    const Span in = span(g[i].grad, i);
    const auto next = std::lower_bound(outs.begin(), outs.end(), Span(in.second, 0));  // the first that starts behind it
    QVH_REQUIRE(next == outs.begin() || std::prev(next)->second <= in.first, w + ": a result overlaps another gradient");
  }
}

void check_gradients(const char* who, const qvh_gradient* g, uint64_t n, bool results) {
  const std::string w(who);
  QVH_REQUIRE(n == 0 || g != nullptr, w + ": null list of gradients");
  QVH_REQUIRE(n <= kMostGradients, w + ": at most 2^20 gradients");
  uint64_t chunks = 0;
  for (uint64_t i = 0; i < n; ++i) {
    require_dtype(who, g[i].dtype);
    QVH_REQUIRE(g[i].count <= (uint64_t{1} << 40), w + ": a gradient has more than 2^40 elements");
    QVH_REQUIRE(g[i].count == 0 || (g[i].grad && (!results || g[i].out)), w + ": null gradient");
    chunks += chunks_of(g[i]);
  }
  QVH_REQUIRE(chunks < (uint64_t{1} << 31), w + ": too many elements in all");
}

/// Calls f(table, work-groups, parts before it) for every launch; from the last gradient to the first where `back`.
template <class F>
uint32_t each_table(const qvh_gradient* g, uint64_t n, bool back, F&& f) {
  uint64_t all = 0;
  for (uint64_t i = 0; i < n; ++i) all += chunks_of(g[i]);
  ClipTable t;
  uint32_t parts = 0;
  const auto flush = [&] {
    const uint32_t groups = groups_of(t.chunks, all);
    f(t, groups, parts);
    parts += groups;
    t.tensors = t.chunks = 0;
  };
  for (uint64_t at = 0; at < n; ++at) {
    const uint64_t i = back ? n - 1 - at : at;
    if (g[i].count == 0) continue;
    const uint32_t k = t.tensors++;
    t.in[k] = g[i].grad;
    t.out[k] = g[i].out;
    t.size[k] = g[i].count;
    t.chunk[k] = t.chunks;
    t.dtype[k] = static_cast<uint8_t>(g[i].dtype);
    t.chunks += static_cast<uint32_t>(chunks_of(g[i]));
    if (t.tensors == kTable) flush();
  }
  if (t.tensors) flush();
  return parts;
}

uint32_t count_parts(const qvh_gradient* g, uint64_t n) {
  return each_table(g, n, false, [](const ClipTable&, uint32_t, uint32_t) {});
}

void run_norm(const qvh_gradient* g, uint64_t n, double* parts, hipStream_t s) {
  each_table(g, n, false, [&](const ClipTable& t, uint32_t groups, uint32_t before) {
    hipLaunchKernelGGL(clip_norm_kernel, dim3(groups), dim3(256), 0, s, t, parts + before);
    QVH_HIP(hipGetLastError());
  });
}

}  // namespace
}  // namespace qvh

extern "C" {

qvh_status qvh_grad_norm_workspace(uint64_t count, uint64_t* bytes) {
  return qvh::guarded([&] {
    using namespace qvh;
    QVH_REQUIRE(bytes != nullptr, "qvh_grad_norm_workspace: null output");
    QVH_REQUIRE(count <= kMostGradients, "qvh_grad_norm_workspace: at most 2^20 gradients");
    // A launch rounds its share of the work-groups up.
    *bytes = count == 0 ? 0 : (kClipGroups + ceil_div(count, kTable)) * sizeof(double);
  });
}

qvh_status qvh_grad_norm_device(const qvh_gradient* grads, uint64_t count, float* d_norm, void* d_workspace,
                                uint64_t workspace_bytes, void* stream) {
  return qvh::guarded([&] {
    using namespace qvh;
    const char* who = "qvh_grad_norm_device";
    check_gradients(who, grads, count, false);
    QVH_REQUIRE(d_norm != nullptr, std::string(who) + ": null norm");
    const uint32_t parts = count_parts(grads, count);
    check_workspace(who, d_workspace, workspace_bytes, parts * sizeof(double));
    const DeviceScope device;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    run_norm(grads, count, static_cast<double*>(d_workspace), s);
    hipLaunchKernelGGL(norm_result_kernel, dim3(1), dim3(256), 0, s, static_cast<const double*>(d_workspace), parts, d_norm);
    QVH_HIP(hipGetLastError());
  });
}

qvh_status qvh_clip_grad_norm_device(const qvh_gradient* grads, uint64_t count, float max_norm, float eps, float* d_norm,
                                     void* d_workspace, uint64_t workspace_bytes, void* stream) {
  return qvh::guarded([&] {
    using namespace qvh;
    const char* who = "qvh_clip_grad_norm_device";
    check_gradients(who, grads, count, true);
    check_apart(who, grads, count);
    QVH_REQUIRE(max_norm >= 0.0f && max_norm < __builtin_huge_valf(), std::string(who) + ": max_norm must be finite and not negative");
    QVH_REQUIRE(eps >= 0.0f && eps < __builtin_huge_valf(), std::string(who) + ": eps must be finite and not negative");
    const uint32_t parts = count_parts(grads, count);
    check_workspace(who, d_workspace, workspace_bytes, parts * sizeof(double));
    const DeviceScope device;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    double* sums = static_cast<double*>(d_workspace);
    if (parts == 0) {  // no elements at all
      if (d_norm) {
        hipLaunchKernelGGL(norm_result_kernel, dim3(1), dim3(256), 0, s, sums, 0u, d_norm);
        QVH_HIP(hipGetLastError());
      }
      return;
    }
    run_norm(grads, count, sums, s);
    uint64_t bytes = 0;
    for (uint64_t i = 0; i < count; ++i) bytes += grads[i].count * dtype_size(grads[i].dtype);
    const auto kernel = bytes >= kStreamed ? clip_scale_kernel<true> : clip_scale_kernel<false>;
    each_table(grads, count, true, [&](const ClipTable& t, uint32_t groups, uint32_t before) {
      hipLaunchKernelGGL(kernel, dim3(groups), dim3(256), 0, s, t, sums, parts, max_norm, eps, before == 0 ? d_norm : nullptr);
      QVH_HIP(hipGetLastError());
    });
  });
}

}  // extern "C"
