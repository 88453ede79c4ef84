// Embedding lookup with scaling and its gradient by sorted tokens.
//
// Lookup: y[t] = scale * table[token[t]], a row of zeros where the token is outside the table. One
// pass that reads each named row and writes each output row; memory traffic is the whole cost.
//
// Gradient: dE[v] = scale * sum of dy[t] over the t with token[t] = v, in fp32. The
// tokens are sorted (stable, least significant digit first), so equal tokens are neighbours; waves
// then sum fixed pieces of the sorted list, and runs that cross a piece are joined in order by a
// second launch. Which partial sums are formed depends on the tokens alone, never on timing, so a
// call repeats bit for bit, and a token that fills half of the batch is spread over many waves.
// A small batch takes one launch instead: every wave owns a few rows of the table and looks through
// all tokens for them.
#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "types16.hpp"

namespace qvh {
namespace {

constexpr uint32_t kMaxDim = 32768;

// ---- lookup -----------------------------------------------------------------------------------

/// Piece c of a row is V elements (vector_width), cpr pieces a row; U pieces per thread, 256 apart, so that each
/// thread has U independent row reads in flight. PAST: the result is stored past the L2s. Bound by memory:
/// 250,007 tokens of 100 fp32 (a fifth of them padding) in a table of 1.18 million rows 22 us, the 182 MB it
/// moves at 8 TB/s, some of the rows from the caches; 24 tokens of 768 bf16 2.4 us, the launch.
template <class T, int V, class I, int U, bool PAST>
__global__ void __launch_bounds__(256) embed_kernel(const T* __restrict__ table, uint64_t rows, uint64_t stride,
                                                    const I* __restrict__ tokens, uint64_t count, uint32_t dim,
                                                    uint32_t cpr, uint32_t magic, float scale, T* __restrict__ out) {
  const uint64_t first = static_cast<uint64_t>(blockIdx.x) * (256 * U);
  const uint64_t t0 = first / cpr;
  const uint32_t lead = static_cast<uint32_t>(first - t0 * cpr);
  const uint64_t total = count * cpr;
  uint64_t at[U], row[U];
  uint32_t col[U];
  int64_t tok[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    // (lead + index) / cpr by a multiplication: exact below 2^32 / cpr.
    const uint32_t i = lead + u * 256 + threadIdx.x;
    const uint32_t q = cpr == 1 ? i : __umulhi(i, magic);
    at[u] = first + u * 256 + threadIdx.x;
    row[u] = t0 + q;
    col[u] = (i - q * cpr) * V;
    col[u] = col[u] < dim - V ? col[u] : dim - V;
    tok[u] = at[u] < total ? static_cast<int64_t>(tokens[t0 + q]) : -1;
  }
  float x[U][V];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (tok[u] >= 0 && static_cast<uint64_t>(tok[u]) < rows) {
      load_floats<T, V>(table + static_cast<uint64_t>(tok[u]) * stride + col[u], x[u]);
#pragma unroll
      for (int i = 0; i < V; ++i) x[u][i] *= scale;
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) x[u][i] = 0.0f;
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (at[u] < total) store_floats<T, V, PAST>(out + row[u] * dim + col[u], x[u]);
  }
}

template <class T, class I>
void launch_embed(const void* table, uint64_t rows, uint32_t dim, uint64_t stride, const void* tokens, uint64_t count,
                  float scale, void* out, hipStream_t s) {
  with_width<T>(vector_width(sizeof(T), dim), [&](auto width) {
    constexpr int V = decltype(width)::value;
    const uint32_t cpr = static_cast<uint32_t>(ceil_div(dim, V));
    const uint32_t magic = cpr == 1 ? 0u : static_cast<uint32_t>((uint64_t{1} << 32) / cpr + 1);
    const uint64_t total = count * cpr;
    const auto go = [&](auto unroll, auto past) {
      constexpr int U = decltype(unroll)::value;
      const uint64_t most = kGridThreads / 2 * U / cpr;  // tokens of a launch
      for (uint64_t t = 0; t < count; t += most) {
        const uint64_t n = std::min(most, count - t);
        hipLaunchKernelGGL((embed_kernel<T, V, I, U, decltype(past)::value>), dim3(static_cast<unsigned>(ceil_div(n * cpr, 256 * U))), dim3(256), 0,
                           s, static_cast<const T*>(table), rows, stride, static_cast<const I*>(tokens) + t, n, dim, cpr,
                           magic, scale, static_cast<T*>(out) + t * dim);
        QVH_HIP(hipGetLastError());
      }
    };
    // Two pieces per thread where the device is full several times over; below, one. Both sides, one and two, with
    // the tables in HBM: 250,007 x 100 fp32 35.1 and 32.0 us, 60,000 x 1,024 bf16 40.3 and 36.0; 16,000 x 100
    // fp32 3.8 and 4.2. (Four: 33.1, 36.4, 4.8.) A result that the L2s cannot hold is stored past them, in whole pieces of 16
    // bytes: 250,007 x 1,024 bf16 162 us through them, 143 past; 250,007 x 100 fp32 31.9 and 32.7; a smaller one,
    // 1,050,000 x 9 bf16, 11.2 either way.
    if (total < (1u << 21)) return go(std::integral_constant<int, 1>{}, std::false_type{});
    if constexpr (V * sizeof(T) == 16) {
      if (count * dim * sizeof(T) >= kStreamed) return go(std::integral_constant<int, 2>{}, std::true_type{});
    }
    go(std::integral_constant<int, 2>{}, std::false_type{});
  });
}

// ---- gradient of a small batch: rows look for their tokens ------------------------------------

constexpr uint32_t kOwnTokens = 2048;  // what LDS has room for

/// Rows per wave: as few as there are waves at once, since a wave's rows follow one another, each waiting for its
/// gradient rows (10,000 rows, 1,000 tokens of 128 fp32: four rows 13 us, two 11).
uint32_t own_rows(uint64_t rows, uint64_t count) {
  const uint64_t lds = std::max<uint64_t>(count, 1) * 24;  // per work-group of four waves
  const uint64_t at_once = 256 * 4 * std::min<uint64_t>(8, 160 * 1024 / lds);
  return static_cast<uint32_t>(std::min<uint64_t>(std::max<uint64_t>(ceil_div(rows, at_once), 1), 64));
}

/// Whether a batch is small enough for rows to look for their tokens: by estimates of both ways, in us. The own way
/// is slow where one wave has many tokens to add, one round of loads after another, or many rows to write; the
/// sorted one is six launches or more. (No dtype: rows of 16-bit and 32-bit elements take as many rounds.) Both
/// sides, own way first: 10,000 rows of 128, fp16, 512 tokens 8.2 and 24.4, 2,048 tokens 29.5 and 26.6; 32,000
/// rows of 1,024, 512 tokens 63 and 35; a million rows of 100, 512 tokens 189 and 58; 1,000 of 64, 2,048 tokens
/// 15.6 and 27.1.
bool rows_look(uint64_t rows, uint32_t dim, uint64_t count) {
  if (count > kOwnTokens) return false;
  const uint64_t pieces = ceil_div(dim, 8), lanes = pieces <= 16 ? 16 : pieces <= 32 ? 32 : 64;
  const uint64_t rounds = ceil_div(count, 64 / lanes * 8) * ceil_div(pieces, lanes);
  const uint64_t waves = ceil_div(rows, own_rows(rows, count));
  const uint64_t turns = ceil_div(waves, 256 * 4 * std::min<uint64_t>(8, 160 * 1024 / (std::max<uint64_t>(count, 1) * 24)));
  const double own = 3.0 + 0.25 * static_cast<double>(rounds) + 1.3 * static_cast<double>(turns * own_rows(rows, count));
  const int passes = rows < 256 ? 1 : rows < 65536 ? 2 : rows < (1u << 24) ? 3 : 4;
  const double sorted = 9.0 + 7.5 * passes + static_cast<double>(rows) * dim / 3e6;
  return own < sorted;
}

/// 1,000 tokens in 10,000 rows of 128 fp32: 9.8 us, where the 5 MB of the table and 0.5 MB of gradients would
/// take 1.1; bound by the chain token, match, gradient row of the wave with the most frequent tokens.
/// One wave per `own` rows (at most 64): lists the batch's tokens that fall into its rows, then per row
/// the positions of its tokens, whose gradient rows are added: 64 / G at a time, each by G lanes that take
/// V columns, every such share in order of position and the shares in order.
template <class T, int V, int G, class I>
__global__ void __launch_bounds__(256) embed_grad_own_kernel(const T* __restrict__ grad, uint64_t stride,
                                                             const I* __restrict__ tokens, uint32_t count, uint32_t rows,
                                                             uint32_t dim, uint32_t own, float scale,
                                                             T* __restrict__ out) {
  constexpr uint32_t kShares = 64 / G, kAhead = V >= 8 ? 8 : 16;
  extern __shared__ uint32_t s_own[];  // per wave: count entries of (row - first) << 16 | position, count positions
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t first = (static_cast<uint64_t>(blockIdx.x) * 4 + wave) * own;
  const uint32_t held = first < rows ? (rows - first < own ? static_cast<uint32_t>(rows - first) : own) : 0u;
  uint32_t* list = s_own + wave * count;
  uint16_t* match = reinterpret_cast<uint16_t*>(s_own + 4 * count) + wave * count;
  uint32_t found = 0;
  const uint64_t below = (uint64_t{1} << lane) - 1;
  constexpr int kScan = 16;  // loads under way
  for (uint32_t b0 = 0; b0 < count; b0 += kScan * 64) {
    int64_t tok[kScan];
#pragma unroll
    for (int u = 0; u < kScan; ++u) {
      const uint32_t t = b0 + u * 64 + lane;
      tok[u] = t < count ? static_cast<int64_t>(tokens[t]) : -1;
    }
#pragma unroll
    for (int u = 0; u < kScan; ++u) {
      const uint64_t r = static_cast<uint64_t>(tok[u]) - first;  // wraps to a large value below the first row
      const bool mine = tok[u] >= 0 && r < held;
      const uint64_t mask = __builtin_amdgcn_ballot_w64(mine);
      if (mine) list[found + __popcll(mask & below)] = static_cast<uint32_t>(r) << 16 | (b0 + u * 64 + lane);
      found += static_cast<uint32_t>(__popcll(mask));
    }
  }
  const uint32_t share = lane / G;
  for (uint32_t r = 0; r < held; ++r) {
    uint32_t n = 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the wave's own LDS accesses stay in order
    for (uint32_t b = 0; b < found; b += 64) {
      const uint32_t e = b + lane < found ? list[b + lane] : 0xFFFFFFFFu;
      const uint64_t mask = __builtin_amdgcn_ballot_w64(e >> 16 == r);
      if (e >> 16 == r) match[n + __popcll(mask & below)] = static_cast<uint16_t>(e);
      n += static_cast<uint32_t>(__popcll(mask));
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (uint32_t c0 = 0; c0 < dim; c0 += G * V) {
      uint32_t c = c0 + lane % G * V;
      const bool in = c < dim;
      c = c < dim - V ? c : dim - V;
      float acc[V] = {};
      for (uint32_t j0 = 0; j0 < n; j0 += kShares * kAhead) {
        float x[kAhead][V];
#pragma unroll
        for (uint32_t u = 0; u < kAhead; ++u) {
          const uint32_t j = j0 + u * kShares + share;
          if (in && j < n) {
            load_floats<T, V>(grad + static_cast<uint64_t>(match[j]) * stride + c, x[u]);
          } else {
#pragma unroll
            for (int k = 0; k < V; ++k) x[u][k] = 0.0f;
          }
        }
#pragma unroll
        for (uint32_t u = 0; u < kAhead; ++u) {
#pragma unroll
          for (int k = 0; k < V; ++k) acc[k] += x[u][k];
        }
      }
#pragma unroll
      for (int off = G; off < 64; off <<= 1) {
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] += __shfl_xor(acc[k], off, 64);
      }
#pragma unroll
      for (int k = 0; k < V; ++k) acc[k] *= scale;
      if (in && share == 0) store_floats<T, V>(out + (first + r) * dim + c, acc);
    }
  }
}

// ---- sorting (key, position) pairs ------------------------------------------------------------
//
// Stable counting passes of at most 8 bits, each a count and a scatter. Each of `parts` work-groups has a
// contiguous part of the list; count[part][digit] gives every part its place per digit. (A scatter that
// also counts the next pass's digits by atomics, knowing where its pairs land, took 33 us of 262,144
// tokens instead of 5 + 7: frequent words all count in one place.) Nor does one work-group that
// makes all passes in its LDS gain: 16 us at 5,651 tokens, the four launches 19 with their gaps.

constexpr uint32_t kParts = 128, kBins = 256;
constexpr uint32_t kSortWaves = 8;

/// The token as a key: its row, or `rows` (sorted behind all of them) outside the table.
template <class I>
__device__ __forceinline__ uint32_t token_key(const I* tokens, uint64_t t, uint32_t rows) {
  const int64_t tok = static_cast<int64_t>(tokens[t]);
  return tok >= 0 && static_cast<uint64_t>(tok) < rows ? static_cast<uint32_t>(tok) : rows;
}

template <class I, bool FIRST>
__global__ void __launch_bounds__(512) count_kernel(const I* __restrict__ tokens, const uint32_t* __restrict__ keys,
                                                    uint32_t count, uint32_t part, uint32_t rows, uint32_t shift,
                                                    uint32_t digit_mask, uint32_t* __restrict__ counts) {
  __shared__ uint32_t s_bins[kBins];
  if (threadIdx.x < kBins) s_bins[threadIdx.x] = 0;
  __syncthreads();
  const uint64_t begin = static_cast<uint64_t>(blockIdx.x) * part;
  const uint64_t end = begin + part < count ? begin + part : count;
#pragma unroll 4
  for (uint64_t t = begin + threadIdx.x; t < end; t += 512) {
    const uint32_t key = FIRST ? token_key(tokens, t, rows) : keys[t];
    atomicAdd(&s_bins[key >> shift & digit_mask], 1u);
  }
  __syncthreads();
  if (threadIdx.x < kBins) counts[blockIdx.x * kBins + threadIdx.x] = s_bins[threadIdx.x];
}

/// Lanes that hold the same digit as this one (those of `in` only).
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, uint32_t bits, bool in) {
  uint64_t same = __builtin_amdgcn_ballot_w64(in);
  for (uint32_t k = 0; k < bits; ++k) {
    const uint64_t ones = __builtin_amdgcn_ballot_w64((digit >> k & 1u) != 0);
    same &= (digit >> k & 1u) ? ones : ~ones;
  }
  return same;
}

/// The place of this lane's pair: *next (the wave's next place for the digit, in LDS) plus its rank among the
/// lanes with the same digit.
__device__ __forceinline__ uint32_t take_place(uint32_t* next, uint64_t same, bool in) {
  const uint32_t rank = static_cast<uint32_t>(__popcll(same & ((uint64_t{1} << (threadIdx.x & 63)) - 1)));
  uint32_t base = 0;
  if (in && rank == 0) base = atomicAdd(next, static_cast<uint32_t>(__popcll(same)));
  base = static_cast<uint32_t>(__shfl(static_cast<int>(base), in ? __builtin_ctzll(same) : 0, 64));
  return base + rank;
}

/// Sum of `v` over the threads below, of the first 256; s_waves has four entries. All threads call it.
__device__ __forceinline__ uint32_t scan_256(uint32_t v, uint32_t* s_waves) {
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t run = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t up = static_cast<uint32_t>(__shfl_up(static_cast<int>(run), d, 64));
    run += lane >= static_cast<uint32_t>(d) ? up : 0u;
  }
  if (wave < 4 && lane == 63) s_waves[wave] = run;
  __syncthreads();
  if (wave < 4) {
    for (uint32_t w = 0; w < wave; ++w) run += s_waves[w];
  }
  return run - v;
}

/// One pass. FIRST reads the tokens themselves (positions are the list's order); HELD: a wave's share is at most
/// kHeld rounds, which are loaded once, at the start.
constexpr uint32_t kHeld = 4;
template <class I, bool FIRST, bool HELD>
__global__ void __launch_bounds__(kSortWaves * 64) scatter_kernel(
    const I* __restrict__ tokens, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ positions,
    uint32_t count, uint32_t part, uint32_t rows, uint32_t shift, uint32_t bits, const uint32_t* __restrict__ counts,
    uint32_t* __restrict__ out_keys, uint32_t* __restrict__ out_positions) {
  __shared__ uint32_t s_at[kSortWaves][kBins];
  __shared__ uint32_t s_half[2][kBins];
  __shared__ uint32_t s_waves[4];
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t digit_mask = (1u << bits) - 1;

  // A wave's share of the part is contiguous: the pairs' order is the waves' order.
  const uint64_t begin = static_cast<uint64_t>(blockIdx.x) * part;
  const uint64_t end = begin + part < count ? begin + part : count;
  const uint32_t share = static_cast<uint32_t>(ceil_div(part, kSortWaves * 64)) * 64;
  const uint64_t w0 = begin + static_cast<uint64_t>(wave) * share;
  const uint64_t w1 = w0 + share < end ? w0 + share : end;
  const auto key_at = [&](uint64_t i) { return i < w1 ? (FIRST ? token_key(tokens, i, rows) : keys[i]) : 0u; };
  const auto position_at = [&](uint64_t i) { return FIRST ? static_cast<uint32_t>(i) : i < w1 ? positions[i] : 0u; };
  uint32_t key[kHeld], pos[kHeld];
  if constexpr (HELD) {
#pragma unroll
    for (uint32_t u = 0; u < kHeld; ++u) {
      key[u] = key_at(w0 + u * 64 + lane);
      pos[u] = position_at(w0 + u * 64 + lane);
    }
  }
  // This part's place per digit: all pairs of smaller digits, and this digit's in earlier parts. Two threads
  // per digit, each over half of the parts.
  const uint32_t digit_of = tid % kBins, half = tid / kBins;
  uint32_t before = 0, all = 0;
  {
    const uint32_t p0 = half ? (gridDim.x + 1) / 2 : 0u, p1 = half ? gridDim.x : (gridDim.x + 1) / 2;
    for (uint32_t p = p0; p < p1; p += 16) {
      uint32_t n[16];  // loads in flight together; past the half's end its last one again, for nothing
#pragma unroll
      for (uint32_t u = 0; u < 16; ++u) n[u] = counts[(p + u < p1 ? p + u : p1 - 1) * kBins + digit_of];
#pragma unroll
      for (uint32_t u = 0; u < 16; ++u) {
        before += p + u < p1 && p + u < blockIdx.x ? n[u] : 0u;
        all += p + u < p1 ? n[u] : 0u;
      }
    }
  }
  for (uint32_t i = tid; i < kSortWaves * kBins; i += kSortWaves * 64) (&s_at[0][0])[i] = 0;
  if (half) {
    s_half[0][digit_of] = before;
    s_half[1][digit_of] = all;
  }
  __syncthreads();
  if constexpr (HELD) {
#pragma unroll
    for (uint32_t u = 0; u < kHeld; ++u) {
      if (w0 + u * 64 + lane < w1) atomicAdd(&s_at[wave][key[u] >> shift & digit_mask], 1u);
    }
  } else {
    for (uint64_t i = w0 + lane; i < w1; i += 64) atomicAdd(&s_at[wave][key_at(i) >> shift & digit_mask], 1u);
  }
  if (!half) {
    before += s_half[0][tid];
    all += s_half[1][tid];
  }
  uint32_t at = scan_256(half ? 0u : all, s_waves) + before;  // its barrier is behind the waves' counts
  if (!half) {
#pragma unroll
    for (uint32_t w = 0; w < kSortWaves; ++w) {
      const uint32_t n = s_at[w][tid];
      s_at[w][tid] = at;
      at += n;
    }
  }
  __syncthreads();
  const auto place = [&](uint64_t i, uint32_t k, uint32_t p) {
    const bool in = i < w1;
    const uint32_t digit = k >> shift & digit_mask;
    const uint32_t to = take_place(&s_at[wave][digit], same_digit(digit, bits, in), in);
    if (in) {
      out_keys[to] = k;
      out_positions[to] = p;
    }
  };
  if constexpr (HELD) {
#pragma unroll
    for (uint32_t u = 0; u < kHeld; ++u) place(w0 + u * 64 + lane, key[u], pos[u]);
  } else {
    for (uint64_t b = w0; b < w1; b += 64) place(b + lane, key_at(b + lane), position_at(b + lane));
  }
}

// ---- sums over the sorted list ----------------------------------------------------------------

constexpr uint32_t kMostEntries = 2048;  // sorted entries of a work-group's pieces
constexpr uint32_t kZeroRows = 64;  // table rows that one work-group checks at a time for having no token
constexpr uint64_t kZeroBlocks = 1u << 22;  // work-groups that do so, at most

struct SumArgs {
  const void* grad;
  uint64_t stride;
  const uint32_t* keys;
  const uint32_t* positions;
  uint32_t count, rows, dim;
  float scale;
  void* out;
  float* partial;  // [piece][2][dim]: the run that came from the piece before, the one that goes on
  uint32_t piece;  // sorted entries that one group of lanes adds
  uint32_t pieces, sum_blocks, zero_blocks, slabs;
  uint32_t cpr;
};

/// First index of [0, n) whose key is not below `key`.
__device__ __forceinline__ uint32_t lower_bound(const uint32_t* keys, uint32_t n, uint32_t key) {
  uint32_t lo = 0;
  while (n > 0) {
    const uint32_t half = n >> 1;
    const bool right = keys[lo + half] < key;
    lo = right ? lo + half + 1 : lo;
    n = right ? n - half - 1 : half;
  }
  return lo;
}

/// The same for a whole wave that looks for one key: 64 probes at a time (a run's end among 262,144 entries
/// in three steps for eighteen: 262,144 x 1,024 joined in 16 us for 19).
__device__ __forceinline__ uint32_t wave_lower_bound(const uint32_t* keys, uint32_t n, uint32_t key) {
  const uint32_t lane = threadIdx.x & 63;
  uint32_t lo = 0;
  while (n > 0) {
    const uint32_t step = (n + 63) / 64, i = (lane + 1) * step - 1;
    const uint32_t c = static_cast<uint32_t>(__popcll(__builtin_amdgcn_ballot_w64(i < n && keys[lo + i] < key)));
    lo += c * step;  // the probe behind it, if there is one, is not below the key
    n = n - c * step < step - 1 ? n - c * step : step - 1;
  }
  return lo;
}

/// Rows without a token become zero (work-groups past the sums').
template <class T, int V>
__device__ __forceinline__ void zero_rows(const SumArgs& a, uint32_t block, uint32_t* s_flag) {
  for (uint64_t r0 = static_cast<uint64_t>(block) * kZeroRows; r0 < a.rows; r0 += static_cast<uint64_t>(a.zero_blocks) * kZeroRows) {
    if (threadIdx.x < kZeroRows) {
      const uint64_t r = r0 + threadIdx.x;
      uint32_t touched = 1;
      if (r < a.rows) {
        const uint32_t i = lower_bound(a.keys, a.count, static_cast<uint32_t>(r));
        touched = i < a.count && a.keys[i] == r ? 1u : 0u;
      }
      s_flag[threadIdx.x] = touched;
    }
    __syncthreads();
    const float zero[V] = {};
    T* out = static_cast<T*>(a.out) + r0 * a.dim;
    for (uint32_t i = threadIdx.x; i < kZeroRows * a.cpr; i += 256) {
      const uint32_t row = i / a.cpr, c = (i - row * a.cpr) * V;
      if (!s_flag[row]) store_floats<T, V>(out + static_cast<uint64_t>(row) * a.dim + (c < a.dim - V ? c : a.dim - V), zero);
    }
    __syncthreads();  // the flags are read
  }
}

/// Groups of G lanes, each adding one piece of the list over G * V columns (slab blockIdx.y). Bound by memory: of
/// 262,144 tokens of 1,024 bf16 in 32,000 rows (537 MB read, 66 MB written) 140 us, 4.3 TB/s, where a copy
/// reaches 4.98; it reads rows in an order of its own, 1 KB of each.
template <class T, int V, int G, bool STREAM>
__global__ void __launch_bounds__(256) embed_grad_sum_kernel(SumArgs a) {
  constexpr uint32_t kGroups = 256 / G;
  constexpr int kAhead = 8;
  __shared__ uint32_t s_key[kMostEntries];
  __shared__ uint32_t s_pos[kMostEntries];
  const uint32_t length = a.piece;
  if (blockIdx.x >= a.sum_blocks) {
    if (blockIdx.y == 0) zero_rows<T, V>(a, blockIdx.x - a.sum_blocks, s_key);
    return;
  }
  const uint64_t block0 = static_cast<uint64_t>(blockIdx.x) * (kGroups * length);
  for (uint32_t i = threadIdx.x; i < kGroups * length; i += 256) {
    const uint64_t e = block0 + i;
    s_key[i] = e < a.count ? a.keys[e] : a.rows;
    s_pos[i] = e < a.count ? a.positions[e] : 0u;
  }
  __syncthreads();
  const uint32_t group = threadIdx.x / G;
  const uint64_t piece = static_cast<uint64_t>(blockIdx.x) * kGroups + group;
  const uint64_t e0 = piece * length;
  uint32_t col = (blockIdx.y * G + threadIdx.x % G) * V;
  if (e0 >= a.count || col >= a.dim) return;
  col = col < a.dim - V ? col : a.dim - V;
  const uint32_t n = a.count - e0 < length ? static_cast<uint32_t>(a.count - e0) : length;
  const uint32_t* key = s_key + group * length;
  const uint32_t* pos = s_pos + group * length;
  const uint32_t from = e0 > 0 ? a.keys[e0 - 1] : a.rows;                // the run that came in, if any
  const uint32_t onto = e0 + n < a.count ? a.keys[e0 + n] : a.rows;      // the run that goes on, if any
  const T* grad = static_cast<const T*>(a.grad) + col;
  T* out = static_cast<T*>(a.out) + col;
  float* partial = a.partial + piece * 2 * a.dim + col;

  float acc[V] = {};
  uint32_t cur = key[0], began = 0;
  const auto flush = [&](uint32_t end) {
    if (cur == a.rows) return;
    const bool came = began == 0 && from == cur, goes = end == n && onto == cur;
    if (came || goes) {
      float* p = partial + (came ? 0u : a.dim);
      constexpr int kWide = V < 4 ? V : 4;
#pragma unroll
      for (int k = 0; k < V; k += kWide) {
        float part[kWide];
#pragma unroll
        for (int e = 0; e < kWide; ++e) part[e] = acc[k + e];
        store_floats<float, kWide>(p + k, part);
      }
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k) acc[k] *= a.scale;
      store_floats<T, V>(out + static_cast<uint64_t>(cur) * a.dim, acc);
    }
  };
  for (uint32_t j = 0; j < n; j += kAhead) {
    float x[kAhead][V];
    uint32_t kk[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      kk[u] = j + u < n ? key[j + u] : a.rows;
      if (kk[u] != a.rows) {
        load_floats<T, V, STREAM>(grad + static_cast<uint64_t>(pos[j + u]) * a.stride, x[u]);
      } else {
#pragma unroll
        for (int k = 0; k < V; ++k) x[u][k] = 0.0f;
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (j + u < n && kk[u] != cur) {
        flush(j + u);
        cur = kk[u];
        began = j + u;
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] = 0.0f;
      }
#pragma unroll
      for (int k = 0; k < V; ++k) acc[k] += x[u][k];
    }
  }
  flush(n);
}

/// Work-group per sixteen pieces and 64 W columns: where a run begins in a piece and goes on, its partial
/// sums are added in order and the row is written. A run of few pieces is its wave's own; a long one is
/// shared by the sixteen waves in contiguous parts, since the longest run decides the time: of 262,144
/// tokens the most frequent has 1,600 pieces of 16, which four waves read in 32 us (a work-group per piece
/// or per four pieces, no matter) and sixteen in 18.
constexpr uint32_t kJoinWaves = 16, kJoinAlone = 16;
template <class T, int W>
__global__ void __launch_bounds__(kJoinWaves * 64) embed_grad_join_kernel(SumArgs a) {
  __shared__ float s_sum[kJoinWaves][64 * W];
  __shared__ uint32_t s_end[kJoinWaves];  // one past a long run's last entry
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t first = blockIdx.x * kJoinWaves;
  uint32_t c = (blockIdx.y * 64 + lane) * W;
  const bool in = c < a.dim;
  c = c < a.dim - W ? c : a.dim - W;
  // Pieces p0 .. p1 of the run that begins in `begin`, where it is the part that goes on.
  const auto add = [&](uint32_t begin, uint32_t p0, uint32_t p1, float (&acc)[W]) {
#pragma unroll 8
    for (uint32_t p = p0; p < p1; ++p) {
      float x[W];
      load_floats<float, W>(a.partial + (static_cast<uint64_t>(p) * 2 + (p == begin ? 1 : 0)) * a.dim + c, x);
#pragma unroll
      for (int k = 0; k < W; ++k) acc[k] += x[k];
    }
  };
  const auto write = [&](uint32_t row, float (&acc)[W]) {
#pragma unroll
    for (int k = 0; k < W; ++k) acc[k] *= a.scale;
    store_floats<T, W>(static_cast<T*>(a.out) + static_cast<uint64_t>(row) * a.dim + c, acc);
  };

  const uint64_t e0 = static_cast<uint64_t>(first + wave) * a.piece, e1 = e0 + a.piece;
  uint32_t shared_end = 0;
  if (e1 < a.count) {  // nothing goes on from the last piece
    const uint32_t cur = a.keys[e1 - 1], next = a.keys[e1], lead = a.keys[e0], from = e0 > 0 ? a.keys[e0 - 1] : a.rows;
    const bool earlier = lead == cur && from == cur;
    if (cur != a.rows && next == cur && !earlier) {
      const uint32_t end = static_cast<uint32_t>(e1) +
                           wave_lower_bound(a.keys + e1, a.count - static_cast<uint32_t>(e1), cur + 1);
      const uint32_t last = (end - 1) / a.piece;
      if (last - (first + wave) < kJoinAlone) {
        float acc[W] = {};
        if (in) {
          add(first + wave, first + wave, last + 1, acc);
          write(cur, acc);
        }
      } else {
        shared_end = end;
      }
    }
  }
  if (lane == 0) s_end[wave] = shared_end;
  __syncthreads();
  for (uint32_t b = 0; b < kJoinWaves; ++b) {
    if (s_end[b] == 0) continue;
    const uint32_t begin = first + b, end = (s_end[b] - 1) / a.piece + 1;  // pieces begin .. end - 1 hold the run
    const uint32_t share = (end - begin + kJoinWaves - 1) / kJoinWaves;
    const uint32_t p0 = begin + wave * share < end ? begin + wave * share : end, p1 = p0 + share < end ? p0 + share : end;
    float acc[W] = {};
    if (in) add(begin, p0, p1, acc);
#pragma unroll
    for (int k = 0; k < W; ++k) s_sum[wave][lane * W + k] = acc[k];
    __syncthreads();
    if (wave == 0 && in) {
#pragma unroll
      for (int k = 0; k < W; ++k) {
        acc[k] = 0.0f;
        for (uint32_t w = 0; w < kJoinWaves; ++w) acc[k] += s_sum[w][lane * W + k];
      }
      write(a.keys[s_end[b] - 1], acc);
    }
    __syncthreads();
  }
}

/// Where the parts of the workspace lie, in bytes.
struct GradLayout {
  uint32_t parts, part, passes, piece;
  size_t counts, keys[2], positions[2], partial, total;
};

GradLayout grad_layout(uint64_t rows, uint32_t dim, uint64_t count) {
  GradLayout l{};
  if (rows_look(rows, dim, count)) return l;
  const auto round = [](size_t b) { return (b + 255) / 256 * 256; };
  l.part = static_cast<uint32_t>(std::max<uint64_t>(ceil_div(count, kParts), 1024));
  l.parts = static_cast<uint32_t>(ceil_div(count, l.part));
  uint32_t bits = 0;
  while (bits < 32 && (rows >> bits) != 0) ++bits;
  l.passes = std::max(1u, (bits + 7) / 8);
  // About 8,192 waves of pieces, where there are so many tokens: long pieces have fewer runs to join, short
  // ones more loads under way (262,144 x 1,024 bf16: 256 entries 263 us a call, 128 208, 64 193). Rows of
  // dim / 8 to dim pieces of 16 bytes: counted as dim / 8 here, for every type.
  const uint64_t lanes = std::min<uint64_t>(std::max<uint64_t>(ceil_div(dim, 8), 8), 64);
  const uint64_t slabs = ceil_div(dim, 512);
  l.piece = 16;
  while (l.piece < 256 && l.piece < 8 * lanes && ceil_div(count, 2 * l.piece) * slabs * lanes >= 8192 * 64) l.piece *= 2;
  size_t at = round(static_cast<size_t>(l.parts) * kBins * 4);
  for (int i = 0; i < 2; ++i) {
    l.keys[i] = at;
    at += round(count * 4);
    l.positions[i] = at;
    at += round(count * 4);
  }
  l.partial = at;
  l.total = at + round(ceil_div(count, l.piece) * 2 * dim * 4);
  return l;
}

template <class T, class I>
void launch_embed_grad(const void* grad, uint64_t stride, const void* tokens, uint64_t count, uint64_t rows,
                       uint32_t dim, float scale, void* out, char* ws, hipStream_t s) {
  const int width = vector_width(sizeof(T), dim);
  if (rows_look(rows, dim, count)) {
    const uint32_t lds = static_cast<uint32_t>(std::max<uint64_t>(count, 1)) * 24, own = own_rows(rows, count);
    with_width<T>(width, [&](auto v) {
      constexpr int V = decltype(v)::value;
      const auto go = [&](auto group) {
        hipLaunchKernelGGL((embed_grad_own_kernel<T, V, decltype(group)::value, I>),
                           dim3(static_cast<unsigned>(ceil_div(rows, 4 * own))), dim3(256), lds, s,
                           static_cast<const T*>(grad), stride, static_cast<const I*>(tokens),
                           static_cast<uint32_t>(count), static_cast<uint32_t>(rows), dim, own, scale,
                           static_cast<T*>(out));
      };
      if constexpr (V * sizeof(T) == 16) {  // narrower rows have one piece or two
        if (ceil_div(dim, V) > 32) return go(std::integral_constant<int, 64>{});
        if (ceil_div(dim, V) > 16) return go(std::integral_constant<int, 32>{});
      }
      go(std::integral_constant<int, 16>{});
    });
    QVH_HIP(hipGetLastError());
    return;
  }
  const GradLayout l = grad_layout(rows, dim, count);
  const uint32_t n = static_cast<uint32_t>(count), r = static_cast<uint32_t>(rows);
  uint32_t bits = 0;
  while (bits < 32 && (rows >> bits) != 0) ++bits;
  const uint32_t digit = (bits + l.passes - 1) / l.passes;
  uint32_t* counts = reinterpret_cast<uint32_t*>(ws + l.counts);
  uint32_t* keys[2] = {reinterpret_cast<uint32_t*>(ws + l.keys[0]), reinterpret_cast<uint32_t*>(ws + l.keys[1])};
  uint32_t* pos[2] = {reinterpret_cast<uint32_t*>(ws + l.positions[0]), reinterpret_cast<uint32_t*>(ws + l.positions[1])};
  const uint32_t sorted = (l.passes - 1) & 1;  // which of the two halves of keys and pos
  const bool held = l.part <= kSortWaves * 64 * kHeld;
  for (uint32_t p = 0; p < l.passes && n > 0; ++p) {  // without tokens there is nothing to sort, and rows to clear all the same
    const uint32_t *ik = keys[(p & 1) ^ 1], *ip = pos[(p & 1) ^ 1];
    const auto pass = [&](auto first, auto hold) {
      constexpr bool F = decltype(first)::value;
      hipLaunchKernelGGL((count_kernel<I, F>), dim3(l.parts), dim3(512), 0, s, static_cast<const I*>(tokens), ik, n, l.part,
                         r, p * digit, (1u << digit) - 1, counts);
      QVH_HIP(hipGetLastError());
      hipLaunchKernelGGL((scatter_kernel<I, F, decltype(hold)::value>), dim3(l.parts), dim3(kSortWaves * 64), 0, s,
                         static_cast<const I*>(tokens), ik, ip, n, l.part, r, p * digit, digit, counts, keys[p & 1],
                         pos[p & 1]);
      QVH_HIP(hipGetLastError());
    };
    const auto either = [&](auto first) { held ? pass(first, std::true_type{}) : pass(first, std::false_type{}); };
    p == 0 ? either(std::true_type{}) : either(std::false_type{});
  }
  with_width<T>(width, [&](auto v) {
    constexpr int V = decltype(v)::value;
    SumArgs a{};
    a.grad = grad;
    a.stride = stride;
    a.keys = keys[sorted];
    a.positions = pos[sorted];
    a.count = n;
    a.rows = r;
    a.dim = dim;
    a.scale = scale;
    a.out = out;
    a.partial = reinterpret_cast<float*>(ws + l.partial);
    a.piece = l.piece;
    a.pieces = static_cast<uint32_t>(ceil_div(count, l.piece));
    a.cpr = static_cast<uint32_t>(ceil_div(dim, V));
    a.zero_blocks = static_cast<uint32_t>(std::min(ceil_div(rows, kZeroRows), kZeroBlocks));
    const auto sum = [&](auto group) {
      constexpr int G = decltype(group)::value;
      QVH_REQUIRE(256 / G * a.piece <= kMostEntries, "qvh_embed_grad_device: pieces past the work-group's memory");
      a.sum_blocks = static_cast<uint32_t>(ceil_div(a.pieces, 256 / G));
      a.slabs = static_cast<uint32_t>(ceil_div(a.cpr, G));
      // Gradients that the L2s cannot hold are read past them, so that the partial sums stay for the join. Both sides,
      // through and past: 250,007 x 100 bf16 146 and 131 us a call, 262,144 x 1,024 193 and 184; 100,000 x 128
      // (26 MB) 44 and 47.
      const dim3 grid(a.sum_blocks + a.zero_blocks, a.slabs);
      if constexpr (V * sizeof(T) == 16) {
        if (count * dim * sizeof(T) >= kStreamed) {
          hipLaunchKernelGGL((embed_grad_sum_kernel<T, V, G, true>), grid, dim3(256), 0, s, a);
          return;
        }
      }
      hipLaunchKernelGGL((embed_grad_sum_kernel<T, V, G, false>), grid, dim3(256), 0, s, a);
    };
    const auto any = [&] {
      if constexpr (V * sizeof(T) == 16) {  // narrower rows have one piece or two
        if (a.cpr > 32) return sum(std::integral_constant<int, 64>{});
        if (a.cpr > 16) return sum(std::integral_constant<int, 32>{});
        if (a.cpr > 8) return sum(std::integral_constant<int, 16>{});
      }
      sum(std::integral_constant<int, 8>{});
    };
    any();
    QVH_HIP(hipGetLastError());
    if (a.pieces > 1) {
      const unsigned blocks = static_cast<unsigned>(ceil_div(a.pieces, kJoinWaves));
      if (dim >= 4) {
        hipLaunchKernelGGL((embed_grad_join_kernel<T, 4>), dim3(blocks, ceil_div(dim, 256)), dim3(kJoinWaves * 64), 0, s, a);
      } else {
        hipLaunchKernelGGL((embed_grad_join_kernel<T, 1>), dim3(blocks, ceil_div(dim, 64)), dim3(kJoinWaves * 64), 0, s, a);
      }
      QVH_HIP(hipGetLastError());
    }
  });
}

void check_embed(const char* who, uint64_t rows, uint32_t dim, int dtype, int index_bytes, uint64_t count) {
  const std::string w(who);
  require_dtype(who, dtype);
  QVH_REQUIRE(index_bytes == 4 || index_bytes == 8, w + ": tokens must be int32 or int64");
  QVH_REQUIRE(dim >= 1 && dim <= kMaxDim, w + ": dim must be in [1, 32768]");
  QVH_REQUIRE(rows < 0xFFFFFFFFu, w + ": rows must be below 2^32 - 1");
  QVH_REQUIRE(count < (uint64_t{1} << 31), w + ": the number of tokens must be below 2^31");
}

}  // namespace
}  // namespace qvh

extern "C" {

qvh_status qvh_embed_device(const void* d_table, uint64_t rows, uint32_t dim, uint64_t row_stride, int dtype,
                            const void* d_tokens, int index_bytes, uint64_t count, float scale, void* d_out,
                            void* stream) {
  return qvh::guarded([&] {
    using namespace qvh;
    check_embed("qvh_embed_device", rows, dim, dtype, index_bytes, count);
    QVH_REQUIRE(reinterpret_cast<uintptr_t>(d_table) % dtype_size(dtype) == 0 && reinterpret_cast<uintptr_t>(d_out) % dtype_size(dtype) == 0 &&
                    reinterpret_cast<uintptr_t>(d_tokens) % index_bytes == 0,
                "qvh_embed_device: a buffer is not aligned to its element type");
    QVH_REQUIRE(row_stride >= dim || rows <= 1, "qvh_embed_device: the row stride must be at least dim");
    if (count == 0) return;
    QVH_REQUIRE((d_table || rows == 0) && d_tokens && d_out, "qvh_embed_device: null buffer");
    const DeviceScope device;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    with_dtype(dtype, [&](auto* t) {
      using T = std::remove_pointer_t<decltype(t)>;
      if (index_bytes == 8) {
        launch_embed<T, int64_t>(d_table, rows, dim, row_stride, d_tokens, count, scale, d_out, s);
      } else {
        launch_embed<T, int32_t>(d_table, rows, dim, row_stride, d_tokens, count, scale, d_out, s);
      }
    });
  });
}

qvh_status qvh_embed_grad_workspace(uint64_t rows, uint32_t dim, uint64_t count, uint64_t* bytes) {
  return qvh::guarded([&] {
    using namespace qvh;
    QVH_REQUIRE(bytes != nullptr, "qvh_embed_grad_workspace: null output");
    check_embed("qvh_embed_grad_workspace", rows, dim, QVH_FP32, 8, count);
    *bytes = grad_layout(rows, dim, count).total;
  });
}

qvh_status qvh_embed_grad_device(const void* d_grad, uint64_t row_stride, const void* d_tokens, int index_bytes,
                                 uint64_t count, uint64_t rows, uint32_t dim, int dtype, float scale, void* d_out,
                                 void* d_workspace, uint64_t workspace_bytes, void* stream) {
  return qvh::guarded([&] {
    using namespace qvh;
    check_embed("qvh_embed_grad_device", rows, dim, dtype, index_bytes, count);
    QVH_REQUIRE(reinterpret_cast<uintptr_t>(d_grad) % dtype_size(dtype) == 0 && reinterpret_cast<uintptr_t>(d_out) % dtype_size(dtype) == 0 &&
                    reinterpret_cast<uintptr_t>(d_tokens) % index_bytes == 0,
                "qvh_embed_grad_device: a buffer is not aligned to its element type");
    QVH_REQUIRE(row_stride >= dim || count <= 1, "qvh_embed_grad_device: the row stride must be at least dim");
    if (rows == 0) return;
    QVH_REQUIRE(((d_grad && d_tokens) || count == 0) && d_out, "qvh_embed_grad_device: null buffer");
    const size_t need = grad_layout(rows, dim, count).total;
    QVH_REQUIRE(need == 0 || (d_workspace != nullptr && workspace_bytes >= need),
                "qvh_embed_grad_device: the workspace is too small");
    QVH_REQUIRE(reinterpret_cast<uintptr_t>(d_workspace) % 16 == 0,
                "qvh_embed_grad_device: the workspace must be 16-byte aligned");
    const DeviceScope device;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    with_dtype(dtype, [&](auto* t) {
      using T = std::remove_pointer_t<decltype(t)>;
      if (index_bytes == 8) {
        launch_embed_grad<T, int64_t>(d_grad, row_stride, d_tokens, count, rows, dim, scale, d_out,
                                      static_cast<char*>(d_workspace), s);
      } else {
        launch_embed_grad<T, int32_t>(d_grad, row_stride, d_tokens, count, rows, dim, scale, d_out,
                                      static_cast<char*>(d_workspace), s);
      }
    });
  });
}

}  // extern "C"
