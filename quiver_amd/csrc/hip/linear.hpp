// Matrix products of the linear layer by element type: one translation unit each.
#pragma once

#include "gemm.hpp"

namespace qvh {

/// How a product's operands are stored: both by rows (forward), the second by k (input gradient), both by
/// k (weight gradient).
enum class Form { kRowsRows, kRowsK, kKK };

void gemm_fp16(Form form, Kind kind, const GemmArgs& g, const LinearEpilogue<half_t>& e, const GemmPlan& p, void* partial,
               hipStream_t s);
void gemm_bf16(Form form, Kind kind, const GemmArgs& g, const LinearEpilogue<bhalf_t>& e, const GemmPlan& p, void* partial,
               hipStream_t s);
/// fp32 operands, or their bf16 planes.
void gemm_fp32(Form form, Kind kind, const GemmArgs& g, const LinearEpilogue<float>& e, const GemmPlan& p, void* partial,
               hipStream_t s);

template <class T, Kind K, class Epi>
void gemm_forms(Form form, const GemmArgs& g, const Epi& e, const GemmPlan& p, void* partial, hipStream_t s) {
  if (form == Form::kRowsRows) return launch_gemm<T, K, false, false>(g, e, p, partial, s);
  if (form == Form::kRowsK) return launch_gemm<T, K, false, true>(g, e, p, partial, s);
  launch_gemm<T, K, true, true>(g, e, p, partial, s);
}

/// A layer of 16-bit elements with results of 32 MB or more, as much as the L2s hold together, stores them past those,
/// whose lines the operands then keep. Only the largest tile does, in one piece: so large a result takes it
/// unless n or k is small, and then there is little of the operands to keep. Both sides, kept and past:
/// 16,384 x 1,024 x 4,096 bf16, GELU, two results of 134 MB 182 and 174 us; three layers of 4,096 x 1,024 x 1,024,
/// 8 MB each, in a row 19.5 and 20.6 us a layer. True where it has launched.
template <class T>
bool gemm_streamed(Form form, const GemmArgs& g, const LinearEpilogue<T>& e, const GemmPlan& p, hipStream_t s) {
  if (form != Form::kRowsRows || p.tile != 2 || p.splits != 1) return false;
  if (static_cast<uint64_t>(g.m) * g.n * sizeof(T) < kStreamed) return false;
  launch_tile<T, false, false, Shapes<Kind::kPlane1>::S2, false>(g, StreamedEpilogue<T>{e}, s);
  return true;
}

}  // namespace qvh
