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

}  // namespace qvh
