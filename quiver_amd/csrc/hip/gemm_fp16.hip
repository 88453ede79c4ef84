// The linear layer's matrix products: fp16.
#include "linear.hpp"

namespace qvh {

void gemm_fp16(Form form, Kind kind, const GemmArgs& g, const LinearEpilogue<half_t>& e, const GemmPlan& p, void* partial,
               hipStream_t s) {
  if (kind == Kind::kNarrow) return gemm_forms<half_t, Kind::kNarrow>(form, g, e, p, partial, s);
  if (gemm_streamed<half_t>(form, g, e, p, s)) return;
  gemm_forms<half_t, Kind::kPlane1>(form, g, e, p, partial, s);
}

}  // namespace qvh
