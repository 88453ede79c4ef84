// The linear layer's matrix products: bf16.
#include "linear.hpp"

namespace qvh {

void gemm_bf16(Form form, Kind kind, const GemmArgs& g, const LinearEpilogue<bhalf_t>& e, const GemmPlan& p, void* partial,
               hipStream_t s) {
  if (kind == Kind::kNarrow) return gemm_forms<bhalf_t, Kind::kNarrow>(form, g, e, p, partial, s);
  if (gemm_streamed<bhalf_t>(form, g, e, p, s)) return;
  gemm_forms<bhalf_t, Kind::kPlane1>(form, g, e, p, partial, s);
}

}  // namespace qvh
