// The linear layer's matrix products: fp32.
#include "linear.hpp"

namespace qvh {

void gemm_fp32(Form form, Kind kind, const GemmArgs& g, const LinearEpilogue<float>& e, const GemmPlan& p, void* partial,
               hipStream_t s) {
  if (kind == Kind::kFloat) return gemm_forms<float, Kind::kFloat>(form, g, e, p, partial, s);
  if (kind == Kind::kFloatNarrow) return gemm_forms<float, Kind::kFloatNarrow>(form, g, e, p, partial, s);
  gemm_forms<bhalf_t, Kind::kPlane3>(form, g, e, p, partial, s);
}

}  // namespace qvh
