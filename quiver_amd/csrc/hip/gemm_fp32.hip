// The linear layer's matrix products: fp32.
#include "linear.hpp"

namespace qvh {

void gemm_fp32(Form form, const GemmArgs& g, const LinearEpilogue<float>& e, const GemmPlan& p, void* partial,
               hipStream_t s) {
  gemm_forms<bhalf_t, 3>(form, g, e, p, partial, s);
}

}  // namespace qvh
