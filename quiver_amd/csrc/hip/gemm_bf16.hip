// The linear layer's matrix products: bf16.
#include "linear.hpp"

namespace qvh {

void gemm_bf16(Form form, const GemmArgs& g, const LinearEpilogue<bhalf_t>& e, const GemmPlan& p, void* partial,
               hipStream_t s) {
  gemm_forms<bhalf_t, 1>(form, g, e, p, partial, s);
}

}  // namespace qvh
