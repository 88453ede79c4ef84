// The linear layer's matrix products: fp16.
#include "linear.hpp"

namespace qvh {

void gemm_fp16(Form form, const GemmArgs& g, const LinearEpilogue<half_t>& e, const GemmPlan& p, void* partial,
               hipStream_t s) {
  gemm_forms<half_t, 1>(form, g, e, p, partial, s);
}

}  // namespace qvh
