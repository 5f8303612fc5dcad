// w4_many_f16.cu — the tensor-core kernel of the 4-bit linear layer on f16 operands.
#include "w4_many.cuh"

namespace fxk {

cudaError_t w4_many_f16(const W4LinearArgs& a, const ManyPlan& p, cudaStream_t s) { return launch_typed<false>(a, p, s); }
cudaError_t w4_many_f16_status(uint32_t* code) { return take_status(code); }

}  // namespace fxk
