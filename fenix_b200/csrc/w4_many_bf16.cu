// w4_many_bf16.cu — the tensor-core kernel of the 4-bit linear layer on bf16 operands.
#include "w4_many.cuh"

namespace fxk {

cudaError_t w4_many_bf16(const W4LinearArgs& a, const ManyPlan& p, cudaStream_t s) { return launch_typed<true>(a, p, s); }
cudaError_t w4_many_bf16_status(uint32_t* code) { return take_status(code); }

}  // namespace fxk
