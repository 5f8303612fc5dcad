// later.cuh — kernels that begin while the one before them in the stream ends.
#pragma once

#include <cuda_runtime.h>

namespace fxk {

#ifdef __CUDACC__
// Waits until that kernel is done and what it wrote is there: nothing in global memory is read or written before, and nothing by
// loads that take memory as constant while a kernel runs.
__device__ __forceinline__ void wait_for_earlier() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// From here on a later kernel of that kind may begin, once every block of this one has come here. Called only after wait_for_earlier
// (so that what the later kernel, perhaps of another library, reads before a wait of its own is there) and where TMEM has been taken
// (or the later one's blocks might take it and wait for this kernel, which waits for TMEM). The norms' kernels whose blocks stay, as
// many as fit, do not ask for it: another's blocks in their places cost more than the begin (100000 x 320 backward 83 us for 59). The
// pairs of the 8-bit linear layer stay too but do ask: one block of few threads an SM, they lose nothing to another's blocks.
__device__ __forceinline__ void let_later_begin() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Launches a kernel that waits for the earlier one by itself.
template <class... P, class... A>
cudaError_t launch_early(void (*kern)(P...), dim3 grid, int threads, int smem, cudaStream_t s, A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, static_cast<P>(args)...);
    return e == cudaSuccess ? cudaGetLastError() : e;
}
#endif

}  // namespace fxk
