// w4_many_bf16.cu — the tensor-core kernel of the 4-bit linear layer on bf16 operands.
#include "w4_many.cuh"

#include <atomic>

namespace fxk {

cudaError_t w4_many_bf16(const W4LinearArgs& a, const ManyPlan& p, cudaStream_t s) { return launch_typed<true>(a, p, s); }
cudaError_t w4_many_bf16_status(uint32_t* code) { return take_status(code); }

cudaError_t w4_many_clusters(int size, int* count) {
    static std::atomic<int> known[64][9];  // by device; 0: not asked yet
    int dev = 0;
    cudaGetDevice(&dev);
    *count = dev < 64 ? known[dev][size].load(std::memory_order_relaxed) : 0;
    if (*count) return cudaSuccess;
    auto* kern = w4_many_kernel<true, false, true, 4, 1, true, false>;  // as any other: a block has its SM to itself
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(size);
    cfg.blockDim = dim3(19 * 32);
    cfg.dynamicSmemBytes = kSmemMax;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = size;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    e = cudaOccupancyMaxActiveClusters(count, kern, &cfg);
    if (e == cudaSuccess && dev < 64) known[dev][size].store(*count, std::memory_order_relaxed);
    return e;
}

}  // namespace fxk
