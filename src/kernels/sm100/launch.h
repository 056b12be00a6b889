// One launch that is a programmatic dependent of the kernel before it: the kernel starts with griddepcontrol.wait.
#pragma once

#include <cuda_runtime.h>

namespace b200ccl::kernels {

// n / d for n below 2^31, as a product.
struct Divisor {
    unsigned d = 0, factor = 0, shift = 0;
    Divisor() = default;
    explicit Divisor(unsigned divisor) : d(divisor) {
        unsigned bits = 0;
        while ((1ull << bits) < d) ++bits;
        shift = 31 + bits;
        factor = (unsigned)((1ull << shift) / d + 1);
    }
    __device__ __forceinline__ unsigned divide(unsigned n) const { return (unsigned)(((unsigned long long)n * factor) >> shift); }
};

template <typename Args>
cudaError_t launch_dependent(void (*kernel)(Args), dim3 grid, unsigned threads, std::size_t shared, cudaStream_t stream, const Args& args) {
    cudaLaunchConfig_t config = {};
    config.gridDim = grid;
    config.blockDim = dim3(threads, 1, 1);
    config.dynamicSmemBytes = shared;
    config.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attr;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, args);
}

}  // namespace b200ccl::kernels
