// One launch that is a programmatic dependent of the kernel before it: the kernel starts with griddepcontrol.wait.
#pragma once

#include <cuda_runtime.h>

namespace b200ccl::kernels {

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
