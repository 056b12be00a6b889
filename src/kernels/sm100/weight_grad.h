// Launch of the weight gradient of a projection whose input was kept in 8 bits (weight_grad.cu). On the current device.
#pragma once

#include "b200ccl/types.h"

#include <cuda_runtime.h>

#include <cstddef>

namespace b200ccl::kernels {

struct WeightGradCall {
    const void* dy = nullptr;  // [tokens, outputs], `stride` elements from one token to the next
    long long stride = 0;
    std::size_t tokens = 0, outputs = 0, inputs = 0;
    DType dtype = DType::Float;
    const unsigned char* codes = nullptr;  // [tokens][inputs rounded up to 32]
    const unsigned char* scales = nullptr;
    void* weight_grad = nullptr;  // [outputs, inputs]
    void* bias_grad = nullptr;    // [outputs], or null
    void* workspace = nullptr;    // weight_grad_workspace() bytes, at a multiple of 256
    unsigned long long wait_ns = 2000000000ull;  // limit of each wait inside the kernel
    cudaStream_t stream = nullptr;
};

// Scratch of one call, on the current device.
std::size_t weight_grad_workspace(const WeightGradCall& call);
// weight_grad[n][k] = sum over tokens of dy[t][n] * x^[t][k], bias_grad[n] = sum of dy[t][n]. Throws std::runtime_error on a failed launch. Where a wait
// inside the kernel runs out, what depends on it is NaN.
void launch_weight_grad(const WeightGradCall& call);
// Whether that happened on `device` since this was last asked.
bool weight_grad_failed(int device);

}  // namespace b200ccl::kernels
