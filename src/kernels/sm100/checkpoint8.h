// Launches of the 8-bit checkpoint kernels (checkpoint8.cu). Every call is one launch without memory of its own, on the current device.
#pragma once

#include "b200ccl/types.h"

#include <cuda_runtime.h>

#include <cstddef>

namespace b200ccl::kernels {

enum class Activation { None = 0, Gelu = 1, GeluTanh = 2 };

// A matrix of rows with `stride` elements from one row to the next, and its 8-bit form: codes[rows][pitch], scales[rows][pitch / 32],
// pitch = columns rounded up to whole blocks of 32.
struct Kept8Call {
    const void* in = nullptr;  // keep: x; read: dy (with an activation) or unused
    long long stride = 0;
    std::size_t rows = 0, columns = 0;
    DType dtype = DType::Float;
    Activation activation = Activation::None;
    unsigned char* codes = nullptr;
    unsigned char* scales = nullptr;
    void* out = nullptr;  // keep: y (with an activation) or unused; read: x^ or dx. Rows without gaps.
    cudaStream_t stream = nullptr;
};

// x -> codes and scales, and y = activation(x) where there is one.
cudaError_t launch_keep8(const Kept8Call& call);
// codes and scales -> x^, or dy * activation'(x^).
cudaError_t launch_read8(const Kept8Call& call);

}  // namespace b200ccl::kernels
