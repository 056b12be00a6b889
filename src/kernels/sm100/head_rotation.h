// Launches of the kernels that rotate queries and keys by their positions, alone or after a norm of each head (head_rotation.cu). On the current device.
#pragma once

#include "b200ccl/types.h"

#include <cuda_runtime.h>

#include <cstddef>

namespace b200ccl::kernels {

constexpr int kMaxHeadDim = 256;
constexpr unsigned kHeadGradCtas = 296;  // at most so many partial sums of a weight's gradient: two CTAs on each of 148 SMs

// [batch, tokens, heads, dim]: elements from one to the next, the last axis without gaps.
struct HeadsView {
    const void* data = nullptr;
    long long batch = 0, token = 0, head = 0;
};

// Queries or keys. heads = 0: none. Outputs have no gaps. The 8-bit form of a head: dim codes in a row of `pitch` (dim rounded up to 16)
// bytes and one scale.
struct HeadsSide {
    int heads = 0;
    HeadsView x;     // forward: input; backward of the norm: the input where it was kept in full
    HeadsView grad;  // backward of the norm: gradient of the output
    void* out = nullptr;  // forward: output; backward: gradient of the input
    const void* weight = nullptr;    // norm: [dim]
    unsigned char* codes = nullptr;  // norm, forward: written unless null; backward: read unless null
    unsigned char* scales = nullptr;
    void* weight_grad = nullptr;  // backward of the norm: [dim]
    float* partial = nullptr;     // backward of the norm: [kHeadGradCtas][dim], scratch
};

struct RotationCall {
    DType dtype = DType::Float;
    long long batch = 0, tokens = 0;
    int dim = 0, rotated = 0;  // even; the first `rotated` elements of a head turn
    bool interleaved = false;  // pairs (2i, 2i+1) instead of (i, i + rotated/2)
    bool inverse = false;      // turn back
    bool norm = false;
    float eps = 0.0f, magnitude = 1.0f;
    const void* positions = nullptr;  // [batch, tokens]
    bool positions64 = true;          // int64, else int32
    long long position_batch = 0, position_token = 0;  // strides in elements
    const double* frequencies = nullptr;  // [rotated / 2], radians per position
    HeadsSide side[2];
    cudaStream_t stream = nullptr;
};

// out = rotation(x), or rotation(norm(x) * weight) and the 8-bit form of x. One launch.
cudaError_t launch_rotate_heads(const RotationCall& call);
// Gradients of the norm and rotation: out = dx, weight_grad. Two launches.
cudaError_t launch_rotate_heads_backward(const RotationCall& call);

}  // namespace b200ccl::kernels
