// Lookup of tokens in an embedding, and its gradient (embedding.cu). On the current device.
#pragma once

#include "b200ccl/types.h"

#include <cuda_runtime.h>

#include <cstddef>

namespace b200ccl::kernels {

struct EmbeddingCall {
    const void* tokens = nullptr;  // `token_stride` elements apart
    bool tokens64 = true;
    long long token_stride = 1;
    std::size_t count = 0, vocabulary = 0, width = 0;
    DType dtype = DType::Float;
    float scale = 1.0f;
    const void* rows = nullptr;  // the matrix, [vocabulary, width]; gradient: what comes back, [count, width]
    long long stride = 0;        // elements from row to row
    void* out = nullptr;         // [count, width], the gradient [vocabulary, width]
    void* workspace = nullptr;   // of the gradient: embedding_workspace() bytes, at a multiple of 256
    cudaStream_t stream = nullptr;
};

cudaError_t launch_embedding(const EmbeddingCall& call);
std::size_t embedding_workspace(const EmbeddingCall& call);
cudaError_t launch_embedding_gradient(const EmbeddingCall& call);

}  // namespace b200ccl::kernels
