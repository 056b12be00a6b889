// Losses over a vocabulary whose logits are never stored, and their gradients (vocabulary_loss.cu). On the current device.
#pragma once

#include "b200ccl/types.h"

#include <cuda_runtime.h>

#include <cstddef>

namespace b200ccl::kernels {

constexpr int kMaxTeacherEntries = 256;

enum class LossReduction : int { None = 0, Mean = 1, Sum = 2 };

// logits z = x weight^T. Cross entropy with targets[token], or distillation from `entries` teacher logits of each token.
struct VocabularyLossCall {
    DType dtype = DType::Float;
    const void* x = nullptr;  // [tokens, width], `x_stride` elements from one token to the next
    long long x_stride = 0;
    const void* weight = nullptr;  // [vocabulary, width]
    long long weight_stride = 0;
    std::size_t tokens = 0, width = 0, vocabulary = 0;
    const void* targets = nullptr;  // [tokens] or [tokens, entries]
    bool targets64 = true;
    long long target_strides[2] = {0, 0};
    bool distillation = false;
    int entries = 0;
    const void* teacher = nullptr;  // [tokens, entries]
    DType teacher_dtype = DType::Float;
    long long teacher_strides[2] = {0, 0};
    float temperature = 1.0f;
    LossReduction reduction = LossReduction::None;
    float* loss = nullptr;  // [tokens], or one
    float* kept = nullptr;  // vocabulary_loss_kept() floats: written by the loss, read by its gradient
    // The gradient.
    const float* loss_grad = nullptr;
    long long loss_grad_stride = 0;
    void* x_grad = nullptr;       // [tokens, width], or null
    void* weight_grad = nullptr;  // [vocabulary, width], or null
    void* workspace = nullptr;    // vocabulary_loss_workspace() bytes, at a multiple of 256
    unsigned long long wait_ns = 2000000000ull;  // limit of each wait inside a kernel
    cudaStream_t stream = nullptr;
};

std::size_t vocabulary_loss_kept(const VocabularyLossCall& call);
std::size_t vocabulary_loss_workspace(const VocabularyLossCall& call, bool gradient);
// Both throw std::runtime_error on a failed launch. Where a wait inside a kernel runs out, what depends on it is NaN, or made again.
void launch_vocabulary_loss(const VocabularyLossCall& call);
void launch_vocabulary_loss_gradient(const VocabularyLossCall& call);
// The loss together with the gradients that are wanted, for a loss_grad of 1: bf16, one loss for all rows. Its workspace; 0 where that is not so, or would take too much of it.
std::size_t vocabulary_loss_both_workspace(const VocabularyLossCall& call);
void launch_vocabulary_loss_both(const VocabularyLossCall& call);
// x_grad and weight_grad, where they are, times loss_grad, in place.
void launch_vocabulary_loss_times(const VocabularyLossCall& call);

}  // namespace b200ccl::kernels
