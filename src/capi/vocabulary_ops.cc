#include "b200ccl/vocabulary_ops.h"

#include "capi/guarded.h"
#include "kernels/sm100/embedding.h"
#include "kernels/sm100/vocabulary_loss.h"
#include "kernels/sm100/wait_status.h"

#include <cmath>

using namespace b200ccl;
using capi::aligned;
using capi::dtype_of;
using capi::guarded;

namespace {

kernels::EmbeddingCall embedding_of(const b2_embedding* e, bool backward, bool sizes_only, void* stream) {
    B2_REQUIRE(e != nullptr, "null call");
    kernels::EmbeddingCall c;
    c.dtype = dtype_of(e->dtype);
    B2_REQUIRE(e->token_bytes == 4 || e->token_bytes == 8, "tokens have 4 or 8 bytes");
    B2_REQUIRE(e->vocabulary > 0 && e->width > 0, "a matrix has at least one row and one column");
    B2_REQUIRE(e->vocabulary < (1ull << 31) && e->width < (1ull << 28) && e->count < (backward ? 1ull << 30 : 1ull << 40),
               "too many tokens, rows or columns");
    c.tokens = e->tokens;
    c.tokens64 = e->token_bytes == 8;
    c.token_stride = e->token_stride;
    c.count = e->count;
    c.vocabulary = e->vocabulary;
    c.width = e->width;
    c.scale = e->scale;
    c.rows = e->rows;
    c.stride = e->stride;
    c.out = e->out;
    c.workspace = e->workspace;
    c.stream = static_cast<cudaStream_t>(stream);
    if (sizes_only) return c;
    const std::size_t bytes = dtype_size(c.dtype);
    if (c.count != 0) {
        B2_REQUIRE(c.tokens != nullptr && c.rows != nullptr, "tokens and rows must be non-null");
        B2_REQUIRE(aligned(c.tokens, (std::size_t)e->token_bytes) && aligned(c.rows, bytes), "a buffer is not aligned to its elements");
        B2_REQUIRE(!backward || (c.workspace != nullptr && aligned(c.workspace, 256)), "the workspace must start at a multiple of 256 bytes");
    }
    if (c.count != 0 || backward) {
        B2_REQUIRE(c.out != nullptr, "the output must be non-null");
        B2_REQUIRE(aligned(c.out, backward ? 16 : bytes), backward ? "the gradient must start at a multiple of 16 bytes" : "a buffer is not aligned to its elements");
    }
    return c;
}

// backward: 0 the loss, 1 its gradient, 2 both at once.
kernels::VocabularyLossCall loss_of(const b2_vocabulary_loss* l, int backward, bool sizes_only, void* stream) {
    B2_REQUIRE(backward >= 0 && backward <= 2, "unknown pass");
    B2_REQUIRE(l != nullptr, "null call");
    kernels::VocabularyLossCall c;
    c.dtype = dtype_of(l->dtype);
    B2_REQUIRE(l->vocabulary > 0 && l->width > 0, "a matrix has at least one row and one column");
    B2_REQUIRE(l->vocabulary < (1ull << 30) && l->width < (1ull << 28) && l->tokens < (1ull << 30), "too many tokens, rows or columns");
    B2_REQUIRE(l->target_bytes == 4 || l->target_bytes == 8, "targets have 4 or 8 bytes");
    B2_REQUIRE(l->reduction >= 0 && l->reduction <= 2, "unknown reduction");
    B2_REQUIRE(l->entries >= 0 && l->entries <= kernels::kMaxTeacherEntries, "a teacher has 1 to 256 entries");
    B2_REQUIRE(l->temperature > 0.0f && std::isfinite(l->temperature), "the temperature must be positive");
    B2_REQUIRE(l->entries != 0 || l->temperature == 1.0f, "cross entropy has no temperature");
    const std::size_t bytes = dtype_size(c.dtype);
    c.x = l->x;
    c.x_stride = l->x_stride;
    c.weight = l->weight;
    c.weight_stride = l->weight_stride;
    c.tokens = l->tokens;
    c.width = l->width;
    c.vocabulary = l->vocabulary;
    c.targets = l->targets;
    c.targets64 = l->target_bytes == 8;
    c.distillation = l->entries != 0;
    c.entries = l->entries;
    c.teacher = l->teacher;
    if (c.distillation && backward != 1) c.teacher_dtype = dtype_of(l->teacher_dtype);
    for (int i = 0; i < 2; ++i) {
        c.target_strides[i] = l->target_strides[i];
        c.teacher_strides[i] = l->teacher_strides[i];
    }
    c.temperature = l->temperature;
    c.reduction = static_cast<kernels::LossReduction>(l->reduction);
    c.loss = l->loss;
    c.kept = l->kept;
    c.loss_grad = l->loss_grad;
    c.loss_grad_stride = l->loss_grad_stride;
    c.x_grad = backward != 0 ? l->x_grad : nullptr;
    c.weight_grad = backward != 0 ? l->weight_grad : nullptr;
    c.workspace = l->workspace;
    c.stream = static_cast<cudaStream_t>(stream);
    // (The sizes depend on where x and the matrix lie: what TMA cannot read is copied.)
    if (c.tokens != 0) {
        B2_REQUIRE(c.x != nullptr && c.weight != nullptr, "x and the matrix must be non-null");
        B2_REQUIRE(aligned(c.x, bytes) && aligned(c.weight, bytes), "a buffer is not aligned to its elements");
        B2_REQUIRE(c.tokens <= 1 || c.x_stride >= 0, "rows that lie backwards are not supported");
        B2_REQUIRE(c.vocabulary <= 1 || c.weight_stride >= 0, "rows that lie backwards are not supported");
    }
    if (sizes_only) return c;
    if (c.tokens != 0) {
        B2_REQUIRE(c.targets != nullptr && c.kept != nullptr, "targets and what is kept must be non-null");
        B2_REQUIRE(aligned(c.targets, (std::size_t)l->target_bytes) && aligned(c.kept, 4), "a buffer is not aligned to its elements");
        B2_REQUIRE(backward == 1 || !c.distillation || (c.teacher != nullptr && aligned(c.teacher, dtype_size(c.teacher_dtype))), "the teacher must be non-null and aligned to its elements");
        B2_REQUIRE(c.workspace != nullptr && aligned(c.workspace, 256), "the workspace must start at a multiple of 256 bytes");
    }
    if (backward != 1) {
        B2_REQUIRE(c.loss != nullptr || (c.tokens == 0 && c.reduction == kernels::LossReduction::None), "loss must be non-null");
        B2_REQUIRE(aligned(c.loss, 4), "a buffer is not aligned to its elements");
    }
    if (backward == 1) B2_REQUIRE(c.tokens == 0 || (c.loss_grad != nullptr && aligned(c.loss_grad, 4)), "loss_grad must be non-null and aligned to its elements");
    if (backward != 0) {
        B2_REQUIRE(aligned(c.x_grad, bytes) && aligned(c.weight_grad, bytes), "a buffer is not aligned to its elements");
    }
    return c;
}

}  // namespace

extern "C" {

int b2_embed(const b2_embedding* call, void* stream) {
    return guarded("embedding", [&] { B2_CUDA(kernels::launch_embedding(embedding_of(call, false, false, stream))); });
}

int b2_embed_backward_workspace(const b2_embedding* call, size_t* bytes) {
    return guarded("embedding", [&] {
        B2_REQUIRE(bytes != nullptr, "bytes must be non-null");
        *bytes = kernels::embedding_workspace(embedding_of(call, true, true, nullptr));
    });
}

int b2_embed_backward(const b2_embedding* call, void* stream) {
    return guarded("embedding", [&] { B2_CUDA(kernels::launch_embedding_gradient(embedding_of(call, true, false, stream))); });
}

int b2_vocabulary_loss_sizes(const b2_vocabulary_loss* call, int backward, size_t* kept_floats, size_t* workspace_bytes) {
    return guarded("vocabulary_loss", [&] {
        const kernels::VocabularyLossCall c = loss_of(call, backward != 0 ? 1 : 0, true, nullptr);
        if (kept_floats != nullptr) *kept_floats = kernels::vocabulary_loss_kept(c);
        if (workspace_bytes != nullptr) *workspace_bytes = kernels::vocabulary_loss_workspace(c, backward != 0);
    });
}

int b2_vocabulary_loss_forward(const b2_vocabulary_loss* call, void* stream) {
    return b2_vocabulary_loss_within(call, 0, kernels::VocabularyLossCall().wait_ns, stream);
}

int b2_vocabulary_loss_backward(const b2_vocabulary_loss* call, void* stream) {
    return b2_vocabulary_loss_within(call, 1, kernels::VocabularyLossCall().wait_ns, stream);
}

int b2_vocabulary_loss_both_workspace(const b2_vocabulary_loss* call, size_t* bytes) {
    return guarded("vocabulary_loss", [&] {
        B2_REQUIRE(bytes != nullptr, "bytes must be non-null");
        *bytes = kernels::vocabulary_loss_both_workspace(loss_of(call, 2, true, nullptr));
    });
}

int b2_vocabulary_loss_both(const b2_vocabulary_loss* call, void* stream) {
    return b2_vocabulary_loss_within(call, 2, kernels::VocabularyLossCall().wait_ns, stream);
}

int b2_vocabulary_loss_times(const b2_vocabulary_loss* call, void* stream) {
    return guarded("vocabulary_loss", [&] {
        kernels::VocabularyLossCall c = loss_of(call, 1, true, stream);
        B2_REQUIRE(c.loss_grad != nullptr && aligned(c.loss_grad, 4), "loss_grad must be non-null and aligned to its elements");
        B2_REQUIRE(aligned(c.x_grad, dtype_size(c.dtype)) && aligned(c.weight_grad, dtype_size(c.dtype)), "a buffer is not aligned to its elements");
        kernels::launch_vocabulary_loss_times(c);
    });
}

int b2_vocabulary_loss_within(const b2_vocabulary_loss* call, int backward, unsigned long long wait_ns, void* stream) {
    return guarded("vocabulary_loss", [&] {
        kernels::VocabularyLossCall c = loss_of(call, backward, false, stream);
        c.wait_ns = wait_ns;
        if (backward == 2) kernels::launch_vocabulary_loss_both(c);
        else if (backward == 1) kernels::launch_vocabulary_loss_gradient(c);
        else kernels::launch_vocabulary_loss(c);
    });
}

int b2_vocabulary_loss_check_async_error(int device) {
    return guarded("vocabulary_loss", [&] {
        if (kernels::waits_failed(kernels::WaitsOf::VocabularyLoss, device))
            throw std::runtime_error("a wait inside a call on device " + std::to_string(device) + " ran out; what depends on it is NaN, unless it was made again");
    });
}

}  // extern "C"
