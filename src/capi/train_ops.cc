#include "b200ccl/train_ops.h"

#include "capi/guarded.h"
#include "kernels/sm100/checkpoint8.h"
#include "kernels/sm100/head_rotation.h"
#include "kernels/sm100/wait_status.h"
#include "kernels/sm100/weight_grad.h"

using namespace b200ccl;
using capi::aligned;
using capi::dtype_of;
using capi::guarded;

namespace {

void check_kept(const void* codes, const void* scales, std::size_t rows, std::size_t columns, bool needed = true) {
    B2_REQUIRE(columns <= (1ull << 30) && rows < (1ull << 31), "more than 2^31 rows or 2^30 columns");
    B2_REQUIRE(rows * ((columns + 31) / 32) < (1ull << 30), "more than 2^30 blocks of 32 elements");
    if (rows == 0 || columns == 0 || !needed) return;
    B2_REQUIRE(codes != nullptr && scales != nullptr, "codes and scales must be non-null");
    B2_REQUIRE(aligned(codes, 32), "codes must start at a multiple of 32 bytes");
}

void run_kept(bool keep, kernels::Activation activation, const void* in, long long stride, std::size_t rows, std::size_t columns, int dtype,
              const void* codes, const void* scales, void* out, void* stream) {
    kernels::Kept8Call c;
    c.dtype = dtype_of(dtype);
    const bool only_activation = keep && activation != kernels::Activation::None && codes == nullptr && scales == nullptr;
    check_kept(codes, scales, rows, columns, !only_activation);
    const bool reads = keep || activation != kernels::Activation::None, writes = !keep || activation != kernels::Activation::None;
    if (rows != 0 && columns != 0) {
        B2_REQUIRE(!reads || in != nullptr, "the input must be non-null");
        B2_REQUIRE(!writes || out != nullptr, "the output must be non-null");
        B2_REQUIRE(aligned(in, dtype_size(c.dtype)) && aligned(out, dtype_size(c.dtype)), "a buffer is not aligned to its elements");
    }
    c.in = reads ? in : nullptr;
    c.stride = reads ? stride : 0;
    c.rows = rows;
    c.columns = columns;
    c.activation = activation;
    c.codes = static_cast<unsigned char*>(const_cast<void*>(codes));
    c.scales = static_cast<unsigned char*>(const_cast<void*>(scales));
    c.out = writes ? out : nullptr;
    c.stream = static_cast<cudaStream_t>(stream);
    B2_CUDA(keep ? kernels::launch_keep8(c) : kernels::launch_read8(c));
}

kernels::Activation gelu_of(int tanh) { return tanh != 0 ? kernels::Activation::GeluTanh : kernels::Activation::Gelu; }

kernels::WeightGradCall weight_grad_of(const b2_weight_grad* g, void* stream) {
    B2_REQUIRE(g != nullptr, "null call");
    kernels::WeightGradCall c;
    c.dtype = dtype_of(g->dtype);
    B2_REQUIRE(g->tokens < (1ull << 31) && g->outputs < (1ull << 31) && g->inputs < (1ull << 31), "more than 2^31 tokens, outputs or inputs");
    c.dy = g->dy;
    c.stride = g->stride;
    c.tokens = g->tokens;
    c.outputs = g->outputs;
    c.inputs = g->inputs;
    c.codes = static_cast<const unsigned char*>(g->codes);
    c.scales = static_cast<const unsigned char*>(g->scales);
    c.weight_grad = g->weight_grad;
    c.bias_grad = g->bias_grad;
    c.workspace = g->workspace;
    c.stream = static_cast<cudaStream_t>(stream);
    return c;
}

kernels::RotationCall rotation_of(const b2_rotation* r, bool backward, void* stream) {
    B2_REQUIRE(r != nullptr, "null call");
    kernels::RotationCall c;
    c.dtype = dtype_of(r->dtype);
    B2_REQUIRE(r->dim >= 2 && r->dim % 2 == 0 && r->dim <= kernels::kMaxHeadDim, "the head dimension must be even, and 2 to 256");
    B2_REQUIRE(r->rotated >= 0 && r->rotated % 2 == 0 && r->rotated <= r->dim, "the rotated part must be even, and at most the head dimension");
    B2_REQUIRE(r->batch >= 0 && r->tokens >= 0 && r->batch < (1ll << 31) && r->tokens < (1ll << 31) && r->batch * r->tokens < (1ll << 31),
               "batch * tokens must be below 2^31");
    B2_REQUIRE(r->position_bytes == 4 || r->position_bytes == 8, "positions have 4 or 8 bytes");
    const bool norm = backward || r->norm != 0, any = r->batch * r->tokens > 0;
    if (any && r->rotated > 0) {
        B2_REQUIRE(r->positions != nullptr && r->frequencies != nullptr, "positions and frequencies must be non-null");
        B2_REQUIRE(aligned(r->positions, (std::size_t)r->position_bytes) && aligned(r->frequencies, 8), "positions or frequencies are not aligned");
    }
    c.batch = r->batch;
    c.tokens = r->tokens;
    c.dim = r->dim;
    c.rotated = r->rotated;
    c.interleaved = r->interleaved != 0;
    c.inverse = backward || r->inverse != 0;
    c.norm = norm;
    c.eps = r->eps;
    c.magnitude = r->magnitude;
    c.positions = r->positions;
    c.positions64 = r->position_bytes == 8;
    c.position_batch = r->position_strides[0];
    c.position_token = r->position_strides[1];
    c.frequencies = r->frequencies;
    const std::size_t bytes = dtype_size(c.dtype);
    int sides = 0, kept = 0;
    for (int i = 0; i < 2; ++i) {
        const b2_heads& h = r->side[i];
        kernels::HeadsSide& s = c.side[i];
        B2_REQUIRE(h.heads >= 0 && h.heads < (1 << 16), "heads must be below 65536");
        s.heads = h.heads;
        if (h.heads == 0) continue;
        ++sides;
        kept += h.codes != nullptr ? 1 : 0;
        const bool full = !backward || h.codes == nullptr;  // x itself is read
        if (any) {
            B2_REQUIRE(h.out != nullptr && (!full || h.x != nullptr), "x and out must be non-null");
            B2_REQUIRE(!norm || h.weight != nullptr, "a norm needs its weight");
            B2_REQUIRE(h.codes == nullptr || (h.scales != nullptr && aligned(h.codes, 16)), "codes must start at a multiple of 16 bytes, and come with scales");
            B2_REQUIRE(!backward || h.grad != nullptr, "grad must be non-null");
            B2_REQUIRE((!full || aligned(h.x, bytes)) && aligned(h.out, bytes) && aligned(h.weight, bytes) && (!backward || aligned(h.grad, bytes)),
                       "a buffer is not aligned to its elements");
        }
        B2_REQUIRE(!backward || (h.weight_grad != nullptr && h.partial != nullptr), "weight_grad and partial must be non-null");
        if (full) s.x = {h.x, h.x_strides[0], h.x_strides[1], h.x_strides[2]};
        if (backward) s.grad = {h.grad, h.grad_strides[0], h.grad_strides[1], h.grad_strides[2]};
        s.out = h.out;
        s.weight = norm ? h.weight : nullptr;
        s.codes = norm ? static_cast<unsigned char*>(h.codes) : nullptr;
        s.scales = norm ? static_cast<unsigned char*>(h.scales) : nullptr;
        s.weight_grad = backward ? h.weight_grad : nullptr;
        s.partial = backward ? static_cast<float*>(h.partial) : nullptr;
    }
    B2_REQUIRE(sides > 0, "neither queries nor keys");
    B2_REQUIRE(!backward || kept == 0 || kept == sides, "both sides are kept in 8 bits, or neither");
    c.stream = static_cast<cudaStream_t>(stream);
    return c;
}

}  // namespace

extern "C" {

int b2_pack8(const void* x, long long stride, size_t rows, size_t columns, int dtype, void* codes, void* scales, void* stream) {
    return guarded("pack8", [&] { run_kept(true, kernels::Activation::None, x, stride, rows, columns, dtype, codes, scales, nullptr, stream); });
}

int b2_unpack8(const void* codes, const void* scales, size_t rows, size_t columns, int dtype, void* out, void* stream) {
    return guarded("unpack8", [&] { run_kept(false, kernels::Activation::None, nullptr, 0, rows, columns, dtype, codes, scales, out, stream); });
}

int b2_gelu8_forward(const void* x, long long stride, size_t rows, size_t columns, int dtype, int tanh, void* y, void* codes, void* scales,
                     void* stream) {
    return guarded("gelu8", [&] { run_kept(true, gelu_of(tanh), x, stride, rows, columns, dtype, codes, scales, y, stream); });
}

int b2_gelu8_backward(const void* dy, long long stride, const void* codes, const void* scales, size_t rows, size_t columns, int dtype, int tanh,
                      void* dx, void* stream) {
    return guarded("gelu8", [&] { run_kept(false, gelu_of(tanh), dy, stride, rows, columns, dtype, codes, scales, dx, stream); });
}

int b2_weight_grad8_workspace(const b2_weight_grad* call, size_t* bytes) {
    return guarded("weight_grad8", [&] {
        B2_REQUIRE(bytes != nullptr, "bytes must be non-null");
        *bytes = kernels::weight_grad_workspace(weight_grad_of(call, nullptr));
    });
}

int b2_weight_grad8(const b2_weight_grad* call, void* stream) { return b2_weight_grad8_within(call, kernels::WeightGradCall().wait_ns, stream); }

int b2_weight_grad8_within(const b2_weight_grad* call, unsigned long long wait_ns, void* stream) {
    return guarded("weight_grad8", [&] {
        kernels::WeightGradCall c = weight_grad_of(call, stream);
        c.wait_ns = wait_ns;
        if (c.outputs != 0 && c.inputs != 0) {
            const std::size_t bytes = dtype_size(c.dtype);
            B2_REQUIRE(c.weight_grad != nullptr, "weight_grad must be non-null");
            B2_REQUIRE(aligned(c.weight_grad, bytes) && aligned(c.bias_grad, bytes) && aligned(c.dy, bytes), "a buffer is not aligned to its elements");
            if (c.tokens != 0) {
                check_kept(c.codes, c.scales, c.tokens, c.inputs);
                B2_REQUIRE(c.dy != nullptr, "dy must be non-null");
                B2_REQUIRE(aligned(c.workspace, 256), "the workspace must start at a multiple of 256 bytes");
            }
        }
        kernels::launch_weight_grad(c);
    });
}

int b2_train_check_async_error(int device) {
    return guarded("weight_grad8", [&] {
        if (kernels::waits_failed(kernels::WaitsOf::WeightGrad, device))
            throw std::runtime_error("a wait inside a call on device " + std::to_string(device) + " ran out; its gradients are NaN");
    });
}

int b2_rotate_heads(const b2_rotation* call, void* stream) {
    return guarded("rotate_heads", [&] { B2_CUDA(kernels::launch_rotate_heads(rotation_of(call, false, stream))); });
}

int b2_rotate_heads_backward(const b2_rotation* call, void* stream) {
    return guarded("rotate_heads_backward", [&] { B2_CUDA(kernels::launch_rotate_heads_backward(rotation_of(call, true, stream))); });
}

}  // extern "C"
