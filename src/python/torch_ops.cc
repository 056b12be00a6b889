// The training operators (include/b200ccl/train_ops.h) on torch tensors: what a raw pointer does not show is checked here, outputs and scratch come from
// torch's allocator (on the current stream of the tensors' device, so a captured call's memory is its graph's), and the call goes to the
// C interface by the addresses handed over in bind().
//
// The operators with a gradient are nodes of autograd here and not Python classes: a backward pass then takes the GIL nowhere. (GELU of 1237 x 1003
// numbers, forward and backward: 67 us as a Python class, 52 us so; the rest is torch's own way to its backward thread and back.)
#include "torch_ops.h"

#include "torch_common.h"

#include "b200ccl/train_ops.h"

#include <ATen/Functions.h>
#include <ATen/autocast_mode.h>
#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <algorithm>
#include <cstdint>
#include <initializer_list>
#include <memory>
#include <optional>
#include <stdexcept>
#include <string>
#include <tuple>
#include <type_traits>
#include <utility>
#include <vector>

namespace b200ccl::python {

namespace {

struct Functions {
    decltype(&b2_pack8) pack8 = nullptr;
    decltype(&b2_unpack8) unpack8 = nullptr;
    decltype(&b2_gelu8_forward) gelu8_forward = nullptr;
    decltype(&b2_gelu8_backward) gelu8_backward = nullptr;
    decltype(&b2_weight_grad8_workspace) weight_grad8_workspace = nullptr;
    decltype(&b2_weight_grad8) weight_grad8 = nullptr;
    decltype(&b2_rotate_heads) rotate_heads = nullptr;
    decltype(&b2_rotate_heads_backward) rotate_heads_backward = nullptr;
} g;

// The 8-bit form in one tensor of bytes: codes, then scales.
struct Kept {
    std::int64_t codes = 0, scales = 0;
};
Kept kept_bytes(std::int64_t rows, std::int64_t columns) {
    const std::int64_t blocks = rows * ((columns + 31) / 32);
    return {blocks * 32, blocks};
}
const at::Tensor& kept_of(const at::Tensor& t, std::int64_t bytes) {
    on_gpu("the 8-bit form", t);
    if (t.scalar_type() != at::kByte || !t.is_contiguous() || t.numel() != bytes)
        refuse("the 8-bit form has " + std::to_string(t.numel()) + " elements, expected " + std::to_string(bytes) + " bytes without gaps");
    return t;
}

at::Tensor pack(const at::Tensor& x) {
    const int dtype = dtype_code("x", x);
    const c10::cuda::CUDAGuard guard(x.device());
    const Rows r = rows_of("x", x);
    const Kept k = kept_bytes(r.rows, r.columns);
    at::Tensor out = new_bytes(x, k.codes + k.scales);
    void* stream = stream_of(x);
    call([&] { return g.pack8(r.t.data_ptr(), r.stride, r.rows, r.columns, dtype, bytes_at(out, 0), bytes_at(out, k.codes), stream); });
    return out;
}

// pack8(x) -> bytes
PyObject* pack8(PyObject* const* args, Py_ssize_t nargs) {
    need_arguments(nargs, 1);
    return THPVariable_Wrap(pack(tensor_of("x", args[0])));
}

// unpack8(bytes, sizes, dtype) -> x^
PyObject* unpack8(PyObject* const* args, Py_ssize_t nargs) {
    need_arguments(nargs, 3);
    if (!PyTuple_Check(args[1]) || PyTuple_GET_SIZE(args[1]) < 1) refuse("the shape must be a tuple of at least one size");
    std::vector<std::int64_t> sizes;
    std::int64_t rows = 1;
    const Py_ssize_t n = PyTuple_GET_SIZE(args[1]);
    for (Py_ssize_t i = 0; i < n; ++i) {
        const long long v = PyLong_AsLongLong(PyTuple_GET_ITEM(args[1], i));
        if (v == -1 && PyErr_Occurred()) throw Raised{};
        if (v < 0) refuse("a size is negative");
        sizes.push_back(v);
        if (i + 1 < n) rows *= v;
    }
    if (sizes.back() == 0) rows = 0;
    if (!THPDtype_Check(args[2])) refuse("the dtype must be a torch.dtype");
    const Kept k = kept_bytes(rows, sizes.back());
    const at::Tensor& kept = kept_of(tensor_of("the 8-bit form", args[0]), k.codes + k.scales);
    const c10::cuda::CUDAGuard guard(kept.device());
    at::Tensor out = at::empty(sizes, kept.options().dtype(reinterpret_cast<THPDtype*>(args[2])->scalar_type));
    const int dtype = dtype_code("the 8-bit form", out);
    void* stream = stream_of(kept);
    call([&] { return g.unpack8(bytes_at(kept, 0), bytes_at(kept, k.codes), rows, sizes.back(), dtype, out.data_ptr(), stream); });
    return THPVariable_Wrap(std::move(out));
}

// (y, bytes where they are kept)
std::pair<at::Tensor, at::Tensor> gelu_forward(const at::Tensor& x, bool tanh, bool keep) {
    const int dtype = dtype_code("x", x);
    const c10::cuda::CUDAGuard guard(x.device());
    const Rows r = rows_of("x", x);
    const Kept k = kept_bytes(r.rows, r.columns);
    at::Tensor y = new_like(x), kept;
    if (keep) kept = new_bytes(x, k.codes + k.scales);
    void* stream = stream_of(x);
    call([&] {
        return g.gelu8_forward(r.t.data_ptr(), r.stride, r.rows, r.columns, dtype, tanh ? 1 : 0, y.data_ptr(), keep ? bytes_at(kept, 0) : nullptr,
                               keep ? bytes_at(kept, k.codes) : nullptr, stream);
    });
    return {std::move(y), std::move(kept)};
}

struct Gelu8 : torch::autograd::Function<Gelu8> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, bool tanh) {
        auto [y, kept] = gelu_forward(x, tanh, true);
        ctx->save_for_backward({kept});
        ctx->saved_data["tanh"] = tanh;
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        return in_backward("gelu8", [&]() -> variable_list {
            const bool tanh = ctx->saved_data["tanh"].toBool();
            const at::Tensor& dy = on_gpu("dy", grads[0]);
            const at::Tensor saved = ctx->get_saved_variables()[0];
            const int dtype = dtype_code("dy", dy);
            const c10::cuda::CUDAGuard guard(dy.device());
            const Rows r = rows_of("dy", dy);
            const Kept k = kept_bytes(r.rows, r.columns);
            const at::Tensor& kept = kept_of(saved, k.codes + k.scales);
            same_place("the 8-bit form", kept, dy);
            at::Tensor dx = new_like(dy);
            void* stream = stream_of(dy);
            call([&] {
                return g.gelu8_backward(r.t.data_ptr(), r.stride, bytes_at(kept, 0), bytes_at(kept, k.codes), r.rows, r.columns, dtype, tanh ? 1 : 0,
                                        dx.data_ptr(), stream);
            });
            return {dx, at::Tensor()};
        });
    }
};

// gelu8(x, tanh) -> y
PyObject* gelu8(PyObject* const* args, Py_ssize_t nargs) {
    need_arguments(nargs, 2);
    const at::Tensor& x = tensor_of("x", args[0]);
    const bool tanh = truth(args[1]);
    return THPVariable_Wrap(wants_gradient({&x}) ? Gelu8::apply(x, tanh) : gelu_forward(x, tanh, false).first);
}

// (dw, db where it is wanted)
std::pair<at::Tensor, at::Tensor> weight_grad(const at::Tensor& dy, const at::Tensor& given, std::int64_t inputs, bool bias) {
    b2_weight_grad c = {};
    c.dtype = dtype_code("dy", dy);
    if (inputs < 1) refuse("a projection has at least one input");
    const c10::cuda::CUDAGuard guard(dy.device());
    const Rows r = rows_of("dy", dy);
    // (Without outputs there are no rows to be counted by dy, and nothing to be made from them.)
    const std::int64_t rows = r.columns == 0 ? 0 : r.rows;
    const Kept k = kept_bytes(rows, inputs);
    const at::Tensor& kept = r.columns == 0 ? on_gpu("the 8-bit form", given) : kept_of(given, k.codes + k.scales);
    same_place("the 8-bit form", kept, dy);
    const auto options = dy.options().requires_grad(false);
    at::Tensor dw = at::empty({r.columns, inputs}, options), db;
    if (bias) db = at::empty({r.columns}, options);
    c.dy = r.t.data_ptr();
    c.stride = r.stride;
    c.tokens = rows;
    c.outputs = r.columns;
    c.inputs = inputs;
    c.codes = bytes_at(kept, 0);
    c.scales = bytes_at(kept, k.codes);
    c.weight_grad = dw.data_ptr();
    c.bias_grad = bias ? db.data_ptr() : nullptr;
    std::size_t bytes = 0;
    call([&] { return g.weight_grad8_workspace(&c, &bytes); });
    at::Tensor workspace;
    if (bytes != 0) {
        workspace = new_bytes(dy, static_cast<std::int64_t>(bytes));
        c.workspace = workspace.data_ptr();
    }
    void* stream = stream_of(dy);
    call([&] { return g.weight_grad8(&c, stream); });
    return {std::move(dw), std::move(db)};
}

// weight_grad8(dy, bytes, inputs, bias) -> (dw, db or None)
PyObject* weight_grad8(PyObject* const* args, Py_ssize_t nargs) {
    need_arguments(nargs, 4);
    const long long inputs = PyLong_AsLongLong(args[2]);
    if (inputs == -1 && PyErr_Occurred()) throw Raised{};
    const at::Tensor& dy = tensor_of("dy", args[0]);
    no_gradient_of("dy", dy);
    auto [dw, db] = weight_grad(dy, tensor_of("the 8-bit form", args[1]), inputs, truth(args[3]));
    return two(std::move(dw), std::move(db));
}

struct Linear8 : torch::autograd::Function<Linear8> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight, const std::optional<at::Tensor>& bias) {
        // What no gradient asks for is not kept: the weight may change then, as behind torch's own.
        ctx->save_for_backward({x.requires_grad() ? weight : at::Tensor(), weight.requires_grad() ? pack(x) : at::Tensor()});
        ctx->saved_data["bias"] = bias.has_value();
        ctx->saved_data["inputs"] = weight.size(1);
        return at::linear(x, weight, bias);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        return in_backward("linear8", [&]() -> variable_list {
            const variable_list saved = ctx->get_saved_variables();
            const at::Tensor &dy = grads[0], &weight = saved[0], &kept = saved[1];
            const at::NoGradGuard no_grad;
            at::Tensor dx, dw, db;
            if (ctx->needs_input_grad(0)) dx = at::matmul(dy, weight);
            const bool bias = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(2);
            if (kept.defined() && (bias || ctx->needs_input_grad(1))) std::tie(dw, db) = weight_grad(on_gpu("dy", dy), kept, ctx->saved_data["inputs"].toInt(), bias);
            else if (bias) db = dy.reshape({-1, dy.size(-1)}).sum(0);  // of a frozen weight
            if (!ctx->needs_input_grad(1)) dw = at::Tensor();
            return {dx, dw, db};
        });
    }
};

// linear8(x, weight, bias or None) -> y
PyObject* linear8(PyObject* const* args, Py_ssize_t nargs) {
    need_arguments(nargs, 3);
    at::Tensor x = tensor_of("x", args[0]), weight = tensor_of("weight", args[1]), bias = maybe_tensor("bias", args[2]);
    const std::optional<c10::impl::ExcludeDispatchKeyGuard> without_autocast = cast_by_autocast(x, {&x, &weight, &bias});
    same_place("weight", weight, x);
    same_dtype("weight", weight, x);
    if (x.dim() < 1 || weight.dim() != 2 || x.size(-1) != weight.size(1)) refuse("the input does not go into the weight");
    if (weight.numel() == 0) refuse("a projection has at least one input and one output");
    if (bias.defined()) {
        same_place("bias", bias, x);
        same_dtype("bias", bias, x);
        if (bias.dim() != 1 || bias.size(0) != weight.size(0)) refuse("the bias does not belong to the weight");
    }
    dtype_code("x", x);
    const std::optional<at::Tensor> b = bias.defined() ? std::optional<at::Tensor>(bias) : std::nullopt;
    return THPVariable_Wrap(wants_gradient({&x, &weight, &bias}) ? Linear8::apply(x, weight, b) : at::linear(x, weight, b));
}

// ---- rotation --------------------------------------------------------------------------------------------

struct Heads {
    at::Tensor t;
    std::int64_t batch = 1, tokens = 0, heads = 0, dim = 0;
    long long strides[3] = {0, 0, 0};
};
Heads heads_of(const char* what, const at::Tensor& given) {
    if (given.dim() != 3 && given.dim() != 4)
        refuse(std::string(what) + " must be [tokens, heads, dim] or [batch, tokens, heads, dim], got " + std::to_string(given.dim()) + " axes");
    Heads h;
    h.t = given.size(-1) == 1 || given.stride(-1) == 1 ? given : given.contiguous();
    const std::int64_t n = h.t.dim();
    h.dim = h.t.size(n - 1);
    h.heads = h.t.size(n - 2);
    h.tokens = h.t.size(n - 3);
    if (n == 4) h.batch = h.t.size(0);
    if (h.heads < 1) refuse(std::string(what) + " needs at least one head");
    if (h.heads > 65535) refuse(std::string(what) + " has " + std::to_string(h.heads) + " heads: at most 65535 are supported");
    // (Axes of one element have any stride: none that counts.)
    h.strides[0] = n == 4 && h.batch > 1 ? h.t.stride(0) : 0;
    h.strides[1] = h.tokens > 1 ? h.t.stride(n - 3) : 0;
    h.strides[2] = h.heads > 1 ? h.t.stride(n - 2) : 0;
    return h;
}

// How to turn: what queries and keys share.
struct Turn {
    at::Tensor positions, frequencies;
    bool interleaved = false;
    double magnitude = 1.0, eps = 0.0;
};

// The arguments that all rotations share; `first` gives place and type.
void shared_arguments(b2_rotation* c, const Heads& first, const Turn& turn) {
    c->dtype = dtype_code("queries or keys", first.t);
    const at::Tensor &positions = turn.positions, &frequencies = turn.frequencies;
    same_place("positions", positions, first.t);
    same_place("frequencies", frequencies, first.t);
    if (positions.scalar_type() != at::kLong && positions.scalar_type() != at::kInt) refuse("positions must be int64 or int32");
    if (frequencies.scalar_type() != at::kDouble || frequencies.dim() != 1 || !frequencies.is_contiguous())
        refuse("frequencies must be a float64 vector without gaps: in 32 bits the angles of far positions are lost");
    const std::int64_t n = positions.dim();
    if ((n != 1 && n != 2) || positions.size(n - 1) != first.tokens || (n == 2 && positions.size(0) != first.batch))
        refuse("positions must be [tokens] or [batch, tokens] of queries and keys");
    if (first.dim < 2 || first.dim % 2 != 0 || first.dim > 256) refuse("the head dimension must be even, and 2 to 256, got " + std::to_string(first.dim));
    if (2 * frequencies.numel() > first.dim)
        refuse(std::to_string(frequencies.numel()) + " frequencies turn " + std::to_string(2 * frequencies.numel()) + " elements, a head has " + std::to_string(first.dim));
    if (first.batch * first.tokens >= (1ll << 31)) refuse("batch * tokens must be below 2^31");
    c->batch = first.batch;
    c->tokens = first.tokens;
    c->dim = static_cast<int>(first.dim);
    c->rotated = static_cast<int>(2 * frequencies.numel());
    c->interleaved = turn.interleaved ? 1 : 0;
    c->magnitude = static_cast<float>(turn.magnitude);
    c->eps = static_cast<float>(turn.eps);
    c->positions = positions.data_ptr();
    c->position_bytes = positions.scalar_type() == at::kLong ? 8 : 4;
    c->position_strides[0] = n == 2 && first.batch > 1 ? positions.stride(0) : 0;
    c->position_strides[1] = first.tokens > 1 ? positions.stride(n - 1) : 0;
    c->frequencies = static_cast<const double*>(frequencies.data_ptr());
}

// Queries and keys, either of which may be left out.
struct Both {
    const char* names[2];
    Heads heads[2];
    bool there[2] = {false, false};
    int first = -1;
    const Heads& any() const { return heads[first]; }
};
Both both_of(const char* q_name, const char* k_name, const at::Tensor& q, const at::Tensor& k) {
    Both b;
    b.names[0] = q_name;
    b.names[1] = k_name;
    const at::Tensor* given[2] = {&q, &k};
    for (int i = 0; i < 2; ++i) {
        if (!given[i]->defined()) continue;
        const at::Tensor& t = on_gpu(b.names[i], *given[i]);
        if (b.first >= 0) {
            same_place(b.names[i], t, b.any().t);
            same_dtype(b.names[i], t, b.any().t);
        }
        const c10::cuda::CUDAGuard guard(t.device());
        b.heads[i] = heads_of(b.names[i], t);
        b.there[i] = true;
        if (b.first < 0) b.first = i;
        const Heads &x = b.any(), &y = b.heads[i];
        if (x.t.dim() != y.t.dim() || x.batch != y.batch || x.tokens != y.tokens || x.dim != y.dim)
            refuse(std::string(b.names[0]) + " and " + b.names[1] + " must agree in all but their heads");
    }
    if (b.first < 0) refuse(std::string(q_name) + " and " + k_name + " are both None");
    return b;
}

// (q, k) turned; what is left out stays undefined.
std::pair<at::Tensor, at::Tensor> rotate(const Both& b, const Turn& turn, bool inverse) {
    const Heads& first = b.any();
    const c10::cuda::CUDAGuard guard(first.t.device());
    b2_rotation c = {};
    shared_arguments(&c, first, turn);
    c.inverse = inverse ? 1 : 0;
    at::Tensor out[2];
    for (int i = 0; i < 2; ++i) {
        if (!b.there[i]) continue;
        const Heads& h = b.heads[i];
        out[i] = new_like(h.t);
        c.side[i].heads = static_cast<int>(h.heads);
        c.side[i].x = h.t.data_ptr();
        std::copy(h.strides, h.strides + 3, c.side[i].x_strides);
        c.side[i].out = out[i].data_ptr();
    }
    void* stream = stream_of(first.t);
    call([&] { return g.rotate_heads(&c, stream); });
    return {std::move(out[0]), std::move(out[1])};
}

// The outputs that are there, and the tuple that a caller gets of them.
variable_list defined_of(std::initializer_list<at::Tensor> tensors) {
    variable_list v;
    for (const at::Tensor& t : tensors)
        if (t.defined()) v.push_back(t);
    return v;
}
PyObject* pair_of(variable_list out, bool q, bool k) {
    at::Tensor first = q ? out.front() : at::Tensor(), second = k ? out.back() : at::Tensor();
    return two(std::move(first), std::move(second));
}
std::optional<at::Tensor> optional_of(const at::Tensor& t) { return t.defined() ? std::optional<at::Tensor>(t) : std::nullopt; }
at::Tensor value_of(const std::optional<at::Tensor>& t) { return t.has_value() ? *t : at::Tensor(); }

// The rest of an autograd node: its Turn, and which sides there are with how many heads.
void save_turn(AutogradContext* ctx, const Turn& turn, std::int64_t q_heads, std::int64_t k_heads) {
    ctx->saved_data["numbers"] = std::vector<double>{turn.magnitude, turn.eps};
    ctx->saved_data["whole"] = std::vector<std::int64_t>{turn.interleaved ? 1 : 0, q_heads, k_heads};
    ctx->set_materialize_grads(false);
}
struct SavedTurn {
    Turn turn;
    std::int64_t heads[2];
    at::Tensor grad[2];  // undefined where an output was not used
};
SavedTurn saved_turn(AutogradContext* ctx, const variable_list& grads, const at::Tensor& positions, const at::Tensor& frequencies) {
    SavedTurn s;
    const std::vector<double> numbers = ctx->saved_data["numbers"].toDoubleVector();
    const std::vector<std::int64_t> whole = ctx->saved_data["whole"].toIntVector();
    s.turn = {positions, frequencies, whole[0] != 0, numbers[0], numbers[1]};
    std::size_t at = 0;
    for (int i = 0; i < 2; ++i) {
        s.heads[i] = whole[1 + i];
        if (s.heads[i] != 0) s.grad[i] = grads[at++];
    }
    return s;
}
std::int64_t heads_in(const at::Tensor& t) { return t.defined() && t.dim() >= 3 ? t.size(-2) : 0; }

using MaybeTensor = std::optional<at::Tensor>;

struct Rotary : torch::autograd::Function<Rotary> {
    static variable_list forward(AutogradContext* ctx, const MaybeTensor& q, const MaybeTensor& k, const at::Tensor& positions, const at::Tensor& frequencies,
                                 bool interleaved, double magnitude) {
        const Turn turn{positions, frequencies, interleaved, magnitude, 0.0};
        const at::Tensor q_ = value_of(q), k_ = value_of(k);
        auto [q_out, k_out] = rotate(both_of("q", "k", q_, k_), turn, false);
        ctx->save_for_backward({positions, frequencies});
        save_turn(ctx, turn, heads_in(q_), heads_in(k_));
        return defined_of({q_out, k_out});
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        return in_backward("rotary", [&]() -> variable_list {
            const variable_list saved = ctx->get_saved_variables();
            const SavedTurn s = saved_turn(ctx, grads, saved[0], saved[1]);
            at::Tensor dq, dk;
            if (s.grad[0].defined() || s.grad[1].defined()) std::tie(dq, dk) = rotate(both_of("dq", "dk", s.grad[0], s.grad[1]), s.turn, true);
            return {dq, dk, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
        });
    }
};

// rotary(q, k, positions, frequencies, interleaved, magnitude) -> (q, k)
PyObject* rotary(PyObject* const* args, Py_ssize_t nargs) {
    need_arguments(nargs, 6);
    const at::Tensor q = maybe_tensor("q", args[0]), k = maybe_tensor("k", args[1]);
    const Turn turn{tensor_of("positions", args[2]), tensor_of("frequencies", args[3]), truth(args[4]), number("magnitude", args[5]), 0.0};
    no_gradient_of("frequencies", turn.frequencies);
    if (wants_gradient({&q, &k}))
        return pair_of(Rotary::apply(optional_of(q), optional_of(k), turn.positions, turn.frequencies, turn.interleaved, turn.magnitude), q.defined(), k.defined());
    auto [q_out, k_out] = rotate(both_of("q", "k", q, k), turn, false);
    return two(std::move(q_out), std::move(k_out));
}

const at::Tensor& weight_of(const char* what, const at::Tensor& w, const Heads& h) {
    if (!w.defined()) refuse(std::string(what) + " is None");
    on_gpu(what, w);
    same_place(what, w, h.t);
    same_dtype(what, w, h.t);
    if (w.dim() != 1 || w.size(0) != h.dim || !w.is_contiguous()) refuse(std::string(what) + " must be a vector of the head dimension without gaps");
    return w;
}

// Bytes of the 8-bit form of queries and keys: codes of both, then scales of both.
struct KeptHeads {
    std::int64_t codes[2] = {0, 0}, scales[2] = {0, 0}, bytes = 0;
};
KeptHeads kept_heads(std::int64_t tokens, std::int64_t q_heads, std::int64_t k_heads, std::int64_t dim) {
    const std::int64_t pitch = (dim + 15) / 16 * 16, q = tokens * q_heads, k = tokens * k_heads;
    KeptHeads h;
    h.codes[1] = q * pitch;
    h.scales[0] = (q + k) * pitch;
    h.scales[1] = h.scales[0] + q;
    h.bytes = h.scales[1] + k;
    return h;
}

constexpr const char* kWeightNames[2] = {"q_weight", "k_weight"};

struct NormRotated {
    at::Tensor out[2], kept;
};
NormRotated norm_rotate(const Both& b, const at::Tensor (&weights)[2], const Turn& turn, bool keep) {
    const Heads& first = b.any();
    const c10::cuda::CUDAGuard guard(first.t.device());
    b2_rotation c = {};
    shared_arguments(&c, first, turn);
    c.norm = 1;
    for (int i = 0; i < 2; ++i)
        if (b.there[i]) c.side[i].weight = weight_of(kWeightNames[i], weights[i], b.heads[i]).data_ptr();
    NormRotated r;
    KeptHeads k8;
    if (keep) {
        k8 = kept_heads(first.batch * first.tokens, b.heads[0].heads, b.heads[1].heads, first.dim);
        r.kept = new_bytes(first.t, k8.bytes);
    }
    for (int i = 0; i < 2; ++i) {
        if (!b.there[i]) continue;
        const Heads& h = b.heads[i];
        r.out[i] = new_like(h.t);
        c.side[i].heads = static_cast<int>(h.heads);
        c.side[i].x = h.t.data_ptr();
        std::copy(h.strides, h.strides + 3, c.side[i].x_strides);
        c.side[i].out = r.out[i].data_ptr();
        if (keep) {
            c.side[i].codes = bytes_at(r.kept, k8.codes[i]);
            c.side[i].scales = bytes_at(r.kept, k8.scales[i]);
        }
    }
    void* stream = stream_of(first.t);
    call([&] { return g.rotate_heads(&c, stream); });
    return r;
}

struct NormRotary : torch::autograd::Function<NormRotary> {
    static variable_list forward(AutogradContext* ctx, const MaybeTensor& q, const MaybeTensor& k, const MaybeTensor& q_weight, const MaybeTensor& k_weight,
                                 const at::Tensor& positions, const at::Tensor& frequencies, bool interleaved, double magnitude, double eps, bool keep8) {
        const Turn turn{positions, frequencies, interleaved, magnitude, eps};
        const at::Tensor q_ = value_of(q), k_ = value_of(k), weights[2] = {value_of(q_weight), value_of(k_weight)};
        const NormRotated r = norm_rotate(both_of("q", "k", q_, k_), weights, turn, keep8);
        ctx->save_for_backward({keep8 ? at::Tensor() : q_, keep8 ? at::Tensor() : k_, r.kept, weights[0], weights[1], positions, frequencies});
        save_turn(ctx, turn, heads_in(q_), heads_in(k_));
        return defined_of({r.out[0], r.out[1]});
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        return in_backward("qk_norm_rotary", [&]() -> variable_list {
            const variable_list saved = ctx->get_saved_variables();
            const SavedTurn s = saved_turn(ctx, grads, saved[5], saved[6]);
            variable_list result(10);
            if (!s.grad[0].defined() && !s.grad[1].defined()) return result;
            const Both b = both_of("dq", "dk", s.grad[0], s.grad[1]);
            const Heads& first = b.any();
            const c10::cuda::CUDAGuard guard(first.t.device());
            b2_rotation c = {};
            shared_arguments(&c, first, s.turn);
            c.norm = 1;
            const at::Tensor& kept = saved[2];
            KeptHeads k8;
            if (kept.defined()) {
                k8 = kept_heads(first.batch * first.tokens, s.heads[0], s.heads[1], first.dim);
                same_place("the 8-bit form", kept_of(kept, k8.bytes), first.t);
            }
            Heads x[2];
            at::Tensor partial[2];
            const auto options = first.t.options().requires_grad(false);
            for (int i = 0; i < 2; ++i) {
                if (!b.there[i]) continue;
                const Heads& h = b.heads[i];
                if (h.heads != s.heads[i]) refuse("a gradient has another shape than its queries or keys");
                b2_heads& side = c.side[i];
                result[i] = new_like(h.t);
                result[2 + i] = at::empty({h.dim}, options);
                partial[i] = at::empty({B2_HEAD_GRAD_PARTIALS * h.dim}, options.dtype(at::kFloat));
                side.heads = static_cast<int>(h.heads);
                side.grad = h.t.data_ptr();
                std::copy(h.strides, h.strides + 3, side.grad_strides);
                side.out = result[i].data_ptr();
                side.weight = weight_of(kWeightNames[i], saved[3 + i], h).data_ptr();
                side.weight_grad = result[2 + i].data_ptr();
                side.partial = partial[i].data_ptr();
                if (kept.defined()) {
                    side.codes = bytes_at(kept, k8.codes[i]);
                    side.scales = bytes_at(kept, k8.scales[i]);
                } else {
                    if (saved[i].sizes() != h.t.sizes()) refuse("a gradient has another shape than its queries or keys");
                    same_place("a gradient", h.t, saved[i]);
                    same_dtype("a gradient", h.t, saved[i]);
                    x[i] = heads_of(i == 0 ? "q" : "k", saved[i]);
                    side.x = x[i].t.data_ptr();
                    std::copy(x[i].strides, x[i].strides + 3, side.x_strides);
                }
            }
            void* stream = stream_of(first.t);
            call([&] { return g.rotate_heads_backward(&c, stream); });
            return result;
        });
    }
};

// qk_norm_rotary(q, k, q_weight, k_weight, positions, frequencies, interleaved, magnitude, eps, keep8) -> (q, k)
PyObject* qk_norm_rotary(PyObject* const* args, Py_ssize_t nargs) {
    need_arguments(nargs, 10);
    const at::Tensor q = maybe_tensor("q", args[0]), k = maybe_tensor("k", args[1]);
    const at::Tensor weights[2] = {maybe_tensor(kWeightNames[0], args[2]), maybe_tensor(kWeightNames[1], args[3])};
    const Turn turn{tensor_of("positions", args[4]), tensor_of("frequencies", args[5]), truth(args[6]), number("magnitude", args[7]), number("eps", args[8])};
    const bool keep8 = truth(args[9]);
    no_gradient_of("frequencies", turn.frequencies);
    if (wants_gradient({&q, &k, &weights[0], &weights[1]}))
        return pair_of(NormRotary::apply(optional_of(q), optional_of(k), optional_of(weights[0]), optional_of(weights[1]), turn.positions, turn.frequencies,
                                         turn.interleaved, turn.magnitude, turn.eps, keep8),
                       q.defined(), k.defined());
    const NormRotated r = norm_rotate(both_of("q", "k", q, k), weights, turn, false);
    return two(r.out[0], r.out[1]);
}

}  // namespace

PyMethodDef train_methods[] = {
    {"pack8", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<pack8>)), METH_FASTCALL, nullptr},
    {"unpack8", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<unpack8>)), METH_FASTCALL, nullptr},
    {"gelu8", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<gelu8>)), METH_FASTCALL, nullptr},
    {"weight_grad8", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<weight_grad8>)), METH_FASTCALL, nullptr},
    {"linear8", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<linear8>)), METH_FASTCALL, nullptr},
    {"rotary", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<rotary>)), METH_FASTCALL, nullptr},
    {"qk_norm_rotary", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<qk_norm_rotary>)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

bool bind_train(PyObject* error_class, PyObject* addresses) {
    constexpr Py_ssize_t kAddresses = 18;
    unsigned long long a[kAddresses];
    if (!PyTuple_Check(addresses) || PyTuple_GET_SIZE(addresses) != kAddresses) {
        PyErr_Format(PyExc_TypeError, "expected a tuple of %zd addresses", kAddresses);
        return false;
    }
    for (Py_ssize_t i = 0; i < kAddresses; ++i) {
        a[i] = PyLong_AsUnsignedLongLong(PyTuple_GET_ITEM(addresses, i));
        if (PyErr_Occurred()) return false;
    }
    const auto take = [](auto& f, unsigned long long v) { f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(static_cast<std::uintptr_t>(v)); };
    take(g_last_error, a[0]);
    take(g.pack8, a[1]);
    take(g.unpack8, a[2]);
    take(g.gelu8_forward, a[3]);
    take(g.gelu8_backward, a[4]);
    take(g.weight_grad8_workspace, a[5]);
    take(g.weight_grad8, a[6]);
    take(g.rotate_heads, a[7]);
    take(g.rotate_heads_backward, a[8]);
    bind_vocabulary(a + 9);
    Py_INCREF(error_class);
    Py_XSETREF(g_error_class, error_class);
    return true;
}

}  // namespace b200ccl::python
