// The operators at the two ends of a training step (include/b200ccl/vocabulary_ops.h) on torch tensors, in the manner of torch_ops.cc.
#include "torch_common.h"

#include "b200ccl/vocabulary_ops.h"

#include <ATen/Functions.h>

#include <type_traits>

namespace b200ccl::python {

namespace {

struct Functions {
    decltype(&b2_embed) embed = nullptr;
    decltype(&b2_embed_backward_workspace) embed_backward_workspace = nullptr;
    decltype(&b2_embed_backward) embed_backward = nullptr;
    decltype(&b2_vocabulary_loss_sizes) loss_sizes = nullptr;
    decltype(&b2_vocabulary_loss_forward) loss_forward = nullptr;
    decltype(&b2_vocabulary_loss_backward) loss_backward = nullptr;
    decltype(&b2_vocabulary_loss_both_workspace) both_workspace = nullptr;
    decltype(&b2_vocabulary_loss_both) both = nullptr;
    decltype(&b2_vocabulary_loss_times) times = nullptr;
} g;

const at::Tensor& whole_numbers(const char* what, const at::Tensor& t) {
    if (t.scalar_type() != at::kLong && t.scalar_type() != at::kInt) refuse(std::string(what) + " must be int64 or int32");
    return t;
}
int bytes_of(const at::Tensor& t) { return t.scalar_type() == at::kLong ? 8 : 4; }

// All elements, evenly apart.
Rows flat_of(const char* what, const at::Tensor& t) { return rows_of(what, t.unsqueeze(-1)); }

Rows matrix_of(const char* what, const at::Tensor& t) {
    if (t.dim() != 2 || t.numel() == 0) refuse(std::string(what) + " must be [vocabulary, width], at least one of each");
    return rows_of(what, t);
}

// ---- embedding -------------------------------------------------------------------------------------------

b2_embedding embedding_call(const Rows& tokens, std::int64_t vocabulary, std::int64_t width, int dtype, double scale) {
    b2_embedding c = {};
    c.dtype = dtype;
    c.tokens = tokens.t.data_ptr();
    c.token_bytes = bytes_of(tokens.t);
    c.token_stride = tokens.stride;
    c.count = tokens.rows;
    c.vocabulary = vocabulary;
    c.width = width;
    c.scale = static_cast<float>(scale);
    return c;
}

at::Tensor embed(const at::Tensor& tokens, const at::Tensor& weight, double scale) {
    const int dtype = dtype_code("weight", weight);
    const c10::cuda::CUDAGuard guard(weight.device());
    const Rows flat = flat_of("tokens", tokens), w = matrix_of("weight", weight);
    std::vector<std::int64_t> sizes = tokens.sizes().vec();
    sizes.push_back(w.columns);
    at::Tensor out = at::empty(sizes, weight.options().requires_grad(false));
    b2_embedding c = embedding_call(flat, w.rows, w.columns, dtype, scale);
    c.rows = w.t.data_ptr();
    c.stride = w.stride;
    c.out = out.data_ptr();
    void* stream = stream_of(weight);
    call([&] { return g.embed(&c, stream); });
    return out;
}

struct Embedding : torch::autograd::Function<Embedding> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& tokens, const at::Tensor& weight, double scale) {
        ctx->save_for_backward({tokens});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["sizes"] = weight.sizes().vec();
        return embed(tokens, weight, scale);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        return in_backward("embedding", [&]() -> variable_list {
            const at::Tensor& dy = on_gpu("dy", grads[0]);
            const at::Tensor tokens = ctx->get_saved_variables()[0];
            const std::vector<std::int64_t> sizes = ctx->saved_data["sizes"].toIntVector();
            same_place("dy", dy, tokens);
            const int dtype = dtype_code("dy", dy);
            const c10::cuda::CUDAGuard guard(dy.device());
            const Rows flat = flat_of("tokens", tokens), r = rows_of("dy", dy);
            if (r.columns != sizes[1] || dy.numel() != tokens.numel() * sizes[1]) refuse("dy has another shape than the result");
            at::Tensor dw = at::empty(sizes, dy.options().requires_grad(false)), workspace;
            b2_embedding c = embedding_call(flat, sizes[0], sizes[1], dtype, ctx->saved_data["scale"].toDouble());
            c.rows = r.t.data_ptr();
            c.stride = r.stride;
            c.out = dw.data_ptr();
            std::size_t bytes = 0;
            call([&] { return g.embed_backward_workspace(&c, &bytes); });
            if (bytes != 0) {
                workspace = new_bytes(dy, static_cast<std::int64_t>(bytes));
                c.workspace = workspace.data_ptr();
            }
            void* stream = stream_of(dy);
            call([&] { return g.embed_backward(&c, stream); });
            return {at::Tensor(), dw, at::Tensor()};
        });
    }
};

// embedding(tokens, weight, scale) -> y
PyObject* embedding(PyObject* const* args, Py_ssize_t nargs) {
    need_arguments(nargs, 3);
    const at::Tensor &tokens = whole_numbers("tokens", tensor_of("tokens", args[0])), &weight = tensor_of("weight", args[1]);
    const double scale = number("scale", args[2]);
    same_place("weight", weight, tokens);
    if (weight.dim() != 2 || weight.numel() == 0) refuse("weight must be [vocabulary, width], at least one of each");
    return THPVariable_Wrap(wants_gradient({&weight}) ? Embedding::apply(tokens, weight, scale) : embed(tokens, weight, scale));
}

// ---- losses ----------------------------------------------------------------------------------------------

// What a loss is asked for beside its tensors.
struct Asked {
    std::int64_t entries = 0;  // 0: cross entropy
    double temperature = 1.0;
    std::int64_t reduction = 0;
};

// Tensors whose memory a call points to.
struct Prepared {
    b2_vocabulary_loss c = {};
    Rows x, weight, targets, teacher;
};

void prepare(Prepared* p, const at::Tensor& x, const at::Tensor& weight, const at::Tensor& targets, const Asked& asked) {
    p->x = rows_of("x", x);
    p->weight = matrix_of("weight", weight);
    p->targets = asked.entries != 0 ? rows_of("teacher_tokens", targets) : flat_of("targets", targets);
    b2_vocabulary_loss& c = p->c;
    c.dtype = dtype_code("x", x);
    c.x = p->x.t.data_ptr();
    c.x_stride = p->x.stride;
    c.weight = p->weight.t.data_ptr();
    c.weight_stride = p->weight.stride;
    c.tokens = p->x.rows;
    c.width = p->x.columns;
    c.vocabulary = p->weight.rows;
    c.targets = p->targets.t.data_ptr();
    c.target_bytes = bytes_of(p->targets.t);
    c.target_strides[0] = p->targets.stride;
    c.target_strides[1] = 1;
    c.entries = static_cast<int>(asked.entries);
    c.temperature = static_cast<float>(asked.temperature);
    c.reduction = static_cast<int>(asked.reduction);
}

struct Lost {
    at::Tensor loss, kept;           // kept: what the backward pass reads
    at::Tensor x_grad, weight_grad;  // made with the loss, but for what comes back to it
};

// wanted: gradients that will be asked for, and may be made with the loss.
Lost loss_forward(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& targets, const at::Tensor& teacher, const Asked& asked, bool x_wanted, bool weight_wanted) {
    const c10::cuda::CUDAGuard guard(x.device());
    Prepared p;
    prepare(&p, x, weight, targets, asked);
    if (asked.entries != 0) {
        p.c.teacher_dtype = dtype_code("teacher_logits", teacher);
        p.teacher = rows_of("teacher_logits", teacher);
        p.c.teacher = p.teacher.t.data_ptr();
        p.c.teacher_strides[0] = p.teacher.stride;
        p.c.teacher_strides[1] = 1;
    }
    const auto options = x.options().dtype(at::kFloat).requires_grad(false);
    Lost r;
    r.loss = at::empty(asked.reduction == 0 ? x.sizes().slice(0, x.dim() - 1).vec() : std::vector<std::int64_t>(), options);
    std::size_t floats = 0, bytes = 0, both = 0;
    call([&] { return g.loss_sizes(&p.c, 0, &floats, &bytes); });
    r.kept = at::empty({static_cast<std::int64_t>(floats)}, options);
    p.c.loss = static_cast<float*>(r.loss.data_ptr());
    p.c.kept = static_cast<float*>(r.kept.data_ptr());
    if ((x_wanted || weight_wanted) && x.scalar_type() == at::kBFloat16 && asked.reduction != 0) {
        // (The size depends on which of them there are, and not on where: they are allocated if they are made.)
        p.c.x_grad = x_wanted ? p.x.t.data_ptr() : nullptr;
        p.c.weight_grad = weight_wanted ? p.weight.t.data_ptr() : nullptr;
        call([&] { return g.both_workspace(&p.c, &both); });
        if (both != 0 && x_wanted) r.x_grad = new_like(x);
        if (both != 0 && weight_wanted) r.weight_grad = new_like(weight);
        p.c.x_grad = r.x_grad.defined() ? r.x_grad.data_ptr() : nullptr;
        p.c.weight_grad = r.weight_grad.defined() ? r.weight_grad.data_ptr() : nullptr;
    }
    at::Tensor workspace = new_bytes(x, static_cast<std::int64_t>(both != 0 ? both : bytes));
    p.c.workspace = workspace.data_ptr();
    void* stream = stream_of(x);
    if (both != 0) call([&] { return g.both(&p.c, stream); });
    else call([&] { return g.loss_forward(&p.c, stream); });
    return r;
}

// The capture that the current stream is part of; 0: none.
std::int64_t capture_of(const at::Tensor& t) {
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    unsigned long long id = 0;
    if (cudaStreamGetCaptureInfo(static_cast<cudaStream_t>(stream_of(t)), &status, &id) != cudaSuccess) {
        (void)cudaGetLastError();
        throw Failed("the stream's capture has failed");
    }
    return status == cudaStreamCaptureStatusNone ? 0 : static_cast<std::int64_t>(id);
}

struct VocabularyLoss : torch::autograd::Function<VocabularyLoss> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight, const at::Tensor& targets, const std::optional<at::Tensor>& teacher,
                              std::int64_t entries, double temperature, std::int64_t reduction) {
        const c10::cuda::CUDAGuard guard(x.device());
        Lost r = loss_forward(x, weight, targets, teacher.has_value() ? *teacher : at::Tensor(), {entries, temperature, reduction}, x.requires_grad(), weight.requires_grad());
        ctx->save_for_backward({x, weight, targets, r.kept});
        // (Not among what is saved: whoever asks for them first takes them away. Only in the capture that they were made in: a graph of the
        // backward pass alone would multiply them at each replay.)
        ctx->saved_data["capture"] = capture_of(x);
        if (r.x_grad.defined()) ctx->saved_data["dx"] = std::move(r.x_grad);
        if (r.weight_grad.defined()) ctx->saved_data["dw"] = std::move(r.weight_grad);
        ctx->saved_data["temperature"] = temperature;
        ctx->saved_data["whole"] = std::vector<std::int64_t>{entries, reduction};
        return r.loss;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        return in_backward("the loss", [&]() -> variable_list {
            const variable_list saved = ctx->get_saved_variables();
            const at::Tensor &x = saved[0], &weight = saved[1], &kept = saved[3], &dloss = on_gpu("dloss", grads[0]);
            const std::vector<std::int64_t> whole = ctx->saved_data["whole"].toIntVector();
            const Asked asked{whole[0], ctx->saved_data["temperature"].toDouble(), whole[1]};
            same_place("dloss", dloss, x);
            if (dloss.scalar_type() != at::kFloat) refuse("dloss must be float32");
            const c10::cuda::CUDAGuard guard(x.device());
            Prepared p;
            prepare(&p, x, weight, saved[2], asked);
            const Rows back = flat_of("dloss", dloss);
            if (dloss.numel() != (asked.reduction == 0 ? p.x.rows : 1)) refuse("dloss has another shape than the loss");
            variable_list result(7);
            p.c.kept = static_cast<float*>(kept.data_ptr());
            p.c.loss_grad = static_cast<const float*>(back.t.data_ptr());
            p.c.loss_grad_stride = back.stride;
            void* stream = stream_of(x);
            // What was made with the loss, once; asked for again, it is made from the logits, as if it had not been.
            constexpr const char* kMade[2] = {"dx", "dw"};
            void** const gradients[2] = {&p.c.x_grad, &p.c.weight_grad};
            for (int i = 0; i < 2; ++i) {
                const auto made = ctx->saved_data.find(kMade[i]);
                if (!ctx->needs_input_grad(i) || made == ctx->saved_data.end() || ctx->saved_data["capture"].toInt() != capture_of(x)) continue;
                result[i] = made->second.toTensor();
                ctx->saved_data.erase(made);
                *gradients[i] = result[i].data_ptr();
            }
            if (p.c.x_grad != nullptr || p.c.weight_grad != nullptr) call([&] { return g.times(&p.c, stream); });
            p.c.x_grad = p.c.weight_grad = nullptr;
            for (int i = 0; i < 2; ++i) {
                if (!ctx->needs_input_grad(i) || result[i].defined()) continue;
                result[i] = new_like(i == 0 ? x : weight);
                *gradients[i] = result[i].data_ptr();
            }
            if (p.c.x_grad == nullptr && p.c.weight_grad == nullptr) return result;
            std::size_t bytes = 0;
            call([&] { return g.loss_sizes(&p.c, 1, nullptr, &bytes); });
            at::Tensor workspace = new_bytes(x, static_cast<std::int64_t>(bytes));
            p.c.workspace = workspace.data_ptr();
            call([&] { return g.loss_backward(&p.c, stream); });
            return result;
        });
    }
};

PyObject* loss_of(at::Tensor x, at::Tensor weight, const at::Tensor& targets, const at::Tensor& teacher, const Asked& asked) {
    const auto without_autocast = cast_by_autocast(x, {&x, &weight});
    same_place("weight", weight, x);
    same_dtype("weight", weight, x);
    dtype_code("x", x);
    if (x.dim() < 1 || weight.dim() != 2 || x.size(-1) != weight.size(1)) refuse("the input does not go into the weight");
    if (weight.numel() == 0) refuse("weight must be [vocabulary, width], at least one of each");
    if (wants_gradient({&x, &weight})) {
        const std::optional<at::Tensor> maybe = teacher.defined() ? std::optional<at::Tensor>(teacher) : std::nullopt;
        return THPVariable_Wrap(VocabularyLoss::apply(x, weight, targets, maybe, asked.entries, asked.temperature, asked.reduction));
    }
    return THPVariable_Wrap(loss_forward(x, weight, targets, teacher, asked, false, false).loss);
}

std::int64_t reduction_of(PyObject* obj) {
    const long v = PyLong_AsLong(obj);
    if (v == -1 && PyErr_Occurred()) throw Raised{};
    return v;
}

// linear_cross_entropy(x, weight, targets, reduction) -> loss
PyObject* linear_cross_entropy(PyObject* const* args, Py_ssize_t nargs) {
    need_arguments(nargs, 4);
    const at::Tensor &x = tensor_of("x", args[0]), &weight = tensor_of("weight", args[1]), &targets = whole_numbers("targets", tensor_of("targets", args[2]));
    same_place("targets", targets, x);
    if (x.dim() < 1 || targets.sizes() != x.sizes().slice(0, x.dim() - 1)) refuse("targets must have one element for each row of x");
    return loss_of(x, weight, targets, at::Tensor(), {0, 1.0, reduction_of(args[3])});
}

// linear_distillation(x, weight, teacher_logits, teacher_tokens, temperature, reduction) -> loss
PyObject* linear_distillation(PyObject* const* args, Py_ssize_t nargs) {
    need_arguments(nargs, 6);
    const at::Tensor &x = tensor_of("x", args[0]), &weight = tensor_of("weight", args[1]), &logits = tensor_of("teacher_logits", args[2]);
    const at::Tensor& tokens = whole_numbers("teacher_tokens", tensor_of("teacher_tokens", args[3]));
    same_place("teacher_logits", logits, x);
    same_place("teacher_tokens", tokens, x);
    no_gradient_of("teacher_logits", logits);
    dtype_code("teacher_logits", logits);
    if (x.dim() < 1 || tokens.dim() != x.dim() || tokens.sizes().slice(0, x.dim() - 1) != x.sizes().slice(0, x.dim() - 1) || logits.sizes() != tokens.sizes())
        refuse("teacher_logits and teacher_tokens must be [..., entries] with one row for each of x");
    const std::int64_t entries = tokens.size(-1);
    if (entries < 1 || entries > 256) refuse("a teacher has 1 to 256 entries, got " + std::to_string(entries));
    return loss_of(x, weight, tokens, logits, {entries, number("temperature", args[4]), reduction_of(args[5])});
}

}  // namespace

PyMethodDef vocabulary_methods[] = {
    {"embedding", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<embedding>)), METH_FASTCALL, nullptr},
    {"linear_cross_entropy", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<linear_cross_entropy>)), METH_FASTCALL, nullptr},
    {"linear_distillation", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<linear_distillation>)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

void bind_vocabulary(const unsigned long long* a) {
    const auto take = [](auto& f, unsigned long long v) { f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(static_cast<std::uintptr_t>(v)); };
    take(g.embed, a[0]);
    take(g.embed_backward_workspace, a[1]);
    take(g.embed_backward, a[2]);
    take(g.loss_sizes, a[3]);
    take(g.loss_forward, a[4]);
    take(g.loss_backward, a[5]);
    take(g.both_workspace, a[6]);
    take(g.both, a[7]);
    take(g.times, a[8]);
}

}  // namespace b200ccl::python
