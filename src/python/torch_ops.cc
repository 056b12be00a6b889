// The training operators (include/b200ccl/train_ops.h) on torch tensors: what a raw pointer does not show is checked here, outputs and scratch come from
// torch's allocator (on the current stream of the tensors' device, so a captured call's memory is its graph's), and the call goes to the
// C interface by the addresses handed over in bind().
#include "torch_ops.h"

#include "b200ccl/train_ops.h"

#include <ATen/Functions.h>
#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdint>
#include <string>
#include <type_traits>
#include <utility>
#include <vector>

namespace b200ccl::python {

namespace {

PyObject* g_error_class = nullptr;
struct Functions {
    const char* (*last_error)() = nullptr;
    decltype(&b2_pack8) pack8 = nullptr;
    decltype(&b2_unpack8) unpack8 = nullptr;
    decltype(&b2_gelu8_forward) gelu8_forward = nullptr;
    decltype(&b2_gelu8_backward) gelu8_backward = nullptr;
    decltype(&b2_weight_grad8_workspace) weight_grad8_workspace = nullptr;
    decltype(&b2_weight_grad8) weight_grad8 = nullptr;
    decltype(&b2_rotate_heads) rotate_heads = nullptr;
    decltype(&b2_rotate_heads_backward) rotate_heads_backward = nullptr;
} g;

// A Python error is set.
struct Raised {};

[[noreturn]] void refuse(const std::string& why) {
    PyErr_SetString(PyExc_ValueError, why.c_str());
    throw Raised{};
}

void need_arguments(Py_ssize_t got, Py_ssize_t want) {
    if (got == want) return;
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, got);
    throw Raised{};
}

int dtype_code(const char* what, const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return 0;
        case at::kHalf: return 1;
        case at::kBFloat16: return 2;
        default: refuse(std::string(what) + " has dtype " + c10::toString(t.scalar_type()) + ": float32, float16 and bfloat16 are supported");
    }
}

const at::Tensor& tensor_of(const char* what, PyObject* obj) {
    if (!THPVariable_Check(obj)) refuse(std::string(what) + " must be a tensor");
    const at::Tensor& t = THPVariable_Unpack(obj);
    if (!t.is_cuda() || t.layout() != at::kStrided) refuse(std::string(what) + " must be a dense CUDA tensor");
    return t;
}

void same_place(const char* what, const at::Tensor& t, const at::Tensor& first) {
    if (t.get_device() != first.get_device())
        refuse(std::string(what) + " lives on cuda:" + std::to_string(t.get_device()) + ", the other tensors on cuda:" + std::to_string(first.get_device()));
}
void same_dtype(const char* what, const at::Tensor& t, const at::Tensor& first) {
    if (t.scalar_type() != first.scalar_type())
        refuse(std::string(what) + " has dtype " + c10::toString(t.scalar_type()) + ", expected " + c10::toString(first.scalar_type()));
}

double number(const char* what, PyObject* obj) {
    const double v = PyFloat_AsDouble(obj);
    if (v == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        refuse(std::string(what) + " must be a number");
    }
    return v;
}
bool truth(PyObject* obj) {
    const int v = PyObject_IsTrue(obj);
    if (v < 0) throw Raised{};
    return v != 0;
}

template <typename F>
void call(F&& f) {
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f();
    Py_END_ALLOW_THREADS
    if (rc != 0) {
        PyErr_SetString(rc == 2 ? PyExc_ValueError : g_error_class, g.last_error());
        throw Raised{};
    }
}

void* stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(t.get_device())).stream(); }

// A tensor as rows of its last axis, `stride` elements apart; a copy without gaps where it does not lie so.
struct Rows {
    at::Tensor t;
    std::int64_t rows = 1, columns = 0, stride = 0;
};
Rows rows_of(const char* what, const at::Tensor& t) {
    if (t.dim() == 0) refuse(std::string(what) + " needs at least one axis");
    Rows r;
    r.columns = t.size(-1);
    bool even = r.columns == 1 || t.stride(-1) == 1;
    std::int64_t step = 0;
    for (std::int64_t d = t.dim() - 2; d >= 0 && even; --d) {
        const std::int64_t n = t.size(d);
        if (n == 1) continue;
        if (r.rows == 1) step = t.stride(d);
        else even = t.stride(d) == step * r.rows;
        r.rows *= n;
    }
    r.t = t;
    r.stride = step;
    if (!even) {
        r.t = t.contiguous();
        r.rows = r.columns == 0 ? 0 : r.t.numel() / r.columns;
        r.stride = r.columns;
    }
    if (t.numel() == 0) r.rows = 0;
    if (r.rows <= 1) r.stride = r.columns;
    return r;
}

// The 8-bit form in one tensor of bytes: codes, then scales.
struct Kept {
    std::int64_t codes = 0, scales = 0;
};
Kept kept_bytes(std::int64_t rows, std::int64_t columns) {
    const std::int64_t blocks = rows * ((columns + 31) / 32);
    return {blocks * 32, blocks};
}
at::Tensor new_bytes(const at::Tensor& like, std::int64_t n) { return at::empty({n}, like.options().dtype(at::kByte).requires_grad(false)); }
unsigned char* bytes_at(const at::Tensor& t, std::int64_t at) { return static_cast<unsigned char*>(t.data_ptr()) + at; }

const at::Tensor& kept_of(PyObject* obj, std::int64_t bytes) {
    const at::Tensor& t = tensor_of("the 8-bit form", obj);
    if (t.scalar_type() != at::kByte || !t.is_contiguous() || t.numel() != bytes)
        refuse("the 8-bit form has " + std::to_string(t.numel()) + " elements, expected " + std::to_string(bytes) + " bytes without gaps");
    return t;
}

// pack8(x) -> bytes
PyObject* pack8(PyObject* const* args, Py_ssize_t nargs) {
    need_arguments(nargs, 1);
    const at::Tensor& x = tensor_of("x", args[0]);
    const int dtype = dtype_code("x", x);
    const c10::cuda::CUDAGuard guard(x.device());
    const Rows r = rows_of("x", x);
    const Kept k = kept_bytes(r.rows, r.columns);
    at::Tensor out = new_bytes(x, k.codes + k.scales);
    void* stream = stream_of(x);
    call([&] { return g.pack8(r.t.data_ptr(), r.stride, r.rows, r.columns, dtype, bytes_at(out, 0), bytes_at(out, k.codes), stream); });
    return THPVariable_Wrap(std::move(out));
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
    const at::Tensor& kept = kept_of(args[0], k.codes + k.scales);
    const c10::cuda::CUDAGuard guard(kept.device());
    at::Tensor out = at::empty(sizes, kept.options().dtype(reinterpret_cast<THPDtype*>(args[2])->scalar_type));
    const int dtype = dtype_code("the 8-bit form", out);
    void* stream = stream_of(kept);
    call([&] { return g.unpack8(bytes_at(kept, 0), bytes_at(kept, k.codes), rows, sizes.back(), dtype, out.data_ptr(), stream); });
    return THPVariable_Wrap(std::move(out));
}

PyObject* two(at::Tensor a, at::Tensor b) {
    PyObject* x = a.defined() ? THPVariable_Wrap(std::move(a)) : Py_NewRef(Py_None);
    PyObject* y = b.defined() ? THPVariable_Wrap(std::move(b)) : Py_NewRef(Py_None);
    PyObject* t = x != nullptr && y != nullptr ? PyTuple_Pack(2, x, y) : nullptr;
    Py_XDECREF(x);
    Py_XDECREF(y);
    return t;
}

at::Tensor new_like(const at::Tensor& t) { return at::empty(t.sizes(), t.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous)); }

// gelu8_forward(x, tanh, keep) -> (y, bytes or None)
PyObject* gelu8_forward(PyObject* const* args, Py_ssize_t nargs) {
    need_arguments(nargs, 3);
    const at::Tensor& x = tensor_of("x", args[0]);
    const int dtype = dtype_code("x", x), tanh = truth(args[1]) ? 1 : 0;
    const bool keep = truth(args[2]);
    const c10::cuda::CUDAGuard guard(x.device());
    const Rows r = rows_of("x", x);
    const Kept k = kept_bytes(r.rows, r.columns);
    at::Tensor y = new_like(x), kept;
    if (keep) kept = new_bytes(x, k.codes + k.scales);
    void* stream = stream_of(x);
    call([&] {
        return g.gelu8_forward(r.t.data_ptr(), r.stride, r.rows, r.columns, dtype, tanh, y.data_ptr(), keep ? bytes_at(kept, 0) : nullptr,
                               keep ? bytes_at(kept, k.codes) : nullptr, stream);
    });
    return two(std::move(y), std::move(kept));
}

// gelu8_backward(dy, bytes, tanh) -> dx
PyObject* gelu8_backward(PyObject* const* args, Py_ssize_t nargs) {
    need_arguments(nargs, 3);
    const at::Tensor& dy = tensor_of("dy", args[0]);
    const int dtype = dtype_code("dy", dy), tanh = truth(args[2]) ? 1 : 0;
    const c10::cuda::CUDAGuard guard(dy.device());
    const Rows r = rows_of("dy", dy);
    const Kept k = kept_bytes(r.rows, r.columns);
    const at::Tensor& kept = kept_of(args[1], k.codes + k.scales);
    same_place("the 8-bit form", kept, dy);
    at::Tensor dx = new_like(dy);
    void* stream = stream_of(dy);
    call([&] {
        return g.gelu8_backward(r.t.data_ptr(), r.stride, bytes_at(kept, 0), bytes_at(kept, k.codes), r.rows, r.columns, dtype, tanh, dx.data_ptr(), stream);
    });
    return THPVariable_Wrap(std::move(dx));
}

// weight_grad8(dy, bytes, inputs, bias) -> (dw, db or None)
PyObject* weight_grad8(PyObject* const* args, Py_ssize_t nargs) {
    need_arguments(nargs, 4);
    const at::Tensor& dy = tensor_of("dy", args[0]);
    b2_weight_grad c = {};
    c.dtype = dtype_code("dy", dy);
    const long long inputs = PyLong_AsLongLong(args[2]);
    if (inputs == -1 && PyErr_Occurred()) throw Raised{};
    if (inputs < 1) refuse("a projection has at least one input");
    const bool bias = truth(args[3]);
    const c10::cuda::CUDAGuard guard(dy.device());
    const Rows r = rows_of("dy", dy);
    // (Without outputs there are no rows to be counted by dy, and nothing to be made from them.)
    std::int64_t rows = r.columns == 0 ? 0 : r.rows;
    const Kept k = kept_bytes(rows, inputs);
    const at::Tensor& kept = r.columns == 0 ? tensor_of("the 8-bit form", args[1]) : kept_of(args[1], k.codes + k.scales);
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
    return two(std::move(dw), std::move(db));
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

// The arguments that all rotations share; `first` gives place and type.
void shared_arguments(b2_rotation* c, const Heads& first, PyObject* positions_obj, PyObject* frequencies_obj, PyObject* interleaved, PyObject* magnitude) {
    c->dtype = dtype_code("queries or keys", first.t);
    const at::Tensor& positions = tensor_of("positions", positions_obj);
    const at::Tensor& frequencies = tensor_of("frequencies", frequencies_obj);
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
    c->interleaved = truth(interleaved) ? 1 : 0;
    c->magnitude = static_cast<float>(number("magnitude", magnitude));
    c->positions = positions.data_ptr();
    c->position_bytes = positions.scalar_type() == at::kLong ? 8 : 4;
    c->position_strides[0] = n == 2 && first.batch > 1 ? positions.stride(0) : 0;
    c->position_strides[1] = first.tokens > 1 ? positions.stride(n - 1) : 0;
    c->frequencies = static_cast<const double*>(frequencies.data_ptr());
}

// Queries and keys, either of which may be None.
struct Both {
    const char* names[2];
    Heads heads[2];
    bool there[2] = {false, false};
    int first = -1;
};
Both both_of(const char* q_name, const char* k_name, PyObject* q, PyObject* k) {
    Both b;
    b.names[0] = q_name;
    b.names[1] = k_name;
    PyObject* objs[2] = {q, k};
    for (int i = 0; i < 2; ++i) {
        if (objs[i] == Py_None) continue;
        const at::Tensor& t = tensor_of(b.names[i], objs[i]);
        if (b.first >= 0) {
            same_place(b.names[i], t, b.heads[b.first].t);
            same_dtype(b.names[i], t, b.heads[b.first].t);
        }
        const c10::cuda::CUDAGuard guard(t.device());
        b.heads[i] = heads_of(b.names[i], t);
        b.there[i] = true;
        if (b.first < 0) b.first = i;
        const Heads &x = b.heads[b.first], &y = b.heads[i];
        if (x.t.dim() != y.t.dim() || x.batch != y.batch || x.tokens != y.tokens || x.dim != y.dim)
            refuse(std::string(b.names[0]) + " and " + b.names[1] + " must agree in all but their heads");
    }
    if (b.first < 0) refuse(std::string(q_name) + " and " + k_name + " are both None");
    return b;
}

const at::Tensor& weight_of(const char* what, PyObject* obj, const Heads& h) {
    const at::Tensor& w = tensor_of(what, obj);
    same_place(what, w, h.t);
    same_dtype(what, w, h.t);
    if (w.dim() != 1 || w.size(0) != h.dim || !w.is_contiguous()) refuse(std::string(what) + " must be a vector of the head dimension without gaps");
    return w;
}

// rotate(q, k, positions, frequencies, interleaved, magnitude, inverse) -> (q, k)
PyObject* rotate(PyObject* const* args, Py_ssize_t nargs) {
    need_arguments(nargs, 7);
    const Both b = both_of("q", "k", args[0], args[1]);
    const Heads& first = b.heads[b.first];
    const c10::cuda::CUDAGuard guard(first.t.device());
    b2_rotation c = {};
    shared_arguments(&c, first, args[2], args[3], args[4], args[5]);
    c.inverse = truth(args[6]) ? 1 : 0;
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
    return two(std::move(out[0]), std::move(out[1]));
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

// norm_rotate(q, k, q_weight, k_weight, positions, frequencies, interleaved, magnitude, eps, keep) -> (q, k, bytes or None)
PyObject* norm_rotate(PyObject* const* args, Py_ssize_t nargs) {
    need_arguments(nargs, 10);
    const Both b = both_of("q", "k", args[0], args[1]);
    const Heads& first = b.heads[b.first];
    const c10::cuda::CUDAGuard guard(first.t.device());
    b2_rotation c = {};
    shared_arguments(&c, first, args[4], args[5], args[6], args[7]);
    c.norm = 1;
    c.eps = static_cast<float>(number("eps", args[8]));
    const bool keep = truth(args[9]);
    at::Tensor out[2], kept;
    KeptHeads k8;
    if (keep) {
        k8 = kept_heads(first.batch * first.tokens, b.there[0] ? b.heads[0].heads : 0, b.there[1] ? b.heads[1].heads : 0, first.dim);
        kept = new_bytes(first.t, k8.bytes);
    }
    for (int i = 0; i < 2; ++i) {
        if (!b.there[i]) continue;
        const Heads& h = b.heads[i];
        out[i] = new_like(h.t);
        c.side[i].heads = static_cast<int>(h.heads);
        c.side[i].x = h.t.data_ptr();
        std::copy(h.strides, h.strides + 3, c.side[i].x_strides);
        c.side[i].out = out[i].data_ptr();
        c.side[i].weight = weight_of(i == 0 ? "q_weight" : "k_weight", args[2 + i], h).data_ptr();
        if (keep) {
            c.side[i].codes = bytes_at(kept, k8.codes[i]);
            c.side[i].scales = bytes_at(kept, k8.scales[i]);
        }
    }
    void* stream = stream_of(first.t);
    call([&] { return g.rotate_heads(&c, stream); });
    PyObject* pair = two(std::move(out[0]), std::move(out[1]));
    if (pair == nullptr) return nullptr;
    PyObject* third = keep ? THPVariable_Wrap(std::move(kept)) : Py_NewRef(Py_None);
    PyObject* t = third != nullptr ? PyTuple_Pack(3, PyTuple_GET_ITEM(pair, 0), PyTuple_GET_ITEM(pair, 1), third) : nullptr;
    Py_DECREF(pair);
    Py_XDECREF(third);
    return t;
}

// norm_rotate_backward(dq, dk, q, k, bytes, q_heads, k_heads, q_weight, k_weight, positions, frequencies, interleaved, magnitude, eps)
//   -> (gradients of q, k, q_weight, k_weight). Where there are bytes, q and k are None, and q_heads and k_heads are those of the kept form
//   (a side whose gradient is None is left out).
PyObject* norm_rotate_backward(PyObject* const* args, Py_ssize_t nargs) {
    need_arguments(nargs, 14);
    const Both b = both_of("dq", "dk", args[0], args[1]);
    const Heads& first = b.heads[b.first];
    const c10::cuda::CUDAGuard guard(first.t.device());
    b2_rotation c = {};
    shared_arguments(&c, first, args[9], args[10], args[11], args[12]);
    c.norm = 1;
    c.eps = static_cast<float>(number("eps", args[13]));
    std::int64_t kept_counts[2];
    for (int i = 0; i < 2; ++i) {
        kept_counts[i] = PyLong_AsLongLong(args[5 + i]);
        if (kept_counts[i] == -1 && PyErr_Occurred()) throw Raised{};
        if (b.there[i] && kept_counts[i] != b.heads[i].heads) refuse("the gradients have another number of heads than queries and keys");
    }
    const bool kept_form = args[4] != Py_None;
    KeptHeads k8;
    if (kept_form) {
        k8 = kept_heads(first.batch * first.tokens, kept_counts[0], kept_counts[1], first.dim);
        same_place("the 8-bit form", kept_of(args[4], k8.bytes), first.t);
    }
    Heads x[2];
    at::Tensor out[2], weight_grad[2], partial[2];
    const auto options = first.t.options().requires_grad(false);
    for (int i = 0; i < 2; ++i) {
        if (!b.there[i]) continue;
        const Heads& h = b.heads[i];
        b2_heads& s = c.side[i];
        out[i] = new_like(h.t);
        weight_grad[i] = at::empty({h.dim}, options);
        partial[i] = at::empty({B2_HEAD_GRAD_PARTIALS * h.dim}, options.dtype(at::kFloat));
        s.heads = static_cast<int>(h.heads);
        s.grad = h.t.data_ptr();
        std::copy(h.strides, h.strides + 3, s.grad_strides);
        s.out = out[i].data_ptr();
        s.weight = weight_of(i == 0 ? "q_weight" : "k_weight", args[7 + i], h).data_ptr();
        s.weight_grad = weight_grad[i].data_ptr();
        s.partial = partial[i].data_ptr();
        if (kept_form) {
            const at::Tensor& kept = THPVariable_Unpack(args[4]);
            s.codes = bytes_at(kept, k8.codes[i]);
            s.scales = bytes_at(kept, k8.scales[i]);
        } else {
            const at::Tensor& t = tensor_of(i == 0 ? "q" : "k", args[2 + i]);
            same_place(i == 0 ? "q" : "k", t, first.t);
            same_dtype(i == 0 ? "q" : "k", t, first.t);
            if (t.sizes() != h.t.sizes()) refuse("a gradient has another shape than its queries or keys");
            x[i] = heads_of(i == 0 ? "q" : "k", t);
            s.x = x[i].t.data_ptr();
            std::copy(x[i].strides, x[i].strides + 3, s.x_strides);
        }
    }
    void* stream = stream_of(first.t);
    call([&] { return g.rotate_heads_backward(&c, stream); });
    PyObject* heads = two(std::move(out[0]), std::move(out[1]));
    PyObject* weights = heads != nullptr ? two(std::move(weight_grad[0]), std::move(weight_grad[1])) : nullptr;
    PyObject* all = weights != nullptr ? PySequence_Concat(heads, weights) : nullptr;
    Py_XDECREF(heads);
    Py_XDECREF(weights);
    return all;
}

template <PyObject* (*kFunction)(PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS  // an allocation that fails raises torch's own error
    if (g.last_error == nullptr) {
        PyErr_SetString(PyExc_RuntimeError, "bind() first");
        return nullptr;
    }
    try {
        return kFunction(args, nargs);
    } catch (const Raised&) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

}  // namespace

PyMethodDef train_methods[] = {
    {"pack8", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<pack8>)), METH_FASTCALL, nullptr},
    {"unpack8", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<unpack8>)), METH_FASTCALL, nullptr},
    {"gelu8_forward", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<gelu8_forward>)), METH_FASTCALL, nullptr},
    {"gelu8_backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<gelu8_backward>)), METH_FASTCALL, nullptr},
    {"weight_grad8", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<weight_grad8>)), METH_FASTCALL, nullptr},
    {"rotate", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<rotate>)), METH_FASTCALL, nullptr},
    {"norm_rotate", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<norm_rotate>)), METH_FASTCALL, nullptr},
    {"norm_rotate_backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<norm_rotate_backward>)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

bool bind_train(PyObject* error_class, PyObject* addresses) {
    unsigned long long a[9];
    if (!PyArg_ParseTuple(addresses, "KKKKKKKKK", &a[0], &a[1], &a[2], &a[3], &a[4], &a[5], &a[6], &a[7], &a[8])) return false;
    const auto take = [](auto& f, unsigned long long v) { f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(static_cast<std::uintptr_t>(v)); };
    take(g.last_error, a[0]);
    take(g.pack8, a[1]);
    take(g.unpack8, a[2]);
    take(g.gelu8_forward, a[3]);
    take(g.gelu8_backward, a[4]);
    take(g.weight_grad8_workspace, a[5]);
    take(g.weight_grad8, a[6]);
    take(g.rotate_heads, a[7]);
    take(g.rotate_heads_backward, a[8]);
    Py_INCREF(error_class);
    Py_XSETREF(g_error_class, error_class);
    return true;
}

}  // namespace b200ccl::python
