// The training operators of the Python package as native calls (torch_ops.cc, vocabulary_ops.cc), part of the module of torch_binding.cc.
#pragma once

#define PY_SSIZE_T_CLEAN
#include <Python.h>

namespace b200ccl::python {

extern PyMethodDef train_methods[];  // ends with an empty entry
extern PyMethodDef vocabulary_methods[];

// The class that a failed call raises, and the addresses of b2_last_error, b2_pack8, b2_unpack8, b2_gelu8_forward, b2_gelu8_backward,
// b2_weight_grad8_workspace, b2_weight_grad8, b2_rotate_heads, b2_rotate_heads_backward, and those of bind_vocabulary(). False with a Python error set.
bool bind_train(PyObject* error_class, PyObject* addresses);
// b2_embed, b2_embed_backward_workspace, b2_embed_backward, b2_vocabulary_loss_sizes, b2_vocabulary_loss_forward, b2_vocabulary_loss_backward,
// b2_vocabulary_loss_both_workspace, b2_vocabulary_loss_both, b2_vocabulary_loss_times.
void bind_vocabulary(const unsigned long long* addresses);

}  // namespace b200ccl::python
