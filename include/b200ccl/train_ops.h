/* C interface of the training operators: activations kept in 8 bits for the backward pass, and the rotation of queries and keys.
 * They work on one GPU's own memory and need no communicator. Same rules as c_api.h: 0 on success, 2 for a rejected argument, 1 for
 * a failure, b2_last_error() has the message; work is enqueued on `stream` of the CURRENT device and the call does not wait for it. Calls keep
 * nothing between them, so any number may run at once, on any streams, or be captured into graphs.
 *
 * dtype: 0 float, 1 fp16, 2 bf16.
 *
 * 8-bit form of a matrix: codes[rows][pitch], pitch = columns rounded up to a multiple of 32, at a multiple of 32 bytes, and scales[rows][pitch / 32],
 * both bytes; a block is 32 neighbouring elements of a row (the last one of a row may be shorter). With largest magnitude
 * 2^a <= amax < 2^(a+1) its step is 2^q, q = max(a - 6, -126) (fp16: -24); its scale is q + 127, a code is sign << 7 | min(rint(|x| / 2^q), 127).
 * A block with an infinity or NaN has scale 255 and codes 0, and reads back as NaN.
 *
 * nano-nccl has no counterpart; these stand beside the data-parallel training layer of the Python package. */
#pragma once

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

/* x: rows of `columns` elements, `stride` elements from row to row. */
int b2_pack8(const void* x, long long stride, size_t rows, size_t columns, int dtype, void* codes, void* scales, void* stream);
/* out: rows without gaps. */
int b2_unpack8(const void* codes, const void* scales, size_t rows, size_t columns, int dtype, void* out, void* stream);

/* y = x Phi(x), or with `tanh` 0.5 x (1 + tanh(sqrt(2/pi) (x + 0.044715 x^3))), and x in 8 bits (not with codes and
 * scales null). y: rows without gaps. */
int b2_gelu8_forward(const void* x, long long stride, size_t rows, size_t columns, int dtype, int tanh, void* y, void* codes, void* scales,
                     void* stream);
/* dx = dy times the derivative at what was kept. dx: rows without gaps. */
int b2_gelu8_backward(const void* dy, long long stride, const void* codes, const void* scales, size_t rows, size_t columns, int dtype, int tanh,
                      void* dx, void* stream);

/* weight_grad[n][k] = sum over tokens t of dy[t][n] * x^[t][k]; bias_grad[n] = sum of dy[t][n]. The pointers other than dy and the 8-bit form are
 * without gaps; bias_grad may be null. `workspace` has the bytes that b2_weight_grad8_workspace gives for the same arguments (it reads no
 * memory; may be 0), at a multiple of 256; it belongs to one call until that call is done. */
typedef struct b2_weight_grad {
    const void* dy;
    long long stride;
    size_t tokens, outputs, inputs;
    int dtype;
    const void* codes; /* of x, [tokens][inputs] */
    const void* scales;
    void* weight_grad; /* [outputs][inputs] */
    void* bias_grad;   /* [outputs] */
    void* workspace;
} b2_weight_grad;
int b2_weight_grad8_workspace(const b2_weight_grad* call, size_t* bytes);
int b2_weight_grad8(const b2_weight_grad* call, void* stream);
/* Every wait inside the kernel is bounded, by two seconds or `wait_ns`. Where one runs out, the gradients that depend on it are NaN (in a replayed graph
 * too), no other call is touched, and the check below says so once: 1, for calls on `device` that are done. */
int b2_weight_grad8_within(const b2_weight_grad* call, unsigned long long wait_ns, void* stream);
int b2_train_check_async_error(int device);

/* Queries and keys [batch][tokens][heads][dim], the last axis without gaps. The first `rotated` elements of a head turn in pairs, (i, i + rotated/2) or with
 * `interleaved` (2i, 2i+1), by position * frequencies[i] radians, and are multiplied with `magnitude`. dim and rotated are even, dim at most 256.
 * `positions` has two strides, in elements; position_bytes is 4 or 8. */
typedef struct b2_heads {
    int heads;              /* 0: none */
    const void* x;
    long long x_strides[3]; /* batch, token, head, in elements */
    const void* grad;       /* backward */
    long long grad_strides[3];
    void* out;              /* without gaps: the turned heads, or the gradient of x */
    const void* weight;     /* norm: [dim] */
    void* codes;            /* norm: x in 8 bits, a head being one block: [batch * tokens * heads][dim rounded up to 16]; null: none */
    void* scales;           /* [batch * tokens * heads] */
    void* weight_grad;      /* backward: [dim] */
    void* partial;          /* backward: B2_HEAD_GRAD_PARTIALS * dim floats of scratch */
} b2_heads;
#define B2_HEAD_GRAD_PARTIALS 296
typedef struct b2_rotation {
    int dtype;
    long long batch, tokens;
    int dim, rotated, interleaved;
    int inverse;            /* turn back: the gradient of a rotation */
    int norm;               /* forward: x * (mean x^2 + eps)^-1/2 * weight before the rotation, and codes where they are given */
    float eps, magnitude;
    const void* positions;
    int position_bytes;
    long long position_strides[2]; /* batch, token */
    const double* frequencies;     /* [rotated / 2] */
    b2_heads side[2];
} b2_rotation;
int b2_rotate_heads(const b2_rotation* call, void* stream);
/* The gradients of the norm and rotation: x is read from `codes` where they are given, from `x` otherwise. `inverse` is not looked at. */
int b2_rotate_heads_backward(const b2_rotation* call, void* stream);

#ifdef __cplusplus
}
#endif
