/* C interface of the operators at the two ends of a training step: the lookup of tokens in an embedding, and losses over a vocabulary whose logits are
 * never stored. Same rules as train_ops.h: 0 on success, 2 for a rejected argument, 1 for a failure, b2_last_error() has the message; work
 * is enqueued on `stream` of the CURRENT device and the call does not wait for it; calls keep nothing between them.
 *
 * dtype: 0 float, 1 fp16, 2 bf16. Tokens and targets have 4 or 8 bytes; negative ones stand for no token. One that is not below `vocabulary` makes NaN.
 * Workspaces have the bytes that the call for them gives for the same arguments (it reads no memory; may be 0), start at a multiple of 256, and belong to one
 * call until that call is done.
 *
 * nano-nccl has no counterpart; these stand beside the data-parallel training layer of the Python package. */
#pragma once

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Forward: out[t] = scale * rows[token[t]], [tokens][width]; zeros where there is no token. Backward: out[v] = scale * sum of rows[t] over the t with
 * token[t] = v, in the order of t, [vocabulary][width], at a multiple of 16 bytes; what is no token has no part in it. `rows` is the matrix, or what comes back
 * to the result; its rows lie `stride` elements apart, those of `out` without gaps. */
typedef struct b2_embedding {
    int dtype;
    const void* tokens;
    int token_bytes;
    long long token_stride; /* elements */
    size_t count, vocabulary, width;
    float scale;
    const void* rows;
    long long stride;
    void* out;
    void* workspace; /* backward */
} b2_embedding;
int b2_embed(const b2_embedding* call, void* stream);
int b2_embed_backward_workspace(const b2_embedding* call, size_t* bytes);
int b2_embed_backward(const b2_embedding* call, void* stream);

/* Logits z = x weight^T. Without `teacher`, cross entropy: log sum exp z - z[target]. With it, distillation: temperature^2 * sum over the entries of
 * p (log p - log q), p the softmax of teacher / temperature over the entries of a token, q that of z / temperature over the vocabulary; entries whose target is
 * negative or whose logit is -infinity are not there, and several may name the same word. A token without a target or entries has no loss and no gradient, and does
 * not count in a mean; without any that count, a mean is 0. */
typedef struct b2_vocabulary_loss {
    int dtype;
    const void* x;
    long long x_stride;
    const void* weight;
    long long weight_stride;
    size_t tokens, width, vocabulary;
    const void* targets;         /* [tokens], with a teacher [tokens][entries] */
    int target_bytes;
    long long target_strides[2]; /* elements */
    int entries;                 /* of the teacher: 1 to 256; otherwise 0 */
    const void* teacher;         /* [tokens][entries]; the backward pass does not look at it */
    int teacher_dtype;
    long long teacher_strides[2];
    float temperature;           /* 1 without a teacher */
    int reduction;               /* 0 none, 1 mean, 2 sum */
    float* loss;                 /* [tokens], or one */
    float* kept;                 /* written by the loss, read by its backward pass: as many floats as the sizes below say */
    /* backward */
    const float* loss_grad;      /* [tokens], or one */
    long long loss_grad_stride;
    void* x_grad;                /* rows without gaps; null: not wanted */
    void* weight_grad;
    void* workspace;
} b2_vocabulary_loss;
int b2_vocabulary_loss_sizes(const b2_vocabulary_loss* call, int backward, size_t* kept_floats, size_t* workspace_bytes);
int b2_vocabulary_loss_forward(const b2_vocabulary_loss* call, void* stream);
int b2_vocabulary_loss_backward(const b2_vocabulary_loss* call, void* stream);
/* bf16, one loss for all tokens (reduction 1 or 2): the loss together with the gradients whose pointers are given, for a loss_grad of 1, which saves making the logits
 * a second time; loss_grad is not looked at. The first call gives the bytes of its workspace, 0 where a call is not of this kind or would need too much: the second refuses it then. The
 * third multiplies gradients (null: not there) by *loss_grad, in place. */
int b2_vocabulary_loss_both_workspace(const b2_vocabulary_loss* call, size_t* bytes);
int b2_vocabulary_loss_both(const b2_vocabulary_loss* call, void* stream);
int b2_vocabulary_loss_times(const b2_vocabulary_loss* call, void* stream);
/* Every wait inside the kernels is bounded, by two seconds or `wait_ns`. Where one runs out, what depends on it is NaN (of gradients made with the loss, what
 * a wait for their first logits left out is made again, and may be right), and the check below says once that a wait ran out: 1, for calls on `device` that are done. */
int b2_vocabulary_loss_within(const b2_vocabulary_loss* call, int backward, unsigned long long wait_ns, void* stream); /* backward: 2 for both at once */
int b2_vocabulary_loss_check_async_error(int device);

#ifdef __cplusplus
}
#endif
