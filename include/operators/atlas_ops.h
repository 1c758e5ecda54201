/*
 * C ABI of the MI355X (gfx950) sequence-layer operators, libatlas_ops_hip.so: layer
 * normalisation, the gated delta rule and the orthogonalised weight update.
 *
 * Every pointer is device memory of the current device unless its comment says otherwise, every
 * call enqueues its kernels on `stream` (a hipStream_t) and returns without waiting; nothing is
 * allocated, kept between calls or read back.  `type` and the other element types are
 * ATLAS_OPS_F32 or ATLAS_OPS_BF16.  Strides count elements.  Return codes are those of the
 * training library: 0 ok, 4 launch failure, 7 invalid argument or host exception, with a message
 * in (error, capacity).  Sizes that a call refuses have a workspace of 0 bytes.
 */
#ifndef ATLAS_OPS_H
#define ATLAS_OPS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define ATLAS_OPS_F32 0
#define ATLAS_OPS_BF16 1

/*
 * Rows of `width` contiguous values.  Row r starts at (r / inner) * outer_stride + (r % inner) *
 * inner_stride; a matrix of one row stride has inner = rows.
 */
typedef struct {
    const void* data;
    int64_t inner, outer_stride, inner_stride;
} AtlasRows;

/* y = (x - mean) * rstd * weight + bias by row, rstd = 1 / sqrt(variance + eps) with the variance
 * over width.  y is rows x width, contiguous, of x's type; weight and bias (either may be NULL)
 * have weight_type; mean and rstd (both or neither NULL) receive f32[rows]. */
int atlas_ops_layer_norm(const AtlasRows* x, int64_t rows, int64_t width, int type, const void* weight, const void* bias,
                         int weight_type, float eps, void* y, float* mean, float* rstd, void* stream, char* error,
                         size_t capacity);

/* Bytes of workspace that atlas_ops_layer_norm_backward needs for dweight and dbias. */
int64_t atlas_ops_layer_norm_workspace(int64_t rows, int64_t width, int type);

/* Gradients of the rows (dx, contiguous, of x's type) and, where not NULL, of weight and bias
 * (weight_type), summed over the rows in a fixed order. */
int atlas_ops_layer_norm_backward(const AtlasRows* grad, const AtlasRows* x, int64_t rows, int64_t width, int type,
                                  const void* weight, int weight_type, const float* mean, const float* rstd, void* dx,
                                  void* dweight, void* dbias, float* workspace, void* stream, char* error,
                                  size_t capacity);

/*
 * The orthogonal factor of `batch` matrices (rows x columns) by `steps` quintic iterations:
 * X = u / (|u|_F + eps), then X <- a X + (b A + c A A) X with A = X X^T and coefficients (a, b, c).
 * u is the matrix, or with a momentum (f32, contiguous, updated in place) momentum <- factor
 * momentum + matrix and u = matrix + factor momentum (nesterov) or the momentum.  The result goes to
 * `out` (contiguous, out_type), or, where out is NULL, into weight (f32, contiguous):
 * weight <- keep weight - rate X.  Element (r, c) of matrix b is at b * batch_stride + r * row_stride + c.
 * Accuracy is float32's for either type.  The coefficients are finite and such that no X before the last, X X^T
 * or b A + c A A passes 4000 for any matrix.  matrix, momentum, weight and out must not share memory.
 */
typedef struct {
    const void* matrix;
    int64_t batch, rows, columns, batch_stride, row_stride;
    float* momentum;
    void* out;
    float* weight;
    int type, out_type, nesterov, steps;
    float factor, eps, keep, rate;
    float coefficients[3];
} AtlasOrthogonal;

/* Bytes of workspace for a call of these sizes: batch 1 to 65535, rows and columns 1 to 2^20 and one of them at most
 * 16384. */
int64_t atlas_ops_orthogonalize_workspace(int64_t batch, int64_t rows, int64_t columns);
int atlas_ops_orthogonalize(const AtlasOrthogonal* problem, void* workspace, void* stream, char* error,
                            size_t capacity);

/*
 * The gated delta rule.  Head h of value_heads keeps a state S (key x value) and reads the queries and
 * keys of head h / (value_heads / heads).  By token, with a = exp(log_decay):
 *   S <- a S,  e = v - S^T k,  S <- S + beta k e^T,  out = scale S^T q.
 * q, k (batch, time, heads, key) and v (batch, time, value_heads, value) have `type` and contiguous
 * last axes, log_decay (NULL: no decay) and beta (batch, time, value_heads) their own types; strides are
 * those of (batch, time, head).  A log_decay below -120 counts as -120, whose exponential is zero in
 * float32: it empties the state.  state (f32, contiguous (batch, value_heads, key, value)) may be NULL
 * for zeros.  lengths (i32[batch], NULL for `time`): tokens from lengths[b] on leave the state as it is
 * and give zeros.  1 <= key <= 128; batch and value_heads up to 65535, value up to 2^20.  In chunks also: time up
 * to 2^29 - 64, batch x value_heads x value (to whole 8 heads and 32 values) below 2^27, with keys up to 64 below 2^28.
 */
typedef struct {
    const void *q, *k, *v, *log_decay, *beta;
    int64_t q_stride[3], k_stride[3], v_stride[3], log_decay_stride[3], beta_stride[3];
    const float* state;
    const int32_t* lengths;
    int64_t batch, time, heads, value_heads, key, value;
    int type, log_decay_type, beta_type;
    float scale;
} AtlasDelta;

/* Token by token: out (contiguous, `type`) and the state after the last token.  final_state may be
 * `state` itself, and shares no memory with the other inputs. */
int atlas_ops_delta_step(const AtlasDelta* delta, void* out, float* final_state, void* stream, char* error,
                         size_t capacity);

/* Bytes of the workspace of a forward pass; with train != 0 of one that a backward pass can use. */
int64_t atlas_ops_delta_workspace(const AtlasDelta* delta, int train);

/* In chunks of 64 tokens: out (contiguous, `type`) and final_state.  With train != 0 the workspace is
 * afterwards the tape of atlas_ops_delta_backward. */
int atlas_ops_delta_forward(const AtlasDelta* delta, int train, void* out, float* final_state, void* workspace,
                            void* stream, char* error, size_t capacity);

/* Bytes of the backward pass's own workspace. */
int64_t atlas_ops_delta_backward_workspace(const AtlasDelta* delta);

/* The gradients of every input, contiguous and of the input's type, from those of out (`type`,
 * strides of (batch, time, head)) and of final_state (f32, contiguous, NULL for zeros).  `delta` and `tape`
 * are those of the forward pass with train != 0, unchanged since.  dlog_decay and dstate may be NULL. */
int atlas_ops_delta_backward(const AtlasDelta* delta, const void* tape, const void* grad_out,
                             const int64_t* grad_out_stride, const float* grad_state, void* dq, void* dk, void* dv,
                             void* dlog_decay, void* dbeta, float* dstate, void* workspace, void* stream, char* error,
                             size_t capacity);

#ifdef __cplusplus
}
#endif

#endif /* ATLAS_OPS_H */
