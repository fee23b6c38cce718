/*
 * tcc_training.h — C-ABI of the operators that a GCN with learned node rows, a
 * deep one or one with a teacher trains with on MI355X (gfx950), beside the
 * block-sparse SpMM of tcc_spmm_cnic.h and the dense products of tcc_gcn.h:
 * rows of an embedding table and their gradient, a group norm over the node
 * rows of each graph and a layer norm of each row, with their activation, a
 * teacher's top logits and the loss against them, the global gradient norm with
 * clipping, and the Adam update that takes the clipped gradient.  The reference trains on a fixed
 * feature table (train/tcgnn_conv_release.py:284-329) and has none of them.
 *
 * Element types (TCC_F32, TCC_BF16, TCC_F16) are those of the tensors in
 * memory; every sum, statistic, norm and moment is held in 32 bits or more
 * and an output is rounded once to its type.  Row strides are in elements;
 * pointers are aligned to their element.  Every function is asynchronous on
 * `stream` (a hipStream_t; NULL = the null stream), allocates nothing and
 * records no memset, so that it can be captured into a HIP graph.  Sums run
 * in an order that sizes, ids, offsets, maxRows and the alignment of addresses
 * and row strides (which decides how many elements a lane takes) fix: the same
 * call gives the same bits, a copy at another alignment may differ in the last
 * ones.  Workspaces are device memory, 16-byte aligned, not shared with a
 * concurrent call, with any contents.
 *
 * Errors as in tcc_swtcf.h: 0 or a TCC_ERR_* code, text in tcc_last_error().
 */
#ifndef TCC_TRAINING_H
#define TCC_TRAINING_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define TCC_F32 0u
#define TCC_BF16 1u
#define TCC_F16 2u

/* ---------------------------------------------------------- embedding rows */

/* out[i] = scale * table[ids[i]] for i < n: table [V x D] (row stride ldt),
 * out [n x D] (ldo), both of `dtype`; ids int32 (idBytes 4) or int64 (8).
 * Rows whose id is `padding` (-1: no such id) are zeros.  So are rows whose
 * id is outside [0, V): they set TCC_DEVERR_FEATURE_INDEX in *deviceError,
 * if it is not NULL.  n and V below 2^32 - 1 and D below 2^32 - 1025
 * (TCC_ERR_UNSUPPORTED above). */
int tcc_embedding_lookup(const void* table, uint64_t ldt, uint32_t dtype, const void* ids, uint32_t idBytes, uint64_t n,
                         uint64_t V, uint32_t D, float scale, int64_t padding, void* out, uint64_t ldo,
                         uint32_t* deviceError, void* stream);

/* Bytes of workspace tcc_embedding_grad needs. */
size_t tcc_embedding_grad_workspace_bytes(uint64_t n, uint64_t V, uint32_t D);

/* grad[v] = scale * sum of dOut[i] over the i with ids[i] = v, for v < V:
 * dOut [n x D] (row stride ldd) and grad [V x D] (ldg) of `dtype`.  Every
 * row of grad is written (accumulate = 0), or the sums are added to grad and
 * only rows that occur are touched (accumulate != 0).  Padding and refused
 * ids as in tcc_embedding_lookup: their rows of dOut are not read.  The rows
 * of one id are added in an order that the ids alone decide.  D below 2^28. */
int tcc_embedding_grad(const void* dOut, uint64_t ldd, uint32_t dtype, const void* ids, uint32_t idBytes, uint64_t n,
                       uint64_t V, uint32_t D, float scale, int64_t padding, void* grad, uint64_t ldg, int accumulate,
                       uint32_t* deviceError, void* workspace, size_t workspaceBytes, void* stream);

/* -------------------------------------------------------------- group norm */

#define TCC_ACT_NONE 0u
#define TCC_ACT_RELU 1u
#define TCC_ACT_SILU 2u
#define TCC_ACT_GELU 3u /* z * Phi(z), with the error function */

/* The rows and channels of a group norm.  Segment b (a graph) holds the rows
 * offsets[b] .. offsets[b+1] (B + 1 non-decreasing device values from 0 to
 * N, int32 or int64 by offsetBytes 4 or 8), or, with offsets NULL, the N / B
 * rows from b * (N / B); a segment may be empty.  Offsets are not checked, only
 * kept within [0, N]: rows that no segment holds are not written.  Group g of its C channels
 * are the C / G from g * (C / G).  x [N x C], row stride ldx, of `dtype`;
 * weight and bias [C] of `paramDtype`, either may be NULL (ones, zeros).
 * `maxRows` is the longest segment's rows where the caller knows it (0: not
 * known); it chooses the split of the work and never the result's meaning.
 * C <= 4096 (TCC_ERR_UNSUPPORTED above). */
typedef struct tcc_group_norm_shape {
    uint64_t N, B, maxRows;
    uint32_t C, G;
    const void* offsets;
    uint32_t offsetBytes;
    uint32_t dtype, paramDtype, activation;
    float eps;
} tcc_group_norm_shape;

/* Bytes of workspace for the forward (backward = 0) or the gradient. */
size_t tcc_group_norm_workspace_bytes(const tcc_group_norm_shape* s, int backward);

/* y = act(z), z = ((x - mean) * rstd) * weight + bias, with mean and
 * rstd = 1 / sqrt(var + eps) over the rows and channels of a segment's group
 * (var over their count; an empty segment gets mean 0, var 0).  y [N x C]
 * (ldy) of x's type; mean and rstd [B x G] fp32, for the gradient. */
int tcc_group_norm(const tcc_group_norm_shape* s, const void* x, uint64_t ldx, const void* weight, const void* bias,
                   void* y, uint64_t ldy, float* mean, float* rstd, void* workspace, size_t workspaceBytes,
                   void* stream);

/* dX [N x C] (lddx) of x's type, and dWeight and dBias [C] fp32 (either may
 * be NULL), from dY [N x C] (lddy) of x's type, x and the forward's mean and
 * rstd.  z is formed with the forward's roundings, so that relu's mask is
 * that of the forward's z (an fp16 output may round to 0 where z does not);
 * what it masks counts as 0, infinities and NaN too. */
int tcc_group_norm_grad(const tcc_group_norm_shape* s, const void* dY, uint64_t lddy, const void* x, uint64_t ldx,
                        const float* mean, const float* rstd, const void* weight, const void* bias, void* dX,
                        uint64_t lddx, float* dWeight, float* dBias, void* workspace, size_t workspaceBytes,
                        void* stream);

/* -------------------------------------------------------------- layer norm */

/* The rows of a layer norm: x [N x C] of `dtype`, weight and bias [C] of
 * `paramDtype`, either may be NULL (ones, zeros).  C <= 16384, N below 2^40
 * (TCC_ERR_UNSUPPORTED above).  Row addresses need only be aligned to their
 * element, and no result depends on them. */
typedef struct tcc_layer_norm_shape {
    uint64_t N;
    uint32_t C;
    uint32_t dtype, paramDtype, activation;
    float eps;
} tcc_layer_norm_shape;

/* y = act(z), z = ((h - mean) * rstd) * weight + bias, of h = x + residual
 * (rounded to x's type; h = x where residual is NULL), with mean and
 * rstd = 1 / sqrt(var + eps) over the channels of each row.  residual, y and
 * sum of x's type, row strides ldr, ldy and lds; h is written to `sum` unless
 * that is NULL.  mean and rstd [N] fp32, for the gradient.  Outputs overlap no
 * input. */
int tcc_layer_norm(const tcc_layer_norm_shape* s, const void* x, uint64_t ldx, const void* residual, uint64_t ldr,
                   const void* weight, const void* bias, void* y, uint64_t ldy, void* sum, uint64_t lds, float* mean,
                   float* rstd, void* stream);

/* Bytes of workspace for dWeight or dBias on the current device. */
size_t tcc_layer_norm_grad_workspace_bytes(const tcc_layer_norm_shape* s);

/* dX [N x C] (lddx) of x's type, the gradient of x and of residual alike, and
 * dWeight and dBias [C] fp32 (either may be NULL; without both no workspace is
 * needed), from dY [N x C] (lddy), h (ldh) and the forward's mean and rstd.
 * dSum [N x C] (ldds), if not NULL, is the gradient that h has from elsewhere:
 * it is added to dX before that is rounded.  z is formed with the forward's
 * roundings, so that relu masks what the forward masked; what it masks counts
 * as 0, infinities and NaN too. */
int tcc_layer_norm_grad(const tcc_layer_norm_shape* s, const void* dY, uint64_t lddy, const void* h, uint64_t ldh,
                        const float* mean, const float* rstd, const void* weight, const void* bias, const void* dSum,
                        uint64_t ldds, void* dX, uint64_t lddx, float* dWeight, float* dBias, void* workspace,
                        size_t workspaceBytes, void* stream);

/* ------------------------------------------------------------ distillation */

/* values and ids [n x K] (row strides ldv, ldi): the K largest of the C logits
 * of each row (ldz) and their classes, largest first, the lowest class first
 * among equals, NaN above all; values of the logits' type.  rest [n], unless it
 * is NULL, is one logit that stands for the other classes at this temperature:
 * rest = T log(sum of exp(z_j / T) over them), -inf where there are none.
 * 1 <= K <= C, K <= 64 (TCC_ERR_UNSUPPORTED above), C below 2^31, the
 * temperature between 1e-18 and 1e18.  Row addresses of the logits need only be
 * aligned to their element. */
int tcc_top_logits(const void* logits, uint64_t ldz, uint32_t dtype, uint64_t n, uint32_t C, uint32_t K,
                   float temperature, void* values, uint64_t ldv, int32_t* ids, uint64_t ldi, float* rest, void* stream);

#define TCC_REDUCE_NONE 0u
#define TCC_REDUCE_MEAN 1u
#define TCC_REDUCE_SUM 2u

/* A distillation of n rows of C logits of `dtype`, each against K entries of a
 * teacher: values of `valueDtype` and ids (classes), int32 or int64 by idBytes 4
 * or 8.  K <= 64, C below 2^31, n below 2^40 (TCC_ERR_UNSUPPORTED above), the
 * temperature between 1e-18 and 1e18. */
typedef struct tcc_distill_shape {
    uint64_t n;
    uint32_t C, K;
    uint32_t dtype, valueDtype, idBytes, reduction;
    float temperature;
} tcc_distill_shape;

/* Bytes of workspace for tcc_distill_loss on the current device. */
size_t tcc_distill_loss_workspace_bytes(const tcc_distill_shape* s);

/* With p = softmax(t / T) over a row's entries t (and its `rest`, if not NULL)
 * and q = softmax(z / T) over its classes, q_rest the sum of q over those that
 * are no entry's:
 *   row loss = w T^2 (sum_k p_k log(p_k / q_id_k) + p_rest log(p_rest / q_rest))
 * with w = weight[row] (1 where weight is NULL).  Terms with p = 0 are 0.  An id
 * of -1 is no entry, and so is any other that is no class: that sets
 * TCC_DEVERR_FEATURE_INDEX in *deviceError, if it is not NULL.  A class may
 * occur in several entries.  A row whose weight is 0 is not read, and it and a
 * row without an entry or rest above -inf have no loss.  The logarithms are
 * differences of fp32 numbers, whose roundings T^2 multiplies: the mean over
 * 20,000 rows of 300 classes is off by 2e-8 at T = 2, 2e-6 at 10, 2e-4 at 100.
 *
 * *loss is the sum of the rows' losses (TCC_REDUCE_SUM) or that divided by the
 * sum of the weights (TCC_REDUCE_MEAN; by n without weights; 0 where that is 0),
 * summed in 64 bits, or loss [n] holds the rows' (TCC_REDUCE_NONE).  *total, if
 * not NULL and the loss is summed, is the sum of the weights.  stats [n][4],
 * 16-byte aligned, is for the gradient: the maximum of the logits, the sum of
 * exp((z - maximum) / T), and both over the classes that are no entry's (0
 * without rest); zeros for rows without a loss. */
int tcc_distill_loss(const tcc_distill_shape* s, const void* logits, uint64_t ldz, const void* values, uint64_t ldv,
                     const void* ids, uint64_t ldi, const float* rest, const float* weight, float* loss, float* total,
                     float* stats, uint32_t* deviceError, void* workspace, size_t workspaceBytes, void* stream);

/* dLogits [n x C] (ldd) of the logits' type, from *dLoss (dLoss [n] with
 * TCC_REDUCE_NONE), the loss's arguments and its stats, and its total where it
 * is a mean with weights (else NULL).  With g = dLoss w T (/ n or / total):
 *   g (q_j - p_j)                  for the entries' classes, p_j the sum over them,
 *   g (q_j - p_rest q_j / q_rest)  for the others (p_rest = 0 without rest).
 * Rows without a loss have zeros.  dLogits overlaps no input. */
int tcc_distill_grad(const tcc_distill_shape* s, const float* dLoss, const void* logits, uint64_t ldz,
                     const void* values, uint64_t ldv, const void* ids, uint64_t ldi, const float* rest,
                     const float* weight, const float* total, const float* stats, void* dLogits, uint64_t ldd,
                     void* stream);

/* ------------------------------------------------ gradient norm, clip, Adam */

/* One tensor of a list, as rows of `cols` elements `ld` apart (a tensor that
 * is dense in memory is one row). */
typedef struct tcc_tensor {
    void* data;
    uint64_t rows, cols, ld;
    uint64_t dtype;
} tcc_tensor;

/* Bytes of workspace for the functions below (whatever the list). */
size_t tcc_grad_norm_workspace_bytes(void);

/* *norm = sqrt of the sum of squares of every element of `count` tensors,
 * summed in 64 bits. */
int tcc_grad_norm(const tcc_tensor* grads, uint32_t count, float* norm, void* workspace, size_t workspaceBytes,
                  void* stream);

/* *norm as tcc_grad_norm, and out[i] = c * grads[i] with
 * c = min(1, maxNorm / (norm + 1e-6)).  out[i] has grads[i]'s rows, cols and
 * type and may be the same memory with the same stride, or memory that no
 * gradient overlaps.  A NaN norm gives NaN, an infinite one 0 (NaN where the
 * gradient is infinite). */
int tcc_clip_grad_norm(const tcc_tensor* grads, const tcc_tensor* out, uint32_t count, float maxNorm, float* norm,
                       void* workspace, size_t workspaceBytes, void* stream);

typedef struct tcc_adam {
    double lr, beta1, beta2, eps, weightDecay;
    double maxNorm; /* clip to it as tcc_clip_grad_norm does; < 0: no clipping */
    int decoupled;  /* weight decay on the parameter (AdamW) instead of in the gradient */
} tcc_adam;

/* One Adam step over `count` parameters: *step (device) becomes t = *step + 1,
 * g = c * grads[i] (+ weightDecay * p unless decoupled),
 * m = beta1 m + (1 - beta1) g, v = beta2 v + (1 - beta2) g^2,
 * p = p (1 - lr weightDecay, where decoupled)
 *     - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps).
 * params and grads of any of the types, expAvg (m) and expAvgSq (v) fp32,
 * each list's i-th with the same rows and cols.  *norm, if not NULL, is the
 * gradients' norm before clipping (formed if norm or maxNorm asks for it).
 * The clipped gradient is not written. */
int tcc_adam_step(const tcc_tensor* params, const tcc_tensor* grads, const tcc_tensor* expAvg,
                  const tcc_tensor* expAvgSq, uint32_t count, const tcc_adam* a, int64_t* step, float* norm,
                  void* workspace, size_t workspaceBytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* TCC_TRAINING_H */
