/*
 * tcc_training.h — C-ABI of the operators that a GCN with learned node rows
 * trains with on MI355X (gfx950), beside the block-sparse SpMM of
 * tcc_spmm_cnic.h and the dense products of tcc_gcn.h: rows of an embedding
 * table and their gradient, a group norm over the node rows of each graph
 * with its activation, the global gradient norm with clipping, and the Adam
 * update that takes the clipped gradient.  The reference trains on a fixed
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
