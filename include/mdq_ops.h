/*
 * mdq_ops.h - C ABI of the training-step operators beside the optimizer step:
 * the memory-bound parts of a language model's step whose gradients the
 * optimizer consumes.
 *
 *   scaled embedding     lookup, and its gradient by sorted tokens
 *   residual norm        the norm after a block with its gate and the
 *                        residual's scale, and the norm before the next block
 *   top-k distillation   loss and gradient against a teacher's top logits
 *
 * No counterpart in ruby320/STREAM-MM2026, whose models come from libraries.
 *
 * The conventions are those of mdq.h: plain pointers and sizes, device memory
 * owned by the caller, nothing allocated here, work enqueued on `stream`, an
 * mdq_status from every entry point and mdq_last_error() for its reason.
 * Arguments are checked before anything is launched.  Sums, statistics and
 * exponentials are held in 32 bits or more; a result is rounded once, when it
 * is stored.  Results do not depend on the order in which blocks run: sums are
 * taken in fixed orders, and where an atomic addition joins a sum to a value in
 * memory, it is the only one of its launch to that value.
 */
#ifndef MDQ_OPS_H_
#define MDQ_OPS_H_

#include "mdq.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------------
 * Scaled embedding: out[n, :] = scale * table[ids[n], :].
 * An id outside [0, vocab) gives a row of zeros, as a shard of a vocabulary
 * wants it (pass ids minus the shard's first id).
 */
typedef struct mdq_embed_desc {
    const void* table;      /* [vocab, dim], table_dtype, rows table_stride apart  */
    const void* ids;        /* [tokens], MDQ_I32 or MDQ_I64                        */
    void* out;              /* [tokens, dim], out_dtype, contiguous                */
    int64_t tokens, vocab, dim;
    int64_t table_stride;   /* elements                                            */
    float scale;
    int32_t table_dtype;    /* MDQ_F32 or MDQ_BF16                                 */
    int32_t out_dtype;      /* MDQ_F32 or MDQ_BF16                                 */
    int32_t ids_dtype;
} mdq_embed_desc;

mdq_status mdq_embed(const mdq_embed_desc* d, cudaStream_t stream);

/*
 * Its gradient: grad[v, :] = scale * sum over n with ids[n] = v of
 * grad_out[n, :], in ascending order of n within fixed groups (the same bits on
 * every call).  Rows of ids that do not occur are written as zeros; with
 * `accumulate` (fp32 grad only) the sums are added to `grad` instead and other
 * rows are not touched.  The addition to `grad` is the L2 cache's, which takes
 * subnormal values as zero (below 1.2e-38 in magnitude).  Ids outside [0, vocab)
 * and ids equal to padding_idx (-1: none) contribute nothing.  tokens < 2^31.
 */
typedef struct mdq_embed_grad_desc {
    const void* grad_out;   /* [tokens, dim], grad_out_dtype, rows stride apart    */
    const void* ids;        /* [tokens], MDQ_I32 or MDQ_I64                        */
    void* grad;             /* [vocab, dim], grad_dtype, contiguous                */
    void* workspace;        /* mdq_embed_grad_workspace_bytes, 16-byte aligned     */
    int64_t workspace_bytes;
    int64_t tokens, vocab, dim;
    int64_t grad_out_stride;
    int64_t padding_idx;
    float scale;
    int32_t grad_out_dtype; /* MDQ_F32 or MDQ_BF16                                 */
    int32_t grad_dtype;     /* MDQ_F32 or MDQ_BF16                                 */
    int32_t ids_dtype;
    int32_t accumulate;
    int32_t reserved;
} mdq_embed_grad_desc;

mdq_status mdq_embed_grad_workspace_bytes(int64_t tokens, int64_t vocab, int64_t dim,
                                          int64_t* bytes);
mdq_status mdq_embed_grad(const mdq_embed_grad_desc* d, cudaStream_t stream);

/* ------------------------------------------------------------------------
 * Residual norm, per row:
 *   x_new = residual_scale * x + gate * (norm(h) * post_weight + post_bias)
 *   n     = norm(x_new) * pre_weight + pre_bias
 * norm is v / sqrt(mean(v^2) + eps) (MDQ_NORM_RMS) or (v - mean(v)) /
 * sqrt(var(v) + eps) (MDQ_NORM_LAYER).  n is computed from x_new before x_new
 * is rounded.  gate has gate_rows rows of dim values, row k for the k-th run of
 * rows / gate_rows consecutive rows; NULL means 1.
 * Without a block (h NULL) x_new = x is not written and n = norm(x) * ...; the
 * pre_weight may be NULL (the model's last block), then n is not written.
 */
typedef enum mdq_norm_kind { MDQ_NORM_RMS = 0, MDQ_NORM_LAYER = 1 } mdq_norm_kind;

typedef struct mdq_residual_norm_desc {
    const void* x;            /* [rows, dim], x_dtype, rows x_stride apart         */
    const void* h;            /* [rows, dim], h_dtype, rows h_stride apart         */
    void* x_new;              /* [rows, dim], x_dtype, contiguous                  */
    void* n;                  /* [rows, dim], h_dtype, contiguous                  */
    float* stats;             /* NULL, or [rows, 4]: mean and 1/deviation of h,
                                 then of x_new (means 0 with MDQ_NORM_RMS),
                                 which the backward pass reads                     */
    const void* post_weight;  /* [dim], param_dtype, as the next four              */
    const void* post_bias;    /* biases: both kinds may have them, or NULL         */
    const void* pre_weight;
    const void* pre_bias;
    const void* gate;         /* [gate_rows, dim], contiguous                      */
    int64_t rows, dim, x_stride, h_stride, gate_rows;
    float residual_scale, eps;
    int32_t x_dtype, h_dtype, param_dtype, kind;
} mdq_residual_norm_desc;

mdq_status mdq_residual_norm(const mdq_residual_norm_desc* d, cudaStream_t stream);

/*
 * Gradients of residual norm, from its inputs and stats (x_new is recomputed,
 * unrounded).  grad_new / grad_n may be NULL for zero.  grad_x and grad_h are
 * written contiguously in x_dtype and h_dtype, the parameters' gradients in
 * param_dtype; each is NULL where the forward argument was.  `f.x_new`, `f.n`
 * are unused.  Without rows the parameters' gradients are zeros and the
 * workspace is not used.
 */
typedef struct mdq_residual_norm_grad_desc {
    mdq_residual_norm_desc f;
    const void* grad_new;     /* [rows, dim], x_dtype, rows grad_new_stride apart  */
    const void* grad_n;       /* [rows, dim], h_dtype, rows grad_n_stride apart    */
    void* grad_x;
    void* grad_h;
    void* grad_post_weight;
    void* grad_post_bias;
    void* grad_pre_weight;
    void* grad_pre_bias;
    void* grad_gate;          /* [gate_rows, dim]                                  */
    void* workspace;          /* 16-byte aligned                                   */
    int64_t workspace_bytes;
    int64_t grad_new_stride, grad_n_stride;
} mdq_residual_norm_grad_desc;

mdq_status mdq_residual_norm_grad_workspace_bytes(int64_t rows, int64_t dim, int64_t gate_rows,
                                                  int64_t* bytes);
mdq_status mdq_residual_norm_grad(const mdq_residual_norm_grad_desc* d, cudaStream_t stream);

/* ------------------------------------------------------------------------
 * Distillation from a teacher's top logits.  For row n with teacher logits
 * t_k at vocabulary indices i_k, k < top:
 *   q   = softmax over the present entries of t_k / temperature
 *   p   = softmax over the vocabulary of logits / temperature
 *   row_loss[n] = c_n * temperature^2 * sum_k q_k (log q_k - log p_{i_k})
 *   grad[n, v]  = u_n * c_n * temperature * (p_v - sum_{k: i_k = v} q_k)
 *   c_n = scale * weight[n],  u_n = upstream[n * upstream_stride]
 * and loss = sum of row_loss.  An entry whose index lies outside [0, vocab) is
 * absent; a row of weight 0, or whose entries are all absent or -infinity, has
 * loss 0 and gradient 0 whatever its logits hold.  Indices may repeat: each
 * counts.  With top = 1 and temperature 1 this is the cross-entropy against
 * the index.
 */
#define MDQ_DISTILL_MAX_TOP 1024

typedef struct mdq_topk_distill_desc {
    const void* logits;     /* [rows, vocab], logits_dtype, rows logits_stride apart */
    const void* teacher;    /* [rows, top], teacher_dtype, contiguous              */
    const void* index;      /* [rows, top], MDQ_I32 or MDQ_I64, contiguous         */
    const float* weight;    /* [rows] or NULL for 1                                */
    const float* upstream;  /* gradient of each row's loss, or NULL for 1          */
    float* row_loss;        /* [rows] or NULL                                      */
    float* loss;            /* [1] or NULL (needs row_loss)                        */
    void* grad;             /* [rows, vocab], logits_dtype, rows grad_stride apart,
                               or NULL; may be `logits` itself (with its stride),
                               else shares nothing with it                     */
    int64_t rows, vocab, logits_stride, grad_stride;
    int64_t upstream_stride;/* 0 (one value for all rows) or 1                     */
    int32_t top;            /* 1..MDQ_DISTILL_MAX_TOP                              */
    float temperature, scale;
    int32_t logits_dtype;   /* MDQ_F32 or MDQ_BF16                                 */
    int32_t teacher_dtype;  /* MDQ_F32 or MDQ_BF16                                 */
    int32_t index_dtype;
} mdq_topk_distill_desc;

mdq_status mdq_topk_distill(const mdq_topk_distill_desc* d, cudaStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* MDQ_OPS_H_ */
