/*
 * agk_losses.h -- C ABI of the losses at the end of a language model, with their
 * gradients: the softmax cross entropy of a vocabulary head, without its logits
 * in memory, and distillation from a teacher's top logits.
 *
 * Implemented by the same library as agk_rmsnorm.h (libagk_rmsnorm.so), with
 * the same conventions: device pointers; row-major tensors; `dtype` is the
 * storage type (AGK_F32 or AGK_BF16); sums, maxima and losses are fp32; work is
 * enqueued on `stream` without synchronising and may be captured into a HIP
 * graph; no global state; deterministic results (no float atomics); an
 * agk_status is returned.  The reference has neither operator: its losses are
 * composed from logsumexp_row and mul (cgadimpl/src/ops/reduction.cpp:54-66)
 * over logits that it keeps.
 *
 * Labels and column indices are int64.  A negative one is an empty place: a row
 * whose label is negative, or without a column of the teacher, has the loss 0
 * and no gradient, whatever its other inputs hold (NaN and infinities too).
 * One at or past the last column cannot be refused by a call that does not read
 * it on the host: its row's loss is NaN, and so is its gradient.  No label or
 * index makes a kernel access memory outside its tensors.
 */
#ifndef AGK_LOSSES_H
#define AGK_LOSSES_H

#include "agk_rmsnorm.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Softmax cross entropy of a linear head, per row:
 *     z = x w^T,  m = max(z),  l = log(sum(exp(z - m))),  loss = (m - z[label]) + l
 * x [rows][ldx], w [vocab][ldw] (the linear layer's (out, in) layout), both of
 * `cols` values of `dtype` per row; labels [rows]; loss [rows] fp32; stats
 * [rows][2] fp32, 8-byte aligned, receives m and l, which the backward reads.
 * z exists in pieces only: bf16 products leave the matrix cores as the maximum
 * and sum of exponentials of each token's logits over a few vocabulary rows, in
 * fp32 and unrounded.  fp32 operands of more than 128 rows are multiplied as two
 * fp16 halves each (in the workspace, a piece of the vocabulary at a time), scaled
 * by a power of two: a product is off by at most 12 * 2^-24 of itself, less than
 * the fp32 sum of the row's products is.  Values below 2^-28 of the largest finite
 * one of their row (backward: of their matrix, x's over the rows that are not left
 * out) are held to 2^-39 of that one.
 * A logit of 2.3e38 and more makes its row's loss NaN.  The stats of a row whose
 * label is negative hold nothing of use.
 * bf16: x and w 16-byte aligned, cols, ldx and ldw multiples of 8 (as
 * agk_linear_bf16); rows and vocab are free.  fp32: any sizes.
 * workspace: agk_linear_xent_fwd_workspace_bytes bytes, 16-byte aligned,
 * scratch.  Calls that share one must not overlap in time.
 * rows == 0 is a no-op; vocab == 0 or cols == 0, or 2^24 rows and more, is
 * AGK_EINVAL.                                                               */
size_t agk_linear_xent_fwd_workspace_bytes(int64_t rows, int64_t vocab, int64_t cols, int dtype);

int agk_linear_xent_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw,
                        const int64_t* labels, float* loss, float* stats, void* workspace,
                        size_t workspace_bytes, int64_t rows, int64_t vocab, int64_t cols,
                        int dtype, agk_stream_t stream);

/* Its gradient for dloss [rows] (fp32, the gradient of each row's loss):
 *     G = dloss * (exp((z - m) - l) - [column == label])
 *     dx (+)= G w,   dw (+)= G^T x
 * with z computed again, `piece` vocabulary rows at a time (0: as many as make
 * G's piece about 512 MiB; others are rounded up to a multiple of 256).  Rows
 * whose label is negative or whose dloss is 0 are left out: dx (+)= 0 and
 * nothing in dw.  dx and dw may not overlap the inputs or each other.
 * dx [rows][cols] of `dtype`; dw [vocab][cols] of dw_dtype (AGK_F32, or
 * AGK_BF16 where dtype is AGK_BF16); either may be NULL.  accumulate:
 * AGK_ACCUM_DX adds into dx, AGK_ACCUM_DGAMMA into dw.
 * bf16: G / max|dloss| is rounded to bf16, the operand type of the two
 * products, and the factor goes into their fp32 results: equal weights then
 * cost no rounding of their own.  dx is summed over the pieces in fp32 and
 * rounded once.  dx 16-byte aligned; rows * ldx at most 2^30 values (AGK_EINVAL).
 * fp32: rows * cols, both rounded up to multiples of 64, at most 2^29.  At most
 * 2^22 rows, fp32 2^21.
 * Other sizes, alignments and the workspace as for the forward;
 * agk_linear_xent_bwd_workspace_bytes takes the same piece and depends on the
 * current device's compute units (few rows are spread over them).
 * rows == 0 zero-fills dw unless it accumulates.                            */
size_t agk_linear_xent_bwd_workspace_bytes(int64_t rows, int64_t vocab, int64_t cols, int dtype,
                                           int64_t piece);

int agk_linear_xent_bwd(const void* x, int64_t ldx, const void* w, int64_t ldw,
                        const int64_t* labels, const float* stats, const float* dloss, void* dx,
                        void* dw, int dw_dtype, void* workspace, size_t workspace_bytes,
                        int64_t rows, int64_t vocab, int64_t cols, int64_t piece, int dtype,
                        int accumulate, agk_stream_t stream);

/* Distillation from a teacher's top logits, per row of student logits z
 * [rows][cols] (dtype), against the teacher's k logits t [rows][k] (t_dtype) of
 * the columns index [rows][k]:
 *     q = softmax(z / T) over all columns,  p = softmax(t / T) over the row's
 *     entries whose index is not negative
 *     loss = T^2 sum_j p_j (log p_j - log q[index_j])
 * T = temperature, 1e-4 to 1e4 (AGK_EINVAL).  The factor T^2 keeps the
 * gradient's size as T grows.  An entry whose t is -inf has p = 0 and adds
 * nothing; a row of such entries alone has no teacher.  A column named by
 * several entries counts for each.  k = 1 is the cross entropy of a label.  loss [rows] fp32;
 * stats [rows][2] fp32, 8-byte aligned, receives max(z) and
 * log(sum(exp((z - max) / T))), for the backward.
 * 0 <= k <= AGK_DISTILL_MAX_K (AGK_EINVAL); any alignment and cols.
 * workspace: agk_distill_topk_workspace_bytes bytes (a few wide rows are spread
 * over several workgroups each), 8-byte aligned, scratch; NULL where that is 0.  Calls that share
 * one must not overlap in time.
 * rows == 0 is a no-op; cols == 0 with rows > 0 is AGK_EINVAL.               */
#define AGK_DISTILL_MAX_K 1024
size_t agk_distill_topk_workspace_bytes(int64_t rows, int64_t cols, int dtype);

int agk_distill_topk_fwd(const void* z, const int64_t* index, const void* t, float* loss,
                         float* stats, void* workspace, size_t workspace_bytes, int64_t rows,
                         int64_t cols, int64_t k, float temperature, int dtype, int t_dtype,
                         agk_stream_t stream);

/* Its gradient for dloss [rows] (fp32):
 *     dz (+)= dloss * T * (q - sum over the entries j of this column of p_j)
 * accumulate: AGK_ACCUM_NONE or AGK_ACCUM_DX.  dz may be z itself (in place),
 * but not overlap it otherwise (AGK_EINVAL).  Rows without a teacher, or with a
 * dloss of 0, get zeros (or stay as they are when accumulating).             */
int agk_distill_topk_bwd(const void* z, const int64_t* index, const void* t, const float* stats,
                         const float* dloss, void* dz, int64_t rows, int64_t cols, int64_t k,
                         float temperature, int dtype, int t_dtype, int accumulate,
                         agk_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* AGK_LOSSES_H */
