/* dvgr_attn.h -- C ABI of multi-head attention to an encoder's states of another length: the words of a question over the frames of
 * its video, clips over words, one word of an answer over everything.  Beside the unit's own attentions (include/dvgr.h), which are
 * fused with their projections and bound to its sizes.
 *
 *     S[l][j] = scale * q_l . k_j        P = softmax of S over the keys j that are there        o_l = sum_j P[l][j] v_j
 *
 * Tensors are (B, L, heads, Dh) of one element type (DVGR_ELEM_*) with strides of their own, so keys and values may lie side by side
 * in one projection's output.  H query heads share Hk key heads, query head h reads key head h / (H / Hk).  Key j of sample b is
 * there if j < lens[b] and mask[b][j] != 0; what lies in the others is never used, NaN included.  A query with no key gives zeros.
 * Scores, softmax statistics and sums are fp32; for bf16 / fp16 the probabilities and the score gradients are rounded to the element
 * type as operands of the matrix unit, as q, k and v are (with many rows taken at up to 2^8 times their size: results are off by 0.0024
 * relative in bf16, rms, where rounding them alone would leave 0.0017).  Finite scores may have any size; the backward knows a row's
 * softmax sum as one fp32 score, so its probabilities are off by up to 2^-22 |scale q.k| relative (keys that share a maximum beyond 2^23
 * count as 1 each).  Conventions as in dvgr.h: nothing is allocated or synchronised, launches go to `stream` of the current device,
 * 0 / DVGR_E_* / hipError_t return codes. */
#ifndef DVGR_ATTN_H
#define DVGR_ATTN_H
#include "dvgr.h"
#ifdef __cplusplus
extern "C" {
#endif

/* element (b, l, h, d) at p[b * sb + l * sl + h * sh + d]; p and the strides of dimensions longer than 1 are multiples of 16 bytes,
 * 0 <= sl < 4 GB */
typedef struct dvgr_attn_view {
  void *p;
  int64_t sb, sl, sh;
} dvgr_attn_view;

typedef struct dvgr_attn_problem {
  int32_t B, Lq, Lk;       /* samples, queries and keys of a sample; any may be 0                        */
  int32_t H, Hk;           /* query heads, key heads; H a multiple of Hk                                 */
  int32_t Dh;              /* head size: a multiple of 8, 8 .. 128.  B Hk (Lq H / Hk / 64 + 1) < 2^24, B Hk (Lk / 128 + 1) <= 2^23 - 8 */
  int32_t elem;            /* DVGR_ELEM_*                                                                */
  float scale;             /* 1e-30 .. 1e30                                                              */
  dvgr_attn_view q, k, v;
  dvgr_attn_view o;        /* written by the forward, read by the backward                               */
  void *o_lo;              /* bf16 / fp16, (B, Lq, H, Dh) contiguous, or NULL: what o's rounding left, rounded to the type.  The forward
                              fills it; with it the backward's rowsum(g_o o) is that of the unrounded output            */
  const int64_t *lens;     /* (B) number of keys, clamped to [0, Lk], or NULL: Lk                        */
  const uint8_t *mask;     /* (B, Lk) 0 / 1, rows `mask_stride` bytes apart, or NULL                     */
  int64_t mask_stride;
  float *lse;              /* (B, H, Lq) fp32, filled by the forward for the backward, or NULL: forward only */
} dvgr_attn_problem;

typedef struct dvgr_attn_grads {
  dvgr_attn_view g_o;              /* upstream gradient                                                  */
  dvgr_attn_view g_q, g_k, g_v;    /* written; keys that are not there get zeros.  g_q.p NULL, or g_k.p and g_v.p NULL: not wanted */
} dvgr_attn_grads;

int dvgr_attn_check(const dvgr_attn_problem *a);
/* 16-byte aligned scratch of either call */
size_t dvgr_attn_forward_workspace_bytes(const dvgr_attn_problem *a);
size_t dvgr_attn_backward_workspace_bytes(const dvgr_attn_problem *a);
int dvgr_attn_forward(const dvgr_attn_problem *a, void *workspace, size_t workspace_bytes, void *stream);
/* No atomics on values: the same inputs give the same bits. */
int dvgr_attn_backward(const dvgr_attn_problem *a, const dvgr_attn_grads *g, void *workspace, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* DVGR_ATTN_H */
