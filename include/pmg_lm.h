/* pmg_lm.h -- C ABI of the training operators around the decoder's vocabulary: the token embedding and
 * its gradient, the cross entropy of a linear vocabulary projection and its gradients, the norm and the
 * clipping of many gradients, and the Adam / AdamW update of many parameters.
 *
 * They do what the learner needs next to the fused recurrence of pmg.h: the reference leaves these steps
 * to torch (embedding and output_layer of the decoder, clip_grad_norm_ and Adam of
 * paccmann_generator/reinforce.py:44-49, reinforce_omics.py:336-341).  NO COUNTERPART IN THE REFERENCE
 * as entry points.  Conventions are those of pmg.h:
 *   - the caller owns every buffer; pointers are DEVICE pointers unless noted, rows are contiguous
 *     (`ld` = elements from one row to the next) and need the alignment of their element type only;
 *   - the library allocates no device memory: scratch comes in through `ws` (16-byte aligned);
 *   - every call is stream-ordered on the caller's stream, on the current device, never synchronises
 *     and can be captured into a graph (a graph keeps its own `ws`);
 *   - return value: 0 ok, <0 argument error (pmg_strerror), >0 a hipError_t;
 *   - sums are held in fp32 or more and taken in a fixed order: equal inputs give equal bits. */
#ifndef PMG_LM_H
#define PMG_LM_H

#include "pmg.h"

#ifdef __cplusplus
extern "C" {
#endif

/* element types */
#define PMG_F32 0
#define PMG_BF16 1
#define PMG_F16 2

/* ------------------------------------------------------------------------------- token embedding */

/* out[n] = scale * weight[ids[n]] (rounded once), n < N.
 *   weight [V,E] of `dtype`, rows ld_weight apart; ids [N], id_bits 32 or 64; out [N,E] contiguous.
 * An id outside [0,V) gives a row of NaN (memory safety; validate on the host). */
int pmg_embedding_fwd(const void* weight, int64_t ld_weight, const void* ids, int id_bits, int64_t N, int64_t V, int64_t E,
                      int dtype, float scale, void* out, pmg_stream stream);

/* Bytes of scratch for pmg_embedding_bwd. */
int pmg_embedding_bwd_workspace(int64_t N, int64_t V, int64_t E, int dtype, size_t* out);

/* grad_weight[v] = scale * (sum of grad[n] over the n with ids[n] == v), summed in fp32, rounded once; zero
 * for tokens that do not occur and for padding_idx (-1: none).  Every row is written; ids outside [0,V) add
 * nothing.
 *   grad [N,E] of `dtype`, rows ld_grad apart; grad_weight [V,E] contiguous; V below 2^30. */
int pmg_embedding_bwd(const void* grad, int64_t ld_grad, const void* ids, int id_bits, int64_t N, int64_t V, int64_t E,
                      int dtype, float scale, int64_t padding_idx, void* grad_weight, void* ws, pmg_stream stream);

/* --------------------------------------------------- cross entropy of a linear vocabulary projection */

#define PMG_REDUCE_NONE 0
#define PMG_REDUCE_SUM 1
#define PMG_REDUCE_MEAN 2 /* over the rows with a target; 0 without any */

/* With logits l = logit_scale (hidden weight^T + bias), kept only where `logits` is given:
 *   lse[n]  = log sum_v exp l[n,v]                     (+inf with a logit of +inf, -inf with nothing but -inf)
 *   nll[n]  = row_weight[n] (lse[n] - l[n,targets[n]]), 0 where targets[n] == ignore_index
 *   loss    = nll [N] (PMG_REDUCE_NONE), its sum, or its sum / count; count[0] = rows with a target
 * and, from grad_loss ([N] or [1], as loss) and grad_lse ([N]; either may be NULL: no slope), the
 * gradients of hidden, weight and bias (each NULL: not formed).  row_weight has no gradient.  A row without
 * a slope (ignored, of weight 0) has a zero gradient and adds nothing to the others, whatever it holds.
 * A target outside [0,V) that is not ignore_index gives NaN (memory safety; validate on the host).
 * dtype PMG_F32 or PMG_BF16; the slopes of the logits are rounded to it once, all sums are fp32.  H up to 65536. */
typedef struct pmg_linear_ce {
  int64_t N, V, H;
  int dtype;               /* of hidden, weight, bias and their gradients */
  int id_bits;             /* of targets: 32 or 64 */
  int reduction;
  float logit_scale;
  int64_t ignore_index;
  int64_t ld_hidden, ld_weight;
  const void* hidden;      /* [N,H] */
  const void* weight;      /* [V,H] */
  const void* bias;        /* [V] or NULL */
  const void* targets;     /* [N] */
  const float* row_weight; /* [N] or NULL */
  float* loss;             /* forward: written */
  float* lse;              /* [N]; forward: written, backward: read */
  float* count;            /* [1]; forward: written unless PMG_REDUCE_NONE (then NULL), backward: read with
                              PMG_REDUCE_MEAN */
  const float* grad_loss;  /* backward */
  const float* grad_lse;
  void* grad_hidden;       /* [N,H] contiguous */
  void* grad_weight;       /* [V,H] contiguous */
  void* grad_bias;         /* [V] */
  float* logits;           /* [N, V rounded up to a multiple of 4], 16-byte aligned, or NULL; forward: written (behind a
                              row's V entries: anything), backward: read in place of forming them again */
} pmg_linear_ce;

/* Bytes of scratch of one direction, for a call with these sizes, strides, operands (their alignment counts)
 * and logits.  It does not grow with N x V, but with the larger of N and V:
 *   forward   statistics of tiles, at most 256 MB or 128 V bytes; 4 N
 *   backward  slopes of a piece of the vocabulary, about 256 MB or 256 N elements; 25 N; where there are several
 *             pieces, fp32 sums of grad_hidden, 4 N H; parts of sums that are split over the chip, some 100 MB
 * and copies of hidden or weight where their rows do not begin and end at multiples of 16 bytes. */
int pmg_linear_ce_workspace(const pmg_linear_ce* a, int backward, size_t* out);
int pmg_linear_ce_fwd(const pmg_linear_ce* a, void* ws, pmg_stream stream);
int pmg_linear_ce_bwd(const pmg_linear_ce* a, void* ws, pmg_stream stream);

/* ---------------------------------------------------------------- norm and clipping of many gradients */

/* Bytes of scratch for pmg_grad_norm over `n` tensors of numel[i] elements (numel: HOST array). */
int pmg_grad_norm_workspace(const int64_t* numel, int n, size_t* out);

/* norm[0] = sqrt(sum of the squares of all elements of all tensors), summed in fp64, stored in fp32.
 *   grads, numel, dtype: HOST arrays of `n` device pointers, element counts (0 allowed) and types. */
int pmg_grad_norm(const void* const* grads, const int64_t* numel, const int* dtype, int n, float* norm, void* ws,
                  pmg_stream stream);

/* The refusals of pmg_grad_clip without its launch: 0 or a negative code. */
int pmg_grad_clip_check(void* const* grads, const int64_t* numel, const int* dtype, int n, float max_norm);

/* Every element of every tensor times min(1, max_norm / (norm[0] + 1e-6)), in place (what
 * clip_grad_norm_ of the reference's update does, reinforce_omics.py:336-340).  A NaN norm makes every
 * element NaN.  Tensors must not overlap. */
int pmg_grad_clip(void* const* grads, const int64_t* numel, const int* dtype, int n, const float* norm, float max_norm,
                  pmg_stream stream);

/* ------------------------------------------------------------------------------ Adam / AdamW update */

#define PMG_STATE_BLOCK 256 /* values of an 8-bit state that share one scale */

/* One update of `n` parameters with t = ++step[0], c = min(1, max_norm / (norm[0] + 1e-6)) (1 without
 * `norm`) and p the 32-bit copy where there is one:
 *   g' = c g            (+ weight_decay p  if !decoupled)
 *   m  = beta1 m + (1 - beta1) g'          v = beta2 v + (1 - beta2) g'^2
 *   p  = (decoupled ? 1 - lr weight_decay : 1) p - lr / (1 - beta1^t) m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
 * Every product, sum, quotient and root is rounded to fp32 by itself; the factors in t, lr and norm are
 * formed in fp64 and rounded once.
 * State in 32 bits: m, v fp32 [numel].  State in 8 bits: m int8, v uint8 [numel], and per block of
 * PMG_STATE_BLOCK values (counted from the tensor's start) a fp32 scale m_top / v_top
 * [ceil(numel / PMG_STATE_BLOCK)], the largest magnitude of the block: a code c stands for
 * sign(c) (c/127)^2 m_top, or (c/255)^4 v_top; codes are rounded to nearest, a positive v keeps a code
 * above zero, a block whose largest magnitude is below the normal numbers is held as zeros, a block with
 * a NaN or infinite value reads back without a finite one.
 * All pointer arrays are HOST arrays of `n` device pointers. */
typedef struct pmg_adamw {
  int n;                /* tensors */
  int dtype;            /* of the parameters */
  int grad_dtype;       /* of the gradients: PMG_F32 or `dtype` */
  int state_bits;       /* 32 or 8 */
  int decoupled;        /* 1: AdamW; 0: the decay joins the gradient (the Adam of reinforce.py:44-49) */
  const int64_t* numel; /* HOST [n], 0 allowed */
  void* const* param;
  const void* const* grad;
  void* const* m;
  void* const* v;
  float* const* m_top;  /* 8 bits only, else NULL */
  float* const* v_top;  /* 8 bits only, else NULL */
  float* const* master; /* 32-bit copies that take the update; the parameter is written rounded.  NULL: none */
  int64_t* step;        /* DEVICE [1]: updates made so far; incremented */
  const float* lr_dev;  /* DEVICE [1] or NULL: overrides lr */
  const float* norm;    /* DEVICE [1] or NULL */
  double lr, beta1, beta2, eps, weight_decay, max_norm;
} pmg_adamw;

/* Scratch: PMG_ADAMW_WS bytes.  Buffers that are written must not overlap anything else of the call
 * (refused: PMG error code, nothing is launched). */
#define PMG_ADAMW_WS 64
int pmg_adamw_step(const pmg_adamw* a, void* ws, pmg_stream stream);

/* out[i] (fp32) = the value that code i of an 8-bit state stands for; is_signed: 1 for m, 0 for v. */
int pmg_adamw_values(const void* code, const float* top, int64_t numel, int is_signed, float* out, pmg_stream stream);

#ifdef __cplusplus
}
#endif
#endif /* PMG_LM_H */
