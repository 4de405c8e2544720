/*
** The loss of a language model's head and its gradients, for the trainer whose optimizer step this
** library is: logits = x W + b over the whole vocabulary, softmax cross entropy against one target per
** row, and the gradients of x, W and b -- written or added where the step reads them, i.e. straight into
** the gradient flat.  W is the head's bf16 twin as the step emits it: row-major [d_model][vocab], the
** reference's w_head (lang/lm_adam.c:117-136).
** The reference computes the same on a device with one matrix product and several passes over stored
** logits (gpu_ce_* of num/gpu.h); here neither logits nor probabilities of the whole vocabulary exist:
** the forward pass keeps a running maximum and sum per row and piece, the backward pass recomputes
** the logits of one piece of the vocabulary at a time.
**
**   lse[t] = log sum_v exp(x[t] W[:,v] + b[v])            nll[t] = lse[t] - (x[t] W[:,target[t]] + b[target[t]])
**   delta[t][v] = grad_scale * weight[t] * (exp(x[t] W[:,v] + b[v] - lse[t]) - [v = target[t]])
**   dx = delta W^T        dw (+)= x^T delta        dbias (+)= column sums of delta
**
** Rows: a target below 0 is ignored (nll 0, no gradient; x[t] may hold anything), a target >= vocab
** gives nll NaN and no gradient, and a row whose factor grad_scale * weight[t] is 0 has no gradient
** either, whatever x[t] holds.  A bias of -inf, or a finite one far below the other logits, masks an entry of
** the vocabulary (its column of W must still be finite); a row with nothing but -inf left has nll NaN and no
** gradient.
**
** Arithmetic: products of bf16 values in fp32 accumulators; maximum, sum, exponentials in fp32.  For
** bf16 gradients delta is rounded once to bf16 as the operand of the two products; for fp32 gradients
** it is carried as three bf16 terms (24 bits), so dx and dw are good to fp32.  dbias is summed in fp32
** from the unrounded delta.  The tensor cores cut sums off instead of rounding them (up to 7e-9 of a sum per term);
** sums are therefore taken in runs that are added up rounded: 512 terms of a logit of the loss, 256 of fp32
** gradients, 16,384 of bf16 gradients and 4096 of the logits behind these.  Sums run in a fixed order: the
** same inputs give the same bits.
**
** Waits inside the kernels are bounded: a block that gives up (two seconds without progress) fills what it
** has not computed with NaN, which shows in nll, dx, dw and dbias.
**
** Nothing is allocated and nothing is kept: all working memory is the caller's, and calls that use
** different workspaces are independent.  Work runs on the current device, which must hold the buffers.
*/
#ifndef ANNI_HEAD_H__
#define ANNI_HEAD_H__

#include "anni_b200.h"
#include "anni_lm_adam.h"

#ifdef __cplusplus
extern "C" {
#endif

#define ANNI_HEAD_ACCUMULATE	1	/* dw and dbias are added to what is there */
#define ANNI_HEAD_MAX_TOKENS	(1 << 24)
#define ANNI_HEAD_MAX_DIM	(1 << 16)
#define ANNI_HEAD_MAX_VOCAB	(1 << 24)

/*
** One call.  ld*: elements from one row to the next, at least the row's length.  Any address and stride
** that the element type allows is taken; x and w on 16-byte addresses with strides that are multiples of
** 8 elements are read in place, others are copied into the workspace first (w: 4 bytes of traffic per
** element); anni_head_loss_grad copies x in any case, with zeros for the rows that have no gradient.
** The loss of one or two rows copies nothing.  Outputs overlap neither each other nor what is read.
*/
typedef struct anni_head_call {
	const void	*x;		/* bf16 [tokens][ldx] */
	int64_t		ldx;
	const void	*w;		/* bf16 [d_model][ldw] */
	int64_t		ldw;
	const float	*bias;		/* fp32 [vocab], or NULL */
	const int32_t	*target;	/* [tokens] */
	int64_t		tokens;		/* 0 <= tokens <= ANNI_HEAD_MAX_TOKENS */
	int32_t		d_model;	/* 1 .. ANNI_HEAD_MAX_DIM */
	int32_t		vocab;		/* 1 .. ANNI_HEAD_MAX_VOCAB */
	float		*nll;		/* [tokens]; written by anni_head_loss */
	float		*lse;		/* [tokens]; written by anni_head_loss, read by anni_head_loss_grad */
	/* gradients */
	const float	*weight;	/* fp32 [tokens] factor of each row, or NULL: 1 */
	double		grad_scale;
	int		grad_dtype;	/* ANNI_DT_F32 or ANNI_DT_BF16: type of dx, dw, dbias */
	int		flags;		/* ANNI_HEAD_* */
	void		*dx;		/* [tokens][lddx], or NULL: not wanted */
	int64_t		lddx;
	void		*dw;		/* [d_model][lddw], or NULL */
	int64_t		lddw;
	void		*dbias;		/* [vocab], or NULL */
	void		*workspace;	/* device memory, 256-byte aligned */
	size_t		workspace_bytes;
} anni_head_call;

/*
** Bytes of workspace that anni_head_loss (grad = 0) or anni_head_loss_grad (grad = 1) of this call need.
** Only sizes, types, addresses and strides of x and w, and which outputs are wanted are looked at: where dw and
** dbias lie, and whether they are added to, makes no difference.
*/
int	anni_head_workspace(const anni_head_call *c, int grad, size_t *bytes);
/*
** nll and lse of every row.  ANNI_E_ARG: a missing or misaligned address, a size or stride out of range,
** a workspace that is too small; ANNI_E_LIMIT: a size beyond its maximum, or more than 2^30 tiles of 128 rows
** and 256 entries.  Nothing is queued then.
*/
int	anni_head_loss(const anni_head_call *c, void *stream);
/* dx, dw, dbias from lse, which an anni_head_loss on the same x, w, bias has written. */
int	anni_head_loss_grad(const anni_head_call *c, void *stream);

/*
** The call's share of an optimizer object (anni_lm_adam.h): W is tensor w_tensor's bf16 twin, the bias tensor
** b_tensor's fp32 weights (b_tensor < 0: none); dw and dbias are their slices of the gradient flat, added to as
** the backward pass of the reference does (lang/lm_train.c:1220-1226), grad_scale is the object's loss
** scale, grad_dtype its gradients' type.  The caller has set d_model and vocab and sets everything else
** (x, target, tokens, nll, lse, weight, dx, workspace) before or after.  The flats live as long as the object;
** its step reads and clears the gradients on the legacy stream: run the head there, or order the two.
** ANNI_E_ARG: not prepared (anni_lm_adam_prepare) or invalidated, a tensor of another size, without a twin, or
** whose gradients still come from the host (anni_lm_adam_alias / _alias_vec end that).
*/
int	anni_lm_adam_head_call(const anni_lm_adam *opt, int w_tensor, int b_tensor, anni_head_call *c);

#ifdef __cplusplus
}
#endif

#endif
