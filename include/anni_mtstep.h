/*
** AdamW over a LIST of tensors that lie wherever their owner put them, with moments in 32 bits or
** in 8: the step of anni_b200.h for a trainer that has no packed arena (tensors allocated one by
** one, adapters beside a frozen model, a parameter subset), and for one whose moments have to fit a
** quarter of the memory.  No counterpart in the reference, whose optimizer knows one flat layout.
**
** One cooperative launch per step, however many tensors: global norm over the whole list, clip factor
** and skip decision on the device, AdamW with decoupled decay by tensor, bf16 twins.  Names, flags,
** hyper-parameters, status and error codes are those of anni_b200.h.
**
** 32-bit moments (ANNI_DT_F32): the arithmetic of anni_optstep_step (moments in double, each product
** and sum rounded on its own, stored as float; parameter update in float): the same bits for the
** same inputs.
**
** 8-bit moments (ANNI_DT_Q8): within a tensor every ANNI_MT_BLOCK consecutive elements share one fp32
** scale for m and one for v; element i of block k is
**     m = e4m3 code * m_scale[k]        v = e5m2 code * v_scale[k]
** (e4m3: sign, 4 exponent and 3 fraction bits, largest 448; e5m2: 5 and 2, largest 57344).  A step
** reads the codes, updates in float, steps the parameter from the unrounded new moments, and codes them
** anew with m_scale = max|m| / 448 and v_scale = max v / 57344 of the block.  A block whose largest
** value is below 2^-100 becomes zero.  A v that is not zero never becomes zero in a block that is
** not: its code is at least the smallest, so that no element divides its m by eps alone.
** Rounding is to nearest, ties to even; with ANNI_STEP_STOCHASTIC it is up with the probability of the
** part cut off, in 16 random bits per element and moment that depend on the caller's seed and the
** element's place in the list alone.  To nearest, a v whose step's change is below half a code (for
** beta2 = 0.999 a change of v by less than a few per cent) stays where it is; stochastic rounding
** follows it on average.
**
** Calls on one handle belong on one stream, one after another (a step changes its tensors in place
** anyway); different handles are independent.  Every call works on the device the handle was created
** on, whichever device is current.  Steps and anni_mtstep_set_grads can be captured into a graph: the
** handle then has to live as long as the graph; the values of hp and seed are those of the capture, and a replayed step takes the gradient addresses that the
** last anni_mtstep_set_grads before it, replayed or not, has left.
*/
#ifndef ANNI_MTSTEP_H__
#define ANNI_MTSTEP_H__

#include "anni_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

#define ANNI_DT_Q8		2	/* moments only: 8-bit codes with a scale per ANNI_MT_BLOCK elements */
#define ANNI_MT_BLOCK		256
#define ANNI_STEP_STOCHASTIC	32	/* per-step flag: stochastic rounding of 8-bit moments */

/*
** One tensor of the list: n >= 0 contiguous elements at any address that its type allows.  The fast step wants
** fp32 buffers (scales and gradients aside) on 16 bytes, twins on 8 and 8-bit moments on 4: one tensor
** off that grid sends the whole list through plain loads (184.7 M elements: 1.64 ms instead of 0.93, in 8
** bits 1.15 instead of 0.57); a gradient off 16 bytes slows its own tensor alone.  grad may be
** NULL: the tensor then sits out (no share in the norm, nothing read or written).  m_scale, v_scale:
** (n + ANNI_MT_BLOCK - 1) / ANNI_MT_BLOCK floats each, with 8-bit moments only.  flags: ANNI_SEG_WD,
** ANNI_SEG_TWIN_BF16 (twin_bf16 then must be given).
*/
typedef struct anni_mt_tensor {
	float	*param;		/* fp32 [n], updated in place */
	void	*grad;		/* grad_dtype [n] */
	void	*m;		/* fp32 [n], or one byte per element */
	void	*v;
	float	*m_scale;
	float	*v_scale;
	void	*twin_bf16;	/* uint16 [n] */
	int64_t	n;
	uint32_t flags;		/* ANNI_SEG_* */
} anni_mt_tensor;

typedef struct anni_mtstep anni_mtstep;

/*
** Lays out the list on the current device (addresses and counts are copied; nothing is read).  What it writes to
** the device is there when it returns: the first step may go to any stream.
** grad_dtype: ANNI_DT_F32 or ANNI_DT_BF16; state_dtype: ANNI_DT_F32 or ANNI_DT_Q8.
** ANNI_E_ARG: n_tensors < 1, an unknown type or flag, a missing or misaligned address, two buffers that
** overlap (the same tensor twice among them).  ANNI_E_LIMIT: more than 2^31 - 1 pieces of 2048 elements.
*/
int	anni_mtstep_create(const anni_mt_tensor *list, int n_tensors, int grad_dtype, int state_dtype,
		anni_mtstep **out);
void	anni_mtstep_destroy(anni_mtstep *h);
/*
** New gradient addresses (n_tensors of them, NULL: sits out) for the steps queued after this call on the
** same stream; the array may be reused at once.  Checks as for create.
*/
int	anni_mtstep_set_grads(anni_mtstep *h, void *const *grads, void *stream);
/*
** One step.  hp as for anni_optstep_step; flags: ANNI_STEP_CHECK_FINITE, ANNI_STEP_ZERO_GRAD,
** ANNI_STEP_STOCHASTIC (ANNI_E_ARG for any other, and for the last without 8-bit moments).  The norm is
** taken, and the gradients read twice, only if hp asks for a clip or the finite check.  With neither,
** non-finite gradients go where the formula takes them; in 8 bits they spoil their whole block.
*/
int	anni_mtstep_step(anni_mtstep *h, const anni_optstep_hyper *hp, uint64_t seed, void *stream);
/* Blocks until `stream` has finished the queued steps, then copies the status. */
int	anni_mtstep_status_read(anni_mtstep *h, anni_optstep_status *out, void *stream);

#ifdef __cplusplus
}
#endif

#endif
