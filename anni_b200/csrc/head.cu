/*
** Loss and gradients of a language model's head (include/anni_head.h).
**
** Forward: the logits of a tile of rows and vocabulary never leave the chip; each tile leaves the maximum and
** the sum of exponentials of its rows, a small kernel joins the tiles of a row.  Backward: for one piece of the
** vocabulary at a time, delta = softmax - one-hot is recomputed from lse and stored as bf16, then multiplied by
** W^T into dx and by x^T into dw.
*/
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>
#include <algorithm>
#include "anni_head.h"
#include "optstep_internal.h"

#define HEAD_TM		64	/* rows and columns of a tile */
#define HEAD_TN		64
#define HEAD_PIECE_BYTES ((size_t)192 << 20)	/* of delta in the workspace */
#define HEAD_TERMS	3	/* bf16 terms of delta for fp32 gradients */

namespace {

struct head_args {
	const __nv_bfloat16	*x;
	int64_t			ldx;
	const __nv_bfloat16	*w;
	int64_t			ldw;
	const float		*bias;
	const int32_t		*target;
	const float		*weight;
	float			scale;
	int			tokens;
	int			d;
	int			vocab;
	float			*nll;
	float			*lse;
	float			*hit;		/* logit of each row's target */
	float2			*part;		/* [tiles over the vocabulary][tokens]: maximum, sum */
	float			*row;		/* factor of each row, 0: no gradient */
	__nv_bfloat16		*delta;		/* [terms][tokens][piece] */
	int			terms;
	int64_t			ldp;
	int			v0;		/* the piece: columns v0 .. v1 - 1 */
	int			v1;
	float			*dxp;		/* fp32 [tokens][d] */
	float			*dbp;		/* fp32 [row tiles][vocab] */
	void			*dx;
	int64_t			lddx;
	void			*dw;
	int64_t			lddw;
	void			*db;
	int			bf16;
	int			add;
	int			*error;
};

/* ---- one 64 x 64 tile of a product in fp32: 256 threads, 4 x 4 results each ----------------------- */

template <typename A, typename B>
__device__ __forceinline__ void tile_product(int k_end, A a, B b, float (&acc)[4][4])
{
	__shared__ float as[16][HEAD_TM + 4];
	__shared__ float bs[16][HEAD_TN + 4];
	const int tm = threadIdx.x / 16 * 4;
	const int tn = threadIdx.x % 16 * 4;

	for (int k0 = 0; k0 < k_end; k0 += 16) {
		for (int i = threadIdx.x; i < 16 * HEAD_TM; i += 256) {
			as[i / HEAD_TM][i % HEAD_TM] = k0 + i / HEAD_TM < k_end ? a(i % HEAD_TM, k0 + i / HEAD_TM) : 0.0f;
			bs[i / HEAD_TN][i % HEAD_TN] = k0 + i / HEAD_TN < k_end ? b(i % HEAD_TN, k0 + i / HEAD_TN) : 0.0f;
		}
		__syncthreads();
		for (int k = 0; k < 16; k++)
			for (int i = 0; i < 4; i++)
				for (int j = 0; j < 4; j++)
					acc[i][j] = fmaf(as[k][tm + i], bs[k][tn + j], acc[i][j]);
		__syncthreads();
	}
}

__device__ __forceinline__ float to_f(__nv_bfloat16 v)
{
	return __bfloat162float(v);
}

/* logits of the tile at (t0, v0), bias included; -inf beyond the vocabulary */
__device__ __forceinline__ void logits_tile(const head_args &h, int t0, int v0, float (*out)[HEAD_TN + 1])
{
	float acc[4][4] = {};
	const int tm = threadIdx.x / 16 * 4;
	const int tn = threadIdx.x % 16 * 4;

	tile_product(h.d, [&](int m, int k) { return t0 + m < h.tokens ? to_f(h.x[(int64_t)(t0 + m) * h.ldx + k]) : 0.0f; },
	    [&](int n, int k) { return v0 + n < h.vocab ? to_f(h.w[(int64_t)k * h.ldw + v0 + n]) : 0.0f; }, acc);
	for (int i = 0; i < 4; i++)
		for (int j = 0; j < 4; j++) {
			const int v = v0 + tn + j;

			out[tm + i][tn + j] = v >= h.vocab ? -INFINITY : acc[i][j] + (h.bias ? h.bias[v] : 0.0f);
		}
	__syncthreads();
}

__global__ void __launch_bounds__(256) loss_kernel(const head_args h)
{
	__shared__ float z[HEAD_TM][HEAD_TN + 1];
	const int t0 = blockIdx.y * HEAD_TM;
	const int v0 = blockIdx.x * HEAD_TN;
	const int t = t0 + threadIdx.x;

	logits_tile(h, t0, v0, z);
	if (threadIdx.x < HEAD_TM && t < h.tokens) {
		float top = -INFINITY;
		float sum = 0.0f;
		const int y = h.target[t];

		for (int j = 0; j < HEAD_TN; j++)
			top = fmaxf(top, z[threadIdx.x][j]);
		for (int j = 0; j < HEAD_TN; j++)
			sum += expf(z[threadIdx.x][j] - (top == -INFINITY ? 0.0f : top));
		h.part[(int64_t)blockIdx.x * h.tokens + t] = make_float2(top, sum);
		if (y >= v0 && y < v0 + HEAD_TN && y < h.vocab)
			h.hit[t] = z[threadIdx.x][y - v0];
	}
}

__global__ void __launch_bounds__(256) join_kernel(const head_args h, int tiles)
{
	const int t = blockIdx.x * blockDim.x + threadIdx.x;
	float top = -INFINITY;
	float sum = 0.0f;
	float lse;
	int y;

	if (t >= h.tokens)
		return;
	for (int k = 0; k < tiles; k++)
		top = fmaxf(top, h.part[(int64_t)k * h.tokens + t].x);
	for (int k = 0; k < tiles; k++) {
		const float2 p = h.part[(int64_t)k * h.tokens + t];

		if (p.x != -INFINITY)
			sum += p.y * expf(p.x - top);
	}
	lse = top + logf(sum);
	y = h.target[t];
	h.lse[t] = lse;
	h.nll[t] = y < 0 ? 0.0f : y >= h.vocab ? NAN : lse - h.hit[t];
}

__global__ void __launch_bounds__(256) row_kernel(const head_args h)
{
	const int t = blockIdx.x * blockDim.x + threadIdx.x;

	if (t < h.tokens) {
		const bool on = h.target[t] >= 0 && h.target[t] < h.vocab && h.lse[t] != -INFINITY;

		h.row[t] = on ? h.scale * (h.weight ? h.weight[t] : 1.0f) : 0.0f;
	}
}

__global__ void __launch_bounds__(256) delta_kernel(const head_args h)
{
	__shared__ float z[HEAD_TM][HEAD_TN + 1];
	const int t0 = blockIdx.y * HEAD_TM;
	const int v0 = h.v0 + blockIdx.x * HEAD_TN;

	logits_tile(h, t0, v0, z);
	for (int i = threadIdx.x; i < HEAD_TM * HEAD_TN; i += 256) {
		const int t = t0 + i / HEAD_TN;
		const int v = v0 + i % HEAD_TN;
		float dl = 0.0f;

		if (t < h.tokens && v < h.v1 && h.row[t] != 0.0f) {
			float rest;

			dl = h.row[t] * (expf(z[i / HEAD_TN][i % HEAD_TN] - h.lse[t]) - (v == h.target[t] ? 1.0f : 0.0f));
			rest = dl;
			for (int k = h.terms - 1; k >= 0; k--) {
				const __nv_bfloat16 q = __float2bfloat16_rn(rest);

				h.delta[((int64_t)k * h.tokens + t) * h.ldp + v - h.v0] = q;
				rest -= to_f(q);
			}
		} else if (t < h.tokens && v < h.v1)
			for (int k = 0; k < h.terms; k++)
				h.delta[((int64_t)k * h.tokens + t) * h.ldp + v - h.v0] = __float2bfloat16_rn(0.0f);
		z[i / HEAD_TN][i % HEAD_TN] = dl;
	}
	__syncthreads();
	if (threadIdx.x < HEAD_TN && v0 + (int)threadIdx.x < h.v1) {
		float s = 0.0f;

		for (int k = 0; k < HEAD_TM; k++)
			s += z[k][threadIdx.x];
		h.dbp[(int64_t)blockIdx.y * h.vocab + v0 + threadIdx.x] = s;
	}
}

__global__ void __launch_bounds__(256) dx_kernel(const head_args h)
{
	float acc[4][4] = {};
	const int t0 = blockIdx.y * HEAD_TM;
	const int d0 = blockIdx.x * HEAD_TN;
	const int tm = threadIdx.x / 16 * 4;
	const int tn = threadIdx.x % 16 * 4;

	for (int p = 0; p < h.terms; p++)
		tile_product(h.v1 - h.v0, [&](int m, int k) { return t0 + m < h.tokens
		    ? to_f(h.delta[((int64_t)p * h.tokens + t0 + m) * h.ldp + k]) : 0.0f; },
		    [&](int n, int k) { return d0 + n < h.d ? to_f(h.w[(int64_t)(d0 + n) * h.ldw + h.v0 + k]) : 0.0f; }, acc);
	for (int i = 0; i < 4; i++)
		for (int j = 0; j < 4; j++)
			if (t0 + tm + i < h.tokens && d0 + tn + j < h.d) {
				float *q = &h.dxp[(int64_t)(t0 + tm + i) * h.d + d0 + tn + j];

				*q = (h.v0 ? *q : 0.0f) + acc[i][j];
			}
}

__device__ __forceinline__ void put(void *base, int64_t i, float v, int bf16, int add)
{
	if (bf16) {
		__nv_bfloat16 *q = static_cast<__nv_bfloat16 *>(base) + i;

		*q = __float2bfloat16_rn(add ? to_f(*q) + v : v);
	} else {
		float *q = static_cast<float *>(base) + i;

		*q = add ? *q + v : v;
	}
}

__global__ void __launch_bounds__(256) dw_kernel(const head_args h)
{
	float acc[4][4] = {};
	const int d0 = blockIdx.y * HEAD_TM;
	const int v0 = h.v0 + blockIdx.x * HEAD_TN;
	const int tm = threadIdx.x / 16 * 4;
	const int tn = threadIdx.x % 16 * 4;

	for (int p = 0; p < h.terms; p++)
		tile_product(h.tokens, [&](int m, int k) { return d0 + m < h.d && h.row[k] != 0.0f
		    ? to_f(h.x[(int64_t)k * h.ldx + d0 + m]) : 0.0f; },
		    [&](int n, int k) { return v0 + n < h.v1
		    ? to_f(h.delta[((int64_t)p * h.tokens + k) * h.ldp + v0 - h.v0 + n]) : 0.0f; }, acc);
	for (int i = 0; i < 4; i++)
		for (int j = 0; j < 4; j++)
			if (d0 + tm + i < h.d && v0 + tn + j < h.v1)
				put(h.dw, (int64_t)(d0 + tm + i) * h.lddw + v0 + tn + j, acc[i][j], h.bf16, h.add);
}

__global__ void __launch_bounds__(256) finish_dx_kernel(const head_args h)
{
	for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < (int64_t)h.tokens * h.d;
	    i += (int64_t)gridDim.x * blockDim.x)
		put(h.dx, i / h.d * h.lddx + i % h.d, h.dxp[i], h.bf16, 0);
}

__global__ void __launch_bounds__(256) finish_db_kernel(const head_args h, int tiles)
{
	const int v = blockIdx.x * blockDim.x + threadIdx.x;
	double s = 0.0;

	if (v >= h.vocab)
		return;
	for (int k = 0; k < tiles; k++)
		s += (double)h.dbp[(int64_t)k * h.vocab + v];
	put(h.db, v, (float)(s + (h.add ? h.bf16 ? (double)to_f(static_cast<__nv_bfloat16 *>(h.db)[v])
	    : (double)static_cast<float *>(h.db)[v] : 0.0)), h.bf16, 0);
}

/* ---- host --------------------------------------------------------------------------------------- */

int64_t up(int64_t n, int64_t to)
{
	return (n + to - 1) / to * to;
}

/* where things lie in the workspace (byte offsets), and how the work is cut */
struct head_plan {
	size_t	hit;
	size_t	part;
	size_t	row;
	size_t	delta;
	size_t	dxp;
	size_t	dbp;
	size_t	bytes;
	int	piece;
	int	terms;
};

int check(const anni_head_call *c, int grad)
{
	if (!c || c->tokens < 0 || c->d_model < 1 || c->vocab < 1)
		return ANNI_E_ARG;
	if (c->tokens > ANNI_HEAD_MAX_TOKENS || c->d_model > ANNI_HEAD_MAX_DIM || c->vocab > ANNI_HEAD_MAX_VOCAB)
		return ANNI_E_LIMIT;
	if (c->ldx < c->d_model || c->ldw < c->vocab || ((uintptr_t)c->x & 1) || ((uintptr_t)c->w & 1))
		return ANNI_E_ARG;
	if (!grad)
		return ANNI_OK;
	if ((c->grad_dtype != ANNI_DT_F32 && c->grad_dtype != ANNI_DT_BF16) || (c->flags & ~ANNI_HEAD_ACCUMULATE))
		return ANNI_E_ARG;
	if ((c->dx && c->lddx < c->d_model) || (c->dw && c->lddw < c->vocab))
		return ANNI_E_ARG;
	if (((uintptr_t)c->dx | (uintptr_t)c->dw | (uintptr_t)c->dbias) & (c->grad_dtype == ANNI_DT_BF16 ? 1 : 3))
		return ANNI_E_ARG;
	return ANNI_OK;
}

/* addresses that a call with something to do must have */
int check_buffers(const anni_head_call *c, int grad, size_t need)
{
	if (!c->x || !c->w || !c->target || !c->lse || (!grad && !c->nll) || !c->workspace)
		return ANNI_E_ARG;
	if (((uintptr_t)c->bias | (uintptr_t)c->target | (uintptr_t)c->lse | (uintptr_t)c->nll | (uintptr_t)c->weight) & 3)
		return ANNI_E_ARG;
	return ((uintptr_t)c->workspace & 255) || c->workspace_bytes < need ? ANNI_E_ARG : ANNI_OK;
}

size_t take(size_t *at, int64_t bytes)
{
	const size_t here = *at;

	*at = (size_t)up((int64_t)here + bytes, 256);
	return here;
}

head_plan plan_of(const anni_head_call *c, int grad)
{
	head_plan p;
	const int64_t t = std::max<int64_t>(c->tokens, 1);

	memset(&p, 0, sizeof(p));
	p.bytes = 256;		/* the error word */
	if (!grad) {
		p.hit = take(&p.bytes, t * 4);
		p.part = take(&p.bytes, up(c->vocab, HEAD_TN) / HEAD_TN * t * 8);
		return p;
	}
	p.terms = c->grad_dtype == ANNI_DT_BF16 ? 1 : HEAD_TERMS;
	p.piece = (int)std::min<int64_t>(up(c->vocab, 256),
	    std::max<int64_t>(256, (int64_t)(HEAD_PIECE_BYTES / (size_t)(t * 2 * p.terms)) / 256 * 256));
	p.row = take(&p.bytes, t * 4);
	p.delta = take(&p.bytes, (int64_t)p.piece * t * 2 * p.terms);
	p.dxp = take(&p.bytes, c->dx ? t * c->d_model * 4 : 0);
	p.dbp = take(&p.bytes, up(t, HEAD_TM) / HEAD_TM * c->vocab * 4);
	return p;
}

head_args args_of(const anni_head_call *c, const head_plan &p)
{
	head_args h;
	char *ws = static_cast<char *>(c->workspace);

	memset(&h, 0, sizeof(h));
	h.x = static_cast<const __nv_bfloat16 *>(c->x);
	h.ldx = c->ldx;
	h.w = static_cast<const __nv_bfloat16 *>(c->w);
	h.ldw = c->ldw;
	h.bias = c->bias;
	h.target = c->target;
	h.weight = c->weight;
	h.scale = (float)c->grad_scale;
	h.tokens = (int)c->tokens;
	h.d = c->d_model;
	h.vocab = c->vocab;
	h.nll = c->nll;
	h.lse = c->lse;
	h.hit = reinterpret_cast<float *>(ws + p.hit);
	h.part = reinterpret_cast<float2 *>(ws + p.part);
	h.row = reinterpret_cast<float *>(ws + p.row);
	h.delta = reinterpret_cast<__nv_bfloat16 *>(ws + p.delta);
	h.terms = p.terms;
	h.ldp = p.piece;
	h.dxp = reinterpret_cast<float *>(ws + p.dxp);
	h.dbp = reinterpret_cast<float *>(ws + p.dbp);
	h.dx = c->dx;
	h.lddx = c->lddx;
	h.dw = c->dw;
	h.lddw = c->lddw;
	h.db = c->dbias;
	h.bf16 = c->grad_dtype == ANNI_DT_BF16;
	h.add = (c->flags & ANNI_HEAD_ACCUMULATE) != 0;
	h.error = reinterpret_cast<int *>(ws);
	return h;
}

unsigned tiles(int64_t n, int64_t of)
{
	return (unsigned)((n + of - 1) / of);
}

int launched(void)
{
	anni_count_launch();
	return cudaGetLastError() == cudaSuccess ? ANNI_OK : ANNI_E_CUDA;
}

}	/* namespace */

extern "C" int anni_head_workspace(const anni_head_call *c, int grad, size_t *bytes)
{
	int rc = check(c, grad);

	if (rc != ANNI_OK || !bytes)
		return rc != ANNI_OK ? rc : ANNI_E_ARG;
	*bytes = plan_of(c, grad).bytes;
	return ANNI_OK;
}

extern "C" int anni_head_loss(const anni_head_call *c, void *stream)
{
	cudaStream_t st = (cudaStream_t)stream;
	int rc = check(c, 0);
	head_plan p;
	head_args h;

	if (rc != ANNI_OK || c->tokens == 0)
		return rc;
	p = plan_of(c, 0);
	rc = check_buffers(c, 0, p.bytes);
	if (rc != ANNI_OK)
		return rc;
	h = args_of(c, p);
	if (cudaMemsetAsync(h.error, 0, 256, st) != cudaSuccess)
		return ANNI_E_CUDA;
	loss_kernel<<<dim3(tiles(h.vocab, HEAD_TN), tiles(h.tokens, HEAD_TM)), 256, 0, st>>>(h);
	rc = launched();
	if (rc == ANNI_OK) {
		join_kernel<<<tiles(h.tokens, 256), 256, 0, st>>>(h, (int)tiles(h.vocab, HEAD_TN));
		rc = launched();
	}
	return rc;
}

/* no rows: the gradients are those of an empty sum */
static int grad_of_nothing(const anni_head_call *c, cudaStream_t st)
{
	const size_t size = c->grad_dtype == ANNI_DT_BF16 ? 2 : 4;

	if (c->flags & ANNI_HEAD_ACCUMULATE)
		return ANNI_OK;
	if (c->dw && cudaMemset2DAsync(c->dw, (size_t)c->lddw * size, 0, (size_t)c->vocab * size, (size_t)c->d_model, st) != cudaSuccess)
		return ANNI_E_CUDA;
	if (c->dbias && cudaMemsetAsync(c->dbias, 0, (size_t)c->vocab * size, st) != cudaSuccess)
		return ANNI_E_CUDA;
	return ANNI_OK;
}

extern "C" int anni_head_loss_grad(const anni_head_call *c, void *stream)
{
	cudaStream_t st = (cudaStream_t)stream;
	int rc = check(c, 1);
	head_plan p;
	head_args h;

	if (rc != ANNI_OK || (!c->dx && !c->dw && !c->dbias))
		return rc;
	if (c->tokens == 0)
		return grad_of_nothing(c, st);
	p = plan_of(c, 1);
	rc = check_buffers(c, 1, p.bytes);
	if (rc != ANNI_OK)
		return rc;
	h = args_of(c, p);
	if (cudaMemsetAsync(h.error, 0, 256, st) != cudaSuccess)
		return ANNI_E_CUDA;
	row_kernel<<<tiles(h.tokens, 256), 256, 0, st>>>(h);
	rc = launched();
	for (h.v0 = 0; rc == ANNI_OK && h.v0 < h.vocab; h.v0 = h.v1) {
		h.v1 = std::min(h.vocab, h.v0 + p.piece);
		delta_kernel<<<dim3(tiles(h.v1 - h.v0, HEAD_TN), tiles(h.tokens, HEAD_TM)), 256, 0, st>>>(h);
		rc = launched();
		if (rc == ANNI_OK && h.dx) {
			dx_kernel<<<dim3(tiles(h.d, HEAD_TN), tiles(h.tokens, HEAD_TM)), 256, 0, st>>>(h);
			rc = launched();
		}
		if (rc == ANNI_OK && h.dw) {
			dw_kernel<<<dim3(tiles(h.v1 - h.v0, HEAD_TN), tiles(h.d, HEAD_TM)), 256, 0, st>>>(h);
			rc = launched();
		}
	}
	if (rc == ANNI_OK && h.dx) {
		finish_dx_kernel<<<std::min(2048u, tiles((int64_t)h.tokens * h.d, 256)), 256, 0, st>>>(h);
		rc = launched();
	}
	if (rc == ANNI_OK && h.db) {
		finish_db_kernel<<<tiles(h.vocab, 256), 256, 0, st>>>(h, (int)tiles(h.tokens, HEAD_TM));
		rc = launched();
	}
	return rc;
}

extern "C" int anni_head_status(const anni_head_call *c, void *stream)
{
	int error = 0;

	if (!c || !c->workspace)
		return ANNI_E_ARG;
	if (cudaStreamSynchronize((cudaStream_t)stream) != cudaSuccess
	    || cudaMemcpy(&error, c->workspace, sizeof(error), cudaMemcpyDeviceToHost) != cudaSuccess)
		return ANNI_E_CUDA;
	return error;
}
