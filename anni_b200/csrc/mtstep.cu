/*
** AdamW over a list of tensors (include/anni_mtstep.h): one cooperative launch per step.
**
** The list is cut into tiles of ANNI_MT_TILE elements that do not cross tensors; a table says which
** tensor a tile belongs to.  A block takes a tile at a time, each of its eight warps one run of
** ANNI_MT_BLOCK = 256 elements -- the run that shares a scale in the 8-bit form, so that the two
** block maxima are reductions inside a warp.
*/
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <stdlib.h>
#include <string.h>
#include <algorithm>
#include <vector>
#include "anni_mtstep.h"
#include "optstep_internal.h"
#include "optstep_device.h"

#define ANNI_MT_TILE		(ANNI_THREADS / 32 * ANNI_MT_BLOCK)
#define ANNI_MT_ADDRS		448	/* gradient addresses per launch of set_grads_kernel */

namespace {

/* one tensor on the device; the gradient's address lives in a table of its own (anni_mtstep_set_grads) */
struct mt_desc {
	float		*p;
	void		*m;
	void		*v;
	float		*ms;
	float		*vs;
	uint16_t	*twin;		/* NULL: none */
	int64_t		n;
	uint64_t	block0;		/* blocks of 256 in the tensors before this one */
	uint32_t	tile0;		/* tiles in the tensors before this one */
	uint32_t	wd;
};

struct mt_launch {
	anni_launch	la;		/* hyper-parameters, flags, control block */
	const mt_desc	*desc;
	void *const	*grad;
	const uint32_t	*tile_of;	/* tensor of each tile */
	uint32_t	tiles;
	uint64_t	seed;
};

/* ---- 8-bit moments ------------------------------------------------------------ */

/* the 32-bit finaliser of MurmurHash3 (A. Appleby, public domain) */
__device__ __forceinline__ uint32_t mix32(uint32_t h)
{
	h = (h ^ (h >> 16)) * 0x85ebca6bu;
	h = (h ^ (h >> 13)) * 0xc2b2ae35u;
	return h ^ (h >> 16);
}

/* random key of a block: of the seed and the block's number in the list */
__device__ __forceinline__ uint32_t block_key(uint64_t seed, uint64_t block)
{
	return mix32((uint32_t)seed ^ mix32((uint32_t)block + (uint32_t)(seed >> 32) * 0x9e3779b9u));
}

/*
** x to KEPT bits of mantissa, up with the probability of the part cut off: 16 random bits are added to
** the top of the bits that go, and the carry decides.  Below LEAST, the smallest normal number of the
** 8-bit type, its numbers are equally spaced; adding LEAST puts x into the binade with that spacing.
*/
template <int KEPT>
__device__ __forceinline__ float stochastic(float x, uint32_t r16, float least)
{
	const int cut = 23 - KEPT;
	const float a = fabsf(x);
	const float add = a < least ? least : 0.0f;
	const uint32_t bits = __float_as_uint(__fadd_rn(a, add)) + (r16 << (cut - 16));
	const float r = __fsub_rn(__uint_as_float(bits >> cut << cut), add);

	return copysignf(r, x);
}

struct q8_hyper {
	float	b1;
	float	omb1;
	float	b2;
	float	omb2;
	float	coef;
};

/* moments in float (their stored form has three and two bits of mantissa), then the shared parameter update */
__device__ __forceinline__ void adam_q8(const anni_launch &a, const q8_hyper &h, float lrwd, float gf, float &p,
	float &m, float &v)
{
	const float g = gf * h.coef;

	m = fmaf(h.b1, m, h.omb1 * g);
	v = fmaf(h.b2, v, h.omb2 * g * g);
	adam_apply(a, lrwd, p, m, v);
}

/* scale of a block from its largest value (as bits, >= 0) and the multiplier that undoes it; a NaN stays one */
__device__ __forceinline__ void q8_scale(uint32_t amax_bits, float top, float &scale, float &inv)
{
	const float amax = __uint_as_float(amax_bits);
	const bool none = amax < 7.8886090522101181e-31f;	/* 2^-100 */

	scale = none ? 0.0f : __fdiv_rn(amax, top);
	inv = none ? 0.0f : __fdiv_rn(top, amax);
}

__device__ __forceinline__ float e4m3_to_float(uint32_t c)
{
	return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E4M3)));
}

__device__ __forceinline__ float e5m2_to_float(uint32_t c)
{
	return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E5M2)));
}

__device__ __forceinline__ uint32_t to_e4m3(float x)
{
	return __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ uint32_t to_e5m2(float x)
{
	return __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E5M2);
}

/* ---- one warp's run of at most 256 elements -------------------------------------- */

/*
** Element-wise: lane l holds elements l, l + 32, ... of the run, so plain accesses coalesce whatever
** the address.
*/
template <typename GradT, bool Q8>
__device__ __forceinline__ void run_scalar(const mt_launch &a, const mt_desc &d, void *grad, int64_t e0, int len,
	double coef, const q8_hyper &h, bool skip)
{
	const int lane = threadIdx.x & 31;
	const float lrwd = d.wd ? a.la.lrwd : 0.0f;
	const int64_t blk = e0 / ANNI_MT_BLOCK;
	float m[8];
	float v[8];
	float ms = 0.0f;
	float vs = 0.0f;
	uint32_t am = 0;
	uint32_t av = 0;

	if (!skip) {
		if (Q8) {
			ms = d.ms[blk];
			vs = d.vs[blk];
		}
#pragma unroll
		for (int j = 0; j < 8; j++) {
			const int i = j * 32 + lane;
			const int64_t e = e0 + i;

			m[j] = v[j] = 0.0f;
			if (i < len) {
				float p = d.p[e];
				const float g = io8<GradT>::load1(grad, e);

				if (Q8) {
					m[j] = e4m3_to_float(static_cast<const uint8_t *>(d.m)[e]) * ms;
					v[j] = e5m2_to_float(static_cast<const uint8_t *>(d.v)[e]) * vs;
					adam_q8(a.la, h, lrwd, g, p, m[j], v[j]);
					am = max(am, __float_as_uint(fabsf(m[j])));
					av = max(av, __float_as_uint(v[j]));
				} else {
					m[j] = static_cast<const float *>(d.m)[e];
					v[j] = static_cast<const float *>(d.v)[e];
					adam_elem<false>(a.la, coef, lrwd, g, p, m[j], v[j]);
					static_cast<float *>(d.m)[e] = m[j];
					static_cast<float *>(d.v)[e] = v[j];
				}
				d.p[e] = p;
				if (d.twin)
					io8<__nv_bfloat16>::store1(d.twin, e, p);
			}
		}
	}
	if (Q8 && !skip) {
		float mi;
		float vi;
		uint32_t key = 0;

		am = __reduce_max_sync(0xffffffffu, am);
		av = __reduce_max_sync(0xffffffffu, av);
		q8_scale(am, 448.0f, ms, mi);
		q8_scale(av, 57344.0f, vs, vi);
		if (lane == 0) {
			d.ms[blk] = ms;
			d.vs[blk] = vs;
		}
		if (a.la.flags & ANNI_STEP_STOCHASTIC)
			key = block_key(a.seed, d.block0 + (uint64_t)blk);
#pragma unroll
		for (int j = 0; j < 8; j++) {
			const int i = j * 32 + lane;
			float x = m[j] * mi;
			float y = v[j] * vi;
			uint32_t c;

			if (i >= len)
				continue;
			if (a.la.flags & ANNI_STEP_STOCHASTIC) {
				const uint32_t r = mix32(key + (uint32_t)i * 0x9e3779b9u);

				x = stochastic<3>(x, r & 0xffffu, 0.015625f);
				y = stochastic<2>(y, r >> 16, 6.103515625e-5f);
			}
			static_cast<uint8_t *>(d.m)[e0 + i] = (uint8_t)to_e4m3(x);
			c = to_e5m2(y);
			if (c == 0 && v[j] > 0.0f && vi > 0.0f)
				c = 1;
			static_cast<uint8_t *>(d.v)[e0 + i] = (uint8_t)c;
		}
	}
	if (a.la.flags & ANNI_STEP_ZERO_GRAD)
		for (int i = lane; i < len; i += 32)
			io8<GradT>::store1(grad, e0 + i, 0.0f);
}

/* where tile t lies for this warp: tensor, first element of the run, its length (0: nothing) */
__device__ __forceinline__ uint32_t run_of(const mt_launch &a, uint32_t t, int64_t &e0, int &len)
{
	const uint32_t s = a.tile_of[t];
	const int64_t left = a.desc[s].n
	    - (e0 = (int64_t)(t - a.desc[s].tile0) * ANNI_MT_TILE + (threadIdx.x >> 5) * ANNI_MT_BLOCK);

	len = left <= 0 ? 0 : left < ANNI_MT_BLOCK ? (int)left : ANNI_MT_BLOCK;
	return s;
}

template <typename GradT>
__device__ __forceinline__ double mt_norm_phase(const mt_launch &a)
{
	const int lane = threadIdx.x & 31;
	double acc = 0.0;

	for (uint32_t t = blockIdx.x; t < a.tiles; t += gridDim.x) {
		int64_t e0;
		int len;
		const void *grad = a.grad[run_of(a, t, e0, len)];

		if (!grad)
			continue;
		for (int i = lane; i < len; i += 32) {
			const double g = (double)io8<GradT>::load1(grad, e0 + i);

			acc = fma(g, g, acc);
		}
	}
	return acc;
}

template <typename GradT, bool Q8>
__global__ void __launch_bounds__(ANNI_THREADS) mt_step_kernel(const mt_launch a)
{
	decision d;
	q8_hyper h;
	double ss = 0.0;

	if (a.la.flags & ANNI_LAUNCH_NEED_NORM) {
		const double s = block_sum(mt_norm_phase<GradT>(a));

		if (threadIdx.x == 0)
			a.la.ctl->partials[blockIdx.x] = s;
		if (!grid_barrier(a.la.ctl, gridDim.x))
			return;
		ss = sum_partials(a.la.ctl, (int)gridDim.x);
	}
	d = decide(a.la, ss, 0.0, 0.0);
	if (blockIdx.x == 0 && threadIdx.x == 0) {
		a.la.ctl->reduce[0] = ss;
		a.la.ctl->reduce[1] = isfinite(ss) ? 0.0 : 1.0;
		a.la.ctl->norm = d.norm;
		a.la.ctl->eff_scale = d.coef;
		a.la.ctl->skipped = d.skip ? 1 : 0;
	}
	h.b1 = (float)a.la.b1;
	h.omb1 = (float)a.la.omb1;
	h.b2 = (float)a.la.b2;
	h.omb2 = (float)a.la.omb2;
	h.coef = (float)d.coef;
	if (!d.skip || (a.la.flags & ANNI_STEP_ZERO_GRAD))
		for (uint32_t t = blockIdx.x; t < a.tiles; t += gridDim.x) {
			int64_t e0;
			int len;
			const uint32_t s = run_of(a, t, e0, len);
			void *grad = a.grad[s];

			if (grad && len > 0)
				run_scalar<GradT, Q8>(a, a.desc[s], grad, e0, len, d.coef, h, d.skip);
		}
	step_epilogue(a.la.ctl, d.skip);
}

struct mt_addrs {
	void	*g[ANNI_MT_ADDRS];
};

/* gradient addresses travel as kernel arguments: in stream order, and part of a capture */
__global__ void set_grads_kernel(void **to, const mt_addrs from, int n)
{
	for (int i = threadIdx.x; i < n; i += blockDim.x)
		to[i] = from.g[i];
}

const void *step_kernel(int grad_dtype, int state_dtype)
{
	if (grad_dtype == ANNI_DT_BF16)
		return state_dtype == ANNI_DT_Q8 ? (const void *)mt_step_kernel<__nv_bfloat16, true>
		    : (const void *)mt_step_kernel<__nv_bfloat16, false>;
	return state_dtype == ANNI_DT_Q8 ? (const void *)mt_step_kernel<float, true>
	    : (const void *)mt_step_kernel<float, false>;
}

struct range {
	uintptr_t	lo;
	uintptr_t	hi;
	bool operator<(const range &o) const { return lo < o.lo; }
};

void add_range(std::vector<range> &v, const void *p, int64_t bytes)
{
	if (bytes > 0)
		v.push_back({ (uintptr_t)p, (uintptr_t)p + (uintptr_t)bytes });
}

/* sorted ranges: does any reach into the next? */
bool overlapping(const std::vector<range> &v)
{
	for (size_t k = 1; k < v.size(); k++)
		if (v[k - 1].hi > v[k].lo)
			return true;
	return false;
}

/* the handle's device for the length of a call */
struct on_device {
	int	was;
	bool	ok;
	explicit on_device(int want) : was(-1), ok(true)
	{
		if (cudaGetDevice(&was) != cudaSuccess)
			ok = false;
		else if (was == want)
			was = -1;
		else
			ok = cudaSetDevice(want) == cudaSuccess;
	}
	~on_device()
	{
		if (was >= 0)
			(void)cudaSetDevice(was);
	}
};

}	/* namespace */

struct anni_mtstep {
	int			device;
	int			grad_dtype;
	int			state_dtype;
	int			n_tensors;
	int			blocks;
	uint32_t		tiles;
	anni_control		*ctl;		/* device, as the next three */
	mt_desc			*desc;
	void			**grad;
	uint32_t		*tile_of;
	std::vector<int64_t>	counts;
	std::vector<range>	written;	/* everything but the gradients, sorted */
};

/* gradients on their type's alignment, clear of each other and of what the step writes */
static int check_grads(const anni_mtstep *h, void *const *grads)
{
	const uintptr_t size = h->grad_dtype == ANNI_DT_BF16 ? 2 : 4;
	std::vector<range> all = h->written;

	for (int i = 0; i < h->n_tensors; i++) {
		if ((uintptr_t)grads[i] & (size - 1))
			return ANNI_E_ARG;
		if (grads[i])
			add_range(all, grads[i], h->counts[i] * (int64_t)size);
	}
	std::inplace_merge(all.begin(), all.begin() + (ptrdiff_t)h->written.size(),
	    (std::sort(all.begin() + (ptrdiff_t)h->written.size(), all.end()), all.end()));
	return overlapping(all) ? ANNI_E_ARG : ANNI_OK;
}

static int send_grads(anni_mtstep *h, void *const *grads, cudaStream_t st)
{
	for (int i = 0; i < h->n_tensors; i += ANNI_MT_ADDRS) {
		const int n = std::min(ANNI_MT_ADDRS, h->n_tensors - i);
		mt_addrs a;

		memcpy(a.g, grads + i, (size_t)n * sizeof(void *));
		memset(a.g + n, 0, (size_t)(ANNI_MT_ADDRS - n) * sizeof(void *));
		set_grads_kernel<<<1, 128, 0, st>>>(h->grad + i, a, n);
		anni_count_launch();
		if (cudaGetLastError() != cudaSuccess)
			return ANNI_E_CUDA;
	}
	return ANNI_OK;
}

/* checks one entry and adds what the step writes of it to `w` */
static int check_tensor(const anni_mt_tensor *t, int state_dtype, std::vector<range> &w)
{
	const bool q8 = state_dtype == ANNI_DT_Q8;
	const int64_t blocks = (t->n + ANNI_MT_BLOCK - 1) / ANNI_MT_BLOCK;
	uintptr_t four;

	if (t->n < 0 || (t->flags & ~(uint32_t)(ANNI_SEG_WD | ANNI_SEG_TWIN_BF16)))
		return ANNI_E_ARG;
	if (t->n == 0)
		return ANNI_OK;
	if (!t->param || !t->m || !t->v || (q8 && (!t->m_scale || !t->v_scale))
	    || ((t->flags & ANNI_SEG_TWIN_BF16) && (!t->twin_bf16 || ((uintptr_t)t->twin_bf16 & 1))))
		return ANNI_E_ARG;
	four = (uintptr_t)t->param;
	four |= q8 ? (uintptr_t)t->m_scale | (uintptr_t)t->v_scale : (uintptr_t)t->m | (uintptr_t)t->v;
	if (four & 3)
		return ANNI_E_ARG;
	add_range(w, t->param, t->n * 4);
	add_range(w, t->m, t->n * (q8 ? 1 : 4));
	add_range(w, t->v, t->n * (q8 ? 1 : 4));
	if (q8) {
		add_range(w, t->m_scale, blocks * 4);
		add_range(w, t->v_scale, blocks * 4);
	}
	if (t->flags & ANNI_SEG_TWIN_BF16)
		add_range(w, t->twin_bf16, t->n * 2);
	return ANNI_OK;
}

static int create(const anni_mt_tensor *list, int n, anni_mtstep *h)
{
	std::vector<mt_desc> desc((size_t)n);
	std::vector<uint32_t> tile_of;
	std::vector<void *> grads((size_t)n);
	uint64_t tiles = 0;
	uint64_t block0 = 0;
	int sms = 0;
	int per_sm = 0;
	int rc;

	for (int i = 0; i < n; i++) {
		rc = check_tensor(&list[i], h->state_dtype, h->written);
		if (rc != ANNI_OK)
			return rc;
		h->counts.push_back(list[i].n);
		grads[i] = list[i].grad;
		desc[i] = { list[i].param, list[i].m, list[i].v, list[i].m_scale, list[i].v_scale,
		    (list[i].flags & ANNI_SEG_TWIN_BF16) ? (uint16_t *)list[i].twin_bf16 : NULL, list[i].n, block0,
		    (uint32_t)tiles, (list[i].flags & ANNI_SEG_WD) ? 1u : 0u };
		tiles += (uint64_t)(list[i].n + ANNI_MT_TILE - 1) / ANNI_MT_TILE;
		block0 += (uint64_t)(list[i].n + ANNI_MT_BLOCK - 1) / ANNI_MT_BLOCK;
		if (tiles > 0x7fffffffu)
			return ANNI_E_LIMIT;
	}
	std::sort(h->written.begin(), h->written.end());
	if (overlapping(h->written))
		return ANNI_E_ARG;
	rc = check_grads(h, grads.data());
	if (rc != ANNI_OK)
		return rc;
	tile_of.reserve((size_t)tiles);
	for (int i = 0; i < n; i++)
		tile_of.insert(tile_of.end(), (size_t)((list[i].n + ANNI_MT_TILE - 1) / ANNI_MT_TILE), (uint32_t)i);
	h->tiles = (uint32_t)tiles;
	if (cudaGetDevice(&h->device) != cudaSuccess
	    || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, h->device) != cudaSuccess
	    || cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, step_kernel(h->grad_dtype, h->state_dtype),
	    ANNI_THREADS, 0) != cudaSuccess || sms < 1 || per_sm < 1
	    || cudaMalloc((void **)&h->ctl, sizeof(anni_control)) != cudaSuccess
	    || cudaMalloc((void **)&h->desc, (size_t)n * sizeof(mt_desc)) != cudaSuccess
	    || cudaMalloc((void **)&h->grad, (size_t)n * sizeof(void *)) != cudaSuccess
	    || cudaMalloc((void **)&h->tile_of, ((size_t)tiles + 1) * sizeof(uint32_t)) != cudaSuccess
	    || cudaMemset(h->ctl, 0, sizeof(anni_control)) != cudaSuccess
	    || cudaMemcpy(h->desc, desc.data(), (size_t)n * sizeof(mt_desc), cudaMemcpyHostToDevice) != cudaSuccess
	    || cudaMemcpy(h->grad, grads.data(), (size_t)n * sizeof(void *), cudaMemcpyHostToDevice) != cudaSuccess
	    || cudaMemcpy(h->tile_of, tile_of.data(), (size_t)tiles * sizeof(uint32_t), cudaMemcpyHostToDevice)
	    != cudaSuccess) {
		(void)cudaGetLastError();
		return ANNI_E_CUDA;
	}
	h->blocks = std::min(sms * per_sm, ANNI_MAX_BLOCKS / sms * sms);
	h->blocks = (int)std::max((uint64_t)1, std::min((uint64_t)h->blocks, tiles));
	return ANNI_OK;
}

extern "C" int anni_mtstep_create(const anni_mt_tensor *list, int n_tensors, int grad_dtype, int state_dtype,
	anni_mtstep **out)
{
	anni_mtstep *h = NULL;
	int rc;

	if (!out)
		return ANNI_E_ARG;
	*out = NULL;
	if (!list || n_tensors < 1 || (grad_dtype != ANNI_DT_F32 && grad_dtype != ANNI_DT_BF16)
	    || (state_dtype != ANNI_DT_F32 && state_dtype != ANNI_DT_Q8))
		return ANNI_E_ARG;
	try {		/* the tables below are std::vectors: no exception may leave a C entry */
		h = new anni_mtstep();
		h->grad_dtype = grad_dtype;
		h->state_dtype = state_dtype;
		h->n_tensors = n_tensors;
		rc = create(list, n_tensors, h);
	} catch (...) {
		rc = ANNI_E_NOMEM;
	}
	if (rc != ANNI_OK) {
		anni_mtstep_destroy(h);
		return rc;
	}
	*out = h;
	return ANNI_OK;
}

extern "C" void anni_mtstep_destroy(anni_mtstep *h)
{
	if (!h)
		return;
	if (h->ctl || h->desc || h->grad || h->tile_of) {
		on_device dev(h->device);

		cudaFree(h->ctl);
		cudaFree(h->desc);
		cudaFree(h->grad);
		cudaFree(h->tile_of);
	}
	delete h;
}

extern "C" int anni_mtstep_set_grads(anni_mtstep *h, void *const *grads, void *stream)
{
	int rc;

	if (!h || !grads)
		return ANNI_E_ARG;
	try {
		rc = check_grads(h, grads);
	} catch (...) {
		rc = ANNI_E_NOMEM;
	}
	if (rc != ANNI_OK)
		return rc;
	on_device dev(h->device);

	return dev.ok ? send_grads(h, grads, (cudaStream_t)stream) : ANNI_E_CUDA;
}

extern "C" int anni_mtstep_step(anni_mtstep *h, const anni_optstep_hyper *hp, uint64_t seed, void *stream)
{
	const int known = ANNI_STEP_CHECK_FINITE | ANNI_STEP_ZERO_GRAD | ANNI_STEP_STOCHASTIC;
	mt_launch a;
	void *args[] = { &a };
	int rc;

	if (!h || !hp || (hp->flags & ~known)
	    || ((hp->flags & ANNI_STEP_STOCHASTIC) && h->state_dtype != ANNI_DT_Q8))
		return ANNI_E_ARG;
	memset(&a, 0, sizeof(a));
	rc = anni_fill_hyper(&a.la, hp);
	if (rc != ANNI_OK)
		return rc;
	a.la.ctl = h->ctl;
	a.desc = h->desc;
	a.grad = h->grad;
	a.tile_of = h->tile_of;
	a.tiles = h->tiles;
	a.seed = seed;
	on_device dev(h->device);

	if (!dev.ok)
		return ANNI_E_CUDA;
	{
		const int slot = anni_op_begin(ANNI_OP_ADAM, stream);

		rc = cudaLaunchCooperativeKernel(step_kernel(h->grad_dtype, h->state_dtype), dim3(h->blocks),
		    dim3(ANNI_THREADS), args, 0, (cudaStream_t)stream) == cudaSuccess ? ANNI_OK : ANNI_E_CUDA;
		anni_op_end(slot, stream);
	}
	if (rc == ANNI_OK)
		anni_count_launch();
	else
		(void)cudaGetLastError();
	return rc;
}

extern "C" int anni_mtstep_status_read(anni_mtstep *h, anni_optstep_status *out, void *stream)
{
	anni_control head;	/* only the scalars in front of partials[] are copied */
	const size_t nb = offsetof(anni_control, partials);

	if (!h || !out)
		return ANNI_E_ARG;
	on_device dev(h->device);

	if (!dev.ok || cudaStreamSynchronize((cudaStream_t)stream) != cudaSuccess
	    || cudaMemcpy(&head, h->ctl, nb, cudaMemcpyDeviceToHost) != cudaSuccess)
		return ANNI_E_CUDA;
	memset(out, 0, sizeof(*out));
	out->sumsq = head.reduce[0];
	out->norm = head.norm;
	out->eff_scale = head.eff_scale;
	out->skipped = head.skipped;
	out->error = head.error;
	out->steps_done = head.steps_done;
	if (head.error != 0) {
		/* a bounded wait gave up: clear the counters so the handle can be used again */
		head.error = 0;
		head.bar_count = 0;
		head.done_ticket = 0;
		if (cudaMemcpy(h->ctl, &head, nb, cudaMemcpyHostToDevice) != cudaSuccess)
			return ANNI_E_CUDA;
	}
	return ANNI_OK;
}
