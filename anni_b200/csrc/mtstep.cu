/*
** AdamW over a list of tensors (include/anni_mtstep.h): one cooperative launch per step.
**
** The list is cut into tiles of ANNI_MT_TILE elements that do not cross tensors; a table says which
** tensor a tile belongs to.  A block takes a tile at a time, each of its eight warps runs of
** ANNI_MT_BLOCK = 256 elements -- the run that shares a scale in the 8-bit form, so that the two
** block maxima are reductions inside a warp.  The step is bound by HBM: 28 bytes per element with 32-bit
** moments, bf16 gradients and twins, 16 with 8-bit moments.
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

#define ANNI_MT_PASS		(ANNI_THREADS / 32 * ANNI_MT_BLOCK)	/* elements a block takes at once */
#define ANNI_MT_TILE		(2 * ANNI_MT_PASS)
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
	uint16_t	wd;
	uint16_t	vec;		/* everything but the gradient on the alignment of the vector accesses */
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

/*
** Moments in float (their stored form has three and two bits of mantissa), every product and sum rounded on its
** own, so that a float restatement of the formula lands on the same codes; then the shared parameter update.
*/
__device__ __forceinline__ void adam_q8(const anni_launch &a, const q8_hyper &h, float lrwd, float gf, float &p,
	float &m, float &v)
{
	const float g = __fmul_rn(gf, h.coef);

	m = __fadd_rn(__fmul_rn(h.b1, m), __fmul_rn(h.omb1, g));
	v = __fadd_rn(__fmul_rn(h.b2, v), __fmul_rn(__fmul_rn(h.omb2, g), g));
	adam_apply(a, lrwd, p, m, v);
}

/* scale of a block from its largest value (as bits, >= 0) and the multiplier that undoes it; a NaN stays one */
__device__ __forceinline__ void q8_scale(uint32_t amax_bits, float top, float &scale, float &inv)
{
	const float amax = __uint_as_float(amax_bits);
	const bool none = amax < 7.8886090522101181e-31f;	/* 2^-100 */

	scale = none ? 0.0f : __fdiv_rn(amax, top);
	inv = none ? 0.0f : __fmul_rn(__frcp_rn(amax), top);
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

/*
** New moments of element i of a block over their scales, as the numbers to code: x by the multiplier, rounded by
** chance if asked for, and a v that is not zero at least the smallest number (its conversion rounds to nearest).
*/
__device__ __forceinline__ void q8_round(bool random, uint32_t key, uint32_t i, float mi, float vi, float &m, float &v)
{
	float x = __fmul_rn(m, mi);
	float y = __fmul_rn(v, vi);

	if (random) {
		const uint32_t r = mix32(key + i * 0x9e3779b9u);

		x = stochastic<3>(x, r & 0xffffu, 0.015625f);		/* 2^-6 */
		y = stochastic<2>(y, r >> 16, 6.103515625e-5f);		/* 2^-14 */
	}
	m = x;
	v = v > 0.0f && vi > 0.0f ? fmaxf(y, 1.52587890625e-5f) : y;	/* 2^-16 */
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

			if (i >= len)
				continue;
			q8_round(a.la.flags & ANNI_STEP_STOCHASTIC, key, (uint32_t)i, mi, vi, m[j], v[j]);
			static_cast<uint8_t *>(d.m)[e0 + i] = (uint8_t)to_e4m3(m[j]);
			static_cast<uint8_t *>(d.v)[e0 + i] = (uint8_t)to_e5m2(v[j]);
		}
	}
	if (a.la.flags & ANNI_STEP_ZERO_GRAD)
		for (int i = lane; i < len; i += 32)
			io8<GradT>::store1(grad, e0 + i, 0.0f);
}

/*
** A whole run on aligned addresses: lane l holds elements 4 l .. 4 l + 3 of each half, so every access of the
** warp is one contiguous piece (512 bytes of fp32, 128 of codes).
*/
template <typename GradT>
__device__ __forceinline__ void run_vec_f32(const mt_launch &a, const mt_desc &d, void *grad, int64_t e0, double coef)
{
	const float lrwd = d.wd ? a.la.lrwd : 0.0f;

#pragma unroll 1
	for (int k = 0; k < 2; k++) {
		const uint64_t e = (uint64_t)e0 + 128 * k + (threadIdx.x & 31) * 4;
		const f32x4 g = io4<GradT>::load(grad, e);
		f32x4 p = io4<float>::load(d.p, e);
		f32x4 m = io4<float>::load(d.m, e);
		f32x4 v = io4<float>::load(d.v, e);

#pragma unroll
		for (int j = 0; j < 4; j++)
			adam_elem<false>(a.la, coef, lrwd, g.x[j], p.x[j], m.x[j], v.x[j]);
		io4<float>::store(d.p, e, p);
		io4<float>::store(d.m, e, m);
		io4<float>::store(d.v, e, v);
		if (d.twin)
			io4<__nv_bfloat16>::store(d.twin, e, p);
		if (a.la.flags & ANNI_STEP_ZERO_GRAD)
			io4<GradT>::zero(grad, e);
	}
}

template <__nv_fp8_interpretation_t KIND>
__device__ __forceinline__ f32x4 decode4(uint32_t q, float scale)
{
	const float2 lo = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(q & 0xffffu), KIND)));
	const float2 hi = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(q >> 16), KIND)));
	f32x4 r;

	r.x[0] = __fmul_rn(lo.x, scale);
	r.x[1] = __fmul_rn(lo.y, scale);
	r.x[2] = __fmul_rn(hi.x, scale);
	r.x[3] = __fmul_rn(hi.y, scale);
	return r;
}

template <__nv_fp8_interpretation_t KIND>
__device__ __forceinline__ uint32_t encode4(const f32x4 &y)
{
	return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(y.x[0], y.x[1]), __NV_SATFINITE, KIND)
	    | ((uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(y.x[2], y.x[3]), __NV_SATFINITE, KIND) << 16);
}

template <typename GradT>
__device__ __forceinline__ void run_vec_q8(const mt_launch &a, const mt_desc &d, void *grad, int64_t e0,
	const q8_hyper &h)
{
	const int lane = threadIdx.x & 31;
	const float lrwd = d.wd ? a.la.lrwd : 0.0f;
	const int64_t blk = e0 / ANNI_MT_BLOCK;
	const uint64_t e = (uint64_t)e0 + lane * 4;
	f32x4 g[2];
	f32x4 p[2];
	f32x4 m[2];
	f32x4 v[2];
	uint32_t qm[2];
	uint32_t qv[2];
	float ms;
	float vs;
	float mi;
	float vi;
	uint32_t am = 0;
	uint32_t av = 0;

#pragma unroll
	for (int k = 0; k < 2; k++) {
		g[k] = io4<GradT>::load(grad, e + 128 * k);
		p[k] = io4<float>::load(d.p, e + 128 * k);
		qm[k] = __ldcs(reinterpret_cast<const uint32_t *>(static_cast<const uint8_t *>(d.m) + e + 128 * k));
		qv[k] = __ldcs(reinterpret_cast<const uint32_t *>(static_cast<const uint8_t *>(d.v) + e + 128 * k));
	}
	ms = d.ms[blk];
	vs = d.vs[blk];
#pragma unroll
	for (int k = 0; k < 2; k++) {
		m[k] = decode4<__NV_E4M3>(qm[k], ms);
		v[k] = decode4<__NV_E5M2>(qv[k], vs);
#pragma unroll
		for (int j = 0; j < 4; j++) {
			adam_q8(a.la, h, lrwd, g[k].x[j], p[k].x[j], m[k].x[j], v[k].x[j]);
			am = max(am, __float_as_uint(fabsf(m[k].x[j])));
			av = max(av, __float_as_uint(v[k].x[j]));
		}
		io4<float>::store(d.p, e + 128 * k, p[k]);
		if (d.twin)
			io4<__nv_bfloat16>::store(d.twin, e + 128 * k, p[k]);
		if (a.la.flags & ANNI_STEP_ZERO_GRAD)
			io4<GradT>::zero(grad, e + 128 * k);
	}
	am = __reduce_max_sync(0xffffffffu, am);
	av = __reduce_max_sync(0xffffffffu, av);
	q8_scale(am, 448.0f, ms, mi);
	q8_scale(av, 57344.0f, vs, vi);
	if (lane == 0) {
		d.ms[blk] = ms;
		d.vs[blk] = vs;
	}
	const bool random = a.la.flags & ANNI_STEP_STOCHASTIC;
	const uint32_t key = random ? block_key(a.seed, d.block0 + (uint64_t)blk) : 0;

#pragma unroll
	for (int k = 0; k < 2; k++) {
#pragma unroll
		for (int j = 0; j < 4; j++)
			q8_round(random, key, (uint32_t)(128 * k + lane * 4 + j), mi, vi, m[k].x[j], v[k].x[j]);
		__stcs(reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(d.m) + e + 128 * k), encode4<__NV_E4M3>(m[k]));
		__stcs(reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(d.v) + e + 128 * k), encode4<__NV_E5M2>(v[k]));
	}
}

template <typename GradT, bool Q8>
__device__ __forceinline__ void mt_update_phase(const mt_launch &a, const decision &dec, const q8_hyper &h)
{
	const int64_t warp0 = (threadIdx.x >> 5) * ANNI_MT_BLOCK;

	/* backwards: the gradients read last by the norm phase are the likeliest to sit in L2 */
	for (uint32_t r = (a.tiles + gridDim.x - 1) / gridDim.x; r > 0; r--) {
		const uint32_t t = (r - 1) * gridDim.x + blockIdx.x;

		if (t >= a.tiles)
			continue;
		const uint32_t s = a.tile_of[t];
		void *grad = a.grad[s];
		const mt_desc &d = a.desc[s];
		const int64_t n = d.n;
		const bool vec = d.vec && ((uintptr_t)grad & 15) == 0 && !dec.skip;
		int64_t e0 = (int64_t)(t - d.tile0) * ANNI_MT_TILE + warp0;

		if (!grad)
			continue;
#pragma unroll 1
		for (int k = 0; k < ANNI_MT_TILE / ANNI_MT_PASS && e0 < n; k++, e0 += ANNI_MT_PASS) {
			const int64_t left = n - e0;

			if (vec && left >= ANNI_MT_BLOCK) {
				if (Q8)
					run_vec_q8<GradT>(a, d, grad, e0, h);
				else
					run_vec_f32<GradT>(a, d, grad, e0, dec.coef);
			} else
				run_scalar<GradT, Q8>(a, d, grad, e0, left < ANNI_MT_BLOCK ? (int)left : ANNI_MT_BLOCK,
				    dec.coef, h, dec.skip);
		}
	}
}

/*
** Sum of squares: a warp takes a tile, so that each lane has several 16-byte loads in flight for one look
** at the tables.
*/
template <typename GradT>
__device__ __forceinline__ double mt_norm_phase(const mt_launch &a)
{
	const int lane = threadIdx.x & 31;
	const uint32_t step = gridDim.x * (ANNI_THREADS / 32);
	double acc0 = 0.0;
	double acc1 = 0.0;

	for (uint32_t t = (threadIdx.x >> 5) * gridDim.x + blockIdx.x; t < a.tiles; t += step) {
		const uint32_t s = a.tile_of[t];
		const void *grad = a.grad[s];
		const int64_t lo = (int64_t)(t - a.desc[s].tile0) * ANNI_MT_TILE;
		const int64_t left = a.desc[s].n - lo;
		const int len = left < ANNI_MT_TILE ? (int)left : ANNI_MT_TILE;
		int i = 0;

		if (!grad)
			continue;
		if (((uintptr_t)grad & 15) == 0)
			for (; i + 1024 <= len; i += 1024) {
				f32x8 g[4];

#pragma unroll
				for (int k = 0; k < 4; k++)
					g[k] = io8<GradT>::load_keep(grad, (uint64_t)lo + i + 256 * k + lane * 8);
#pragma unroll
				for (int k = 0; k < 4; k++)
					norm_accumulate<GradT>(g[k], acc0, acc1);
			}
		for (i += lane; i < len; i += 32) {
			const double g = (double)io8<GradT>::load1(grad, (uint64_t)lo + i);

			acc0 = fma(g, g, acc0);
		}
	}
	return acc0 + acc1;
}

template <typename GradT, bool Q8>
__global__ void __launch_bounds__(ANNI_THREADS, 4) mt_step_kernel(const mt_launch a)
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
		mt_update_phase<GradT, Q8>(a, d, h);
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

/* 16-byte accesses of fp32, 8-byte of twins, 4-byte of codes */
bool aligned(const mt_desc &d, bool q8)
{
	const uintptr_t mv = (uintptr_t)d.m | (uintptr_t)d.v;

	return (((uintptr_t)d.p | (q8 ? 0 : mv)) & 15) == 0 && (mv & 3) == 0 && ((uintptr_t)d.twin & 7) == 0;
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
		    (uint32_t)tiles, (uint16_t)((list[i].flags & ANNI_SEG_WD) ? 1 : 0), 0 };
		desc[i].vec = aligned(desc[i], h->state_dtype == ANNI_DT_Q8);
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
