/*
** AdamW over a list of tensors (include/anni_mtstep.h): one cooperative launch per step.
**
** Every tensor is cut into whole tiles of ANNI_MT_TILE elements, which a table lists with their tensors, and
** what is left of it, which a second table lists: two loops, the first without a thought for ends.  A block
** takes a tile at a time, each of its eight warps a run of ANNI_MT_BLOCK = 256 elements -- the run that
** shares a scale in the 8-bit form, so that the two block maxima are reductions inside a warp.  The step is
** bound by HBM: 28 bytes per element with 32-bit moments, bf16 gradients and twins, 16 with 8-bit moments.
** 184.7 M elements, with the norm: 0.95 ms (0.83 of the copy rate for those bytes) and 0.60 ms (0.75); 98.5 M,
** fp32 gradients, stochastic, no norm: 0.32 ms (0.76).
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

#define ANNI_MT_TILE		(ANNI_THREADS / 32 * ANNI_MT_BLOCK)	/* elements a block takes at once */
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
	uint32_t	tile0;		/* whole tiles in the tensors before this one */
	uint32_t	wd;
};

static_assert(sizeof(mt_desc) % 8 == 0, "mt_held keeps the gradient's address behind it");

struct mt_launch {
	anni_launch	la;		/* hyper-parameters, flags, control block */
	const mt_desc	*desc;
	void *const	*grad;
	const uint32_t	*tile_of;	/* tensor of each whole tile */
	const uint32_t	*rest_of;	/* tensors that do not end with a whole tile */
	uint32_t	tiles;
	uint32_t	rests;
	uint64_t	seed;
	float		b1;		/* beta1, 1 - beta1, beta2, 1 - beta2 for the 8-bit form */
	float		omb1;
	float		b2;
	float		omb2;
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
** x >= 0 to KEPT bits of mantissa, up with the probability of the part cut off: 16 random bits are added to
** the top of the bits that go, and the carry decides.  Below LEAST, the smallest normal number of the
** 8-bit type, its numbers are equally spaced; adding LEAST puts x into the binade with that spacing.
*/
template <int KEPT>
__device__ __forceinline__ float stochastic(float x, uint32_t r16, float least)
{
	const int cut = 23 - KEPT;
	const float add = x < least ? least : 0.0f;
	const uint32_t bits = __float_as_uint(__fadd_rn(x, add)) + (r16 << (cut - 16));

	return __fsub_rn(__uint_as_float(bits >> cut << cut), add);
}

/* two floats in one instruction each, every result rounded on its own */
typedef unsigned long long f32x2;

__device__ __forceinline__ f32x2 pair(float lo, float hi)
{
	f32x2 r;

	asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
	return r;
}

__device__ __forceinline__ void unpair(f32x2 x, float &lo, float &hi)
{
	asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x));
}

__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b)
{
	f32x2 r;

	asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
	return r;
}

/*
** Sums of products that are to be rounded on their own: two plain additions.  (The assembler contracts a packed
** product and a packed sum into one fused operation, whatever rounding they name: checked on a million pairs.)
*/
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b)
{
	float a0;
	float a1;
	float b0;
	float b1;

	unpair(a, a0, a1);
	unpair(b, b0, b1);
	return pair(__fadd_rn(a0, b0), __fadd_rn(a1, b1));
}

__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c)
{
	f32x2 r;

	asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
	return r;
}

/*
** Two elements of the 8-bit form.  Moments in float (their stored form has three and two bits of mantissa),
** every product and sum rounded on its own, so that a float restatement of the formula lands on the same codes;
** then the parameter update of adam_apply, operation for operation.
*/
__device__ __forceinline__ void adam_q8(const mt_launch &a, float coef, float lrwd, float g0, float g1, float &p0,
	float &p1, f32x2 &m, f32x2 &v)
{
	const f32x2 g = mul2(pair(g0, g1), pair(coef, coef));
	f32x2 p = pair(p0, p1);
	float s0;
	float s1;
	float d0;
	float d1;

	m = add2(mul2(pair(a.b1, a.b1), m), mul2(pair(a.omb1, a.omb1), g));
	v = add2(mul2(pair(a.b2, a.b2), v), mul2(mul2(pair(a.omb2, a.omb2), g), g));
	unpair(mul2(v, pair(a.la.ibc2_s24, a.la.ibc2_s24)), s0, s1);
	unpair(fma2(pair(sqrt_approx_ftz(s0), sqrt_approx_ftz(s1)), pair(268435456.0f, 268435456.0f),
	    pair(a.la.eps_s40, a.la.eps_s40)), d0, d1);
	p = fma2(mul2(mul2(pair(a.la.lrbc1_s40, a.la.lrbc1_s40), m), pair(rcp_approx_ftz(d0), rcp_approx_ftz(d1))),
	    pair(-1.0f, -1.0f), p);
	p = fma2(pair(-lrwd, -lrwd), p, p);
	unpair(p, p0, p1);
}

/* scale of a block from its largest value (as bits, >= 0) and the multiplier that undoes it; a NaN stays one */
__device__ __forceinline__ void q8_scale(uint32_t amax_bits, float top, float &scale, float &inv)
{
	const float amax = __uint_as_float(amax_bits);
	const bool none = amax < 7.8886090522101181e-31f;	/* 2^-100 */

	scale = none ? 0.0f : __fmul_rn(amax, 1.0f / top);
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
** What is coded for element i of a block, from its new moments over their scales x and y: rounded by chance if
** asked for, and y at least the smallest number unless v is zero (the conversions round to nearest).
*/
__device__ __forceinline__ void q8_round(bool random, uint32_t key, uint32_t i, float v, float vi, float &x, float &y)
{
	if (random) {
		const uint32_t r = mix32(key + i * 0x9e3779b9u);

		x = copysignf(stochastic<3>(fabsf(x), r & 0xffffu, 0.015625f), x);	/* 2^-6 */
		y = stochastic<2>(y, r >> 16, 6.103515625e-5f);		/* 2^-14 */
	}
	if (v > 0.0f && vi > 0.0f)
		y = fmaxf(y, 1.52587890625e-5f);	/* 2^-16 */
}

/* ---- one warp's run of at most 256 elements -------------------------------------- */

/*
** Tensors on addresses that only their type allows: element-wise, lane l on elements l, l + 32, ... of the
** run, so that plain accesses coalesce.
*/
template <typename GradT, bool Q8>
__device__ __forceinline__ void run_scalar(const mt_launch &a, const mt_desc &d, void *grad, int64_t e0, int len,
	double coef)
{
	const int lane = threadIdx.x & 31;
	const float lrwd = d.wd ? a.la.lrwd : 0.0f;
	const int64_t blk = e0 / ANNI_MT_BLOCK;
	const float old_ms = Q8 ? d.ms[blk] : 0.0f;
	const float old_vs = Q8 ? d.vs[blk] : 0.0f;
	float m[8];
	float v[8];
	uint32_t am = 0;
	uint32_t av = 0;

#pragma unroll
	for (int j = 0; j < 8; j++) {
		const int64_t e = e0 + j * 32 + lane;

		m[j] = v[j] = 0.0f;
		if (j * 32 + lane < len) {
			float p = d.p[e];
			const float g = io8<GradT>::load1(grad, e);

			if (Q8) {
				f32x2 m2 = pair(__fmul_rn(e4m3_to_float(static_cast<const uint8_t *>(d.m)[e]), old_ms), 0.0f);
				f32x2 v2 = pair(__fmul_rn(e5m2_to_float(static_cast<const uint8_t *>(d.v)[e]), old_vs), 0.0f);
				float none = 0.0f;

				adam_q8(a, (float)coef, lrwd, g, 0.0f, p, none, m2, v2);
				unpair(m2, m[j], none);
				unpair(v2, v[j], none);
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
			if (a.la.flags & ANNI_STEP_ZERO_GRAD)
				io8<GradT>::store1(grad, e, 0.0f);
		}
	}
	if (Q8) {
		float ms;
		float vs;
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
			float x = __fmul_rn(m[j], mi);
			float y = __fmul_rn(v[j], vi);

			if (i >= len)
				continue;
			q8_round(a.la.flags & ANNI_STEP_STOCHASTIC, key, (uint32_t)i, v[j], vi, x, y);
			static_cast<uint8_t *>(d.m)[e0 + i] = (uint8_t)to_e4m3(x);
			static_cast<uint8_t *>(d.v)[e0 + i] = (uint8_t)to_e5m2(y);
		}
	}
}

/*
** The same on elements e .. e + 3 of which the first `left` exist (ALL: four do); what does not exist reads as
** zero.  Only the last lane with elements of a tensor takes the element-wise road.
*/
template <typename T, bool ALL>
__device__ __forceinline__ f32x4 load_some(const void *base, uint64_t e, int left)
{
	f32x4 r;

	if (ALL || left >= 4)
		return io4<T>::load(base, e);
#pragma unroll
	for (int j = 0; j < 4; j++)
		r.x[j] = j < left ? io8<T>::load1(base, e + j) : 0.0f;
	return r;
}

template <typename T, bool ALL>
__device__ __forceinline__ void store_some(void *base, uint64_t e, const f32x4 &r, int left)
{
	if (ALL || left >= 4) {
		io4<T>::store(base, e, r);
		return;
	}
#pragma unroll
	for (int j = 0; j < 4; j++)
		if (j < left)
			io8<T>::store1(base, e + j, r.x[j]);
}

/* gradients: `vec` says whether their address allows the vector accesses */
template <typename T, bool ALL>
__device__ __forceinline__ f32x4 load_grad(const void *base, uint64_t e, int left, bool vec)
{
	f32x4 r;

	if (vec)
		return load_some<T, ALL>(base, e, left);
#pragma unroll
	for (int j = 0; j < 4; j++)
		r.x[j] = ALL || j < left ? io8<T>::load1(base, e + j) : 0.0f;
	return r;
}

template <typename T, bool ALL>
__device__ __forceinline__ void zero_grad(void *base, uint64_t e, int left, bool vec)
{
	if (vec) {
		store_some<T, ALL>(base, e, f32x4{}, left);
		return;
	}
#pragma unroll
	for (int j = 0; j < 4; j++)
		if (ALL || j < left)
			io8<T>::store1(base, e + j, 0.0f);
}

template <bool ALL>
__device__ __forceinline__ uint32_t load_codes(const void *base, uint64_t e, int left)
{
	const uint8_t *p = static_cast<const uint8_t *>(base) + e;
	uint32_t q = 0;

	if (ALL || left >= 4)
		return __ldcs(reinterpret_cast<const uint32_t *>(p));
#pragma unroll
	for (int j = 0; j < 4; j++)
		if (j < left)
			q |= (uint32_t)p[j] << (8 * j);
	return q;
}

template <bool ALL>
__device__ __forceinline__ void store_codes(void *base, uint64_t e, uint32_t q, int left)
{
	uint8_t *p = static_cast<uint8_t *>(base) + e;

	if (ALL || left >= 4) {
		__stcs(reinterpret_cast<uint32_t *>(p), q);
		return;
	}
#pragma unroll
	for (int j = 0; j < 4; j++)
		if (j < left)
			p[j] = (uint8_t)(q >> (8 * j));
}

/*
** A run of len elements on aligned addresses: lane l holds elements 4 l .. 4 l + 3 of each half, so every access of the
** warp is one contiguous piece (512 bytes of fp32, 128 of codes).
*/
template <typename GradT, bool ALL>
__device__ __forceinline__ void run_vec_f32(const mt_launch &a, const mt_desc &d, void *grad, int64_t e0, int len,
	double coef)
{
	const float lrwd = d.wd ? a.la.lrwd : 0.0f;
	float *const pp = d.p;		/* copies: the compiler cannot know that the stores leave d alone */
	void *const mp = d.m;
	void *const vp = d.v;
	uint16_t *const tp = d.twin;
	const bool gvec = ((uintptr_t)grad & 15) == 0;

#pragma unroll 1
	for (int k = 0; k < 2; k++) {
		const int i = 128 * k + (threadIdx.x & 31) * 4;
		const int left = len - i;
		const uint64_t e = (uint64_t)e0 + i;

		if (!ALL && left <= 0)
			break;
		const f32x4 g = load_grad<GradT, ALL>(grad, e, left, gvec);
		f32x4 p = load_some<float, ALL>(pp, e, left);
		f32x4 m = load_some<float, ALL>(mp, e, left);
		f32x4 v = load_some<float, ALL>(vp, e, left);

#pragma unroll
		for (int j = 0; j < 4; j++)
			adam_elem<false>(a.la, coef, lrwd, g.x[j], p.x[j], m.x[j], v.x[j]);
		store_some<float, ALL>(pp, e, p, left);
		store_some<float, ALL>(mp, e, m, left);
		store_some<float, ALL>(vp, e, v, left);
		if (tp)
			store_some<__nv_bfloat16, ALL>(tp, e, p, left);
		if (a.la.flags & ANNI_STEP_ZERO_GRAD)
			zero_grad<GradT, ALL>(grad, e, left, gvec);
	}
}

template <__nv_fp8_interpretation_t KIND>
__device__ __forceinline__ f32x2 decode2(uint32_t q, float scale)
{
	const float2 x = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)q, KIND)));

	return mul2(pair(x.x, x.y), pair(scale, scale));
}

template <__nv_fp8_interpretation_t KIND>
__device__ __forceinline__ uint32_t encode2(float lo, float hi)
{
	return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, KIND);
}

/*
** WHOLE: the block's eight warps are on the eight runs of a whole tile, block-uniformly; their new scales are
** then stored by one warp, two full 32-byte sectors, instead of by each warp, four bytes twice.  Single-lane
** stores into sectors that other warps load at the same time cost a quarter of the step (184.7 M elements
** without arithmetic: 574 us against 447 us without those stores; 474 us this way).
*/
template <typename GradT, bool WHOLE>
__device__ __forceinline__ void run_vec_q8(const mt_launch &a, const mt_desc &d, void *grad, int64_t e0,
	int len, float coef, float (*slot)[ANNI_THREADS / 32])
{
	const int lane = threadIdx.x & 31;
	const float lrwd = d.wd ? a.la.lrwd : 0.0f;
	const int64_t blk = e0 / ANNI_MT_BLOCK;
	const uint64_t e = (uint64_t)e0 + lane * 4;
	const bool gvec = ((uintptr_t)grad & 15) == 0;
	const int left = len - lane * 4;	/* of this lane's four, and 128 more than of its second four */
	f32x4 g[2];
	f32x4 p[2];
	f32x2 m[4];
	f32x2 v[4];
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
		g[k] = load_grad<GradT, WHOLE>(grad, e + 128 * k, left - 128 * k, gvec);
		p[k] = load_some<float, WHOLE>(d.p, e + 128 * k, left - 128 * k);
		qm[k] = load_codes<WHOLE>(d.m, e + 128 * k, left - 128 * k);
		qv[k] = load_codes<WHOLE>(d.v, e + 128 * k, left - 128 * k);
	}
	ms = d.ms[blk];
	vs = d.vs[blk];
#pragma unroll
	for (int k = 0; k < 2; k++) {
#pragma unroll
		for (int j = 0; j < 2; j++) {
			f32x2 &mm = m[2 * k + j];
			f32x2 &vv = v[2 * k + j];
			float lo;
			float hi;

			mm = decode2<__NV_E4M3>((qm[k] >> (16 * j)) & 0xffffu, ms);
			vv = decode2<__NV_E5M2>((qv[k] >> (16 * j)) & 0xffffu, vs);
			adam_q8(a, coef, lrwd, g[k].x[2 * j], g[k].x[2 * j + 1], p[k].x[2 * j], p[k].x[2 * j + 1], mm, vv);
			unpair(mm, lo, hi);
			am = max(am, max(__float_as_uint(fabsf(lo)), __float_as_uint(fabsf(hi))));
			unpair(vv, lo, hi);
			av = max(av, max(__float_as_uint(lo), __float_as_uint(hi)));
		}
		store_some<float, WHOLE>(d.p, e + 128 * k, p[k], left - 128 * k);
		if (d.twin)
			store_some<__nv_bfloat16, WHOLE>(d.twin, e + 128 * k, p[k], left - 128 * k);
		if (a.la.flags & ANNI_STEP_ZERO_GRAD)
			zero_grad<GradT, WHOLE>(grad, e + 128 * k, left - 128 * k, gvec);
	}
	am = __reduce_max_sync(0xffffffffu, am);
	av = __reduce_max_sync(0xffffffffu, av);
	q8_scale(am, 448.0f, ms, mi);
	q8_scale(av, 57344.0f, vs, vi);
	if (WHOLE) {
		const int w = threadIdx.x >> 5;

		/* the caller alternates two slots: one barrier per tile keeps writers and the reader apart */
		if (lane == 0) {
			slot[0][w] = ms;
			slot[1][w] = vs;
		}
		__syncthreads();
		if (w == 0 && lane < 2 * (ANNI_THREADS / 32))
			(lane < ANNI_THREADS / 32 ? d.ms : d.vs)[blk + (lane & (ANNI_THREADS / 32 - 1))] =
			    slot[lane / (ANNI_THREADS / 32)][lane & (ANNI_THREADS / 32 - 1)];
	} else if (lane == 0) {
		d.ms[blk] = ms;
		d.vs[blk] = vs;
	}
	const bool random = a.la.flags & ANNI_STEP_STOCHASTIC;
	const uint32_t key = random ? block_key(a.seed, d.block0 + (uint64_t)blk) : 0;

#pragma unroll
	for (int k = 0; k < 2; k++) {
		uint32_t cm = 0;
		uint32_t cv = 0;

#pragma unroll
		for (int j = 0; j < 2; j++) {
			const uint32_t i = (uint32_t)(128 * k + lane * 4 + 2 * j);
			float x0;
			float x1;
			float y0;
			float y1;
			float v0;
			float v1;

			unpair(mul2(m[2 * k + j], pair(mi, mi)), x0, x1);
			unpair(mul2(v[2 * k + j], pair(vi, vi)), y0, y1);
			unpair(v[2 * k + j], v0, v1);
			q8_round(random, key, i, v0, vi, x0, y0);
			q8_round(random, key, i + 1, v1, vi, x1, y1);
			cm |= encode2<__NV_E4M3>(x0, x1) << (16 * j);
			cv |= encode2<__NV_E5M2>(y0, y1) << (16 * j);
		}
		store_codes<WHOLE>(d.m, e + 128 * k, cm, left - 128 * k);
		store_codes<WHOLE>(d.v, e + 128 * k, cv, left - 128 * k);
	}
}

/* the entry of a tensor in shared memory */
struct mt_held {
	mt_desc	d;
	void	*grad;
};

__device__ __forceinline__ void fetch(const mt_launch &a, uint32_t s, mt_held &to)
{
	const uint32_t i = threadIdx.x;
	const uint32_t words = sizeof(mt_desc) / 4;

	if (i < words + 2) {
		const uint32_t *from = i < words ? reinterpret_cast<const uint32_t *>(a.desc + s) + i
		    : reinterpret_cast<const uint32_t *>(a.grad + s) + (i - words);

		asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" :: "r"((uint32_t)__cvta_generic_to_shared(
		    reinterpret_cast<uint32_t *>(&to) + i)), "l"(from) : "memory");
	}
}

__device__ __forceinline__ void fetched(void)
{
	asm volatile("cp.async.wait_all;" ::: "memory");
	__syncthreads();
}

/*
** Blocks take the entries of a table round-robin, backwards: the whole grid works inside one small window of
** every buffer, and the gradients read last by the norm phase are the likeliest to sit in L2.  An entry's tensor is
** looked up one step ahead, what there is to know of it is loaded into shared memory while the entry before is
** worked on.  work(tensor, gradient, entry) is called with the block together.
*/
template <typename F>
__device__ __forceinline__ void walk(const mt_launch &a, const uint32_t *table, uint32_t entries, mt_held (&held)[2], F work)
{
	const uint32_t G = gridDim.x;
	uint32_t r = (entries + G - 1) / G;
	uint32_t s;		/* tensor of this entry */
	uint32_t next;		/* and of the next */
	int cur = 0;

	if (blockIdx.x >= entries)
		return;
	if ((r - 1) * G + blockIdx.x >= entries)
		r--;
	s = table[(r - 1) * G + blockIdx.x];
	next = r > 1 ? table[(r - 2) * G + blockIdx.x] : s;
	__syncthreads();
	fetch(a, s, held[0]);
	fetched();
	for (; r > 0; r--) {
		const uint32_t t = (r - 1) * G + blockIdx.x;
		const bool change = next != s;

		s = next;
		if (r > 2)
			next = table[t - 2 * G];
		if (change)
			fetch(a, s, held[cur ^ 1]);
		if (held[cur].grad)
			work(held[cur].d, held[cur].grad, t);
		if (change) {
			cur ^= 1;
			fetched();
		}
	}
}

/*
** ALIGNED: every address but the gradients' allows the vector accesses; otherwise everything goes element by
** element.  A gradient's address may change between two replays of a captured step, so it is looked at here.
*/
template <typename GradT, bool Q8, bool ALIGNED>
__device__ __forceinline__ void mt_update_phase(const mt_launch &a, const decision &dec)
{
	__shared__ float slots[2][2][ANNI_THREADS / 32];	/* new scales of m and v, two tiles */
	__shared__ mt_held held[2];				/* this entry's tensor and the next one */
	const int64_t mine = (threadIdx.x >> 5) * ANNI_MT_BLOCK;
	const float coef = (float)dec.coef;
	int odd = 0;

	walk(a, a.tile_of, a.tiles, held, [&](const mt_desc &d, void *grad, uint32_t t) {
		const int64_t e0 = (int64_t)(t - d.tile0) * ANNI_MT_TILE + mine;

		if (!ALIGNED)
			run_scalar<GradT, Q8>(a, d, grad, e0, ANNI_MT_BLOCK, dec.coef);
		else if (Q8) {
			run_vec_q8<GradT, true>(a, d, grad, e0, ANNI_MT_BLOCK, coef, slots[odd]);
			odd ^= 1;
		} else
			run_vec_f32<GradT, true>(a, d, grad, e0, ANNI_MT_BLOCK, dec.coef);
	});
	walk(a, a.rest_of, a.rests, held, [&](const mt_desc &d, void *grad, uint32_t) {
		const int64_t e0 = d.n / ANNI_MT_TILE * ANNI_MT_TILE + mine;
		const int len = (int)min((int64_t)ANNI_MT_BLOCK, d.n - e0);

		if (len <= 0)
			return;
		if (!ALIGNED)
			run_scalar<GradT, Q8>(a, d, grad, e0, len, dec.coef);
		else if (Q8)
			run_vec_q8<GradT, false>(a, d, grad, e0, len, coef, NULL);
		else
			run_vec_f32<GradT, false>(a, d, grad, e0, len, dec.coef);
	});
}

/* a skipped step that leaves the gradients zeroed */
template <typename GradT>
__device__ __forceinline__ void mt_zero_phase(const mt_launch &a)
{
	for (uint32_t t = blockIdx.x; t < a.tiles + a.rests; t += gridDim.x) {
		const uint32_t s = t < a.tiles ? a.tile_of[t] : a.rest_of[t - a.tiles];
		const int64_t n = a.desc[s].n;
		const int64_t e0 = t < a.tiles ? (int64_t)(t - a.desc[s].tile0) * ANNI_MT_TILE : n / ANNI_MT_TILE * ANNI_MT_TILE;

		if (a.grad[s])
			for (int64_t e = e0 + threadIdx.x; e < min(n, e0 + ANNI_MT_TILE); e += ANNI_THREADS)
				io8<GradT>::store1(a.grad[s], e, 0.0f);
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

	for (uint32_t t = (threadIdx.x >> 5) * gridDim.x + blockIdx.x; t < a.tiles + a.rests; t += step) {
		const bool whole = t < a.tiles;
		const uint32_t s = whole ? a.tile_of[t] : a.rest_of[t - a.tiles];
		const void *grad = a.grad[s];
		const int64_t n = a.desc[s].n;
		const int64_t lo = whole ? (int64_t)(t - a.desc[s].tile0) * ANNI_MT_TILE : n / ANNI_MT_TILE * ANNI_MT_TILE;
		const int len = whole ? ANNI_MT_TILE : (int)(n - lo);
		const bool vec = ((uintptr_t)grad & 15) == 0;
		int i = 0;

		if (!grad)
			continue;
		if (vec)
			for (; i + 256 <= len; i += 1024) {
				f32x8 g[4];

#pragma unroll
				for (int k = 0; k < 4; k++)
					if (i + 256 * k + 256 <= len)
						g[k] = io8<GradT>::load_keep(grad, (uint64_t)lo + i + 256 * k + lane * 8);
#pragma unroll
				for (int k = 0; k < 4; k++)
					if (i + 256 * k + 256 <= len)
						norm_accumulate<GradT>(g[k], acc0, acc1);
			}
		/* what is left of the last 256, or everything on other addresses */
		for (i = vec ? len & ~255 : 0; i < len; i += 256) {
			float g[8];

#pragma unroll
			for (int k = 0; k < 8; k++)
				g[k] = i + 32 * k + lane < len ? io8<GradT>::load1(grad, (uint64_t)lo + i + 32 * k + lane) : 0.0f;
#pragma unroll
			for (int k = 0; k < 8; k++)
				acc0 = fma((double)g[k], (double)g[k], acc0);
		}
	}
	return acc0 + acc1;
}

/*
** Resident blocks per SM: as in the arena step, fewer where a thread has more bytes in flight (184.7 M elements,
** 32-bit moments: 3 blocks 0.935 ms, 4 blocks 0.987 ms; 8-bit moments: 4 blocks 0.581 ms, 3 blocks 0.602 ms).
*/
template <typename GradT, bool Q8, bool ALIGNED>
__global__ void __launch_bounds__(ANNI_THREADS, Q8 ? 4 : 3) mt_step_kernel(const mt_launch a)
{
	decision d;
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
	if (!d.skip)
		mt_update_phase<GradT, Q8, ALIGNED>(a, d);
	else if (a.la.flags & ANNI_STEP_ZERO_GRAD)
		mt_zero_phase<GradT>(a);
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

template <typename GradT, bool Q8>
const void *step_kernel_of(bool aligned)
{
	return aligned ? (const void *)mt_step_kernel<GradT, Q8, true> : (const void *)mt_step_kernel<GradT, Q8, false>;
}

const void *step_kernel(int grad_dtype, int state_dtype, bool aligned)
{
	if (grad_dtype == ANNI_DT_BF16)
		return state_dtype == ANNI_DT_Q8 ? step_kernel_of<__nv_bfloat16, true>(aligned)
		    : step_kernel_of<__nv_bfloat16, false>(aligned);
	return state_dtype == ANNI_DT_Q8 ? step_kernel_of<float, true>(aligned) : step_kernel_of<float, false>(aligned);
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
	uint32_t		rests;
	bool			aligned;	/* everything but the gradients, which come and go */
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
	std::vector<uint32_t> table;	/* tensors of the whole tiles, then of the rests */
	std::vector<uint32_t> rest;
	std::vector<void *> grads((size_t)n);
	uint64_t tiles = 0;
	uint64_t block0 = 0;
	int sms = 0;
	int per_sm = 0;
	int rc;

	h->aligned = true;
	for (int i = 0; i < n; i++) {
		rc = check_tensor(&list[i], h->state_dtype, h->written);
		if (rc != ANNI_OK)
			return rc;
		h->counts.push_back(list[i].n);
		grads[i] = list[i].grad;
		desc[i] = { list[i].param, list[i].m, list[i].v, list[i].m_scale, list[i].v_scale,
		    (list[i].flags & ANNI_SEG_TWIN_BF16) ? (uint16_t *)list[i].twin_bf16 : NULL, list[i].n, block0,
		    (uint32_t)tiles, (list[i].flags & ANNI_SEG_WD) ? 1u : 0u };
		if (list[i].n > 0 && !aligned(desc[i], h->state_dtype == ANNI_DT_Q8))
			h->aligned = false;
		tiles += (uint64_t)list[i].n / ANNI_MT_TILE;
		block0 += (uint64_t)(list[i].n + ANNI_MT_BLOCK - 1) / ANNI_MT_BLOCK;
		if (list[i].n % ANNI_MT_TILE)
			rest.push_back((uint32_t)i);
		if (tiles + rest.size() > 0x7fffffffu)
			return ANNI_E_LIMIT;
	}
	std::sort(h->written.begin(), h->written.end());
	if (overlapping(h->written))
		return ANNI_E_ARG;
	rc = check_grads(h, grads.data());
	if (rc != ANNI_OK)
		return rc;
	table.reserve((size_t)tiles + rest.size() + 1);
	for (int i = 0; i < n; i++)
		table.insert(table.end(), (size_t)(list[i].n / ANNI_MT_TILE), (uint32_t)i);
	table.insert(table.end(), rest.begin(), rest.end());
	h->tiles = (uint32_t)tiles;
	h->rests = (uint32_t)rest.size();
	if (cudaGetDevice(&h->device) != cudaSuccess
	    || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, h->device) != cudaSuccess || sms < 1
	    || cudaMalloc((void **)&h->ctl, sizeof(anni_control)) != cudaSuccess
	    || cudaMalloc((void **)&h->desc, (size_t)n * sizeof(mt_desc)) != cudaSuccess
	    || cudaMalloc((void **)&h->grad, (size_t)n * sizeof(void *)) != cudaSuccess
	    || cudaMalloc((void **)&h->tile_of, (table.size() + 1) * sizeof(uint32_t)) != cudaSuccess
	    || cudaMemset(h->ctl, 0, sizeof(anni_control)) != cudaSuccess
	    || cudaMemcpy(h->desc, desc.data(), (size_t)n * sizeof(mt_desc), cudaMemcpyHostToDevice) != cudaSuccess
	    || cudaMemcpy(h->grad, grads.data(), (size_t)n * sizeof(void *), cudaMemcpyHostToDevice) != cudaSuccess
	    || cudaMemcpy(h->tile_of, table.data(), table.size() * sizeof(uint32_t), cudaMemcpyHostToDevice) != cudaSuccess
	    || !anni_landed()) {
		(void)cudaGetLastError();
		return ANNI_E_CUDA;
	}
	if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, step_kernel(h->grad_dtype, h->state_dtype, h->aligned),
	    ANNI_THREADS, 0) != cudaSuccess || per_sm < 1) {
		(void)cudaGetLastError();
		return ANNI_E_CUDA;
	}
	h->blocks = std::min(sms * per_sm, ANNI_MAX_BLOCKS / sms * sms);
	h->blocks = (int)std::max((uint64_t)1, std::min((uint64_t)h->blocks, tiles + rest.size()));
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
	a.rest_of = h->tile_of + h->tiles;
	a.tiles = h->tiles;
	a.rests = h->rests;
	a.seed = seed;
	a.b1 = (float)a.la.b1;
	a.omb1 = (float)a.la.omb1;
	a.b2 = (float)a.la.b2;
	a.omb2 = (float)a.la.omb2;
	on_device dev(h->device);

	if (!dev.ok)
		return ANNI_E_CUDA;
	{
		const int slot = anni_op_begin(ANNI_OP_ADAM, stream);


		rc = cudaLaunchCooperativeKernel(step_kernel(h->grad_dtype, h->state_dtype, h->aligned), dim3(h->blocks),
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
		if (cudaMemcpy(h->ctl, &head, nb, cudaMemcpyHostToDevice) != cudaSuccess || !anni_landed())
			return ANNI_E_CUDA;
	}
	return ANNI_OK;
}
