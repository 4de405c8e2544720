/*
** Device code shared by the step kernels (optstep.cu, mtstep.cu): typed loads and stores, fixed-order
** sums, the bounded grid barrier, the clip / skip decision, AdamW on one element, and the block that
** closes a step.  Everything is in an anonymous namespace: each source file compiles its own copy.
*/
#ifndef ANNI_OPTSTEP_DEVICE_H__
#define ANNI_OPTSTEP_DEVICE_H__

#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include "optstep_internal.h"

namespace {

/* ---- small device helpers ------------------------------------------------ */

struct f32x8 {
	float	x[ANNI_VEC];
};

struct f32x4 {
	float	x[ANNI_UVEC];
};

__device__ __forceinline__ uint32_t ld_acquire_u32(const uint32_t *p)
{
	uint32_t v;

	asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
	return v;
}

/*
** The SFU's square root and reciprocal in their single-instruction forms.  These flush
** subnormal inputs and results to zero; the caller keeps its operands out of that range by
** scaling with powers of two (exact), which the forms without .ftz would do with extra
** instructions around the same SFU operation.
*/
__device__ __forceinline__ float sqrt_approx_ftz(float x)
{
	float r;

	asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
	return r;
}

__device__ __forceinline__ float rcp_approx_ftz(float x)
{
	float r;

	asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
	return r;
}

__device__ __forceinline__ f32x8 unpack_bf16x8(uint4 q)
{
	f32x8 r;

	r.x[0] = __uint_as_float(q.x << 16);
	r.x[1] = __uint_as_float(q.x & 0xffff0000u);
	r.x[2] = __uint_as_float(q.y << 16);
	r.x[3] = __uint_as_float(q.y & 0xffff0000u);
	r.x[4] = __uint_as_float(q.z << 16);
	r.x[5] = __uint_as_float(q.z & 0xffff0000u);
	r.x[6] = __uint_as_float(q.w << 16);
	r.x[7] = __uint_as_float(q.w & 0xffff0000u);
	return r;
}

__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi)
{
	__nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);	/* round to nearest even */

	return *reinterpret_cast<uint32_t *>(&h);
}

__device__ __forceinline__ uint4 pack_bf16x8(const f32x8 &r)
{
	uint4 q;

	q.x = pack_bf16x2(r.x[0], r.x[1]);
	q.y = pack_bf16x2(r.x[2], r.x[3]);
	q.z = pack_bf16x2(r.x[4], r.x[5]);
	q.w = pack_bf16x2(r.x[6], r.x[7]);
	return q;
}

/* eight consecutive elements starting at element index e of a typed buffer */
template <typename T> struct io8;

template <> struct io8<float> {
	static __device__ __forceinline__ f32x8 load(const void *base, uint64_t e)
	{
		const uint4 *p = reinterpret_cast<const uint4 *>(static_cast<const float *>(base) + e);
		uint4 a = __ldcs(p);
		uint4 b = __ldcs(p + 1);
		f32x8 r;

		r.x[0] = __uint_as_float(a.x);
		r.x[1] = __uint_as_float(a.y);
		r.x[2] = __uint_as_float(a.z);
		r.x[3] = __uint_as_float(a.w);
		r.x[4] = __uint_as_float(b.x);
		r.x[5] = __uint_as_float(b.y);
		r.x[6] = __uint_as_float(b.z);
		r.x[7] = __uint_as_float(b.w);
		return r;
	}
	/* same, default cache policy: the norm phase wants its last reads to stay in L2 */
	static __device__ __forceinline__ f32x8 load_keep(const void *base, uint64_t e)
	{
		const uint4 *p = reinterpret_cast<const uint4 *>(static_cast<const float *>(base) + e);
		uint4 a = p[0];
		uint4 b = p[1];
		f32x8 r;

		r.x[0] = __uint_as_float(a.x);
		r.x[1] = __uint_as_float(a.y);
		r.x[2] = __uint_as_float(a.z);
		r.x[3] = __uint_as_float(a.w);
		r.x[4] = __uint_as_float(b.x);
		r.x[5] = __uint_as_float(b.y);
		r.x[6] = __uint_as_float(b.z);
		r.x[7] = __uint_as_float(b.w);
		return r;
	}
	static __device__ __forceinline__ void store(void *base, uint64_t e, const f32x8 &r)
	{
		uint4 *p = reinterpret_cast<uint4 *>(static_cast<float *>(base) + e);

		__stcs(p, make_uint4(__float_as_uint(r.x[0]), __float_as_uint(r.x[1]),
		    __float_as_uint(r.x[2]), __float_as_uint(r.x[3])));
		__stcs(p + 1, make_uint4(__float_as_uint(r.x[4]), __float_as_uint(r.x[5]),
		    __float_as_uint(r.x[6]), __float_as_uint(r.x[7])));
	}
	static __device__ __forceinline__ void zero(void *base, uint64_t e)
	{
		uint4 *p = reinterpret_cast<uint4 *>(static_cast<float *>(base) + e);

		__stcs(p, make_uint4(0, 0, 0, 0));
		__stcs(p + 1, make_uint4(0, 0, 0, 0));
	}
	static __device__ __forceinline__ float load1(const void *base, uint64_t e)
	{
		return static_cast<const float *>(base)[e];
	}
	static __device__ __forceinline__ void store1(void *base, uint64_t e, float x)
	{
		static_cast<float *>(base)[e] = x;
	}
};

template <> struct io8<__nv_bfloat16> {
	static __device__ __forceinline__ f32x8 load(const void *base, uint64_t e)
	{
		return unpack_bf16x8(__ldcs(reinterpret_cast<const uint4 *>(
		    static_cast<const uint16_t *>(base) + e)));
	}
	static __device__ __forceinline__ f32x8 load_keep(const void *base, uint64_t e)
	{
		return unpack_bf16x8(*reinterpret_cast<const uint4 *>(
		    static_cast<const uint16_t *>(base) + e));
	}
	static __device__ __forceinline__ void store(void *base, uint64_t e, const f32x8 &r)
	{
		__stcs(reinterpret_cast<uint4 *>(static_cast<uint16_t *>(base) + e), pack_bf16x8(r));
	}
	static __device__ __forceinline__ void zero(void *base, uint64_t e)
	{
		__stcs(reinterpret_cast<uint4 *>(static_cast<uint16_t *>(base) + e),
		    make_uint4(0, 0, 0, 0));
	}
	static __device__ __forceinline__ float load1(const void *base, uint64_t e)
	{
		return __uint_as_float((uint32_t)static_cast<const uint16_t *>(base)[e] << 16);
	}
	static __device__ __forceinline__ void store1(void *base, uint64_t e, float x)
	{
		__nv_bfloat16 h = __float2bfloat16_rn(x);

		static_cast<uint16_t *>(base)[e] = *reinterpret_cast<uint16_t *>(&h);
	}
};

/* four consecutive elements starting at element index e: one 16-byte (fp32) or 8-byte (bf16) access */
template <typename T> struct io4;

template <> struct io4<float> {
	static __device__ __forceinline__ f32x4 load(const void *base, uint64_t e)
	{
		const uint4 a = __ldcs(reinterpret_cast<const uint4 *>(static_cast<const float *>(base) + e));
		f32x4 r;

		r.x[0] = __uint_as_float(a.x);
		r.x[1] = __uint_as_float(a.y);
		r.x[2] = __uint_as_float(a.z);
		r.x[3] = __uint_as_float(a.w);
		return r;
	}
	static __device__ __forceinline__ void store(void *base, uint64_t e, const f32x4 &r)
	{
		__stcs(reinterpret_cast<uint4 *>(static_cast<float *>(base) + e),
		    make_uint4(__float_as_uint(r.x[0]), __float_as_uint(r.x[1]), __float_as_uint(r.x[2]),
		    __float_as_uint(r.x[3])));
	}
	/* same, default cache policy: for lines that are read again soon and should wait in L2 */
	static __device__ __forceinline__ void store_keep(void *base, uint64_t e, const f32x4 &r)
	{
		*reinterpret_cast<uint4 *>(static_cast<float *>(base) + e) =
		    make_uint4(__float_as_uint(r.x[0]), __float_as_uint(r.x[1]), __float_as_uint(r.x[2]),
		    __float_as_uint(r.x[3]));
	}
	static __device__ __forceinline__ void zero(void *base, uint64_t e)
	{
		__stcs(reinterpret_cast<uint4 *>(static_cast<float *>(base) + e), make_uint4(0, 0, 0, 0));
	}
};

template <> struct io4<__nv_bfloat16> {
	static __device__ __forceinline__ f32x4 load(const void *base, uint64_t e)
	{
		const uint2 q = __ldcs(reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(base) + e));
		f32x4 r;

		r.x[0] = __uint_as_float(q.x << 16);
		r.x[1] = __uint_as_float(q.x & 0xffff0000u);
		r.x[2] = __uint_as_float(q.y << 16);
		r.x[3] = __uint_as_float(q.y & 0xffff0000u);
		return r;
	}
	static __device__ __forceinline__ void store(void *base, uint64_t e, const f32x4 &r)
	{
		__stcs(reinterpret_cast<uint2 *>(static_cast<uint16_t *>(base) + e),
		    make_uint2(pack_bf16x2(r.x[0], r.x[1]), pack_bf16x2(r.x[2], r.x[3])));
	}
	static __device__ __forceinline__ void zero(void *base, uint64_t e)
	{
		__stcs(reinterpret_cast<uint2 *>(static_cast<uint16_t *>(base) + e), make_uint2(0, 0));
	}
};

__device__ __forceinline__ double warp_sum(double v)
{
#pragma unroll
	for (int k = 16; k > 0; k >>= 1)
		v += __shfl_down_sync(0xffffffffu, v, k);
	return v;
}

/* Block sum in a fixed order; the result is valid in thread 0. */
__device__ __forceinline__ double block_sum(double v)
{
	__shared__ double s_w[ANNI_THREADS / 32];
	const int lane = threadIdx.x & 31;
	const int w = threadIdx.x >> 5;

	v = warp_sum(v);
	if (lane == 0)
		s_w[w] = v;
	__syncthreads();
	if (threadIdx.x == 0) {
		v = 0.0;
#pragma unroll
		for (int k = 0; k < ANNI_THREADS / 32; k++)
			v += s_w[k];
	}
	return v;
}

/*
** Device-wide barrier with a bounded wait.  All blocks of the grid are
** co-resident (cooperative launch), so the wait ends as soon as the slowest
** block arrives; the poll limit only matters if something is badly wrong, in
** which case the block records the error and the kernel returns without
** touching the parameters.  Returns false on timeout (uniform over the block).
*/
__device__ __forceinline__ bool grid_barrier(anni_control *ctl, uint32_t target,
	uint32_t max_polls = ANNI_WAIT_POLLS)
{
	__shared__ int s_ok;

	__syncthreads();
	if (threadIdx.x == 0) {
		uint32_t polls = 0;
		int ok = 1;

		__threadfence();
		atomicAdd(&ctl->bar_count, 1u);
		while (ld_acquire_u32(&ctl->bar_count) < target) {
			__nanosleep(32);
			if (++polls > max_polls) {
				ok = 0;
				atomicExch(&ctl->error, ANNI_E_BARRIER_TIMEOUT);
				break;
			}
		}
		__threadfence();
		s_ok = ok;
	}
	__syncthreads();
	return s_ok != 0;
}

/* Sum of the block partials in index order; every thread of the block gets it. */
__device__ __forceinline__ double sum_partials(const anni_control *ctl, int nparts)
{
	__shared__ double s_total;

	if (threadIdx.x < 32) {
		const volatile double *p = ctl->partials;
		double v = 0.0;

		for (int k = threadIdx.x; k < nparts; k += 32)
			v += p[k];
		v = warp_sum(v);
		if (threadIdx.x == 0)
			s_total = v;
	}
	__syncthreads();
	return s_total;
}

/* ---- phase A: sum of squares of this block's chunks ---------------------- */

template <typename GradT>
__device__ __forceinline__ void norm_accumulate(const f32x8 &g, double &acc0, double &acc1)
{
	/* squares and their sum in double: the skip decision and the clip factor then
	** agree with a double accumulation to the last bits */
#pragma unroll
	for (int k = 0; k < ANNI_VEC; k += 2) {
		const double g0 = (double)g.x[k];
		const double g1 = (double)g.x[k + 1];

		acc0 = fma(g0, g0, acc0);
		acc1 = fma(g1, g1, acc1);
	}
}

/* ---- the decision every block takes from the same bits --------------------- */

struct decision {
	double	coef;	/* multiplier of the raw gradient */
	double	norm;
	bool	skip;
};

__device__ __forceinline__ decision decide(const anni_launch &a, double ss, double nonfinite,
	double loss_scale)
{
	decision d;
	double gs = a.grad_scale;

	if ((a.flags & ANNI_STEP_DEV_LOSS_SCALE) && loss_scale > 0.0)
		gs = gs / loss_scale;
	d.coef = gs;
	d.norm = 0.0;
	d.skip = false;
	if (a.flags & ANNI_LAUNCH_NEED_NORM) {
		d.norm = sqrt(ss) * fabs(gs);
		if ((a.flags & ANNI_STEP_CHECK_FINITE) && (!isfinite(d.norm) || nonfinite > 0.0))
			d.skip = true;
		else if (a.clip > 0.0 && d.norm > a.clip)
			d.coef = gs * (a.clip / (d.norm + 1e-12));
	}
	return d;
}

/* ---- phase B: AdamW on one element ----------------------------------------- */

/* p -= lr * (m/bc1) / (sqrt(v/bc2) + eps), then p -= lr*wd*p, in float with the SFU's square root and reciprocal */
__device__ __forceinline__ void adam_apply(const anni_launch &a, float lrwd, float &p, float m, float v)
{
	/*
	** den = sqrt(v / bc2) + eps and upd = (lr / bc1 * m) / den, carried at other binary
	** scales: s = sqrt(2^24 v / bc2) = 2^12 sqrt(v / bc2), so no subnormal v is flushed;
	** den40 = 2^28 s + 2^40 eps = 2^40 den in one fused step (the same single rounding as
	** the plain sum), never subnormal unless it is zero; the factor 2^40 returns through lr.
	*/
	const float s = sqrt_approx_ftz(__fmul_rn(v, a.ibc2_s24));
	const float den40 = __fmaf_rn(s, 268435456.0f, a.eps_s40);
	const float upd = __fmul_rn(__fmul_rn(a.lrbc1_s40, m), rcp_approx_ftz(den40));

	p = __fsub_rn(p, upd);
	p = __fmaf_rn(-lrwd, p, p);
}

template <bool EXACT>
__device__ __forceinline__ void adam_elem(const anni_launch &a, double coef, float lrwd,
	float gf, float &p, float &m, float &v)
{
	/* moments: the reference's double expression, each product and the sum rounded on its own */
	const double g = __dmul_rn((double)gf, coef);
	const double md = __dadd_rn(__dmul_rn(a.b1, (double)m), __dmul_rn(a.omb1, g));
	const double vd = __dadd_rn(__dmul_rn(a.b2, (double)v), __dmul_rn(__dmul_rn(a.omb2, g), g));

	m = __double2float_rn(md);
	v = __double2float_rn(vd);
	/*
	** p -= lr * (m/bc1) / (sqrt(v/bc2) + eps), then p -= lr*wd*p on the stored
	** value.  The quotient uses the SFU square root and reciprocal (about one
	** ulp each): the update term carries a relative error of a few 1e-7, which
	** moves p by far less than one ulp unless p itself is of the size of the
	** update.  Every product is rounded on its own (no contraction).
	*/
	if (EXACT) {
		/*
		** The reference's double expression lr*(m/bc1)/(sqrt(v/bc2)+eps) from the
		** rounded float moments: reciprocal square root and reciprocal start from
		** the SFU's 64-bit seeds (about 20 bits) and take one Newton step each
		** (relative error ~1e-12), so p - u rounds to the reference's float in
		** all but about one element in ten million.
		*/
		const double vr = (double)v;
		const double x = vr * a.ibc2d;
		const double hx = vr * (0.5 * a.ibc2d);
		double y;
		double q;

		asm("rsqrt.approx.ftz.f64 %0, %1;" : "=d"(y) : "d"(x));
		y = y * fma(-hx * y, y, 1.5);
		const double dn = (v > 0.0f ? x * y : 0.0) + a.epsd;

		asm("rcp.approx.ftz.f64 %0, %1;" : "=d"(q) : "d"(dn));
		q = fma(fma(-dn, q, 1.0), q, q);
		const float p1 = __double2float_rn((double)p - (a.lrbc1d * (double)m) * q);

		/* decay on the stored float, in double as the reference does, rounded once */
		p = lrwd != 0.0f ? __double2float_rn(fma(-a.lrwdd, (double)p1, (double)p1)) : p1;
		return;
	}
	adam_apply(a, lrwd, p, m, v);
}

/* ---- epilogue: the last block to finish closes the step --------------------- */

__device__ __forceinline__ void step_epilogue(anni_control *ctl, bool skipped)
{
	__syncthreads();
	if (threadIdx.x != 0)
		return;
	__threadfence();
	if (atomicAdd(&ctl->done_ticket, 1u) != gridDim.x - 1)
		return;
	/* every block has read the loss scale and passed every barrier by now */
	if (ctl->loss_scale > 0.0) {
		if (skipped) {
			double s = ctl->loss_scale * ctl->ls_backoff;

			ctl->loss_scale = s < ctl->ls_min ? ctl->ls_min : s;
			ctl->good_steps = 0;
		} else if (++ctl->good_steps >= ctl->ls_interval && ctl->ls_interval > 0) {
			double s = ctl->loss_scale * ctl->ls_growth;

			ctl->loss_scale = s > ctl->ls_max ? ctl->ls_max : s;
			ctl->good_steps = 0;
		}
	}
	ctl->steps_done++;
	ctl->bar_count = 0;
	ctl->done_ticket = 0;
	__threadfence();
}

}	/* namespace */

#endif
