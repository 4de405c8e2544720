/*
** Loss and gradients of a language model's head (include/anni_head.h).
**
** Four matrix products on the tensor cores, in three persistent kernels:
**   loss    logits of a tile of rows and vocabulary; its epilogue keeps the maximum and the sum of exponentials
**           of each row and drops the logits.  A small kernel joins the tiles of a row.
**   delta   the same logits again for one piece of the vocabulary; softmax - one-hot from lse, stored as bf16
**           (three terms of it for fp32 gradients), and its column sums for dbias
**   grad    dx = delta W^T of the piece, added to an fp32 sum over the pieces, and dw = x^T delta of the piece, stored
**           or added to the gradient; together, so that the tiles of one fill the rounds that the other leaves open
** Bound by the tensor cores: 2 T D V operations each (the logits twice, since they are not kept).  4096 rows of 1536
** against 100,000 entries: loss 838 us (1.50 PFLOP/s, 0.89 of the rate of a library product), delta 902, dx and dw 1.7 ms
** one by one; back to back at the power limit 4.1 ms in all, where four library products would take 3.6 ms.
**
** Two blocks (a cluster on two neighbouring SMs) work on a 256 x 256 tile: each keeps 128 rows of the result
** and loads its 128 rows of the one operand and 128 of the other by TMA into a ring of HEAD_STAGES stages; one
** thread of the first block issues tcgen05.mma for both SMs, which read half of the second operand from each
** other's shared memory, into one of two accumulators in tensor memory, while eight warps of each block empty
** the other one.  An operand whose rows run along the summed dimension ("K-major") is loaded as one box
** of 64 k x rows, one whose rows run along the result ("MN-major") as boxes of 64 mn x 64 k, so nothing is
** transposed in memory.  Lengths that are no multiple of a tile end in zeros that TMA fills in.
**
** The tensor cores cut their running sums off instead of rounding them: over K terms a result drifts towards zero
** by about 3e-9 K of its size (measured: log-sum-exp of 1001 terms low by 3.6e-6, an fp32 gradient over 8192
** rows off by 2.5e-5; terms of one sign: up to 7e-9 K, 5.6 % of a sum over 8.4 M rows).  A sum is therefore taken in
** runs: the warps that empty an accumulator add it to sums in their registers, rounded, and the next run starts from
** zero.  A run has 512 terms for the loss, 256 for fp32 gradients, and for bf16 gradients, whose rounding is 2^-8, as
** many as cost nothing that could be measured: 16,384, and 4096 of a logit (4096 x 1536 x 100,000: 4.07 ms, in one run 4.08).
*/
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>
#include <algorithm>
#include <atomic>
#include <mutex>
#include "anni_head.h"
#include "head_plan.h"
#include "optstep_internal.h"

#define HEAD_STAGES	6
#define HEAD_A_BYTES	(HEAD_HALF * HEAD_TK * 2)
#define HEAD_B_BYTES	(HEAD_HALF * HEAD_TK * 2)
#define HEAD_STAGE_BYTES (HEAD_A_BYTES + HEAD_B_BYTES)
#define HEAD_MN_BYTES	(64 * HEAD_TK * 2)	/* one MN-major box */
#define HEAD_EPI	256	/* threads that empty accumulators: 128 rows x 2 halves of the columns */
#define HEAD_THREADS	(128 + HEAD_EPI)
#define HEAD_RUN	8	/* stages in one run of a sum: 512 terms of a logit, */
#define HEAD_RUN_F32	4	/* 256 of an fp32 gradient, */
#define HEAD_RUN_BF16	256	/* 16,384 of one that is rounded to bf16, */
#define HEAD_RUN_DELTA	64	/* 4096 of a logit whose exponential is rounded to bf16 */
#define ROWS_DEEP	64	/* rows of W that a block has at least, */
#define ROWS_START	512	/* and those that a round of blocks takes in time to start and end */
#define HEAD_WAIT_NS	2000000000ull	/* a wait inside a kernel gives up after this long */

namespace {

enum { LOSS, DELTA, GRAD };

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
	__nv_bfloat16		*delta;		/* [terms][tokens][ldp] */
	int			terms;
	int64_t			ldp;
	int			v0;		/* the piece: columns v0 .. v1 - 1 */
	int			v1;
	float			*dxp;		/* fp32 [splits][tokens][ldd], or NULL: straight into dx */
	int			ldd;
	int			splits;
	float			*dbp;		/* fp32 [row tiles][vocab] */
	void			*dx;
	int64_t			lddx;
	void			*dw;
	int64_t			lddw;
	void			*db;
	int			bf16;
	int			add;
};

/* one product: operands, tiles, and how its sums are cut */
struct product_args {
	CUtensorMap	a;
	CUtensorMap	b;
	int		m_tiles;
	int		n_tiles;
	int		k_blocks;	/* of one term */
	int		run;		/* ... of them that one accumulator adds up */
	int		total;		/* tiles, times the parts of dx */
};

struct gemm_args {
	product_args	p[2];		/* GRAD: dx and dw; otherwise the first alone */
	head_args	h;
	int		first;		/* GRAD: the product with the longer tiles, which go first */
	int		extra;		/* tiles of the other that a pair with one fewer of those gets for it */
};

/* ---- PTX ------------------------------------------------------------------------------------------ */

__device__ __forceinline__ uint32_t smem_of(const void *p)
{
	return (uint32_t)__cvta_generic_to_shared(p);
}

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count)
{
	asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(bar), "r"(count) : "memory");
}

/* the same variable in the shared memory of block `rank` of the cluster */
__device__ __forceinline__ uint32_t smem_in(uint32_t addr, uint32_t rank)
{
	uint32_t r;

	asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
	return r;
}

__device__ __forceinline__ float load_in(uint32_t cluster_addr)
{
	float v;

	asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr) : "memory");
	return v;
}

__device__ __forceinline__ void mbar_arrive_in(uint32_t cluster_bar)
{
	asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" :: "r"(cluster_bar) : "memory");
}

__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes)
{
	asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(bar), "r"(bytes) : "memory");
}

__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity)
{
	uint32_t ok;

	asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
	    : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
	return ok != 0;
}

__device__ __forceinline__ uint64_t now_ns(void)
{
	uint64_t t;

	asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
	return t;
}

/*
** Waits for the barrier's phase of this parity.  Gives up, and says so to the whole block through `stop`, after
** HEAD_WAIT_NS, or as soon as another thread of the block has given up (stop NULL: only the time counts).  What a
** block has not computed by then it fills with NaN.
*/
__device__ __noinline__ bool mbar_wait_long(uint32_t bar, uint32_t parity, volatile int *stop)
{
	const uint64_t end = now_ns() + HEAD_WAIT_NS;

	for (;;) {
		for (int k = 0; k < 64; k++)
			if (mbar_try(bar, parity))
				return true;
		if (stop && *stop)
			return false;
		if (now_ns() > end) {
			if (stop)
				*stop = 1;
			return false;
		}
	}
}

__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int *stop)
{
	return mbar_try(bar, parity) || mbar_wait_long(bar, parity, stop);
}

/* into this block's memory, counted by a barrier of either block of the pair */
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap *map, uint32_t bar, int c0, int c1, int c2)
{
	asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
	    :: "r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2) : "memory");
}

/*
** Shared-memory descriptor of an operand tile with 128-byte swizzle (all distances in units of 16 bytes).
** K-major: rows of 128 bytes, eight rows to a swizzle atom, atoms 1024 bytes apart (the stride field); the
** leading field is not used.  MN-major: boxes of 64 mn x 64 k; eight k to an atom, atoms 1024 bytes apart
** (the stride field), the next 64 mn one box further (the leading field).
*/
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, bool mn)
{
	const uint64_t lead = mn ? HEAD_MN_BYTES >> 4 : 1;

	return (uint64_t)((addr & 0x3ffff) >> 4) | lead << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

/* D (fp32) = A B, both bf16: M 256 and N 256 over the pair, and which of them are MN-major */
__device__ __forceinline__ constexpr uint32_t instr_desc(bool a_mn, bool b_mn)
{
	return 1u << 4 | 1u << 7 | 1u << 10 | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) | (uint32_t)(HEAD_TN >> 3) << 17
	    | (uint32_t)(HEAD_TM >> 4) << 24;
}

__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add)
{
	asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
	    "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
	    :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add) : "memory");
}

/* arrives on this barrier of both blocks when the products issued so far are done */
__device__ __forceinline__ void mma_commit(uint32_t bar)
{
	asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
	    :: "r"(bar), "h"((uint16_t)3) : "memory");
}

/* 32 columns of this warp's 32 lanes of tensor memory: lane l gets row l; valid after tmem_wait() */
__device__ __forceinline__ void tmem_load(uint32_t addr, float (&v)[32])
{
	asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
	    "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
	    "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
	    : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
	    "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
	    "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
	    "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31]) : "r"(addr));
}

/* the values of the loads before are there: nothing that uses them may be moved ahead of it */
__device__ __forceinline__ void tmem_wait(float (&v)[32])
{
	asm volatile("tcgen05.wait::ld.sync.aligned;" : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]),
	    "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]),
	    "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]),
	    "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31]) :: "memory");
}

__device__ __forceinline__ float exp2_approx(float x)
{
	float r;

	asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
	return r;
}

/* two floats in one instruction: a += b, a *= b */
__device__ __forceinline__ void add2(float &a0, float &a1, float b0, float b1)
{
	asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\tadd.rn.f32x2 x, x, y;\n\t"
	    "mov.b64 {%0, %1}, x;\n\t}" : "+f"(a0), "+f"(a1) : "f"(b0), "f"(b1));
}

__device__ __forceinline__ void mul2(float &a0, float &a1, float b)
{
	asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %2};\n\tmul.rn.f32x2 x, x, y;\n\t"
	    "mov.b64 {%0, %1}, x;\n\t}" : "+f"(a0), "+f"(a1) : "f"(b));
}

__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi)
{
	const __nv_bfloat162 q = __floats2bfloat162_rn(lo, hi);

	return *reinterpret_cast<const uint32_t *>(&q);
}

/* 32 bytes at a time: a whole sector per lane where each lane writes a row of its own */
__device__ __forceinline__ void store32(void *p, const uint32_t (&r)[8])
{
	asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" :: "l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]),
	    "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}

__device__ __forceinline__ void load32(const void *p, uint32_t (&r)[8])
{
	/* not volatile: nothing that a kernel loads this way has been stored by it before, so loads may go ahead of stores */
	asm("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]),
	    "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "l"(p));
}

__device__ __forceinline__ float to_f(__nv_bfloat16 v)
{
	return __bfloat162float(v);
}

#define LOG2E	1.44269504088896340736f

/* ---- which tile, and what of it a stage holds ---------------------------------------------------- */

struct tile_at {
	int	which;	/* GRAD: DX or DW */
	int	m0;	/* this block's rows */
	int	n0;
	int	b0;	/* its share of the second operand */
	int	k0;	/* k blocks lo .. hi - 1 of each term */
	int	k1;
	int	split;
};

/* how many of 0 .. n - 1 are at + i * step */
__device__ __forceinline__ int count_of(int n, int at, int step)
{
	return at < n ? (n - at + step - 1) / step : 0;
}

/*
** The i-th tile of a pair of blocks; false: there is none.
**
** loss, delta: all row tiles (32 at most) of one column tile after another, dealt round-robin, so that W is read
** once while x stays in L2.  grad: the longer tiles round-robin; the pairs that get one fewer of them take `extra`
** of the shorter ones for it, the rest of those go round-robin again.  Within dx the column tiles of a row
** tile come together, within dw the row tiles of a column tile, so that delta is read once.
*/
template <int KIND>
__device__ __forceinline__ bool tile_of(const gemm_args &g, int i, int rank, int pair, int pairs, tile_at &r)
{
	int t;
	int m;
	int n;

	r.split = 0;
	r.which = 0;
	if (KIND == GRAD) {
		const int n_long = g.p[g.first].total;
		const int n_short = g.p[1 - g.first].total;
		const int own = count_of(n_long, pair, pairs);
		const int full = n_long % pairs;		/* pairs with one more */
		const int lack = pairs - full;
		const int fill = min(n_short, lack * g.extra);
		const int own_fill = pair >= full ? count_of(fill, pair - full, lack) : 0;

		if (i < own) {
			r.which = g.first;
			t = pair + i * pairs;
		} else {
			i -= own;
			r.which = 1 - g.first;
			t = i < own_fill ? pair - full + i * lack : fill + (pair + lack) % pairs + (i - own_fill) * pairs;
			if (t >= n_short)
				return false;
		}
	} else {
		t = pair + i * pairs;
		if (t >= g.p[0].total)
			return false;
	}
	const product_args &p = g.p[r.which];

	r.k0 = 0;
	r.k1 = p.k_blocks;
	if (KIND == GRAD && r.which == DX) {
		n = t % p.n_tiles;
		m = t / p.n_tiles % p.m_tiles;
		r.split = t / (p.n_tiles * p.m_tiles);
		r.k0 = part_begin(p.k_blocks, r.split, g.h.splits);
		r.k1 = part_begin(p.k_blocks, r.split + 1, g.h.splits);
	} else if (KIND == GRAD) {
		m = t % p.m_tiles;
		n = t / p.m_tiles;
	} else {
		const int group = t / (32 * p.n_tiles);
		const int rows = min(32, p.m_tiles - group * 32);

		t -= group * 32 * p.n_tiles;
		m = group * 32 + t % rows;
		n = t / rows;
	}
	r.m0 = m * HEAD_TM + rank * HEAD_HALF;
	r.n0 = n * HEAD_TN;
	r.b0 = r.n0 + rank * HEAD_HALF;
	return true;
}

template <int KIND>
__device__ __forceinline__ void load_stage(const gemm_args &g, const tile_at &t, int term, int k, uint32_t dst, uint32_t bar)
{
	const product_args &p = g.p[t.which];
	const uint32_t b = dst + HEAD_A_BYTES;

	if (KIND != GRAD) {
		tma_load(dst, &p.a, bar, k, t.m0, 0);
#pragma unroll
		for (int j = 0; j < HEAD_HALF / 64; j++)
			tma_load(b + j * HEAD_MN_BYTES, &p.b, bar, g.h.v0 + t.b0 + 64 * j, k, 0);
	} else if (t.which == DX) {
		tma_load(dst, &p.a, bar, k, t.m0, term);
		tma_load(b, &p.b, bar, g.h.v0 + k, t.b0, 0);
	} else {
#pragma unroll
		for (int j = 0; j < HEAD_HALF / 64; j++)
			tma_load(dst + j * HEAD_MN_BYTES, &p.a, bar, t.m0 + 64 * j, k, 0);
#pragma unroll
		for (int j = 0; j < HEAD_HALF / 64; j++)
			tma_load(b + j * HEAD_MN_BYTES, &p.b, bar, t.b0 + 64 * j, k, term);
	}
}

/* ---- epilogues: a thread has 128 columns of one row, as four times 32 --------------------------------- */

struct epi_smem {
	float	bias[2][HEAD_TN];	/* of two tiles; -inf beyond the vocabulary */
	float	sums[2][4][HEAD_TN];	/* delta: column sums of each quarter of the rows */
	float2	half[2][HEAD_HALF];	/* loss: maximum and sum of the second half of the columns */
};

__device__ __forceinline__ void epi_barrier(void)
{
	asm volatile("bar.sync 1, 256;" ::: "memory");
}

/* row of the block's 128, first column of the tile's 256, and number among the epilogue's threads */
__device__ __forceinline__ int epi_row(void)
{
	return threadIdx.x & (HEAD_HALF - 1);
}

__device__ __forceinline__ int epi_thread(void)
{
	return threadIdx.x - 128;
}

__device__ __forceinline__ int epi_col(void)
{
	return epi_thread() / HEAD_HALF * 128;
}

/* biases of the tile's columns */
__device__ __forceinline__ void stage_bias(const head_args &h, int v0, int end, float *to)
{
	const int i = epi_thread();

	to[i] = v0 + i >= end ? -INFINITY : h.bias ? __ldg(h.bias + v0 + i) : 0.0f;
	epi_barrier();
}

/* v[i] + sum over the warp's rows: lane l ends with the sum of column l, rows added in a fixed tree */
__device__ __forceinline__ float column_sums(float (&v)[32])
{
	const int lane = threadIdx.x & 31;

#pragma unroll
	for (int s = 16; s > 0; s >>= 1) {
		const bool up = lane & s;

#pragma unroll
		for (int i = 0; i < s; i++) {
			const float send = up ? v[i] : v[i + s];
			const float keep = up ? v[i + s] : v[i];

			v[i] = keep + __shfl_xor_sync(0xffffffffu, send, s);
		}
	}
	return v[0];
}

/* one pass over the columns with a running maximum and a sum that follows it */
__device__ __forceinline__ void loss_epilogue(const gemm_args &g, const tile_at &at, float (&acc)[4][32], const float *bias,
	float2 *half)
{
	const head_args &h = g.h;
	const int t = at.m0 + epi_row();
	const int y = t < h.tokens ? h.target[t] : -1;
	const int c0 = epi_col();
	const int rel = y >= at.n0 + c0 && y < h.vocab && y < at.n0 + c0 + 128 ? y - at.n0 - c0 : -1;
	float top = -INFINITY;
	float sum = 0.0f;
	float sum1 = 0.0f;

#pragma unroll
	for (int c = 0; c < 4; c++) {
		float (&v)[32] = acc[c];
		float high;
		float base;

#pragma unroll
		for (int i = 0; i < 32; i += 4) {
			const float4 b = *reinterpret_cast<const float4 *>(bias + c0 + c * 32 + i);

			add2(v[i], v[i + 1], b.x, b.y);
			add2(v[i + 2], v[i + 3], b.z, b.w);
		}
		if (__any_sync(0xffffffffu, rel >= c * 32 && rel < c * 32 + 32)) {	/* one in vocab / 32 chunks of a row */
#pragma unroll
			for (int i = 0; i < 32; i++)
				if (rel == c * 32 + i)
					h.hit[t] = v[i];
		}
		high = v[0];
#pragma unroll
		for (int i = 1; i < 32; i++)
			high = fmaxf(high, v[i]);	/* a NaN shows in the sum */
		high = fmaxf(high, top);
		base = high == -INFINITY ? 0.0f : high;
		mul2(sum, sum1, exp2_approx((top - base) * LOG2E));
		top = high;
#pragma unroll
		for (int i = 0; i < 32; i += 2) {	/* the difference first: a rounded product of a mask's size is anything */
			add2(v[i], v[i + 1], -base, -base);
			mul2(v[i], v[i + 1], LOG2E);
			add2(sum, sum1, exp2_approx(v[i]), exp2_approx(v[i + 1]));
		}
	}
	sum += sum1;
	if (c0)
		half[epi_row()] = make_float2(top, sum);
	epi_barrier();
	if (!c0 && t < h.tokens) {
		const float2 p = half[epi_row()];
		const float high = fmaxf(top, p.x);
		const float base = high == -INFINITY ? 0.0f : high;

		sum = sum * exp2_approx((top - base) * LOG2E) + p.y * exp2_approx((p.x - base) * LOG2E);
		h.part[(int64_t)(at.n0 / HEAD_TN) * h.tokens + t] = make_float2(high, sum);
	}
}

/*
** Softmax minus one-hot, times the row's factor.  As an operand of a bf16 product it has to be bf16: for bf16 gradients
** one term, whose rounding is as large as that of the result and adds to it as an independent one (off from 64 bits by
** 1.9e-3 of the norm at 8192 x 1024 x 16,384, where the rounding of the result alone makes 1.7e-3; a second term would
** take six products instead of four); for fp32 gradients three terms, which hold all 24 bits.
*/
__device__ __forceinline__ void delta_epilogue(const gemm_args &g, const tile_at &at, float (&acc)[4][32], const float *bias,
	float (*sums)[HEAD_TN])
{
	const head_args &h = g.h;
	const int lane = threadIdx.x & 31;
	const int c0 = epi_col();
	const int t = at.m0 + epi_row();
	const float f = t < h.tokens ? h.row[t] : 0.0f;
	const float lse = f != 0.0f ? -h.lse[t] : -INFINITY;	/* negated; no gradient: all exponentials 0 */
	const int y = f != 0.0f ? h.target[t] - h.v0 - at.n0 - c0 : -1;
	__nv_bfloat16 *out = h.delta + (int64_t)t * h.ldp + at.n0 + c0;

#pragma unroll
	for (int c = 0; c < 4; c++) {
		float (&v)[32] = acc[c];

#pragma unroll
		for (int i = 0; i < 32; i += 4) {
			const float4 b = *reinterpret_cast<const float4 *>(bias + c0 + c * 32 + i);

			add2(v[i], v[i + 1], b.x, b.y);
			add2(v[i + 2], v[i + 3], b.z, b.w);
		}
#pragma unroll
		for (int i = 0; i < 32; i += 2) {
			add2(v[i], v[i + 1], lse, lse);
			mul2(v[i], v[i + 1], LOG2E);
			v[i] = exp2_approx(v[i]);
			v[i + 1] = exp2_approx(v[i + 1]);
		}
		if (__any_sync(0xffffffffu, y >= c * 32 && y < c * 32 + 32)) {
#pragma unroll
			for (int i = 0; i < 32; i++)
				if (y == c * 32 + i)
					v[i] -= 1.0f;
		}
#pragma unroll
		for (int i = 0; i < 32; i += 2)
			mul2(v[i], v[i + 1], f);
		if (t < h.tokens) {
			__nv_bfloat16 *q = out + c * 32;

			for (int n = 1; n < h.terms; n++) {	/* fp32 gradients: first the terms that correct the largest */
#pragma unroll
				for (int i = 0; i < 32; i += 16) {
					uint32_t r[8];

#pragma unroll
					for (int j = 0; j < 8; j++) {
						float lo = v[i + 2 * j];
						float hi = v[i + 2 * j + 1];

#pragma unroll 1
						for (int k = 0; k < n; k++) {
							lo -= to_f(__float2bfloat16_rn(lo));
							hi -= to_f(__float2bfloat16_rn(hi));
						}
						r[j] = bf16_pair(lo, hi);
					}
					store32(q + (int64_t)n * h.tokens * h.ldp + i, r);
				}
			}
#pragma unroll
			for (int i = 0; i < 32; i += 16) {
				uint32_t r[8];

#pragma unroll
				for (int j = 0; j < 8; j++)
					r[j] = bf16_pair(v[i + 2 * j], v[i + 2 * j + 1]);
				store32(q + i, r);
			}
		}
		if (h.db)
			sums[threadIdx.x >> 5 & 3][c0 + c * 32 + lane] = column_sums(v);
		asm volatile("" ::: "memory");	/* one 32 after the other: what is read ahead is spilled */
	}
	if (h.db) {
		const int i = epi_thread();

		epi_barrier();
		if (at.m0 < h.tokens && h.v0 + at.n0 + i < h.v1)
			h.dbp[(int64_t)(at.m0 / HEAD_HALF) * h.vocab + h.v0 + at.n0 + i] =
			    (sums[0][i] + sums[1][i]) + (sums[2][i] + sums[3][i]);
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

__device__ __forceinline__ float2 unpack2(uint32_t q)
{
	return make_float2(__uint_as_float(q << 16), __uint_as_float(q & 0xffff0000u));
}

/* 32 x 32 values of a warp, lane l with row l, so that lane l has column l: v[i] is then of row i */
__device__ __forceinline__ void transpose(float (&v)[32])
{
	const int lane = threadIdx.x & 31;

#pragma unroll
	for (int s = 16; s > 0; s >>= 1)
#pragma unroll
		for (int i = 0; i < 32; i++)
			if (!(i & s)) {
				const bool up = lane & s;
				const float got = __shfl_xor_sync(0xffffffffu, up ? v[i] : v[i + s], s);

				if (up)
					v[i] = got;
				else
					v[i + s] = got;
			}
}

/*
** A warp's 32 x 32 results, lane l with row l, stored or added to what is there: at (row, col) of a matrix of which
** `rows` rows and `left` of these columns exist.  Rows on 32 bytes: every lane whole sectors of its own row; on 16 bytes: half
** sectors; others: transposed, the warp row by row, so that its accesses are one piece whatever the address.
*/
__device__ __forceinline__ void put_block(void *base, int64_t ld, int row, int rows, int64_t col, int left, float (&v)[32],
	bool bf16, bool add)
{
	const int lane = threadIdx.x & 31;
	const int size = bf16 ? 2 : 4;

	if (left >= 32 && (((uintptr_t)base | (uintptr_t)(ld * size) | (uintptr_t)(col * size)) & 31) == 0) {
		char *out = static_cast<char *>(base) + ((int64_t)(row + lane) * ld + col) * size;

		if (row + lane >= rows)
			return;
		if (bf16) {
#pragma unroll
			for (int i = 0; i < 32; i += 16) {
				uint32_t r[8] = { 0, 0, 0, 0, 0, 0, 0, 0 };

				if (add)
					load32(out + i * 2, r);
#pragma unroll
				for (int j = 0; j < 8; j++) {
					const float2 q = unpack2(r[j]);

					r[j] = bf16_pair(q.x + v[i + 2 * j], q.y + v[i + 2 * j + 1]);
				}
				store32(out + i * 2, r);
			}
		} else {
#pragma unroll
			for (int i = 0; i < 32; i += 8) {
				uint32_t r[8] = { 0, 0, 0, 0, 0, 0, 0, 0 };

				if (add)
					load32(out + i * 4, r);
#pragma unroll
				for (int j = 0; j < 8; j++)
					r[j] = __float_as_uint(__uint_as_float(r[j]) + v[i + j]);
				store32(out + i * 4, r);
			}
		}
		return;
	}
	if (left >= 32 && (((uintptr_t)base | (uintptr_t)(ld * size) | (uintptr_t)(col * size)) & 15) == 0) {
		char *out = static_cast<char *>(base) + ((int64_t)(row + lane) * ld + col) * size;

		if (row + lane >= rows)
			return;
#pragma unroll
		for (int i = 0; i < 32; i += 4) {
			if (bf16) {
				uint2 r = add ? *reinterpret_cast<const uint2 *>(out + i * 2) : make_uint2(0, 0);
				const float2 p = unpack2(r.x);
				const float2 q = unpack2(r.y);

				r.x = bf16_pair(p.x + v[i], p.y + v[i + 1]);
				r.y = bf16_pair(q.x + v[i + 2], q.y + v[i + 3]);
				*reinterpret_cast<uint2 *>(out + i * 2) = r;
			} else {
				float4 r = add ? *reinterpret_cast<const float4 *>(out + i * 4) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);

				r.x += v[i];
				r.y += v[i + 1];
				r.z += v[i + 2];
				r.w += v[i + 3];
				*reinterpret_cast<float4 *>(out + i * 4) = r;
			}
		}
		return;
	}
	transpose(v);
	if (lane >= left)
		return;
	if (bf16) {
		__nv_bfloat16 *out = static_cast<__nv_bfloat16 *>(base) + (int64_t)row * ld + col + lane;

#pragma unroll
		for (int i = 0; i < 32; i += 4) {
			float old[4];

#pragma unroll
			for (int j = 0; j < 4; j++)
				old[j] = add && row + i + j < rows ? to_f(out[j * ld]) : 0.0f;
#pragma unroll
			for (int j = 0; j < 4; j++)
				if (row + i + j < rows)
					out[j * ld] = __float2bfloat16_rn(old[j] + v[i + j]);
			out += 4 * ld;
			asm volatile("" ::: "memory");
		}
	} else {
		float *out = static_cast<float *>(base) + (int64_t)row * ld + col + lane;

#pragma unroll
		for (int i = 0; i < 32; i += 4) {
			float old[4];

#pragma unroll
			for (int j = 0; j < 4; j++)
				old[j] = add && row + i + j < rows ? out[j * ld] : 0.0f;
#pragma unroll
			for (int j = 0; j < 4; j++)
				if (row + i + j < rows)
					out[j * ld] = old[j] + v[i + j];
			out += 4 * ld;
			asm volatile("" ::: "memory");
		}
	}
}

/*
** Results that are added to what is there: this thread's piece of its row on its way to the L2 while the products
** run.  (Fetched from HBM when they are needed, piece by piece, they made an epilogue of 6,000 cycles one of 24,000.)
*/
__device__ __forceinline__ void fetch_ahead(const gemm_args &g, const tile_at &at)
{
	const head_args &h = g.h;
	const bool dx = at.which == DX;
	const int row = at.m0 + epi_row();
	const int col = (dx ? 0 : h.v0) + at.n0 + epi_col();
	const int size = !dx && h.bf16 ? 2 : 4;
	const int left = min(128, (dx ? h.ldd : h.v1) - col);
	const char *base = reinterpret_cast<const char *>(dx ? h.dxp + (int64_t)at.split * h.tokens * h.ldd : h.dw);

	if (dx ? !h.dxp || h.v0 == 0 : !h.add)
		return;
	if (row >= (dx ? h.tokens : h.d))
		return;
	base += ((int64_t)row * (dx ? h.ldd : h.lddw) + col) * size;
	for (int i = 0; i < left * size; i += 128)
		asm volatile("prefetch.global.L2 [%0];" :: "l"(base + i));
}

__device__ __forceinline__ void grad_epilogue(const gemm_args &g, const tile_at &at, float (&acc)[4][32])
{
	const head_args &h = g.h;
	const int row = at.m0 + (epi_row() & ~31);	/* this warp's first */
	const bool dx = at.which == DX;
	const bool parts = dx && h.dxp;
	/* dx: its fp32 sum, or where one part of one piece is all of it, dx itself */
	void *const base = parts ? h.dxp + (int64_t)at.split * h.tokens * h.ldd : dx ? h.dx : h.dw;
	const int64_t ld = parts ? h.ldd : dx ? h.lddx : h.lddw;
	const int rows = dx ? h.tokens : h.d;
	const int cols = parts ? h.ldd : dx ? h.d : h.v1;
	const bool add = parts ? h.v0 != 0 : !dx && h.add;
	const int col = (dx ? 0 : h.v0) + at.n0 + epi_col();

#pragma unroll
	for (int c = 0; c < 4; c++)
		if (col + c * 32 < cols && row < rows) {
			put_block(base, ld, row, rows, col + c * 32, cols - col - c * 32, acc[c], h.bf16 && !parts, add);
			asm volatile("" ::: "memory");	/* one 32 after the other: what is read ahead is spilled */
		}
}

/* dbias of the columns from, from + step, ... below `to`: delta's column sums of all rows of tiles, in order */
__device__ __forceinline__ void finish_db(const head_args &h, int from, int to, int step)
{
	const int tiles = (h.tokens + HEAD_HALF - 1) / HEAD_HALF;

	for (int v = from; v < to; v += step) {
		double s = 0.0;

#pragma unroll 8
		for (int k = 0; k < tiles; k++)
			s += (double)h.dbp[(int64_t)k * h.vocab + v];
		if (h.add)
			s += h.bf16 ? (double)to_f(static_cast<__nv_bfloat16 *>(h.db)[v]) : (double)static_cast<float *>(h.db)[v];
		put(h.db, v, (float)s, h.bf16, 0);
	}
}

/* ---- the product -------------------------------------------------------------------------------------- */

struct gemm_smem {
	uint64_t	full[HEAD_STAGES];	/* a stage has been loaded */
	uint64_t	empty[HEAD_STAGES];	/* ... and consumed */
	uint64_t	ready[2];		/* an accumulator is complete */
	uint64_t	drained[2];		/* ... and read out */
	uint64_t	quiet;			/* after a give-up: the products in flight are done */
	uint32_t	tmem;
	int		stop;			/* somebody has given up */
	epi_smem	epi;
};

/*
** Loads this block's shares.  The first block's barrier counts both blocks' bytes, since the products of both
** are issued there.  Returns after a give-up only when the copies in flight have landed, or the time is up.
*/
template <int KIND>
__device__ __forceinline__ void producer(const gemm_args &g, gemm_smem *s, uint32_t ring, int rank, int pair, int pairs)
{
	const int terms = KIND == GRAD ? g.h.terms : 1;
	uint32_t n = 0;		/* stages loaded so far */
	tile_at at;

	for (int tile = 0; tile_of<KIND>(g, tile, rank, pair, pairs, at); tile++) {
		const int run = g.p[at.which].run;
		int k = at.k0;
		int term = 0;
		int from = k;	/* of this run */

		/* all terms of a run, the small ones first, then the next run */
		while (from < at.k1) {
			const uint32_t i = n % HEAD_STAGES;

			if (!mbar_wait(smem_of(&s->empty[i]), (n / HEAD_STAGES & 1) ^ 1, &s->stop)) {
				if (rank == 0)
					for (uint32_t j = n < HEAD_STAGES ? 0 : n - HEAD_STAGES; j < n; j++)
						(void)mbar_wait(smem_of(&s->full[j % HEAD_STAGES]), j / HEAD_STAGES & 1, NULL);
				else {
					/* counted elsewhere: no copy is under way for this long */
					for (const uint64_t end = now_ns() + HEAD_WAIT_NS / 100; now_ns() < end; )
						__nanosleep(1000);
				}
				return;
			}
			if (rank == 0)
				mbar_expect(smem_of(&s->full[i]), 2 * HEAD_STAGE_BYTES);
			load_stage<KIND>(g, at, terms - 1 - term, k * HEAD_TK, ring + i * HEAD_STAGE_BYTES,
			    smem_in(smem_of(&s->full[i]), 0));
			n++;
			if (++k == min(from + run, at.k1)) {
				if (++term == terms) {
					term = 0;
					from = k;
				}
				k = from;
			}
		}
	}
}

/* the first block's: issues the products of both */
template <int KIND>
__device__ __forceinline__ void multiplier(const gemm_args &g, gemm_smem *s, uint32_t ring, int pair, int pairs)
{
	uint32_t n = 0;
	uint32_t done = 0;	/* runs */
	tile_at at;

	for (int tile = 0; tile_of<KIND>(g, tile, 0, pair, pairs, at); tile++) {
		const bool a_mn = KIND == GRAD && at.which == DW;
		const bool b_mn = KIND != GRAD || at.which == DW;
		const uint32_t idesc = instr_desc(a_mn, b_mn);
		/* 16 k a time: 32 bytes further in a K-major row, 16 rows of 128 bytes further in an MN-major box */
		const uint32_t a_step = a_mn ? 2048 : 32;
		const uint32_t b_step = b_mn ? 2048 : 32;
		const int run = g.p[at.which].run;

		for (int from = at.k0; from < at.k1; from += run, done++) {
			const int steps = (min(from + run, at.k1) - from) * (KIND == GRAD ? g.h.terms : 1);
			const uint32_t acc = s->tmem + (done & 1) * HEAD_TN;
			bool ok = mbar_wait(smem_of(&s->drained[done & 1]), (done / 2 & 1) ^ 1, &s->stop);

			asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
			for (int k = 0; ok && k < steps; k++, n++) {
				const uint32_t i = n % HEAD_STAGES;
				const uint32_t base = ring + i * HEAD_STAGE_BYTES;

				ok = mbar_wait(smem_of(&s->full[i]), n / HEAD_STAGES & 1, &s->stop);
				if (!ok)
					break;
				asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
				for (int j = 0; j < HEAD_TK / 16; j++)
					mma(acc, smem_desc(base + j * a_step, a_mn),
					    smem_desc(base + HEAD_A_BYTES + j * b_step, b_mn), idesc, k > 0 || j > 0);
				mma_commit(smem_of(&s->empty[i]));
			}
			if (!ok) {
				mma_commit(smem_of(&s->quiet));
				(void)mbar_wait(smem_of(&s->quiet), 0, NULL);
				return;
			}
			mma_commit(smem_of(&s->ready[done & 1]));
		}
	}
}

template <int KIND>
__device__ __forceinline__ void drainer(const gemm_args &g, gemm_smem *s, int rank, int pair, int pairs)
{
	const uint32_t lanes = (uint32_t)(threadIdx.x >> 5 & 3) << 21;	/* this warp's quarter of the lanes: 32 w << 16 */
	uint32_t done = 0;
	uint32_t b = 0;
	tile_at at;

	for (int tile = 0; tile_of<KIND>(g, tile, rank, pair, pairs, at); tile++, b ^= 1) {
		const int run = g.p[at.which].run;
		float acc[4][32];

		if (KIND == LOSS)
			stage_bias(g.h, at.n0, g.h.vocab, s->epi.bias[b]);
		if (KIND == DELTA)
			stage_bias(g.h, g.h.v0 + at.n0, g.h.v1, s->epi.bias[b]);
		if (KIND == GRAD)
			fetch_ahead(g, at);
#pragma unroll 1
		for (int from = at.k0; from < at.k1; from += run, done++) {
			const uint32_t addr = s->tmem + lanes + (done & 1) * HEAD_TN + epi_col();

			/* the warps keep step with each other even after a give-up, for the barriers' sake */
			(void)__all_sync(0xffffffffu, mbar_wait(smem_of(&s->ready[done & 1]), done / 2 & 1, &s->stop));
			asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
			if (from == at.k0) {
#pragma unroll
				for (int c = 0; c < 4; c++)
					tmem_load(addr + c * 32, acc[c]);
#pragma unroll
				for (int c = 0; c < 4; c++)
					tmem_wait(acc[c]);
			} else {
#pragma unroll
				for (int c = 0; c < 4; c++) {
					float v[32];

					tmem_load(addr + c * 32, v);
					tmem_wait(v);
#pragma unroll
					for (int i = 0; i < 32; i++)
						acc[c][i] += v[i];
				}
			}
			asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
			__syncwarp();
			if ((threadIdx.x & 31) == 0)
				mbar_arrive_in(smem_in(smem_of(&s->drained[done & 1]), 0));
		}
		if (*static_cast<volatile int *>(&s->stop))	/* somebody gave up: nothing here is to be believed */
#pragma unroll
			for (int i = 0; i < 128; i++)
				acc[i / 32][i % 32] = NAN;
		__syncwarp();
		if (KIND == LOSS)
			loss_epilogue(g, at, acc, s->epi.bias[b], s->epi.half[b]);
		else if (KIND == DELTA)
			delta_epilogue(g, at, acc, s->epi.bias[b], s->epi.sums[b]);
		else
			grad_epilogue(g, at, acc);
	}
}

/* everything the kernels ahead in the stream have done is visible after this; the next kernel may set itself up */
__device__ __forceinline__ void dependent(void)
{
	asm volatile("griddepcontrol.launch_dependents;\n\tgriddepcontrol.wait;" ::: "memory");
}

__device__ __forceinline__ void cluster_barrier(void)
{
	asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <int KIND>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(HEAD_THREADS, 1) product_kernel(const __grid_constant__ gemm_args g)
{
	extern __shared__ uint8_t dynamic[];
	__shared__ gemm_smem s;
	const uint32_t ring = (smem_of(dynamic) + 1023) & ~1023u;	/* swizzle atoms lie on 1024 bytes */
	const int warp = threadIdx.x >> 5;
	const int rank = blockIdx.x & 1;
	const int pair = blockIdx.x >> 1;
	const int pairs = gridDim.x >> 1;

	if (threadIdx.x == 0) {
		for (int i = 0; i < HEAD_STAGES; i++) {
			mbar_init(smem_of(&s.full[i]), 1);
			mbar_init(smem_of(&s.empty[i]), 1);
		}
		for (int i = 0; i < 2; i++) {
			mbar_init(smem_of(&s.ready[i]), 1);
			mbar_init(smem_of(&s.drained[i]), 2 * HEAD_EPI / 32);	/* the warps of both blocks */
		}
		mbar_init(smem_of(&s.quiet), 1);
		s.stop = 0;
		asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
		asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
	}
	__syncwarp();
	if (warp == 2) {
		asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" :: "r"(smem_of(&s.tmem)) : "memory");
		asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
	}
	asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
	__syncthreads();
	cluster_barrier();
	asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
	dependent();
	if (warp < 4) {
		if (warp == 0 && (threadIdx.x & 31) == 0)
			producer<KIND>(g, &s, ring, rank, pair, pairs);
		if (warp == 1 && (threadIdx.x & 31) == 0 && rank == 0)
			multiplier<KIND>(g, &s, ring, pair, pairs);
		/* nothing waits for dbias: a warp that is idle otherwise, beside the products */
		if (KIND == GRAD && warp == 3 && g.h.db)
			finish_db(g.h, g.h.v0 + blockIdx.x * 32 + (threadIdx.x & 31), g.h.v1, gridDim.x * 32);
	} else
		drainer<KIND>(g, &s, rank, pair, pairs);
	__syncwarp();
	asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
	__syncthreads();
	cluster_barrier();	/* neither block leaves, nor gives its tensor memory back, while the other may need it */
	asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
	if (warp == 2)
		asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" :: "r"(s.tmem) : "memory");
}

/* maximum and sum of one part of a row taken into those of the others */
__device__ __forceinline__ void join(float &top, float &sum, float2 p)
{
	const float high = fmaxf(top, p.x);
	const float base = high == -INFINITY ? 0.0f : high;

	sum = sum * exp2f((top - base) * LOG2E) + p.y * exp2f((p.x - base) * LOG2E);
	top = high;
}

/* ---- a few rows ------------------------------------------------------------------------------------------- */

/*
** The loss of one row or two: W is read once and little is computed, so HBM is the bound, and a product whose
** tiles have 256 rows spends longer on the empty ones (one row, 1536 x 100,000: 58 us here, 89 there, and reading W
** alone takes 47; 1536 x 4097, off the 16-byte grid: 10 and 21; 2560 x 32,768: 32 and 53).
** A block takes `width` entries of the vocabulary and `deep` rows of W, each of its eight warps every eighth of these:
** ROWS x 8 sums a thread, in fp32, added up over the warps and then over the blocks of a cluster, which
** share the rows of the same entries, in order.
** Loads are of 16-byte granules.  In rows off that grid a warp's granules all begin the same number of entries ahead of
** the tile, since eight rows on an address is the same modulo 16 bytes: its sums just belong to entries that many
** places to the left, and a tile has eight entries less.  What such granules hold of other rows goes into
** sums that nobody reads; those that reach out of W are read one entry at a time.
*/
template <int ROWS>
__global__ void __launch_bounds__(256) rows_kernel(const head_args h, int width, int deep, int parts)
{
	extern __shared__ float xs[];		/* [deep][ROWS] */
	__shared__ float red[8][HEAD_TN];
	__shared__ float sums[ROWS][HEAD_TN];
	__shared__ float2 warps[8];
	const int lane = threadIdx.x & 31;
	const int w = threadIdx.x >> 5;
	const int tile = blockIdx.x / parts;
	const int rank = blockIdx.x % parts;	/* in the cluster */
	const int v0 = tile * width;
	const int lo = min(rank * deep, h.d);
	const int hi = min(lo + deep, h.d);
	const int shift = (int)((uintptr_t)(h.w + (int64_t)(lo + w) * h.ldw) & 15) / 2;
	const int c0 = v0 - shift + lane * 8;	/* this thread's entries */
	const int64_t total = (int64_t)(h.d - 1) * h.ldw + h.vocab;
	const int mine = v0 + threadIdx.x;
	float acc[ROWS][8];

	dependent();
	for (int i = threadIdx.x; i < (hi - lo) * ROWS; i += 256)
		xs[i] = to_f(h.x[(int64_t)(i % ROWS) * h.ldx + lo + i / ROWS]);
#pragma unroll
	for (int r = 0; r < ROWS; r++)
#pragma unroll
		for (int j = 0; j < 8; j++)
			acc[r][j] = 0.0f;
	__syncthreads();
	for (int d0 = lo + w; d0 < hi; d0 += 64) {
		uint32_t q[8][4];

#pragma unroll
		for (int k = 0; k < 8; k++) {
			const int64_t e = (int64_t)(d0 + k * 8) * h.ldw + c0;

#pragma unroll
			for (int j = 0; j < 4; j++)
				q[k][j] = 0;
			if (d0 + k * 8 >= hi || c0 >= h.vocab)
				continue;
			if (e >= 0 && e + 8 <= total) {
				const uint4 r = __ldcs(reinterpret_cast<const uint4 *>(h.w + e));

				q[k][0] = r.x;
				q[k][1] = r.y;
				q[k][2] = r.z;
				q[k][3] = r.w;
			} else
#pragma unroll
				for (int j = 0; j < 8; j++)
					if (c0 + j >= 0 && c0 + j < h.vocab)
						q[k][j / 2] |= (uint32_t)reinterpret_cast<const uint16_t *>(h.w)[e + j] << (j % 2 * 16);
		}
#pragma unroll
		for (int k = 0; k < 8; k++) {
			if (d0 + k * 8 >= hi)
				break;
#pragma unroll
			for (int j = 0; j < 8; j += 2) {
				const float2 b = unpack2(q[k][j / 2]);

#pragma unroll
				for (int r = 0; r < ROWS; r++) {
					const float a = xs[(d0 + k * 8 - lo) * ROWS + r];

					acc[r][j] = fmaf(a, b.x, acc[r][j]);
					acc[r][j + 1] = fmaf(a, b.y, acc[r][j + 1]);
				}
			}
		}
	}
#pragma unroll
	for (int r = 0; r < ROWS; r++) {
		float z = 0.0f;

		__syncthreads();
#pragma unroll
		for (int j = 0; j < 8; j++)
			if (lane * 8 + j >= shift)
				red[w][lane * 8 + j - shift] = acc[r][j];
		__syncthreads();
		if ((int)threadIdx.x < width)
#pragma unroll
			for (int k = 0; k < 8; k++)
				z += red[k][threadIdx.x];
		sums[r][threadIdx.x] = z;
	}
	if (parts > 1) {
		cluster_barrier();
		if (rank == 0)
#pragma unroll
			for (int r = 0; r < ROWS; r++) {
				float z = sums[r][threadIdx.x];

				for (int k = 1; k < parts; k++)
					z += load_in(smem_in(smem_of(&sums[r][threadIdx.x]), k));
				sums[r][threadIdx.x] = z;
			}
		cluster_barrier();	/* nobody leaves before its sums have been read */
		if (rank != 0)
			return;
	}
#pragma unroll
	for (int r = 0; r < ROWS; r++) {
		float z = -INFINITY;
		float top;
		float sum;

		if ((int)threadIdx.x < width && mine < h.vocab) {
			z = sums[r][threadIdx.x] + (h.bias ? h.bias[mine] : 0.0f);
			if (h.target[r] == mine)
				h.hit[r] = z;
		}
		top = z;
#pragma unroll
		for (int k = 16; k > 0; k >>= 1)
			top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
		sum = exp2_approx((z - (top == -INFINITY ? 0.0f : top)) * LOG2E);
#pragma unroll
		for (int k = 16; k > 0; k >>= 1)
			sum += __shfl_xor_sync(0xffffffffu, sum, k);
		__syncthreads();
		if (lane == 0)
			warps[w] = make_float2(top, sum);
		__syncthreads();
		if (threadIdx.x == 0) {
			for (int k = 1; k < 8; k++)
				join(top, sum, warps[k]);
			h.part[(int64_t)tile * h.tokens + r] = make_float2(top, sum);
		}
	}
}

/* ---- what goes before and after the products ------------------------------------------------------------ */

/* joins the tiles of a row: 32 warps share the tiles of 32 rows */
__global__ void __launch_bounds__(1024) join_kernel(const head_args h, int tiles)
{
	__shared__ float2 s[32][33];
	const int lane = threadIdx.x & 31;
	const int w = threadIdx.x >> 5;
	int t = blockIdx.x * 32 + lane;
	float top = -INFINITY;
	float sum = 0.0f;

	dependent();
	if (t < h.tokens) {
#pragma unroll 4
		for (int k = w; k < tiles; k += 32)
			join(top, sum, h.part[(int64_t)k * h.tokens + t]);
	}
	s[lane][w] = make_float2(top, sum);
	__syncthreads();
	/* warp w now joins row w */
	t = blockIdx.x * 32 + w;
	top = s[w][lane].x;
	sum = s[w][lane].y;
#pragma unroll
	for (int k = 16; k > 0; k >>= 1)
		join(top, sum, make_float2(__shfl_down_sync(0xffffffffu, top, k), __shfl_down_sync(0xffffffffu, sum, k)));
	if (lane == 0 && t < h.tokens) {
		const float lse = top + logf(sum);
		const int y = h.target[t];

		h.lse[t] = lse;
		h.nll[t] = y < 0 ? 0.0f : y >= h.vocab ? NAN : lse - h.hit[t];
	}
}

/* factor of each row: 0 where there is no gradient */
__device__ __forceinline__ float row_factor(const head_args &h, int t)
{
	const int y = h.target[t];

	return y >= 0 && y < h.vocab && h.lse[t] != -INFINITY ? h.scale * (h.weight ? h.weight[t] : 1.0f) : 0.0f;
}

/* a matrix to be copied to rows on the 16-byte grid, by so many blocks */
struct pack_job {
	__nv_bfloat16		*to;
	const __nv_bfloat16	*from;
	int64_t			ldf;
	int			ldt;
	int			rows;
	int			cols;
	int			blocks;
};

/*
** The copies of x and w, 16 bytes a thread.  With `factors` also those of x's rows, and zeros for the rows
** without a gradient, so that whatever they hold meets a delta of 0 as 0.
*/
__global__ void __launch_bounds__(256) pack_kernel(const head_args h, const pack_job x, const pack_job w, int factors)
{
	const bool is_x = (int)blockIdx.x < x.blocks;
	const pack_job &p = is_x ? x : w;
	const int block = is_x ? blockIdx.x : blockIdx.x - x.blocks;
	const int per = p.ldt / 8;
	const int64_t total = (int64_t)p.rows * per;

	dependent();
	for (int64_t i = (int64_t)block * 256 + threadIdx.x; i < total; i += (int64_t)p.blocks * 256) {
		const int r = (int)(i / per);
		const int c = (int)(i - (int64_t)r * per) * 8;
		const float f = is_x && factors ? row_factor(h, r) : 1.0f;
		const __nv_bfloat16 *src = p.from + (int64_t)r * p.ldf + c;
		uint32_t q[4] = { 0, 0, 0, 0 };

		if (is_x && factors && c == 0)
			h.row[r] = f;
		if (f != 0.0f) {
			if (c + 8 <= p.cols && ((uintptr_t)src & 15) == 0)
				*reinterpret_cast<uint4 *>(q) = *reinterpret_cast<const uint4 *>(src);
			else
#pragma unroll
				for (int j = 0; j < 8; j++)
					if (c + j < p.cols)
						q[j / 2] |= (uint32_t)reinterpret_cast<const uint16_t *>(src)[j] << (j % 2 * 16);
		}
		*reinterpret_cast<uint4 *>(p.to + (int64_t)r * p.ldt + c) = make_uint4(q[0], q[1], q[2], q[3]);
	}
}

/* the parts of dx added up in order; a block takes a row at a time */
__global__ void __launch_bounds__(128) finish_dx_kernel(const head_args h)
{
	dependent();
	for (int t = blockIdx.x; t < h.tokens; t += gridDim.x) {
		const int size = h.bf16 ? 2 : 4;
		char *out = static_cast<char *>(h.dx) + (int64_t)t * h.lddx * size;

		for (int d = threadIdx.x * 4; d < h.d; d += 128 * 4) {
			float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);

			for (int k = 0; k < h.splits; k++) {
				const float4 q = *reinterpret_cast<const float4 *>(h.dxp + ((int64_t)k * h.tokens + t) * h.ldd + d);

				v.x += q.x;
				v.y += q.y;
				v.z += q.z;
				v.w += q.w;
			}
			if (d + 4 <= h.d && ((uintptr_t)out & 15) == 0) {
				if (h.bf16)
					*reinterpret_cast<uint2 *>(out + d * 2) = make_uint2(bf16_pair(v.x, v.y), bf16_pair(v.z, v.w));
				else
					*reinterpret_cast<float4 *>(out + d * 4) = v;
			} else {
				const float e[4] = { v.x, v.y, v.z, v.w };

#pragma unroll
				for (int j = 0; j < 4; j++)
					if (d + j < h.d)
						put(out, d + j, e[j], h.bf16, 0);
			}
		}
	}
}

/* where no product of gradients follows, which would do it */
__global__ void __launch_bounds__(256) finish_db_kernel(const head_args h)
{
	dependent();
	finish_db(h, blockIdx.x * blockDim.x + threadIdx.x, h.vocab, gridDim.x * blockDim.x);
}

/* ---- host --------------------------------------------------------------------------------------- */

int check(const anni_head_call *c, int grad)
{
	if (!c || c->tokens < 0 || c->d_model < 1 || c->vocab < 1)
		return ANNI_E_ARG;
	if (c->tokens > ANNI_HEAD_MAX_TOKENS || c->d_model > ANNI_HEAD_MAX_DIM || c->vocab > ANNI_HEAD_MAX_VOCAB)
		return ANNI_E_LIMIT;
	if ((up(c->tokens, HEAD_TM) / HEAD_TM) * (up(c->vocab, HEAD_TN) / HEAD_TN) > 0x3fffffff)
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

head_args args_of(const anni_head_call *c, const head_plan &p)
{
	head_args h;
	char *ws = static_cast<char *>(c->workspace);

	memset(&h, 0, sizeof(h));
	h.x = p.copy_x ? reinterpret_cast<const __nv_bfloat16 *>(ws + p.x) : static_cast<const __nv_bfloat16 *>(c->x);
	h.ldx = p.copy_x ? p.ldx : c->ldx;
	h.w = p.copy_w ? reinterpret_cast<const __nv_bfloat16 *>(ws + p.w) : static_cast<const __nv_bfloat16 *>(c->w);
	h.ldw = p.copy_w ? p.ldw : c->ldw;
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
	h.dxp = p.parts ? reinterpret_cast<float *>(ws + p.dxp) : NULL;
	h.ldd = p.ldd;
	h.splits = p.splits;
	h.dbp = reinterpret_cast<float *>(ws + p.dbp);
	h.dx = c->dx;
	h.lddx = c->lddx;
	h.dw = c->dw;
	h.lddw = c->lddw;
	h.db = c->dbias;
	h.bf16 = c->grad_dtype == ANNI_DT_BF16;
	h.add = (c->flags & ANNI_HEAD_ACCUMULATE) != 0;
	return h;
}

unsigned tiles(int64_t n, int64_t of)
{
	return (unsigned)((n + of - 1) / of);
}

/*
** Launches a kernel that may start before the one ahead of it in the stream has ended: its blocks set themselves
** up meanwhile and wait (dependent()) before they touch memory.
*/
template <typename... P, typename... A>
int launch_clusters(void (*kernel)(P...), int64_t grid, int threads, int smem, cudaStream_t st, int cluster, A... args)
{
	cudaLaunchConfig_t cfg = {};
	cudaLaunchAttribute attrs[2];

	attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
	attrs[0].val.programmaticStreamSerializationAllowed = 1;
	attrs[1].id = cudaLaunchAttributeClusterDimension;
	attrs[1].val.clusterDim.x = (unsigned)cluster;
	attrs[1].val.clusterDim.y = 1;
	attrs[1].val.clusterDim.z = 1;
	cfg.gridDim = dim3((unsigned)grid);
	cfg.blockDim = dim3((unsigned)threads);
	cfg.dynamicSmemBytes = (size_t)smem;
	cfg.stream = st;
	cfg.attrs = attrs;
	cfg.numAttrs = cluster > 1 ? 2 : 1;	/* 1: none, or the kernel's own */
	if (cudaLaunchKernelEx(&cfg, kernel, P(args)...) != cudaSuccess) {
		(void)cudaGetLastError();
		return ANNI_E_CUDA;
	}
	anni_count_launch();
	return ANNI_OK;
}

template <typename... P, typename... A>
int launch(void (*kernel)(P...), int64_t grid, int threads, int smem, cudaStream_t st, A... args)
{
	return launch_clusters(kernel, grid, threads, smem, st, 1, args...);
}

/* blocks of 256 threads with 16 bytes each */
int64_t blocks(int64_t rows, int64_t ld)
{
	return std::min<int64_t>((rows * ld / 8 + 255) / 256, 16 * 2 * HEAD_PAIRS);
}

typedef CUresult (*encode_fn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
    const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
    CUtensorMapFloatOOBfill);
encode_fn g_encode;
std::once_flag g_encode_once;

void find_encode(void)
{
	void *p = NULL;
	cudaDriverEntryPointQueryResult st;

	if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &st) == cudaSuccess
	    && st == cudaDriverEntryPointSuccess)
		g_encode = reinterpret_cast<encode_fn>(p);
	else
		(void)cudaGetLastError();
}

/* bf16 [deep][rows][ld], of which `cols` columns exist, in boxes of 64 columns and `box` rows, 128-byte swizzle */
int tensor_map(CUtensorMap *m, const void *base, int64_t cols, int64_t rows, int64_t ld, int deep, int box)
{
	const cuuint64_t dims[3] = { (cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)deep };
	const cuuint64_t strides[2] = { (cuuint64_t)ld * 2, (cuuint64_t)ld * 2 * (cuuint64_t)rows };
	const cuuint32_t boxes[3] = { 64, (cuuint32_t)box, 1 };
	const cuuint32_t one[3] = { 1, 1, 1 };

	std::call_once(g_encode_once, find_encode);
	if (!g_encode)
		return ANNI_E_CUDA;
	return g_encode(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(base), dims, strides, boxes, one,
	    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
	    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? ANNI_OK : ANNI_E_CUDA;
}

/*
** Number of SMs of the current device, and the kernel's shared memory allowed on it; asked for once per device
** (devices beyond the table are asked every time).
*/
#define HEAD_DEVICES	16
std::atomic<int> known[3][HEAD_DEVICES];
std::atomic<int> known_rows[2][HEAD_DEVICES];

template <typename K>
int ready(K kernel, int smem, int *sms, std::atomic<int> (*seen)[HEAD_DEVICES])
{
	int dev = 0;
	int n = 0;

	if (cudaGetDevice(&dev) != cudaSuccess)
		return ANNI_E_CUDA;
	n = dev < HEAD_DEVICES ? (*seen)[dev].load(std::memory_order_relaxed) : 0;
	if (n == 0) {
		if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess
		    || cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) {
			(void)cudaGetLastError();
			return ANNI_E_CUDA;
		}
		if (dev < HEAD_DEVICES)
			(*seen)[dev].store(n, std::memory_order_relaxed);
	}
	*sms = n;
	return ANNI_OK;
}

/* the products of one kind over the piece h.v0 .. h.v1 of the vocabulary */
template <int KIND>
int product(const head_args &h, cudaStream_t st)
{
	const int smem = HEAD_STAGES * HEAD_STAGE_BYTES + 1024;
	const int width = h.v1 - h.v0;
	const bool f32 = h.terms > 1;
	gemm_args g;
	int sms;
	int rc = ANNI_OK;

	memset(&g, 0, sizeof(g));
	g.h = h;
	if (KIND == GRAD) {
		const int splits = g.h.splits = parts_of(h.splits, width);
		const grad_work w = work_of(h.tokens, h.d, width, h.terms, h.dx != NULL, h.dw != NULL, splits,
		    epilogue_of_dw(h.dw, h.lddw, h.bf16, h.add));
		product_args &x = g.p[DX];
		product_args &y = g.p[DW];

		order(w, &g.first, &g.extra);
		x.m_tiles = (int)tiles(h.tokens, HEAD_TM);
		x.n_tiles = (int)tiles(h.d, HEAD_TN);
		x.k_blocks = (int)tiles(width, HEAD_TK);
		y.m_tiles = (int)tiles(h.d, HEAD_TM);
		y.n_tiles = (int)tiles(width, HEAD_TN);
		y.k_blocks = (int)tiles(h.tokens, HEAD_TK);
		/* fp32 gradients are to be good to fp32; 1.1e-4 of a sum is a thirty-fifth of half a step of bf16 */
		x.run = y.run = f32 ? HEAD_RUN_F32 : HEAD_RUN_BF16;
		x.total = (int)w.tiles[DX];
		y.total = (int)w.tiles[DW];
		rc = tensor_map(&x.a, h.delta, width, h.tokens, h.ldp, h.terms, HEAD_HALF);
		rc = rc ? rc : tensor_map(&x.b, h.w, h.vocab, h.d, h.ldw, 1, HEAD_HALF);
		rc = rc ? rc : tensor_map(&y.a, h.x, h.d, h.tokens, h.ldx, 1, HEAD_TK);
		rc = rc ? rc : tensor_map(&y.b, h.delta, width, h.tokens, h.ldp, h.terms, HEAD_TK);
	} else {
		product_args &z = g.p[0];

		z.m_tiles = (int)tiles(h.tokens, HEAD_TM);
		z.n_tiles = (int)tiles(width, HEAD_TN);
		z.k_blocks = (int)tiles(h.d, HEAD_TK);
		/* a logit's error is a relative one of delta: of a logit of 20 a seventh of half a step of bf16 */
		z.run = KIND == LOSS || f32 ? HEAD_RUN : HEAD_RUN_DELTA;
		z.total = z.m_tiles * z.n_tiles;
		rc = tensor_map(&z.a, h.x, h.d, h.tokens, h.ldx, 1, HEAD_HALF);
		rc = rc ? rc : tensor_map(&z.b, h.w, h.vocab, h.d, h.ldw, 1, HEAD_TK);
	}
	rc = rc ? rc : ready(product_kernel<KIND>, smem, &sms, &known[KIND]);
	if (rc != ANNI_OK)
		return rc;
	return launch(product_kernel<KIND>, 2 * std::min<int64_t>(sms / 2, (int64_t)g.p[0].total + g.p[1].total), HEAD_THREADS, smem,
	    st, g);
}

template <int ROWS>
int loss_rows(const head_args &h, int width, cudaStream_t st)
{
	const int n = (int)tiles(h.vocab, width);
	int64_t least = 0;
	int parts = 1;
	int deep;
	int sms;
	int rc = ready(rows_kernel<ROWS>, ROWS * HEAD_FEW_DIM * 4, &sms, &known_rows[ROWS - 1]);

	/*
	** Few entries: the rows of W are split, so that every SM has blocks that read (1536 x 300, 8 us, unsplit 44).  Blocks
	** that run at a time: four an SM with one row (61 registers), three with two (68); a round that few blocks
	** are left for costs as much as a full one (two rows, 1536 x 65,536: 59 us in 512 blocks, 51 in 256).
	*/
	for (int p = 1; p <= 8 && (p == 1 || h.d >= p * ROWS_DEEP); p++) {
		const int64_t rounds = ((int64_t)n * p + (5 - ROWS) * 2 * HEAD_PAIRS - 1) / ((5 - ROWS) * 2 * HEAD_PAIRS);
		const int64_t time = rounds * (h.d / p + ROWS_START);

		if (p == 1 || time < least) {
			least = time;
			parts = p;
		}
	}
	deep = (int)up((h.d + parts - 1) / parts, 8);	/* a warp's rows are then eight apart from block to block, too */
	return rc ? rc : launch_clusters(rows_kernel<ROWS>, (int64_t)n * parts, 256, deep * ROWS * 4, st, parts, h, width, deep, parts);
}

/* the copies that the plan asks for, in one launch; x's with the factors of the rows when gradients follow */
int pack(const anni_head_call *c, const head_plan &p, const head_args &h, bool grad, cudaStream_t st)
{
	const pack_job x = { const_cast<__nv_bfloat16 *>(h.x), static_cast<const __nv_bfloat16 *>(c->x), c->ldx, (int)p.ldx, h.tokens,
	    h.d, p.copy_x ? (int)blocks(h.tokens, p.ldx) : 0 };
	const pack_job w = { const_cast<__nv_bfloat16 *>(h.w), static_cast<const __nv_bfloat16 *>(c->w), c->ldw, (int)p.ldw, h.d,
	    h.vocab, p.copy_w ? (int)blocks(h.d, p.ldw) : 0 };

	return x.blocks + w.blocks == 0 ? ANNI_OK : launch(pack_kernel, x.blocks + w.blocks, 256, 0, st, h, x, w, (int)grad);
}

}	/* namespace */

extern "C" int anni_head_workspace(const anni_head_call *c, int grad, size_t *bytes)
{
	int rc = check(c, grad);

	if (rc != ANNI_OK || !bytes)
		return rc != ANNI_OK ? rc : ANNI_E_ARG;
	*bytes = workspace_of(c, grad);
	return ANNI_OK;
}

extern "C" int anni_head_loss(const anni_head_call *c, void *stream)
{
	cudaStream_t st = (cudaStream_t)stream;
	int rc = check(c, 0);
	head_plan p;
	head_args h;
	int width = HEAD_TN;

	if (rc != ANNI_OK || c->tokens == 0)
		return rc;
	p = plan_of(c, 0);
	rc = check_buffers(c, 0, p.bytes);
	if (rc != ANNI_OK)
		return rc;
	h = args_of(c, p);
	rc = pack(c, p, h, false, st);
	h.v1 = h.vocab;
	if (rc == ANNI_OK && p.few) {
		width = (h.ldw & 7) || ((uintptr_t)h.w & 15) ? ROWS_ODD_TN : HEAD_TN;
		rc = h.tokens == 1 ? loss_rows<1>(h, width, st) : loss_rows<2>(h, width, st);
	} else if (rc == ANNI_OK)
		rc = product<LOSS>(h, st);
	if (rc == ANNI_OK)
		rc = launch(join_kernel, tiles(h.tokens, 32), 1024, 0, st, h, (int)tiles(h.vocab, width));
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
	rc = pack(c, p, h, true, st);
	for (h.v0 = 0; rc == ANNI_OK && h.v0 < h.vocab; h.v0 = h.v1) {
		h.v1 = std::min(h.vocab, h.v0 + p.piece);
		rc = product<DELTA>(h, st);
		if (rc == ANNI_OK && (h.dx || h.dw))
			rc = product<GRAD>(h, st);
	}
	if (rc == ANNI_OK && h.dxp)
		rc = launch(finish_dx_kernel, std::min(h.tokens, 16384), 128, 0, st, h);
	if (rc == ANNI_OK && h.db && !h.dx && !h.dw)
		rc = launch(finish_db_kernel, tiles(h.vocab, 256), 256, 0, st, h);
	return rc;
}
