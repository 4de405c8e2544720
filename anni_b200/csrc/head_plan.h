/*
** How the work of a call of the head (include/anni_head.h) is cut: pieces of the vocabulary, parts of dx's sum
** over a piece, and what lies where in the workspace.  Host arithmetic on sizes, types and addresses alone.
*/
#ifndef ANNI_HEAD_PLAN_H__
#define ANNI_HEAD_PLAN_H__

#include <stddef.h>
#include <stdint.h>
#include <string.h>
#include <algorithm>
#include "anni_head.h"

#define HEAD_TM		256	/* rows and columns of a tile */
#define HEAD_TN		256
#define HEAD_HALF	128	/* rows of the result, and of either operand, in each block of the pair */
#define HEAD_TK		64	/* 128 bytes of bf16: the widest swizzle */
#define HEAD_PAIRS	74	/* pairs of SMs that the work is cut for; any number of them runs it */
#define HEAD_PIECE_BYTES ((size_t)256 << 20)	/* of delta in the workspace */
#define HEAD_TERMS	3	/* bf16 terms of delta for fp32 gradients */
#define HEAD_FEW_DIM	8192	/* rows_kernel keeps two rows of x in shared memory */
#define ROWS_ODD_TN	(HEAD_TN - 8)	/* its tile where the rows of W are off the 16-byte grid */

#ifdef __CUDACC__
#define HEAD_BOTH	__host__ __device__
#else
#define HEAD_BOTH
#endif

namespace {

enum { DX, DW };	/* the products of the gradients */

int64_t up(int64_t n, int64_t to)
{
	return (n + to - 1) / to * to;
}

/* the loss by rows_kernel, which takes x and w as they are */
bool few_rows(const anni_head_call *c)
{
	return c->tokens <= 2 && c->d_model <= HEAD_FEW_DIM;
}

/* where things lie in the workspace (byte offsets), and how the work is cut */
struct head_plan {
	size_t	x;		/* copies of x and w on a 16-byte grid, where needed */
	size_t	w;
	int	few;		/* rows_kernel */
	int	copy_x;
	int	copy_w;
	int64_t	ldx;
	int64_t	ldw;
	size_t	hit;
	size_t	part;
	size_t	row;
	size_t	delta;
	size_t	dxp;
	size_t	dbp;
	size_t	bytes;
	int	piece;
	int	terms;
	int	splits;
	int	parts;		/* dx is added up in fp32 in the workspace */
	int	ldd;
};

size_t take(size_t *at, int64_t bytes)
{
	const size_t here = *at;

	*at = (size_t)up((int64_t)here + bytes, 256);
	return here;
}

/*
** Tiles of the two products of the gradients over one piece of `width` columns, and how long a tile takes, in
** stages of 512 cycles: its stages (all terms), but no less than its epilogue (`least`, for dw): 6,000 cycles, 14,000
** where it adds to what is there, 20,000 where the rows of the result are off the 16-byte grid.
*/
struct grad_work {
	int64_t	tiles[2];
	int64_t	stages[2];
};

#define HEAD_EPI_STAGES		12
#define HEAD_EPI_STAGES_ADD	28
#define HEAD_EPI_STAGES_ODD	40

/* an epilogue of dw, in stages */
int epilogue_of_dw(const void *base, int64_t ld, bool bf16, bool add)
{
	return (((uintptr_t)base | (uintptr_t)(ld * (bf16 ? 2 : 4))) & 15) != 0 ? HEAD_EPI_STAGES_ODD
	    : add ? HEAD_EPI_STAGES_ADD : HEAD_EPI_STAGES;
}

grad_work work_of(int64_t tokens, int64_t d, int64_t width, int terms, bool dx, bool dw, int splits, int least)
{
	grad_work w;

	w.tiles[DX] = dx ? up(tokens, HEAD_TM) / HEAD_TM * (up(d, HEAD_TN) / HEAD_TN) * splits : 0;
	w.tiles[DW] = dw ? up(d, HEAD_TM) / HEAD_TM * (up(width, HEAD_TN) / HEAD_TN) : 0;
	w.stages[DX] = std::max<int64_t>((up(width, HEAD_TK) / HEAD_TK * terms + splits - 1) / splits, HEAD_EPI_STAGES);
	w.stages[DW] = std::max<int64_t>(up(tokens, HEAD_TK) / HEAD_TK * terms, least);
	return w;
}

/* where part `part` of a sum over `stages` begins, of so many parts */
HEAD_BOTH inline int part_begin(int stages, int part, int parts)
{
	return (int)((int64_t)stages * part / parts);
}

/*
** Parts of dx's sum over a piece of `width` columns.  The last piece may be as short as one column and have fewer
** stages than a full one has parts; every part must have one, since an accumulator that nothing was multiplied into
** holds no zero.
*/
inline int parts_of(int splits, int64_t width)
{
	return (int)std::min<int64_t>(splits, up(width, HEAD_TK) / HEAD_TK);
}

/* which product goes first, and how many tiles of the other make up for one of it */
void order(const grad_work &w, int *first, int *extra)
{
	*first = w.stages[DX] >= w.stages[DW] ? DX : DW;
	*extra = (int)((w.stages[*first] + w.stages[1 - *first] / 2) / w.stages[1 - *first]);
}

/*
** Into how many parts the sum over the vocabulary in dx is cut: as many as make the busiest pair of SMs finish
** first.  A stage takes a pair 512 cycles (0.27 us); every part is written and read once more as fp32, at 6.5 TB/s.
** With dw's tiles to fill the rounds one part is best for many rows; a few rows have few tiles of dx, whose sums
** are as long as the vocabulary (128 rows of 1536 against 100,000 entries: 6 tiles of 1563 stages).
*/
int split_dx(int64_t tokens, int64_t d, int64_t width, int terms, bool dw, int least_dw)
{
	const int64_t stages = up(width, HEAD_TK) / HEAD_TK;
	int best = 1;
	double least = 0.0;

	for (int n = 1; n <= HEAD_PAIRS && (n == 1 || stages / n >= 4); n++) {
		const grad_work w = work_of(tokens, d, width, terms, true, dw, n, least_dw);
		int first;
		int extra;
		int64_t full;
		int64_t fill;
		int64_t most;
		int64_t least_long;
		double time;

		order(w, &first, &extra);
		full = w.tiles[first] % HEAD_PAIRS;
		least_long = w.tiles[first] / HEAD_PAIRS * w.stages[first];
		fill = std::min(w.tiles[1 - first], (HEAD_PAIRS - full) * extra);
		/* pairs with one more of the long tiles, and those that got short ones for it; then the rest for all */
		most = std::max(full ? least_long + w.stages[first] : 0,
		    least_long + (fill + HEAD_PAIRS - full - 1) / (HEAD_PAIRS - full) * w.stages[1 - first]);
		most += (w.tiles[1 - first] - fill + HEAD_PAIRS - 1) / HEAD_PAIRS * w.stages[1 - first];
		time = (double)most * 0.27 + (n > 1 ? 3.0 + n * (double)tokens * (double)d * 8.0 / 6.5e6 : 0.0);
		if (n == 1 || time < least * 0.98) {
			least = time;
			best = n;
		}
	}
	return best;
}

/* `least`: stages of an epilogue of dw */
head_plan plan_of(const anni_head_call *c, int grad, int least)
{
	head_plan p;
	const int64_t t = std::max<int64_t>(c->tokens, 1);

	memset(&p, 0, sizeof(p));
	p.few = !grad && few_rows(c);
	p.copy_x = grad || (!p.few && ((c->ldx & 7) || ((uintptr_t)c->x & 15)));
	p.copy_w = !p.few && ((c->ldw & 7) || ((uintptr_t)c->w & 15));
	p.ldx = up(c->d_model, 8);
	p.ldw = up(c->vocab, 8);
	p.x = take(&p.bytes, p.copy_x ? t * p.ldx * 2 : 0);
	p.w = take(&p.bytes, p.copy_w ? c->d_model * p.ldw * 2 : 0);
	if (!grad) {
		p.hit = take(&p.bytes, t * 4);
		p.part = take(&p.bytes, up(c->vocab, ROWS_ODD_TN) / ROWS_ODD_TN * t * 8);
		return p;
	}
	p.terms = c->grad_dtype == ANNI_DT_BF16 ? 1 : HEAD_TERMS;
	/* as many columns of delta as HEAD_PIECE_BYTES hold, then pieces of about the same size */
	p.piece = (int)std::max<int64_t>(HEAD_TN, (int64_t)(HEAD_PIECE_BYTES / (size_t)(t * 2 * p.terms)) / HEAD_TN * HEAD_TN);
	p.piece = (int)up((c->vocab + (c->vocab + p.piece - 1) / p.piece - 1) / ((c->vocab + p.piece - 1) / p.piece), HEAD_TN);
	p.row = take(&p.bytes, t * 4);
	p.delta = take(&p.bytes, (int64_t)p.piece * t * 2 * p.terms);
	p.ldd = (int)up(c->d_model, 8);
	p.splits = c->dx ? split_dx(t, c->d_model, std::min(p.piece, c->vocab), p.terms, c->dw != NULL, least) : 1;
	p.parts = c->dx && (p.splits > 1 || p.piece < c->vocab);
	p.dxp = take(&p.bytes, p.parts ? p.splits * t * p.ldd * 4 : 0);
	p.dbp = take(&p.bytes, c->dbias ? up(t, HEAD_HALF) / HEAD_HALF * c->vocab * 4 : 0);
	return p;
}

head_plan plan_of(const anni_head_call *c, int grad)
{
	return plan_of(c, grad, epilogue_of_dw(c->dw, c->lddw, c->grad_dtype == ANNI_DT_BF16,
	    (c->flags & ANNI_HEAD_ACCUMULATE) != 0));
}

/* bytes of workspace wherever dw lies, and whether it is added to or not: the parts of dx depend on it */
size_t workspace_of(const anni_head_call *c, int grad)
{
	size_t most = 0;

	for (int least : { HEAD_EPI_STAGES, HEAD_EPI_STAGES_ADD, HEAD_EPI_STAGES_ODD })
		most = std::max(most, plan_of(c, grad, least).bytes);
	return most;
}

}	/* namespace */

#endif
