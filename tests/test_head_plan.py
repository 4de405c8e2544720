"""How a call of the head's gradients is cut (csrc/head_plan.h), walked on the CPU over many sizes."""
import os
import subprocess

from conftest import ROOT

WALK = r"""
#include <stdio.h>
#include <stdlib.h>
#include "head_plan.h"

/* one call: every piece of the vocabulary, every part of dx's sum over it */
static int walk(int64_t t, int d, int v, int dtype, int dw, int add, int odd)
{
	anni_head_call c;
	head_plan p;
	int v0;

	memset(&c, 0, sizeof(c));
	c.tokens = t, c.d_model = d, c.vocab = v, c.ldx = d, c.ldw = v, c.lddx = d, c.lddw = v + odd;
	c.grad_dtype = dtype, c.flags = add ? ANNI_HEAD_ACCUMULATE : 0;
	c.x = c.w = (void *)4096;
	c.dx = (void *)4096;
	c.dw = dw ? (void *)4096 : NULL;
	p = plan_of(&c, 1);
	for (v0 = 0; v0 < v; v0 += p.piece) {
		const int width = std::min(p.piece, v - v0);
		const int stages = (width + HEAD_TK - 1) / HEAD_TK;
		const int parts = parts_of(p.splits, width);
		int at = 0;
		int k;

		/* the first piece stores, so it has every part that is added up in the end */
		if (parts < 1 || parts > p.splits || (v0 == 0 && parts != p.splits) || (parts > 1 && !p.parts))
			return printf("%ld %d %d: %d parts of %d in the piece at %d\n", (long)t, d, v, parts, p.splits, v0), 1;
		for (k = 0; k < parts; k++) {
			if (part_begin(stages, k, parts) != at || part_begin(stages, k + 1, parts) <= at)
				return printf("%ld %d %d type %d: part %d of %d is empty in the piece of %d columns at %d\n",
				    (long)t, d, v, dtype, k, parts, width, v0), 1;
			at = part_begin(stages, k + 1, parts);
		}
		if (at != stages)
			return printf("%ld %d %d: stages left over\n", (long)t, d, v), 1;
	}
	return 0;
}

static double uniform(void)
{
	return rand() / (RAND_MAX + 1.0);
}

int main(void)
{
	static const int known[][4] = { { 18083, 512, 258078, ANNI_DT_BF16 }, { 6000, 256, 207936, ANNI_DT_F32 },
	    { 12288, 512, 46593, ANNI_DT_F32 }, { 8192, 64, 107521, ANNI_DT_F32 }, { 27600, 64, 92190, ANNI_DT_BF16 },
	    { 12288, 64, 50257, ANNI_DT_F32 }, { 24576, 64, 50257, ANNI_DT_F32 }, { 8192, 64, 107541, ANNI_DT_F32 } };
	int bad = 0;
	int i;

	for (i = 0; i < 8; i++)
		bad += walk(known[i][0], known[i][1], known[i][2], known[i][3], 0, 0, 0)
		    + walk(known[i][0], known[i][1], known[i][2], known[i][3], 1, 0, 0);
	srand(1);
	for (i = 0; i < 20000; i++) {
		const int64_t t = (int64_t)exp2(uniform() * 20);
		const int d = (int)exp2(uniform() * 13);
		const int v = (int)exp2(uniform() * 20);
		const int r = rand() >> 8;

		bad += walk(t, d, v, r & 1 ? ANNI_DT_F32 : ANNI_DT_BF16, r >> 1 & 1, r >> 2 & 1, r >> 3 & 1);
	}
	return bad != 0;
}
"""


def test_no_part_of_a_sum_is_empty(tmp_path):
    src, exe = tmp_path / "walk.cpp", tmp_path / "walk"
    src.write_text("#include <math.h>\n" + WALK)
    subprocess.run(["g++", "-O1", "-std=c++17", "-I", os.path.join(ROOT, "include"),
                    "-I", os.path.join(ROOT, "anni_b200", "csrc"), "-o", str(exe), str(src)], check=True)
    got = subprocess.run([str(exe)], capture_output=True, text=True)
    assert got.returncode == 0, got.stdout[-2000:]
