"""The size of the head's workspace: of sizes, types, addresses of x and w, and of which outputs are wanted, and nothing else."""
import ctypes as C
import random

import pytest

from anni_b200 import capi, head
from test_head import _c


def need(**kw):
    n = C.c_size_t()
    assert head.lib().anni_head_workspace(C.byref(_c(**kw)), 1, C.byref(n)) == capi.OK
    return n.value


@pytest.mark.parametrize("seed", range(4))
def test_where_dw_lies_makes_no_difference(seed):
    """Asked for before dw's address and stride are known, or for a first call that does not add yet."""
    r = random.Random(seed)
    for _ in range(400):
        t, d, v = (int(2 ** r.uniform(0, k)) for k in (14, 12, 18))
        kind = r.choice((capi.DT_F32, capi.DT_BF16))
        sizes = dict(tokens=t, d_model=d, vocab=v, ldx=d, ldw=v, lddx=d, grad_dtype=kind)
        got = {need(**sizes, dw=dw, lddw=ld, flags=flags) for dw in (0x50000000, 0x50000004) for ld in (v, v + 1, -(-v // 8) * 8)
               for flags in (0, head.HEAD_ACCUMULATE)}
        assert len(got) == 1, (sizes, got)
