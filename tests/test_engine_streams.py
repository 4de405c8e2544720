"""The arena engine next to other streams."""
import pytest
import torch

from anni_b200.capi import DT_BF16, check
from anni_b200.engine import LM_SHAPES, OptStep, lm_segments

gpu = pytest.mark.gpu
CYCLES = 200_000_000            # about 100 ms of a stream kept busy


@gpu
def test_tables_are_there_when_creation_returns():
    """Creation, and a change of the loss scale, behind a busy default stream: a step on a non-blocking one may follow."""
    segs = lm_segments(**LM_SHAPES["tiny"], wd="matrices")
    torch.cuda.synchronize()
    torch.cuda._sleep(CYCLES)
    eng = OptStep(segs, grad_dtype=DT_BF16)
    assert torch.cuda.default_stream().query()
    eng.allocate()
    torch.cuda.synchronize()
    torch.cuda._sleep(CYCLES)
    check("anni_optstep_loss_scale_init", eng.L.anni_optstep_loss_scale_init(eng.h, 8.0, 100, 2.0, 0.5, 1.0, 64.0))
    assert torch.cuda.default_stream().query()
    assert eng.status().loss_scale == 8.0
