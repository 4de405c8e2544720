"""The list step next to other streams."""
import pytest
import torch

from anni_b200.capi import DT_BF16, DT_F32, DT_Q8
from test_mtstep import HYP, Case, hyper

gpu = pytest.mark.gpu
CYCLES = 20_000_000             # about 10 ms of a stream kept busy


@gpu
@pytest.mark.parametrize("state_dtype", [DT_F32, DT_Q8])
def test_tables_are_there_when_creation_returns(state_dtype):
    """Creation behind a busy default stream: nothing of it is under way any more when a non-blocking stream steps."""
    st = torch.cuda.Stream()
    c = Case([300, 5000, 70001], DT_BF16, state_dtype, seed=51)
    torch.cuda.synchronize()
    torch.cuda._sleep(CYCLES)
    c.step = type(c.step)(c.p, grads=c.g, state_dtype=state_dtype, decay=c.decay, twins=c.twin, moments=(c.m, c.v),
                          scales=(c.ms, c.vs) if c.eight else None)
    assert torch.cuda.default_stream().query()
    c.step.step(hyper(0.1), stream=st)
    torch.cuda.synchronize()
    c.check(HYP, clip=0.1)
