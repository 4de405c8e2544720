"""The list step next to other streams."""
import pytest
import torch

from anni_b200.capi import DT_BF16, DT_F32, DT_Q8
from test_mtstep import HYP, Case, hyper

gpu = pytest.mark.gpu
CYCLES = 200_000_000            # about 100 ms of a stream kept busy


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


@gpu
@pytest.mark.parametrize("how", ["step", "set_grads", "constructor"])
def test_gradients_outlive_the_step(how):
    """A step queued on a busy stream, its gradients replaced and dropped at once: their memory is not handed out yet."""
    sizes = [1 << 20, 700001]
    c = Case(sizes, DT_F32, DT_F32, seed=52)
    st = torch.cuda.Stream()
    g = [x.clone() for x in c.g]
    c.step = type(c.step)(c.p, grads=g if how == "constructor" else c.g, decay=c.decay, twins=c.twin, moments=(c.m, c.v))
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        torch.cuda._sleep(CYCLES)
    if how == "step":
        c.step.step(hyper(0.1), grads=g, stream=st)
    else:
        if how == "set_grads":
            c.step.set_grads(g, stream=st)
        c.step.step(hyper(0.1), stream=st)
    c.step.set_grads(c.g, stream=st)
    del g
    kept = [torch.full((n,), float("nan"), device="cuda") for n in sizes]
    torch.cuda.synchronize()
    c.check(HYP, clip=0.1)
    assert c.step.status().skipped == 0 and all(x.isnan().all() for x in kept)
