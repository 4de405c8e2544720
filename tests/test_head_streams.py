"""The head on a stream that is not its tensors' own: their memory is not handed out again before it is done with them.

What is given to the call dies right after it, while the stream is still busy with something else; memory of the same
sizes, allocated next, is overwritten at once.
"""
import pytest
import torch

from anni_b200.head import head_loss, head_loss_grad
from test_head import BF, inputs

gpu = pytest.mark.gpu
CYCLES = 200_000_000            # about 100 ms of a stream kept busy
T, D, V = 2048, 512, 4096       # blocks of megabytes, which the allocator hands out whole


def spoil(*shapes_and_types):
    return [torch.full(s, float("nan") if k.is_floating_point else -7, dtype=k, device="cuda") for s, k in shapes_and_types]


@gpu
def test_inputs_outlive_the_call():
    x, w, target, b = inputs(T, D, V, seed=60)
    nll, lse = head_loss(x, w, target, bias=b)
    dx, dw = torch.zeros(T, D, dtype=BF, device="cuda"), torch.zeros(D, V, dtype=BF, device="cuda")
    head_loss_grad(x, w, target, lse, bias=b, dx=dx, dw=dw)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    given = [a.clone() for a in (x, w, target, b)]
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        torch.cuda._sleep(CYCLES)
    got = head_loss(*given[:3], bias=given[3], stream=st)
    del given
    kept = spoil(((T, D), BF), ((D, V), BF), ((T,), torch.int32), ((V,), torch.float32))
    torch.cuda.synchronize()
    assert torch.equal(got[0], nll) and torch.equal(got[1], lse)
    del kept

    given = [a.clone() for a in (x, w, target, b, lse)]
    mine = torch.empty_like(dx), torch.empty_like(dw)
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        torch.cuda._sleep(CYCLES)
    head_loss_grad(*given[:3], given[4], bias=given[3], dx=mine[0], dw=mine[1], stream=st)
    del given
    kept = spoil(((T, D), BF), ((D, V), BF), ((T,), torch.int32), ((V,), torch.float32), ((T,), torch.float32))
    torch.cuda.synchronize()
    assert torch.equal(mine[0], dx) and torch.equal(mine[1], dw)
    del kept


@gpu
def test_results_outlive_their_stream():
    """nll and lse, allocated on the given stream and read on the caller's, which is behind."""
    t = 1 << 19
    x, w, target, _ = inputs(t, 8, 16, seed=61)
    want, _ = head_loss(x, w, target)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    nll, lse = head_loss(x, w, target, stream=st)
    torch.cuda.current_stream().wait_stream(st)
    torch.cuda._sleep(CYCLES)
    got = nll + 0
    del nll, lse
    with torch.cuda.stream(st):
        kept = spoil(((2, t), torch.float32))
    torch.cuda.synchronize()
    assert torch.equal(got, want) and kept[0].isnan().all()
