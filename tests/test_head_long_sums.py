"""Sums of the head's bf16 gradients over more terms than one run of the tensor cores may take."""
import pytest
import torch

from anni_b200.head import head_loss, head_loss_grad
from test_head import BF, Exact, both, check_grads, check_loss, inputs

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("t,d,v", [(130, 4096, 520), (130, 4097, 520), (70, 9001, 300), (300, 64, 40000), (2050, 1000, 33000),
                                   (16384, 64, 300), (16385, 64, 300), (40000, 72, 264)])
def test_a_run_and_one_term_more(t, d, v):
    """Each of the three sums at the length of one run, just beyond it, and of several."""
    x, w, target, b = inputs(t, d, v, seed=41)
    nll, lse, dx, dw, db = both(x, w, target, b, BF)
    ex = Exact(x, w, target, b)
    check_loss(ex, nll, lse)
    check_grads(ex, BF, dx=dx, dw=dw, db=db)


@gpu
def test_dw_over_eight_million_rows():
    """dw of sums that do not cancel (x > 0, one target for all rows) against 64 bits.

    Off by at most: delta's rounding and the result's, 2^-8 each; delta itself, whose logits have 8 terms, 2^-19; a
    run of at most 16,384 terms in fp32, cut off: 16,384 / 16 + 8 additions of 2^-23; the 512 runs added up, 2^-24 each.
    """
    t, d, v = 1 << 23, 8, 16
    g = torch.Generator(device="cuda").manual_seed(40)
    x = (torch.rand(t, d, generator=g, device="cuda") + 0.5).bfloat16()
    w = (torch.randn(d, v, generator=g, device="cuda") * 0.3).bfloat16()
    target = torch.zeros(t, dtype=torch.int32, device="cuda")
    _, lse = head_loss(x, w, target)
    dw = torch.empty(d, v, dtype=torch.bfloat16, device="cuda")
    head_loss_grad(x, w, target, lse, dw=dw, grad_scale=1 / 1024)
    want = torch.zeros(d, v, dtype=torch.float64, device="cuda")
    for a in range(0, t, 1 << 20):
        xd = x[a:a + (1 << 20)].double()
        p = torch.softmax(xd @ w.double(), 1)
        p[:, 0] -= 1.0
        want += xd.t() @ p / 1024
    bound = 2 * 2.0 ** -8 + 2.0 ** -16 + 2.0 ** -19 + (16384 / 16 + 8) * 2.0 ** -23 + 512 * 2.0 ** -24
    off = (dw.double() / want - 1).abs()
    assert (off <= bound).all(), float(off.max())
