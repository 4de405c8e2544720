"""How the head's gradients are cut into pieces of the vocabulary, and a piece's sum over the vocabulary into parts."""
import pytest
import torch

from anni_b200.head import head_loss, head_loss_grad
from test_head import BF, F32, Exact, check_grads, inputs

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("t,d,v,kind,with_dw", [(12288, 64, 50257, F32, False), (12288, 512, 46593, F32, False),
                                                (6000, 256, 207936, F32, True), (18083, 512, 258078, BF, True)])
def test_last_piece_shorter_than_the_parts(t, d, v, kind, with_dw):
    """dx where the last piece has fewer blocks of 64 entries than a full piece's sum has parts.

    The rows after the first 64 are ignored: with few rows the definition in 64 bits takes little memory, and the cut
    depends on the number of rows alone."""
    x, w, target, b = inputs(t, d, v, seed=30, ignored=0.0)
    target[64:] = -1
    lse = torch.zeros(t, device="cuda")
    _, lse[:64] = head_loss(x[:64], w, target[:64], bias=b)
    dx = torch.full((t, d), float("nan"), dtype=kind, device="cuda")
    dw = torch.full((d, v), float("nan"), dtype=kind, device="cuda") if with_dw else None
    for _ in range(3):
        head_loss_grad(x, w, target, lse, bias=b, dx=dx, dw=dw)
        ex = Exact(x[:64], w, target[:64], b)
        ex.t = t                # terms of dw's sum
        check_grads(ex, kind, dx=dx[:64])
        assert not dx[64:].any()
        if with_dw:
            check_grads(ex, kind, dw=dw)
