"""State handed to the list step, and state asked of it."""
import pytest
import torch

from anni_b200 import mtstep
from anni_b200.capi import DT_F32, DT_Q8
from anni_b200.mtstep import MultiStep

gpu = pytest.mark.gpu


def test_8_bit_moments_without_scales_are_refused():
    """Codes mean nothing without their scales; zeros in their place would lose the moments silently."""
    p = torch.zeros(300)
    m, v = (torch.ones(300).to(k) for k in (torch.float8_e4m3fn, torch.float8_e5m2))
    with pytest.raises(ValueError, match="scales"):
        MultiStep([p], state_dtype=DT_Q8, moments=([m], [v]))


@gpu
@pytest.mark.parametrize("state_dtype", [DT_F32, DT_Q8])
@pytest.mark.parametrize("given", [False, True])
def test_moments_have_the_parameters_shapes(state_dtype, given):
    p = [torch.zeros(3, 5, 7, device="cuda"), torch.zeros((), device="cuda"), torch.zeros(0, 4, device="cuda")]
    flat = [torch.rand(x.numel(), generator=torch.Generator().manual_seed(1)) + 0.5 for x in p]
    kw = {}
    if given and state_dtype == DT_F32:
        kw = dict(moments=([x.cuda() for x in flat], [x.cuda() for x in flat]))
    elif given:
        m, v = ([mtstep.encode(x, k) for x in flat] for k in (torch.float8_e4m3fn, torch.float8_e5m2))
        kw = dict(moments=([x.cuda() for x, _ in m], [x.cuda() for x, _ in v]), scales=([s.cuda() for _, s in m], [s.cuda() for _, s in v]))
    s = MultiStep(p, state_dtype=state_dtype, **kw)
    for got in s.moments():
        assert [x.shape for x in got] == [x.shape for x in p] and all(x.dtype == torch.float32 for x in got)
        for a, b in zip(got, flat):
            assert ((a.cpu().view(-1) - (b if given else 0)).abs() <= (2.0 ** -3 if state_dtype == DT_Q8 else 0) * b).all()
