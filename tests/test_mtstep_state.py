"""State handed to the list step."""
import pytest
import torch

from anni_b200.capi import DT_Q8
from anni_b200.mtstep import MultiStep


def test_8_bit_moments_without_scales_are_refused():
    """Codes mean nothing without their scales; zeros in their place would lose the moments silently."""
    p = torch.zeros(300)
    m, v = (torch.ones(300).to(k) for k in (torch.float8_e4m3fn, torch.float8_e5m2))
    with pytest.raises(ValueError, match="scales"):
        MultiStep([p], state_dtype=DT_Q8, moments=([m], [v]))
