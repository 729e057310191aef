"""Edges of the language-model operators that need no GPU."""

import pytest
import torch

from heatvit_amd.device import DeviceF8Weight


def test_weight_exponent_minus_128_is_refused():
    f8 = torch.ones(144, 130).to(torch.float8_e4m3fn)
    e = torch.full((2, 2), -127, dtype=torch.int8)
    assert DeviceF8Weight(f8, e, device="cpu").exps[1, 1] == -127
    e[1, 0] = -128
    with pytest.raises(ValueError):
        DeviceF8Weight(f8, e, device="cpu")
