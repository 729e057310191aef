"""Edges of the language-model operators that need no GPU."""

import math

import pytest
import torch

import lm_kernels
from heatvit_amd import lm
from heatvit_amd.device import DeviceF8Weight, quantise_f8_weight


def test_weight_exponent_minus_128_is_refused():
    f8 = torch.ones(144, 130).to(torch.float8_e4m3fn)
    e = torch.full((2, 2), -127, dtype=torch.int8)
    assert DeviceF8Weight(f8, e, device="cpu").exps[1, 1] == -127
    e[1, 0] = -128
    with pytest.raises(ValueError):
        DeviceF8Weight(f8, e, device="cpu")


@pytest.mark.parametrize("value", (math.inf, -math.inf, math.nan))
def test_weight_not_finite_stays_alone(value):
    """A NaN or an infinity in a weight is NaN where it stands; the rest of
    its block has the values and the exponent that it has without it."""
    w = torch.randn(300, 140, generator=torch.Generator().manual_seed(3)) * 700
    w[5, 7], w[200, 139], w[299, 0] = 0, 0, 0
    want, e_want = quantise_f8_weight(w)
    for k, n in ((5, 7), (200, 139), (299, 0)):
        w[k, n] = value
    w[128:256, 128:] = torch.where(torch.arange(12) == 11, value, 0.0)  # nothing else in a block
    want.view(torch.uint8)[128:256, 128:] = 0
    e_want[1, 1] = -127
    q, e = quantise_f8_weight(w)
    assert torch.equal(e, e_want)
    finite = w.isfinite()
    assert q.float()[~finite].isnan().all()
    assert torch.equal(q.view(torch.uint8)[finite], want.view(torch.uint8)[finite])


@pytest.mark.parametrize("scale_exp,temperature", ((2000, 1.0), (1024, 3.0), (10 ** 30, 1.0)))
def test_answer_scale_out_of_range(scale_exp, temperature):
    with pytest.raises(ValueError, match="out of range"):
        lm.log_probs(torch.zeros(3, 50), scale_exp=scale_exp, temperature=temperature)


def test_product_kernels_by_size():
    """The rule that picks a product's kernel: the sizes that the GPU tests
    hold each kernel to take it, and rows too far apart for a tile do not."""
    import test_gpu_lm_kernels as gpu
    assert {n for k, n in gpu.CALLS if k != "f32"} == set(gpu.SIZES16)
    assert {n for k, n in gpu.CALLS if k == "f32"} == set(gpu.SIZES32)
    assert set(gpu.SIZES16) | set(gpu.SIZES32) == set(lm_kernels.NAMES)
    for f32, sizes in ((False, gpu.SIZES16), (True, gpu.SIZES32)):
        for name, (m, n) in sizes.items():
            for lda in (16, 400, (1 << 22) - 16):
                assert lm_kernels.kernel_of(f32, m, n, lda) == name
            assert lm_kernels.kernel_of(f32, m, n, 1 << 22) in ("rows16", "rows16x2")
