"""Edges of the language-model operators (heatvit_amd.lm): exponents, weights,
squares and differences at the ends of their ranges."""

import numpy as np
import pytest
import torch

import lm_reference as ref

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _whole(shape, seed, high=3):
    """Small whole numbers as e4m3: every partial sum is exact in 32 bits."""
    return torch.randint(-high, high + 1, shape, generator=_gen(seed)).float().to(
        torch.float8_e4m3fn)


def _exps(shape, seed, low, high):
    return torch.randint(low, high + 1, shape, generator=_gen(seed)).to(torch.int8)


# ------------------------------------------------------------------ gemm_f8

@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("size", ((5, 64, 400), (40, 4200, 400), (600, 600, 400), (600, 600, 8576)),
                         ids=str)
def test_gemm_exponent_minus_128(size, kind):
    """An exponent of -128 is no number: its row is NaN, over a block of
    zeros too, and every other row and the row's other blocks keep theirs."""
    from heatvit_amd import lm
    from heatvit_amd.device import DeviceF8Weight
    m, n, k = size
    kb, nb = -(-k // 128), -(-n // 128)
    a, w = _whole((m, k), 1, 1), _whole((k, n), 2, 1)
    ae, we = _exps((m, kb), 3, -2, 0), _exps((kb, nb), 4, -2, 0)
    dw = DeviceF8Weight(w, we)
    s = torch.from_numpy(ref.spread(ae.numpy(), 128, k)).float().cuda()
    t = torch.from_numpy(np.repeat(ref.spread(we.numpy(), 128, n), 128, 0)[:k]).float().cuda()
    # exact: whole multiples of 2^-4, at most k of them
    want = ((a.float().cuda() * s) @ (w.float().cuda() * t)).to(TYPES[kind])
    bad = torch.zeros(m, dtype=torch.bool)
    for row, block in ((0, 0), (1, kb - 1), (3, 1), (m - 1, kb // 2)):
        ae[row, block] = -128
        bad[row] = True
    a[3, 128:256] = 0
    bad = bad.cuda()
    got = lm.gemm_f8(a.cuda(), ae.cuda(), dw, out_dtype=TYPES[kind])
    assert got[bad].isnan().all()
    assert torch.equal(got[~bad], want[~bad])


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("size", ((5, 300, 400), (40, 4200, 400), (600, 600, 400)), ids=str)
def test_gemm_weight_exponent_minus_128(size, kind):
    """The same in a weight that was changed behind the constructor's check:
    the block's 128 channels are NaN, the others keep their values."""
    from heatvit_amd import lm
    from heatvit_amd.device import DeviceF8Weight
    m, n, k = size
    kb, nb = -(-k // 128), -(-n // 128)
    a, w = _whole((m, k), 1), _whole((k, n), 2)
    ae, we = _exps((m, kb), 3, -2, 0), _exps((kb, nb), 4, -3, 0)
    want, _ = ref.gemm_f8(a, ae.numpy(), w, we.numpy(), None, None)
    dw = DeviceF8Weight(w, we)
    dw.exps[2, 1] = -128
    got = lm.gemm_f8(a.cuda(), ae.cuda(), dw, out_dtype=TYPES[kind]).cpu()
    assert got[:, 128:256].isnan().all()
    want = torch.from_numpy(want).to(TYPES[kind])
    assert torch.equal(got[:, :128], want[:, :128]) and torch.equal(got[:, 256:], want[:, 256:])


# ------------------------------------------------------------------ rms_norm_q8

@pytest.mark.parametrize("residual", (False, True))
@pytest.mark.parametrize("kind", ("bf16", "f32"))
@pytest.mark.parametrize("size", ((20, 100), (5, 100), (5, 300), (3, 1500), (600, 700), (2, 4096)),
                         ids=str)
def test_norm_squares_outside_float32(size, kind, residual):
    """Rows whose squares, or their sum, lie above or below float32's numbers:
    the factor is that of the formula all the same."""
    from heatvit_amd import lm
    rows, width = size
    dtype = TYPES[kind]
    row = torch.arange(rows)
    # the rows' sizes go through 2^-140 .. 2^126, some rows' values all alike
    size_of = -140 + (row * 37 + width) % 267
    x = torch.randn(rows, width, generator=_gen(width)).clamp(-1.9, 1.9)
    x[row % 4 == 1] = 1.0
    x = torch.ldexp(x.double(), size_of[:, None]).to(dtype)
    x[rows - 1] = 0
    if rows > 4:
        x[2, width // 2] = float("inf")
        x[3, 1] = float("nan")
    w = torch.ones(width, dtype=dtype)
    # without a residual's own values the sum is x itself
    r = torch.zeros(rows, width, dtype=dtype).cuda() if residual else None
    for eps in (0.0, 1e-36, 1e-6):
        for fmt, block in (("e4m3", 128), ("int8", 0)):
            got = lm.rms_norm_q8(x.cuda(), w.cuda(), residual=r, eps=eps, fmt=fmt, block=block)
            with np.errstate(all="ignore"):
                eps32 = float(np.float32(eps))
                want = 1.0 / np.sqrt(np.square(x.double().numpy()).mean(1) + eps32)
            g = got.scale.cpu().double().numpy()
            assert np.array_equal(np.isnan(g), np.isnan(want))
            far = want > float(np.finfo(np.float32).max)  # 1 / 0 among them
            assert np.array_equal(np.isposinf(g), far)
            fine = ~np.isnan(want) & ~far
            # half a step of the numbers below the normal ones
            bound = ref.scale_bound(width) * want + 2.0 ** -149
            assert (np.abs(g - want)[fine] <= bound[fine]).all(), (eps, fmt)
            q, exps, _, _ = ref.rms_norm_q8(x, w, None, eps, fmt, block)
            assert np.array_equal(got.exps.cpu().numpy(), exps)
            if fmt == "int8":
                assert torch.equal(got.q.cpu(), q)


@pytest.mark.parametrize("size", ((3, 200), (3, 700), (3, 1500), (600, 3000), (2, 20000)), ids=str)
def test_norm_squares_outside_float32_in_place(size):
    """The same with the residual's sum in its place: what is squared a second
    time is what the row's other threads have written."""
    from heatvit_amd import lm
    rows, width = size
    for power in (-100, 80):
        g = _gen(width)
        x, r = (torch.ldexp(torch.randn(rows, width, generator=g).double(),
                            torch.tensor(power)).to(torch.bfloat16) for _ in range(2))
        h = (x.float() + r.float()).to(torch.bfloat16)
        kept = r.cuda()
        out = lm.Q8Rows(torch.empty((rows, width), dtype=torch.int8, device="cuda"),
                        torch.empty((rows, 1), dtype=torch.int8, device="cuda"),
                        torch.empty(rows, device="cuda"), kept)
        lm.rms_norm_q8(x.cuda(), torch.ones(width, dtype=torch.bfloat16).cuda(), residual=kept,
                       eps=0.0, fmt="int8", block=0, out=out)
        assert torch.equal(kept.cpu(), h)
        want = 1.0 / np.sqrt(np.square(h.double().numpy()).mean(1))
        off = np.abs(out.scale.cpu().double().numpy() - want)
        assert (off <= ref.scale_bound(width) * want).all(), power
        q, exps, _, _ = ref.rms_norm_q8(h, torch.ones(width).to(h.dtype), None, 0.0, "int8", 0)
        assert np.array_equal(out.exps.cpu().numpy(), exps) and torch.equal(out.q.cpu(), q)


def test_int8_rows_through_the_int8_product():
    """int8 rows of very different sizes through hv_gemm_i8 on the device: its
    sums, times 2^exps and scale of each row, are the normalised rows' product.
    q is off by half a step of 2^exps, scale by its roundings."""
    from heatvit_amd import _lib, lm
    from heatvit_amd.device import pack_mfma32
    m, n, k = 70, 40, 192
    x = torch.randn(m, k, generator=_gen(3)) * torch.exp2(torch.arange(m) % 23 - 11.0)[:, None]
    x, w = x.to(torch.bfloat16), (1 + 0.3 * torch.randn(k, generator=_gen(4))).to(torch.bfloat16)
    rows = lm.rms_norm_q8(x.cuda(), w.cuda(), fmt="int8", block=0)
    assert rows.exps.unique().numel() > 10
    b = np.random.default_rng(2).integers(-128, 128, (k, n)).astype(np.int8)
    packed = torch.from_numpy(pack_mfma32(b)).cuda()
    sums = torch.empty((m, n), dtype=torch.int32, device="cuda")
    d = _lib.GemmDesc()
    d.a, d.b_packed, d.c = rows.q.data_ptr(), packed.data_ptr(), sums.data_ptr()
    d.m, d.n, d.k, d.lda, d.ldc, d.ldr = m, n, k, k, n, n
    d.a_mode, d.epilogue = _lib.HV_A_ROWS, _lib.HV_EPI_I32
    _lib.check(_lib.lib().hv_gemm_i8(d, torch.cuda.current_stream().cuda_stream), "gemm")
    step = torch.exp2(rows.exps[:, 0].double().cpu()) * rows.scale.double().cpu()
    got = sums.cpu().double() * step[:, None]
    h = x.double()
    normal = h * w.double() / torch.sqrt(h.square().mean(1, keepdim=True) + 1e-6)
    want = normal @ torch.from_numpy(b).double()
    size = normal.abs() @ torch.from_numpy(b).double().abs()
    half = step[:, None] / 2 * torch.from_numpy(b).double().abs().sum(0)
    assert ((got - want).abs() <= (half + size * ref.scale_bound(k)) * (1 + 2.0 ** -20)).all()


# ------------------------------------------------------------------ log_probs

@pytest.mark.parametrize("kind", ("bf16", "f32"))
@pytest.mark.parametrize("size", ((1, 131072), (3, 900), (600, 3000)), ids=str)
def test_answer_differences_beyond_the_largest_number(size, kind):
    """Logits over the whole range of their type with a scale that brings them
    near each other: their differences are twice the largest number."""
    from heatvit_amd import lm
    rows, width = size
    x = (torch.rand(rows, width, generator=_gen(rows)) * 2 - 1) * 3.38e38
    x = x.to(TYPES[kind])
    x[0, 5], x[0, 9] = torch.finfo(TYPES[kind]).max, torch.finfo(TYPES[kind]).min
    t = torch.randint(0, width, (rows, 2), generator=_gen(1)).to(torch.int32)
    t[0, 0], t[0, 1] = 5, 9
    got = lm.log_probs(x.cuda(), t.cuda(), scale_exp=-126, top=7)
    want = ref.log_probs(x.double().numpy(), t.numpy().astype(np.int64), 2.0 ** -126, 7)
    for name in ("entropy", "logp", "top_logp"):
        off = np.abs(getattr(got, name).cpu().double().numpy() - want[name])
        assert (off <= want[name + "_bound"]).all(), name
    assert np.array_equal(got.top_index.cpu().numpy(), want["top_index"])
