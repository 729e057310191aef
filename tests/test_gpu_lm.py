"""The language-model operators (heatvit_amd.lm) against their plain 64-bit
forms (lm_reference), at the sizes, strides, masks and values where they can
go wrong, and a run of them together."""

import numpy as np
import pytest
import torch

import lm_reference as ref

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _bytes(t):
    return t.contiguous().cpu().view(torch.uint8).numpy()


# ------------------------------------------------------------------ rms_norm_q8

def _norm_inputs(rows, width, dtype, residual, seed):
    g = _gen(seed)
    channel = torch.exp(torch.randn(width, generator=g))
    x = (torch.randn(rows, width, generator=g) * channel).to(dtype)
    r = (torch.randn(rows, width, generator=g) * 3).to(dtype) if residual else None
    w = (1 + 0.3 * torch.randn(width, generator=g)).to(dtype)
    return x, r, w


def _check_norm(got, x, w, r, eps, fmt, block, rows=None):
    q, exps, scale, kept = ref.rms_norm_q8(x, w, r, eps, fmt, block)
    rows = slice(0, rows)
    assert np.array_equal(got.exps.cpu().numpy()[rows], exps[rows])
    gq, rq = _bytes(got.q)[rows], _bytes(q)[rows]
    if fmt == "e4m3":  # one NaN: 0x7f with either sign
        nan = (rq & 0x7F) == 0x7F
        assert np.array_equal((gq & 0x7F) == 0x7F, nan)
        gq, rq = np.where(nan, 0, gq), np.where(nan, 0, rq)
    assert np.array_equal(gq, rq)
    gs, rs = got.scale.cpu().double().numpy()[rows], scale[rows]
    assert np.array_equal(np.isnan(gs), np.isnan(rs))
    fine = ~np.isnan(rs)
    assert (np.abs(gs - rs)[fine] <= ref.scale_bound(x.shape[1]) * rs[fine]).all()
    if r is not None:
        assert np.array_equal(_bytes(got.residual)[rows], _bytes(kept)[rows])


@pytest.mark.parametrize("residual", (False, True))
@pytest.mark.parametrize("block", (128, 0))
@pytest.mark.parametrize("fmt", ("e4m3", "int8"))
@pytest.mark.parametrize("kind", TYPES)
def test_norm_sizes(kind, fmt, block, residual):
    from heatvit_amd import lm
    for rows, width in ((1, 1), (3, 7), (2, 8), (5, 127), (4, 128), (2, 129), (7, 192), (1, 1000),
                        (3, 2047), (2, 2048), (3, 2056), (1, 4096), (2, 5001), (1, 8200),
                        (1, 16384), (2, 20000)):
        x, r, w = _norm_inputs(rows, width, TYPES[kind], residual, rows * width)
        print(f"norm {kind} {fmt} block {block} {rows} x {width}", flush=True)
        got = lm.rms_norm_q8(x.cuda(), w.cuda(), residual=None if r is None else r.cuda(),
                             eps=1e-5, fmt=fmt, block=block)
        _check_norm(got, x, w, r, 1e-5, fmt, block)


@pytest.mark.parametrize("rows", (63, 64, 255, 256, 257, 1025, 5000))
def test_norm_many_rows(rows):
    from heatvit_amd import lm
    for width, kind in ((192, "bf16"), (96, "f32"), (264, "f16"), (1000, "bf16")):
        x, r, w = _norm_inputs(rows, width, TYPES[kind], True, rows + width)
        got = lm.rms_norm_q8(x.cuda(), w.cuda(), residual=r.cuda())
        _check_norm(got, x, w, r, 1e-6, "e4m3", 128)


@pytest.mark.parametrize("fmt", ("e4m3", "int8"))
@pytest.mark.parametrize("kind", TYPES)
def test_norm_values_at_the_edges(kind, fmt):
    """Rows of zeros, of the smallest and the largest values, of exact block
    borders (a maximum of L 2^k and its neighbours), ties of the rounding,
    and infinities and NaN beside ordinary blocks."""
    from heatvit_amd import lm
    dtype = TYPES[kind]
    width = 384
    info = torch.finfo(dtype)
    x = torch.zeros(12, width)
    g = _gen(5)
    x[1] = torch.randn(width, generator=g)
    x[1, 128:256] = 0                       # an empty block between others
    x[2] = info.tiny
    x[3, ::5] = info.smallest_normal / 4    # below the normal numbers
    x[4] = torch.randn(width, generator=g) * 1e-3
    top = ref.LARGEST[fmt]
    step = 2 * info.eps
    x[5, 0], x[5, 128], x[5, 256] = top / 16, top / 16 * (1 + step), top / 16 * (1 - step)
    x[5, 1:128] = torch.linspace(-top / 16, top / 16, 127)
    x[6] = (torch.arange(width) % 33 - 16) * 0.5 + 0.25  # ties
    x[6, ::128] = top
    x[7] = torch.randn(width, generator=g)
    x[7, 5] = float("inf")
    x[8] = torch.randn(width, generator=g)
    x[8, 200] = float("nan")
    x[9] = torch.randn(width, generator=g)
    x[9, 383] = -float("inf")
    x[10] = 1e4 * torch.randn(width, generator=g).clamp(-4, 4)
    x[11, 17] = -1.0
    x = x.to(dtype)
    w = torch.ones(width).to(dtype)
    for block in (128, 0):
        got = lm.rms_norm_q8(x.cuda(), w.cuda(), fmt=fmt, block=block)
        _check_norm(got, x, w, None, 1e-6, fmt, block)


@pytest.mark.parametrize("kind", TYPES)
def test_norm_strides_alignment_and_in_place(kind):
    """Rows apart in memory, rows that start off 16 bytes, the residual
    updated in place, bytes around the outputs left alone."""
    from heatvit_amd import lm
    dtype = TYPES[kind]
    for rows, width, pad, off in ((5, 256, 64, 0), (4, 256, 3, 1), (3, 250, 6, 0), (6, 136, 8, 4)):
        x, r, w = _norm_inputs(rows, width, dtype, True, width + pad)
        big = torch.full((rows, width + pad + off), 7.0).to(dtype).cuda()
        xs = big[:, off:off + width]
        xs.copy_(x)
        kept = torch.full((rows, width + pad + off), 3.0).to(dtype).cuda()
        ks = kept[:, off:off + width]
        ks.copy_(r)
        blocks = -(-width // 128)
        q = torch.full((rows, width + 24), 0x11, dtype=torch.uint8, device="cuda")
        e = torch.full((rows, blocks + 2), 99, dtype=torch.int8, device="cuda")
        s = torch.empty(rows, device="cuda")
        out = lm.Q8Rows(q.view(torch.float8_e4m3fn)[:, off:off + width], e[:, 1:1 + blocks], s, ks)
        got = lm.rms_norm_q8(xs, w.cuda(), residual=ks, out=out)
        _check_norm(got, x, w, r, 1e-6, "e4m3", 128)
        assert (q[:, :off] == 0x11).all() and (q[:, off + width:] == 0x11).all()
        assert (e[:, 0] == 99).all() and (e[:, -1] == 99).all()
        assert (kept[:, :off] == 3).all() and (kept[:, off + width:] == 3).all()
        assert torch.equal(xs.cpu(), x)


def test_norm_live_rows():
    from heatvit_amd import lm
    for rows, width, block in ((9, 192, 128), (300, 64, 0), (70, 4096, 128)):
        for live in (0, 1, 7, rows, rows + 5):
            x, r, w = _norm_inputs(rows, width, torch.bfloat16, True, live)
            blocks = -(-width // 128) if block else 1
            out = lm.Q8Rows(torch.full((rows, width), 5, dtype=torch.int8, device="cuda"),
                            torch.full((rows, blocks), 6, dtype=torch.int8, device="cuda"),
                            torch.full((rows,), 7.0, device="cuda"),
                            torch.full((rows, width), 8.0, dtype=torch.bfloat16, device="cuda"))
            lm.rms_norm_q8(x.cuda(), w.cuda(), residual=r.cuda(), fmt="int8", block=block, out=out,
                           live_rows=torch.tensor([live], dtype=torch.int32, device="cuda"))
            n = min(live, rows)
            if n:
                _check_norm(out, x, w, r, 1e-6, "int8", block, n)
            for t, v in zip(out, (5, 6, 7, 8)):
                assert (t[n:] == v).all()


def test_norm_into_the_int8_product():
    """int8 rows with one exponent a row through the framework's int8 GEMM."""
    from heatvit_amd import lm, ops
    x, r, w = _norm_inputs(70, 192, torch.bfloat16, True, 3)
    got = lm.rms_norm_q8(x.cuda(), w.cuda(), residual=r.cuda(), fmt="int8", block=0)
    m = np.random.default_rng(2).integers(-128, 128, (192, 40)).astype(np.int8)
    acc = ops.gemm_writeback(got.q.cpu().numpy(), m, None, 0, 0, 32)
    assert np.array_equal(acc, got.q.cpu().numpy().astype(np.int64) @ m)


# ------------------------------------------------------------------ gemm_f8

def _whole(shape, seed, high=3):
    """Small whole numbers as e4m3: every partial sum is exact in 32 bits."""
    return torch.randint(-high, high + 1, shape, generator=_gen(seed)).float().to(
        torch.float8_e4m3fn)


def _exps(shape, seed, low, high):
    return torch.randint(low, high + 1, shape, generator=_gen(seed)).to(torch.int8)


GEMM_SIZES = ((1, 1, 16), (1, 64, 128), (3, 17, 48), (16, 64, 192), (17, 65, 144), (5, 130, 512),
              (33, 200, 1040), (64, 256, 256), (65, 127, 384), (100, 129, 128), (128, 128, 2048),
              (129, 300, 640), (200, 1000, 192), (256, 256, 256), (257, 513, 400), (300, 70, 1152),
              (520, 260, 272), (1, 1000, 4096), (40, 4100, 512), (70, 1030, 1664), (1030, 300, 528),
              (24, 1030, 1040), (32, 4200, 256), (8, 9000, 128), (2100, 1030, 384), (4000, 4100, 144),
              (4100, 4000, 272), (600, 600, 256), (1500, 2100, 128))


@pytest.mark.parametrize("size", GEMM_SIZES, ids=str)
def test_gemm_whole_numbers_exactly(size):
    """Whole numbers and exponents whose sums are exact: every bit of the
    outputs is right, whatever the order of the additions."""
    from heatvit_amd import lm
    from heatvit_amd.device import DeviceF8Weight
    m, n, k = size
    kb, nb = -(-k // 128), -(-n // 128)
    a, w = _whole((m, k), 1), _whole((k, n), 2)
    # |sum| <= 9 k 2^4 < 2^24 units of 2^-6 up to k = 4096
    ae, we = _exps((m, kb), 3, -2, 0), _exps((kb, nb), 4, -3, 0)
    want, _ = ref.gemm_f8(a, ae.numpy(), w, we.numpy(), None, None)
    dw = DeviceF8Weight(w, we)
    got = lm.gemm_f8(a.cuda(), ae.cuda(), dw, out_dtype=torch.float32)
    assert np.array_equal(got.cpu().double().numpy(), want)
    # products of at most 9 lose nothing to the 8-bit matrix cores' alignment
    # either: the 16-bit outputs are these sums, rounded once
    for dtype in (torch.bfloat16, torch.float16):
        got = lm.gemm_f8(a.cuda(), ae.cuda(), dw, out_dtype=dtype)
        assert torch.equal(got.cpu(), torch.from_numpy(want).to(dtype))


@pytest.mark.parametrize("size", GEMM_SIZES, ids=str)
@pytest.mark.parametrize("kind", TYPES)
def test_gemm_values(kind, size):
    from heatvit_amd import lm
    from heatvit_amd.device import DeviceF8Weight
    m, n, k = size
    g = _gen(m + n + k)
    kb, nb = -(-k // 128), -(-n // 128)
    a = (torch.randn(m, k, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    w = (torch.randn(k, n, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    ae, we = _exps((m, kb), 3, -12, -4), _exps((kb, nb), 4, -14, -8)
    scale = torch.rand(m, generator=g) + 0.5
    bias = torch.randn(n, generator=g)
    dw = DeviceF8Weight(w, we)
    for s, b in ((None, None), (scale, bias)):
        y, bound = ref.gemm_f8(a, ae.numpy(), w, we.numpy(), None if s is None else
                               s.double().numpy(), None if b is None else b.double().numpy(),
                               fast=kind != "f32")
        got = lm.gemm_f8(a.cuda(), ae.cuda(), dw, row_scale=None if s is None else s.cuda(),
                         bias=None if b is None else b.cuda(), out_dtype=TYPES[kind])
        off = np.abs(got.cpu().double().numpy() - y)
        # the rounding of an output smaller than the type's normal numbers
        tiny = torch.finfo(TYPES[kind]).tiny * torch.finfo(TYPES[kind]).eps
        assert (off <= bound + (np.abs(y) + bound) * ref.HALF[TYPES[kind]] + tiny).all()


@pytest.mark.parametrize("size", ((5, 64, 16400), (70, 200, 8208), (1100, 1030, 8336),
                                  (4100, 4100, 8464), (70, 64, 20000), (600, 260, 16640)), ids=str)
def test_gemm_long_inner(size):
    """Inner sizes past the exponents that a tile holds at once (64 blocks),
    and at every number of blocks modulo the stages."""
    from heatvit_amd import lm
    from heatvit_amd.device import DeviceF8Weight
    m, n, k = size
    for cut in (0, 128, 256, 384):
        kk = k - cut
        kb, nb = -(-kk // 128), -(-n // 128)
        a, w = _whole((m, kk), 1, 1), _whole((kk, n), 2, 1)
        # |sum| <= k < 2^24 units of 2^-4
        ae, we = _exps((m, kb), 3, -2, 0), _exps((kb, nb), 4, -2, 0)
        dw = DeviceF8Weight(w, we)
        s = torch.from_numpy(ref.spread(ae.numpy(), 128, kk)).float().cuda()
        t = torch.from_numpy(np.repeat(ref.spread(we.numpy(), 128, n), 128, 0)[:kk]).float().cuda()
        want = (a.float().cuda() * s) @ (w.float().cuda() * t)  # exact: whole multiples of 2^-4
        for dtype in (torch.bfloat16, torch.float32):
            got = lm.gemm_f8(a.cuda(), ae.cuda(), dw, out_dtype=dtype)
            assert torch.equal(got, want.to(dtype)), (cut, dtype)


def test_gemm_every_exponent():
    """Exponents over their whole range: the scales multiply as powers of
    two, sums that stay within float32's normal numbers are exact."""
    from heatvit_amd import lm
    from heatvit_amd.device import DeviceF8Weight
    a, w = _whole((255, 128), 1), _whole((128, 128), 2)
    ae = torch.arange(-127, 128).to(torch.int8)[:, None]
    for e in (-127, -60, -1, 0, 1, 60, 120):
        dw = DeviceF8Weight(w, torch.full((1, 1), e, dtype=torch.int8))
        got = lm.gemm_f8(a.cuda(), ae.cuda(), dw, out_dtype=torch.float32).cpu().double().numpy()
        want, _ = ref.gemm_f8(a, ae.numpy(), w, np.full((1, 1), e, np.int8), None, None)
        total = ae[:, 0].numpy().astype(int) + e
        fine = (total >= -126) & (total <= 114)
        assert np.array_equal(got[fine], want[fine]), e


@pytest.mark.parametrize("size", ((255, 32000), (16, 8300)), ids=str)
def test_gemm_far_exponents_beside_near_ones(size):
    """The same where a float32 output's conversion applies the factors, with
    rows of factors inside and outside what it takes beside each other, and a
    far smaller block behind another (264 additions of 2^-23 each)."""
    from heatvit_amd import lm
    from heatvit_amd.device import DeviceF8Weight
    m, n = size
    a, w = _whole((m, 256), 1), _whole((256, n), 2)
    ae = torch.arange(-127, 128).to(torch.int8)[torch.arange(m) * (255 // m)][:, None]
    w64 = w.double().cuda()
    for e in (-127, -60, 0, 60, 120):
        for second in (None, -127):
            exps = ae.repeat(1, 2)
            if second is not None:
                exps[:, 1] = second
            dw = DeviceF8Weight(w, torch.full((2, -(-n // 128)), e, dtype=torch.int8))
            got = lm.gemm_f8(a.cuda(), exps.cuda(), dw, out_dtype=torch.float32)
            factor = torch.exp2(exps.double().cuda() + e)
            x = a.double().cuda()
            want = (x[:, :128] * factor[:, :1]) @ w64[:128]
            total = ae[:, 0].int() + e
            fine = (total >= -126) & (total <= 113)
            want += (x[:, 128:] * factor[:, -1:]) @ w64[128:]
            if second is None:  # whole multiples, below 2^12, of one unit: exact
                assert torch.equal(got[fine.cuda()], want[fine.cuda()].float()), e
                continue
            size = (x[:, :128].abs() * factor[:, :1]) @ w64[:128].abs() + \
                (x[:, 128:].abs() * factor[:, -1:]) @ w64[128:].abs()
            off = (got.double() - want).abs()
            assert (off <= size * 264 * 2.0 ** -23 + 2.0 ** -126)[fine.cuda()].all(), e


def test_gemm_nan_stays_in_its_row():
    """NaN in a row of `a`, at the last of k and in what follows the rows in
    memory, reaches that row alone."""
    from heatvit_amd import lm
    from heatvit_amd.device import DeviceF8Weight
    for m, n, k in ((40, 70, 144), (300, 300, 208), (3, 64, 272)):
        a, w = _whole((m, k + 112), 1), _whole((k, n), 2)
        nan = torch.full((m, k + 112), float("nan")).to(torch.float8_e4m3fn)
        a[:, k:] = nan[:, k:]
        kb = -(-k // 128)
        ae, we = _exps((m, kb), 3, -2, 0), _exps((kb, -(-n // 128)), 4, -3, 0)
        want, _ = ref.gemm_f8(a[:, :k], ae.numpy(), w, we.numpy(), None, None)
        bad = m // 2
        a[bad, k - 1] = nan[0, 0]
        dw = DeviceF8Weight(w, we)
        da = a.cuda()[:, :k]
        got = lm.gemm_f8(da, ae.cuda(), dw, out_dtype=torch.float32).cpu().double().numpy()
        assert np.isnan(got[bad]).all()
        keep = np.arange(m) != bad
        assert np.array_equal(got[keep], want[keep])


def test_gemm_strides_live_rows_and_nothing_outside():
    from heatvit_amd import lm
    from heatvit_amd.device import DeviceF8Weight
    for m, n, k, kind in ((37, 100, 192, "bf16"), (300, 260, 400, "f16"), (150, 65, 256, "f32"),
                          (2, 500, 128, "bf16")):
        dtype = TYPES[kind]
        kb, nb = -(-k // 128), -(-n // 128)
        a, w = _whole((m, k), 1), _whole((k, n), 2)
        ae, we = _exps((m, kb), 3, -2, 0), _exps((kb, nb), 4, -3, 0)
        want, _ = ref.gemm_f8(a, ae.numpy(), w, we.numpy(), None, None)
        want = torch.from_numpy(want).to(dtype)
        dw = DeviceF8Weight(w.t().contiguous().t(), we)  # a checkpoint's [N][K]
        da = torch.full((m, k + 48), 0x7F, dtype=torch.uint8, device="cuda")
        da = da.view(torch.float8_e4m3fn)
        da[:, 16:16 + k] = a.cuda()
        de = torch.full((m, kb + 3), 100, dtype=torch.int8, device="cuda")
        de[:, 2:2 + kb] = ae.cuda()
        for live in (0, 1, m - 1, m, m + 9):
            for pad in (0, 1, 4):
                c = torch.full((m, n + 8), 55.0, dtype=dtype, device="cuda")
                lm.gemm_f8(da[:, 16:16 + k], de[:, 2:2 + kb], dw, out_dtype=dtype,
                           out=c[:, pad:pad + n],
                           live_rows=torch.tensor([live], dtype=torch.int32, device="cuda"))
                rows = min(live, m)
                assert torch.equal(c[:rows, pad:pad + n].cpu(), want[:rows]), (m, live, pad)
                assert (c[rows:] == 55).all()
                assert (c[:, :pad] == 55).all() and (c[:, pad + n:] == 55).all()


def test_gemm_rows_far_apart():
    """Rows 2^22 and more bytes apart, where a tile's 32-bit offsets end."""
    from heatvit_amd import lm
    from heatvit_amd.device import DeviceF8Weight
    m, n, k = 70, 130, 400
    a, w = _whole((m, k), 1), _whole((k, n), 2)
    ae, we = _exps((m, 4), 3, -2, 0), _exps((4, 2), 4, -3, 0)
    want, _ = ref.gemm_f8(a, ae.numpy(), w, we.numpy(), None, None)
    for ld in (1 << 22, (1 << 22) - 16):
        far = torch.zeros((m, ld), dtype=torch.uint8, device="cuda")
        far[:, :k] = a.view(torch.uint8).cuda()
        got = lm.gemm_f8(far.view(torch.float8_e4m3fn)[:, :k], ae.cuda(), DeviceF8Weight(w, we),
                         out_dtype=torch.float32)
        assert np.array_equal(got.cpu().double().numpy(), want)


def test_weight_quantised_here():
    """A float weight: every value within half an e4m3 step of its block."""
    from heatvit_amd.device import quantise_f8_weight
    w = torch.randn(200, 300, generator=_gen(9))
    w[:128, 128:256] = 0
    q, e = quantise_f8_weight(w.cuda())
    s = np.repeat(ref.spread(e.cpu().numpy(), 128, 300), 128, axis=0)[:200]
    back = q.cpu().double().numpy() * s
    off = np.abs(back - w.double().numpy())
    assert (off <= np.maximum(np.abs(w.numpy()) * 2.0 ** -4, s * 2.0 ** -10)).all()
    flat = torch.zeros(256, 384)
    flat[:200, :300] = w
    flat = flat.view(2, 128, 3, 128).permute(0, 2, 1, 3).reshape(6, -1).double().numpy()
    assert np.array_equal(e.cpu().numpy().reshape(-1),
                          ref.block_exps(flat, 0, 448.0).reshape(-1))


# ------------------------------------------------------------------ log_probs

def _check_answer(got, x, tokens, scale, top, rows=None):
    want = ref.log_probs(x, None if tokens is None else
                         tokens.reshape(len(x), -1).astype(np.int64), scale, top)
    rows = slice(0, rows)
    names = ["entropy"] + (["logp"] if tokens is not None else []) + (["top_logp"] if top else [])
    for name in names:
        g = getattr(got, name).cpu().double().numpy().reshape(len(x), -1)[rows]
        w, b = (want[k].reshape(len(x), -1)[rows] for k in (name, name + "_bound"))
        assert np.array_equal(np.isnan(g), np.isnan(w)), name
        assert np.array_equal(np.isneginf(g), np.isneginf(w)), name
        fine = np.isfinite(w)
        assert (np.abs(g - w)[fine] <= b[fine]).all(), (name, np.max((np.abs(g - w) / b)[fine]))
    if top:
        assert np.array_equal(got.top_index.cpu().numpy()[rows], want["top_index"][rows])


def _logits(rows, width, kind, seed, spread=3.0):
    x = torch.randn(rows, width, generator=_gen(seed)) * spread
    if kind == "i32":
        return torch.round(x * 2 ** 14).to(torch.int32)
    return x.to(TYPES[kind])


ANSWER_SIZES = ((1, 1), (2, 2), (3, 5), (5, 63), (4, 64), (3, 65), (7, 255), (2, 257), (256, 1000),
                (3, 1023), (3, 4096), (2, 5003), (1, 8192), (9, 20001), (1, 50001), (2, 131072),
                (1, 262144), (40, 3001), (1, 16384), (1, 16385))


@pytest.mark.parametrize("kind", ("bf16", "f16", "f32", "i32"))
def test_answer_sizes(kind):
    from heatvit_amd import lm
    for rows, width in ANSWER_SIZES:
        x = _logits(rows, width, kind, rows + width)
        e = -14 if kind == "i32" else 0
        for count, top in ((1, 0), (3, min(width, 5)), (0, min(width, 64)), (2, min(width, 32))):
            print(f"answer {kind} {rows} x {width} tokens {count} top {top}", flush=True)
            t = torch.randint(0, width, (rows, count), generator=_gen(1)).to(torch.int32)
            got = lm.log_probs(x.cuda(), t.cuda(), scale_exp=e, top=top)
            _check_answer(got, x.double().numpy(), t.numpy(), 2.0 ** e, top)


@pytest.mark.parametrize("width", (40, 1000, 30000))
@pytest.mark.parametrize("kind", ("bf16", "f32", "i32"))
def test_answer_orders(kind, width):
    """Rows in rising and falling order, flat rows, rows of few values, a row
    whose largest come last: alternatives in order, ties by the lower index."""
    from heatvit_amd import lm
    r = torch.arange(width).float()
    x = torch.stack([r / width * 8, -r / width * 8, torch.zeros(width), (r % 3), -(r % 7),
                     torch.where(r >= width - 70, r - width, torch.tensor(-90.0)),
                     torch.where(r % 2 == 0, 0.0, -0.0), (r * 7919 % width) / width])
    x = torch.round(x * 1024).to(torch.int32) if kind == "i32" else x.to(TYPES[kind])
    e = -10 if kind == "i32" else 0
    for top in (1, 20, 33):
        got = lm.log_probs(x.cuda(), scale_exp=e, top=top)
        _check_answer(got, x.double().numpy(), None, 2.0 ** e, top)


@pytest.mark.parametrize("kind", ("bf16", "f32", "i32"))
def test_answer_more_equal_logits_than_candidates(kind):
    """Rows that are flat, or flat but for a few logits, past what the
    alternatives are picked from, the largest values of the type among them."""
    from heatvit_amd import lm
    width = 20000
    x = torch.zeros(6, width)
    x[1, 19990:] = 1.0
    x[2, ::2] = -3.0
    x[4] = torch.arange(width) % 2
    x = x.to(torch.int32) if kind == "i32" else x.to(TYPES[kind])
    x[3] = 2 ** 31 - 1 if kind == "i32" else torch.finfo(TYPES[kind]).max
    x[5] = -2 ** 31 if kind == "i32" else torch.finfo(TYPES[kind]).min
    for rows in (slice(0, 6), slice(3, 4), slice(4, 6)):
        part = x[rows]
        got = lm.log_probs(part.cuda(), scale_exp=-2, top=17)
        _check_answer(got, part.double().numpy(), None, 0.25, 17)
    big = x.repeat(100, 1)  # a row to each workgroup
    got = lm.log_probs(big.cuda(), scale_exp=-2, top=3)
    _check_answer(got, big.double().numpy(), None, 0.25, 3)


@pytest.mark.parametrize("rows", (1, 600))
def test_answer_nan_and_few_left_in_wide_rows(rows):
    """NaN at either end of a wide row (in parts, and a row to a workgroup),
    and rows whose mask leaves fewer logits than alternatives."""
    from heatvit_amd import lm
    width = 20011
    for at in (0, 9000, width - 1):
        x = torch.randn(rows, width, generator=_gen(at))
        x[-1, at] = float("nan")
        got = lm.log_probs(x.cuda(), top=4)
        assert got.entropy[-1].isnan() and got.top_logp[-1].isnan().all()
        want = x[-1].clone()
        want[at] = float("inf")
        assert got.top_index[-1].tolist() == torch.sort(want, descending=True, stable=True)[1][:4].tolist()
    x = torch.full((rows, width), -float("inf"))
    x[:, 7], x[:, 12345] = 1.0, 2.0
    got = lm.log_probs(x.cuda(), torch.full((rows,), 7, dtype=torch.int32).cuda(), top=20)
    _check_answer(got, x.double().numpy(), np.full((rows, 1), 7), 1.0, 20)


def test_answer_int32_range():
    """int32 logits over their whole range: differences past 2^31."""
    from heatvit_amd import lm
    x = torch.randint(-2 ** 31, 2 ** 31, (4, 700), generator=_gen(3)).to(torch.int32)
    x[0, 5], x[0, 9], x[1] = -2 ** 31, 2 ** 31 - 1, -2 ** 31
    for e in (-31, -26, -14, 0):
        got = lm.log_probs(x.cuda(), torch.tensor([[5], [9], [0], [1]], dtype=torch.int32).cuda(),
                           scale_exp=e, top=9)
        _check_answer(got, x.double().numpy(), np.array([[5], [9], [0], [1]]), 2.0 ** e, 9)


@pytest.mark.parametrize("kind", ("bf16", "f16", "f32"))
def test_answer_masks(kind):
    """Masked tokens (-inf, the type's lowest), rows with nothing left, with
    one token left, NaN and +inf, tokens outside the row."""
    from heatvit_amd import lm
    inf, width = float("inf"), 900
    low = torch.finfo(TYPES[kind]).min
    x = _logits(9, width, kind, 4)
    x[0, ::2] = -inf
    x[1] = -inf
    x[2] = -inf
    x[2, 321] = 1.5
    x[3, 1::3] = low
    x[4] = low
    x[5, 700:] = -inf
    x[6, :899] = -inf
    t = torch.tensor([[0, 1, -1], [3, 900, -7], [321, 320, 0], [1, 0, 4], [0, 5, 899],
                      [699, 700, 2 ** 31 - 1], [899, 0, -2 ** 31], [1, 2, 3], [4, 5, 6]],
                     dtype=torch.int32)
    for top in (0, 3, 40):
        got = lm.log_probs(x.cuda(), t.cuda(), top=top)
        one = np.arange(9) != 1
        sub = lm.LogProbs(*[None if v is None else v[torch.from_numpy(one).cuda()] for v in got])
        _check_answer(sub, x.double().numpy()[one], t.numpy()[one], 1.0, top)
        # nothing left: no probability anywhere, no uncertainty
        assert got.entropy[1] == 0
        lp = got.logp[1].cpu()
        assert lp[0] == -inf and lp[1].isnan() and lp[2] == 0
        if top:
            assert (got.top_logp[1] == -inf).all()
            assert got.top_index[1].tolist() == list(range(top))
    for value in (float("nan"), inf):
        y = x[7:].clone()
        y[0, 77] = value
        got = lm.log_probs(y.cuda(), t[7:].cuda(), top=2)
        assert got.logp[0].isnan().all() and got.entropy[0].isnan()
        assert got.top_index[0, 0] == 77 and got.top_logp[0].isnan().all()
        assert torch.isfinite(got.logp[1]).all() and torch.isfinite(got.entropy[1])


def test_answer_temperature_strides_and_live_rows():
    from heatvit_amd import lm
    for kind, rows, width, off in (("bf16", 6, 1001, 3), ("f32", 5, 5000, 1), ("f16", 3, 777, 0)):
        x = _logits(rows, width, kind, 8)
        big = torch.full((rows, width + 7), 90.0).to(TYPES[kind]).cuda()
        big[:, off:off + width] = x.cuda()
        t = torch.randint(0, width, (rows,), generator=_gen(1)).to(torch.int32)
        for temperature in (0.25, 1.0, 3.7):
            for live in (0, 2, rows, rows + 1):
                out = lm.LogProbs(torch.full((rows,), 5.0).cuda(), torch.full((rows,), 6.0).cuda(),
                                  torch.full((rows, 4), 7.0).cuda(),
                                  torch.full((rows, 4), 8, dtype=torch.int32).cuda())
                lm.log_probs(big[:, off:off + width], t.cuda(), temperature=temperature, top=4,
                             live_rows=torch.tensor([live], dtype=torch.int32).cuda(), out=out)
                n = min(live, rows)
                if n:
                    _check_answer(out, x.double().numpy(), t.numpy(), 1.0 / temperature, 4, n)
                for v, want in zip(out, (5, 6, 7, 8)):
                    assert (v[n:] == want).all()


# ------------------------------------------------------------------ together

def _step(lm, x, r, w, weight, tokens, live=None):
    n = lm.rms_norm_q8(x, w, residual=r, live_rows=live)
    logits = lm.gemm_f8(n.q, n.exps, weight, row_scale=n.scale, live_rows=live)
    return n, logits, lm.log_probs(logits, tokens, top=5, live_rows=live)


@pytest.mark.parametrize("rows", (1, 37, 300))
def test_norm_product_answer(rows):
    """The end of a language model's step: the last norm, the product onto
    the vocabulary and the answer, against the plain forms in turn."""
    from heatvit_amd import lm
    from heatvit_amd.device import DeviceF8Weight, quantise_f8_weight
    width, vocab = 576, 2011
    x, r, w = _norm_inputs(rows, width, torch.bfloat16, True, rows)
    m = torch.randn(width, vocab, generator=_gen(6)) * 0.1
    weight = DeviceF8Weight(m.cuda())
    tokens = torch.randint(0, vocab, (rows,), generator=_gen(2)).to(torch.int32)
    n, logits, answer = _step(lm, x.cuda(), r.cuda(), w.cuda(), weight, tokens.cuda())
    _check_norm(n, x, w, r, 1e-6, "e4m3", 128)
    q, e = quantise_f8_weight(m)
    y, bound = ref.gemm_f8(n.q.cpu(), n.exps.cpu().numpy(), q, e.numpy(),
                           n.scale.cpu().double().numpy(), None, fast=True)
    off = np.abs(logits.cpu().double().numpy() - y)
    assert (off <= bound + (np.abs(y) + bound) * 2.0 ** -8).all()
    _check_answer(answer, logits.cpu().double().numpy(), tokens.numpy(), 1.0, 5)


def test_model_scores():
    """The classifier's answers: HeatViTModel.score_batch on the logits that
    infer_batch gives, for int8 and for float images."""
    from heatvit_amd import synth
    from heatvit_amd.model import HeatViTModel
    images, params = synth.pruned_workload(5)
    model = HeatViTModel()
    logits = model.infer_batch(images, params).logits
    labels = np.random.default_rng(4).integers(0, 1000, (5, 3))
    labels[:, 0] = logits.argmax(1)
    want = ref.log_probs(logits.astype(np.float64), labels, 2.0 ** -14, 5)
    floats = np.asarray(images, np.float32).reshape(5, 224, 224, 3).transpose(0, 3, 1, 2) * \
        np.float32(2.0 ** params.patch.image_scale_exp)
    for x in (images, np.ascontiguousarray(floats)):
        got = model.score_batch(x, params, labels)
        for name in ("logp", "entropy", "top_logp"):
            off = np.abs(getattr(got, name).astype(np.float64) - want[name])
            assert (off <= want[name + "_bound"]).all(), name
        assert np.array_equal(got.top_index, want["top_index"])
        assert np.array_equal(got.top_index[:, 0], labels[:, 0])
    one = model.score_batch(images, params, labels[:, 1], top=0)
    assert np.array_equal(one.logp, got.logp[:, 1]) and one.top_index is None
    assert model.score_batch(images, params, top=1).logp is None
    for bad, error in ((labels[:4], ValueError), (labels + 1000, ValueError), (-labels - 1, ValueError),
                       (labels.astype(float), TypeError)):
        with pytest.raises(error):
            model.score_batch(images, params, bad)
    with pytest.raises(ValueError):
        model.score_batch(images, params, top=65)


def test_step_in_a_graph_and_on_streams():
    """The step captured into two graphs that are replayed in turn, with the
    program's own eager steps between, and on a stream of its own: the bits
    of the eager results each time."""
    from heatvit_amd import lm
    from heatvit_amd.device import DeviceF8Weight
    width, vocab, rows = 512, 40000, 3
    weight = DeviceF8Weight((torch.randn(width, vocab, generator=_gen(6)) * 0.1).cuda())
    w = torch.ones(width, dtype=torch.bfloat16, device="cuda")
    sets = []
    for i in range(3):
        x, r, _ = _norm_inputs(rows, width, torch.bfloat16, True, 50 + i)
        t = torch.randint(0, vocab, (rows,), generator=_gen(i)).to(torch.int32)
        sets.append((x.cuda(), r.cuda(), t.cuda()))

    def flat(n, logits, answer):
        return [v for v in (*n, logits, *answer)]

    eager = [[v.clone() for v in flat(*_step(lm, x, r, w, weight, t))] for x, r, t in sets]
    held = [[v.clone() for v in s] for s in sets[:2]]
    graphs = []
    for x, r, t in held:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = flat(*_step(lm, x, r, w, weight, t))
        graphs.append((g, out))
    for rep in range(4):
        for i, (g, out) in enumerate(graphs):
            s = (rep + i) % 3
            for dst, src in zip(held[i], sets[s]):
                dst.copy_(src)
            g.replay()
            other = flat(*_step(lm, sets[2][0], sets[2][1], w, weight, sets[2][2]))
            torch.cuda.synchronize()
            for a, b in zip(out, eager[s]):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), (rep, i)
            for a, b in zip(other, eager[2]):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), (rep, i)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for s, (x, r, t) in zip(streams, sets):
        with torch.cuda.stream(s):
            outs.append([flat(*_step(lm, x, r, w, weight, t)) for _ in range(4)])
    torch.cuda.synchronize()
    for many, want in zip(outs, eager):
        for out in many:
            for a, b in zip(out, want):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_numbers_that_no_descriptor_holds():
    from heatvit_amd import lm
    x = torch.zeros(2, 64).cuda()
    for call in (lambda: lm.rms_norm_q8(x, x[0], eps=1e300), lambda: lm.rms_norm_q8(x, x[0], eps=-1.0),
                 lambda: lm.log_probs(x, temperature=1e-300), lambda: lm.log_probs(x, scale_exp=200)):
        with pytest.raises(ValueError):
            call()
