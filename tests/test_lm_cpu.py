"""The language-model operators without a GPU: the packed weight layout, the
weight quantiser, and every refusal, of the Python entry points (before any
GPU is touched) and of the C entry points (before any launch)."""

import ctypes as C
import struct
from pathlib import Path

import numpy as np
import pytest
import torch

import lm_reference as ref
from heatvit_amd import _lib, lm
from heatvit_amd.device import DeviceF8Weight, pack_f8x64, quantise_f8_weight

LIB = Path(__file__).resolve().parents[1] / "heatvit_amd" / "libheatvit_hip.so"


# ------------------------------------------------------------------ weights

@pytest.mark.parametrize("size", ((16, 1), (128, 64), (144, 65), (400, 200)))
def test_f8x64_layout(size):
    """Element (k, n) lies where include/heatvit_hip.h says, the rest is 0."""
    k, n = size
    rng = np.random.default_rng(k)
    raw = rng.integers(1, 127, (k, n)).astype(np.uint8)
    w = torch.from_numpy(raw).view(torch.float8_e4m3fn)
    kb, ng = -(-k // 128), -(-n // 64)
    want = np.zeros(ng * kb * 8192, np.uint8)
    for kk in range(k):
        for nn in range(n):
            lane = 4 * (nn % 32 // 8) + nn % 4 + 16 * (kk % 64 // 16)
            part = nn % 64 // 32 * 2 + nn % 8 // 4
            at = ((nn // 64) * kb + kk // 128) * 8192 + part * 2048 + \
                (kk % 128 // 64) * 1024 + lane * 16 + kk % 16
            want[at] = raw[kk, nn]
    assert np.array_equal(pack_f8x64(w).numpy(), want)
    assert np.array_equal(pack_f8x64(w.t().contiguous().t()).numpy(), want)


def test_quantised_weight_values():
    g = torch.Generator().manual_seed(3)
    w = torch.randn(300, 140, generator=g) * 5
    w[:128, :128] = 0
    w[130, 130] = 448.0 * 4          # a block's border
    w[140, 20] = 448.0 * 4 + 0.25    # just past it
    q, e = quantise_f8_weight(w)
    flat = torch.zeros(384, 256)
    flat[:300, :140] = w
    flat = flat.view(3, 128, 2, 128).permute(0, 2, 1, 3).reshape(6, -1).double().numpy()
    assert np.array_equal(e.numpy().reshape(-1), ref.block_exps(flat, 0, 448.0).reshape(-1))
    s = np.repeat(ref.spread(e.numpy(), 128, 140), 128, axis=0)[:300]
    want = torch.from_numpy((w.double().numpy() / s).astype(np.float32)).to(torch.float8_e4m3fn)
    assert torch.equal(q.view(torch.uint8), want.view(torch.uint8))


def test_weight_refusals():
    f8 = torch.zeros(32, 40).to(torch.float8_e4m3fn)
    e = torch.zeros(1, 1, dtype=torch.int8)
    for bad in (lambda: DeviceF8Weight(torch.zeros(17, 4), device="cpu"),
                lambda: DeviceF8Weight(torch.zeros(4), device="cpu"),
                lambda: DeviceF8Weight(torch.zeros(0, 4), device="cpu"),
                lambda: DeviceF8Weight(f8, torch.zeros(1, 2, dtype=torch.int8), device="cpu")):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: DeviceF8Weight(torch.zeros(16, 4, dtype=torch.int8), device="cpu"),
                lambda: DeviceF8Weight(f8, e.int(), device="cpu"),
                lambda: DeviceF8Weight(f8.float(), e, device="cpu")):
        with pytest.raises(TypeError):
            bad()
    assert DeviceF8Weight(f8, e, device="cpu").packed.numel() == 8192


# ------------------------------------------------------------------ Python refusals

def _norm(**k):
    a = dict(x=torch.zeros(3, 130), weight=torch.ones(130))
    a.update(k)
    return lm.rms_norm_q8(a.pop("x"), a.pop("weight"), **a)


def test_norm_refusals():
    r = torch.zeros(3, 130)
    out = lm.Q8Rows(torch.zeros(3, 130).to(torch.float8_e4m3fn), torch.zeros(3, 2, dtype=torch.int8),
                    torch.zeros(3), None)
    for k in (dict(x=torch.zeros(130)), dict(x=torch.zeros(3, 0), weight=torch.ones(0)),
              dict(x=torch.zeros(130, 3).t()), dict(x=torch.zeros(1, 130).expand(3, 130)),
              dict(weight=torch.ones(129)), dict(weight=torch.ones(260)[::2]),
              dict(residual=torch.zeros(2, 130)), dict(residual=torch.zeros(130, 3).t()),
              dict(fmt="e5m2"), dict(block=64),
              dict(out=out._replace(exps=torch.zeros(3, 1, dtype=torch.int8))),
              dict(out=out._replace(scale=torch.zeros(2))), dict(residual=r, out=out),
              dict(out=out._replace(residual=r)),
              dict(live_rows=torch.zeros(2, dtype=torch.int32)),
              dict()):  # not on a GPU
        with pytest.raises(ValueError):
            _norm(**k)
    for k in (dict(x=np.zeros((3, 130))), dict(x=torch.zeros(3, 130).double()),
              dict(x=torch.zeros(3, 130, dtype=torch.int8)), dict(weight=torch.ones(130).half()),
              dict(residual=r.half()), dict(out=out._replace(q=torch.zeros(3, 130))),
              dict(fmt="int8", out=out)):
        with pytest.raises(TypeError):
            _norm(**k)


def _gemm(**k):
    a = dict(a=torch.zeros(3, 144).to(torch.float8_e4m3fn), e=torch.zeros(3, 2, dtype=torch.int8),
             w=DeviceF8Weight(torch.zeros(144, 20), device="cpu"))
    a.update(k)
    return lm.gemm_f8(a.pop("a"), a.pop("e"), a.pop("w"), **a)


def test_gemm_refusals():
    f8 = torch.float8_e4m3fn
    for k in (dict(a=torch.zeros(3, 128).to(f8)), dict(a=torch.zeros(144).to(f8)),
              dict(a=torch.zeros(144, 3).to(f8).t()), dict(e=torch.zeros(3, 1, dtype=torch.int8)),
              dict(e=torch.zeros(2, 2, dtype=torch.int8)), dict(row_scale=torch.zeros(2)),
              dict(bias=torch.zeros(3)), dict(bias=torch.zeros(40)[::2]),
              dict(out=torch.zeros(3, 21, dtype=torch.bfloat16)),
              dict(out=torch.zeros(20, 3, dtype=torch.bfloat16).t()), dict()):
        with pytest.raises(ValueError):
            _gemm(**k)
    for k in (dict(a=torch.zeros(3, 144)), dict(e=torch.zeros(3, 2)), dict(w=torch.zeros(144, 20)),
              dict(out_dtype=torch.int8), dict(row_scale=torch.zeros(3).half()),
              dict(out=torch.zeros(3, 20))):
        with pytest.raises(TypeError):
            _gemm(**k)


def _answer(logits=None, tokens=None, **k):
    return lm.log_probs(torch.zeros(3, 50) if logits is None else logits, tokens, **k)


def test_answer_refusals():
    t = torch.zeros(3, dtype=torch.int32)
    out = lm.LogProbs(torch.zeros(3), torch.zeros(3), None, None)
    for k in (dict(logits=torch.zeros(50)), dict(logits=torch.zeros(3, 0)),
              dict(logits=torch.zeros(50, 3).t()), dict(tokens=t[:2]),
              dict(tokens=torch.zeros(3, 4, dtype=torch.int32)[:, ::2]), dict(top=51),
              dict(top=-1), dict(logits=torch.zeros(3, 500), top=65), dict(temperature=0.0),
              dict(temperature=-1.0), dict(temperature=float("nan")),
              dict(temperature=float("inf")), dict(out=out), dict(tokens=t, top=2, out=out),
              dict(tokens=t, out=out._replace(entropy=torch.zeros(2))), dict(tokens=t)):
        with pytest.raises(ValueError):
            _answer(**k)
    for k in (dict(logits=torch.zeros(3, 50).double()), dict(tokens=t.long()),
              dict(tokens=[0, 1, 2]), dict(tokens=t, out=out._replace(logp=t))):
        with pytest.raises(TypeError):
            _answer(**k)


# ------------------------------------------------------------------ C refusals

@pytest.fixture(scope="module")
def library():
    if not LIB.exists():
        pytest.skip("library not built")
    L = C.CDLL(str(LIB))
    _lib._declare(L)
    return L


def _refused(L, rc, cls):
    assert rc == _lib.HV_EVALUE
    assert L.hv_last_error_class() == cls
    assert L.hv_last_error()


@pytest.mark.parametrize("desc", (_lib.RmsNormDesc, _lib.GemmF8Desc, _lib.LogProbsDesc))
def test_packed_descriptors(desc):
    """The packed bytes are the structure's, and a value too wide is an error."""
    values = [0.5 if t is C.c_float else 3 + i for i, (_, t) in enumerate(desc._fields_)]
    pack = _lib.packer(desc)
    assert pack(*values) == bytes(desc(*values))
    at = [t for _, t in desc._fields_].index(C.c_int32)
    values[at] = 1 << 31
    with pytest.raises(struct.error):
        pack(*values)


PTR = 4096  # never read: every call is refused, or has no rows


def test_norm_c_refusals(library):
    L = library

    def desc(**k):
        v = dict(x=PTR, weight=PTR, q=PTR, exps=PTR, scale=PTR, x_ld=256, q_ld=256, exps_ld=2,
                 rows=4, width=256, type=_lib.HV_T_BF16, format=_lib.HV_Q_E4M3, block=128, eps=1e-6)
        v.update(k)
        return C.byref(_lib.RmsNormDesc(**v))

    _refused(L, L.hv_rms_norm_q8(None, None), _lib.HV_ERR_ADDRESS)
    for k in (dict(type=3), dict(type=-1), dict(format=2)):
        _refused(L, L.hv_rms_norm_q8(desc(**k), None), _lib.HV_ERR_OPCODE)
    for k in (dict(block=64), dict(rows=-1), dict(rows=1 << 24), dict(width=0),
              dict(width=(1 << 20) + 1),
              dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(x_ld=255),
              dict(q_ld=8), dict(exps_ld=1), dict(residual=PTR, residual_out=PTR, residual_ld=8,
                                                  residual_out_ld=256)):
        _refused(L, L.hv_rms_norm_q8(desc(**k), None), _lib.HV_ERR_DIMENSION)
    for k in (dict(x=None), dict(weight=None), dict(q=None), dict(exps=None), dict(scale=None),
              dict(residual=PTR, residual_ld=256, residual_out_ld=256), dict(residual_out=PTR),
              dict(x=PTR + 1), dict(scale=PTR + 2)):
        _refused(L, L.hv_rms_norm_q8(desc(**k), None), _lib.HV_ERR_ADDRESS)
    assert L.hv_rms_norm_q8(desc(rows=0), None) == _lib.HV_OK


def test_gemm_c_refusals(library):
    L = library

    def call(**k):
        v = dict(a=PTR, a_exps=PTR, w_packed=PTR, w_exps=PTR, c=PTR, lda=256, a_exps_ld=2, ldc=64,
                 m=4, n=64, k=256, type=_lib.HV_T_BF16)
        v.update(k)
        return L.hv_gemm_f8(C.byref(_lib.GemmF8Desc(**v)), None)

    _refused(L, L.hv_gemm_f8(None, None), _lib.HV_ERR_ADDRESS)
    for k in (dict(type=3), dict(type=-1)):
        _refused(L, call(**k), _lib.HV_ERR_OPCODE)
    for k in (dict(m=-1), dict(n=0), dict(k=0), dict(k=250), dict(n=(1 << 22) + 1),
              dict(m=(1 << 24) + 1), dict(lda=240), dict(lda=264), dict(a_exps_ld=1),
              dict(ldc=63)):
        _refused(L, call(**k), _lib.HV_ERR_DIMENSION)
    for k in (dict(a=None), dict(a_exps=None), dict(w_packed=None), dict(w_exps=None),
              dict(c=None), dict(a=PTR + 8), dict(w_packed=PTR + 4), dict(c=PTR + 1),
              dict(bias=PTR + 2), dict(row_scale=PTR + 1)):
        _refused(L, call(**k), _lib.HV_ERR_ADDRESS)
    assert call(m=0) == _lib.HV_OK


def test_answer_c_refusals(library):
    L = library

    def call(**k):
        v = dict(logits=PTR, tokens=PTR, logp=PTR, entropy=PTR, top_logp=PTR, top_index=PTR,
                 logits_ld=100, tokens_ld=2, rows=4, width=100, type=_lib.HV_T_F32, n_tokens=2,
                 top=5, scale=1.0)
        v.update(k)
        return L.hv_log_probs(C.byref(_lib.LogProbsDesc(**v)), None, 0, None)

    _refused(L, L.hv_log_probs(None, None, 0, None), _lib.HV_ERR_ADDRESS)
    for k in (dict(type=4), dict(type=-1)):
        _refused(L, call(**k), _lib.HV_ERR_OPCODE)
    for k in (dict(rows=-1), dict(rows=1 << 24), dict(width=0), dict(n_tokens=-1),
              dict(width=(1 << 30) + 1, logits_ld=1 << 31),
              dict(n_tokens=(1 << 30) + 1, tokens_ld=1 << 31),
              dict(logits_ld=99), dict(tokens_ld=1), dict(top=-1), dict(top=65), dict(top=101), dict(scale=0.0),
              dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf"))):
        _refused(L, call(**k), _lib.HV_ERR_DIMENSION)
    for k in (dict(logits=None), dict(entropy=None), dict(tokens=None), dict(logp=None),
              dict(top_logp=None), dict(top_index=None), dict(logits=PTR + 2),
              dict(entropy=PTR + 1)):
        _refused(L, call(**k), _lib.HV_ERR_ADDRESS)
    assert call(rows=0) == _lib.HV_OK
