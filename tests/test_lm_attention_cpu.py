"""The attention operators without a GPU: where rows, keys and pages lie for
good and bad offsets, lengths and tables, and every refusal, of the Python
entry points (before any GPU is touched) and of the C entry points (before any
launch)."""

import ctypes as C
import math
from pathlib import Path

import numpy as np
import pytest
import torch

import lm_attention_kernels
from heatvit_amd import _lib, lm

ROOT = Path(__file__).resolve().parents[1]
LIB = ROOT / "heatvit_amd" / "libheatvit_hip.so"
BF, HF = torch.bfloat16, torch.float16
F8 = torch.float8_e4m3fn


# ------------------------------------------------------------------ places

@pytest.fixture(scope="module")
def places():
    return lm_attention_kernels.library()


def test_rows_stay_inside(places):
    """Whatever the offsets are, a sequence's rows lie in [0, rows)."""
    rng = np.random.default_rng(0)
    out = np.zeros(2, np.int32)
    for _ in range(300):
        rows = int(rng.integers(0, 50))
        starts = rng.choice([-2 ** 31, -5, 0, 3, 7, 20, 49, 50, 51, 2 ** 31 - 1], 6).astype(np.int32)
        for b in range(5):
            places.seq_rows_of(starts.ctypes.data, b, rows, out.ctypes.data)
            first, count = out
            assert count >= 0 and first >= 0 and first + count <= rows
            lo, hi = np.clip(starts[b:b + 2].astype(np.int64), 0, rows)
            assert count == max(hi - lo, 0)
    places.seq_rows_of(None, 3, 5, out.ctypes.data)
    assert out.tolist() == [3, 1]
    places.seq_rows_of(None, 5, 5, out.ctypes.data)
    assert out[1] == 0


def test_pages(places):
    table = np.array([4, 0, -1, 5, 2 ** 31 - 1, -2 ** 31], np.int32)
    shift, pages, most = 4, 5, 6

    def page(position):
        return places.page_at(pages, shift, most, table.ctypes.data, position)

    assert [page(16 * i + 15) for i in range(6)] == [4, 0, -1, -1, -1, -1]
    for bad in (-1, -2 ** 40, 96, 2 ** 31, 2 ** 40):
        assert page(bad) == -1
    assert places.keys_of(pages, shift, most, 96) == 96
    assert places.keys_of(pages, shift, most, 97) == -1
    assert places.keys_of(pages, shift, most, 2 ** 31 - 1) == -1
    for none in (0, -1, -2 ** 31):
        assert places.keys_of(pages, shift, most, none) == 0
    assert places.keys_of(pages, shift, 0, 1) == -1
    for heads, p, h, at in ((3, 4, 2, 17), (1, 0, 0, 0), (4096, 2 ** 20, 4095, 2 ** 31 - 1)):
        assert places.row_at(pages, shift, heads, p, h, at) == (p * heads + h) * 16 + at % 16


def test_what_a_row_sees(places):
    out = np.zeros(2, np.int32)
    for n in (1, 2, 5):
        for keys in (0, 1, 2, 5, 9):
            for causal, window in ((0, 0), (1, 0), (1, 1), (1, 3), (1, 2 ** 31 - 1)):
                for i in range(n):
                    places.seen_at(i, n, keys, causal, window, out.ctypes.data)
                    want = [j for j in range(keys) if not causal or
                            (j <= keys - n + i and (not window or j > keys - n + i - window))]
                    assert list(range(*out)) == want
    places.seen_at(0, 2 ** 24, 2 ** 31 - 1, 1, 0, out.ctypes.data)
    assert out.tolist() == [0, 2 ** 31 - 1 - 2 ** 24 + 1]


def test_kernels():
    """Few rows a sequence, or tiles; shares where tiles leave the card idle and
    the keys are many; a workspace where there may be shares, and only there."""
    of = lm_attention_kernels.kernel_of
    assert of(1, 1, 32, 8, 128, 32768) == "few in shares"
    assert of(8, 8, 16, 16, 64, 1008) == "few"
    assert of(4096, 4096, 8, 8, 64, 4096) == "few"
    assert of(8192, 1, 32, 8, 128, 8192) == "tiles"
    assert of(50432, 256, 3, 3, 64, 50432) == "tiles"
    assert of(100, 1, 4, 1, 64, 100) == "tiles"
    assert of(648, 4, 32, 8, 128, 16384) == "tiles in shares"
    for rows, batch, heads, kv, width in ((1, 1, 1, 1, 8), (4096, 4096, 8, 8, 64), (648, 4, 32, 8, 128),
                                          (8192, 1, 32, 8, 128), (300, 1, 4, 4, 256)):
        size = lm_attention_kernels.library().attention_workspace(rows, batch, heads, kv, width)
        if "shares" in of(rows, batch, heads, kv, width, 1 << 30):
            assert 0 < size < 1 << 28
        else:
            assert size == 0


def test_kernels_by_the_longest_sequence():
    """Many short sequences are no long one: neither their keys' sum nor a wide
    table that the caller says more about cuts their work into shares."""
    L, of = lm_attention_kernels.library(), lm_attention_kernels.kernel_of
    for rows, batch, heads, kv, width in ((8 * 512, 8, 4, 4, 128), (16 * 100, 16, 8, 1, 64),
                                          (32 * 128, 32, 8, 2, 128), (8 * 300, 8, 8, 2, 64),
                                          (4 * 1024, 4, 8, 2, 128)):
        assert of(rows, batch, heads, kv, width, rows) == "tiles in shares"
        assert of(rows, batch, heads, kv, width, L.packed_keys(0, rows, batch)) == "tiles"
    assert of(3200, 200, 8, 8, 128, 3200) == "few in shares"
    assert of(3200, 200, 8, 8, 128, L.packed_keys(0, 3200, 200)) == "few"
    assert of(4096, 1, 8, 8, 128, L.packed_keys(0, 4096, 1)) == "tiles in shares"
    assert of(8, 8, 16, 4, 128, L.packed_keys(0, 4700, 8)) == "few"
    assert of(8, 8, 16, 4, 128, L.packed_keys(4000, 4700, 8)) == "few in shares"
    assert of(4, 4, 16, 4, 64, L.packed_keys(0, 16300, 4)) == "few in shares"
    for rows, heads, kv, width, kind in ((512, 32, 8, 128, "tiles"), (1, 32, 8, 128, "few")):
        assert of(rows, 1, heads, kv, width, L.table_keys(0, 131072)) == kind + " in shares"
        assert of(rows, 1, heads, kv, width, L.table_keys(512, 131072)) == kind
    assert L.table_keys(0, 96) == 96 and L.table_keys(7, 96) == 7
    for said, total, batch, want in ((0, 0, 5, 0), (0, 1, 5, 1), (0, 10, 1, 10), (0, 10, 2, 10), (0, 10, 5, 4),
                                     (3, 10, 5, 3), (0, 2 ** 24, 3, 2 * 5592406), (2 ** 31 - 1, 1, 1, 2 ** 31 - 1)):
        assert L.packed_keys(said, total, batch) == want


def test_runs():
    """Workgroups in runs take every place once, and an XCD's are side by side."""
    L = lm_attention_kernels.library()
    for run in (2, 6, 9, 12, 20):
        places = np.array([L.place_in_runs(b, run) for b in range(3 * 8 * run)])
        assert (np.sort(places) == np.arange(places.size)).all()
        for xcd in range(8):
            assert (places[xcd::8].reshape(3, run) ==
                    np.arange(3)[:, None] * 8 * run + xcd * run + np.arange(run)).all()
    assert L.attention_run(256 * 197, 256, 3, 3, 64, 0) == 6
    assert L.attention_run(256 * 577, 256, 3, 3, 64, 0) == 12
    for none in ((256 * 197, 256, 16, 8, 64, 0), (4096, 4096, 12, 3, 64, 0), (8192, 1, 4, 4, 128, 0),
                 (256 * 197, 256, 3, 3, 64, 1)):
        assert L.attention_run(*none) == 0


def test_shares():
    """Shares of the work cover it, one behind the other, and a tile's parts are
    the shares that it reaches into."""
    L = lm_attention_kernels.library()
    out = np.zeros(4, np.int32)

    def numbers(cost, groups, share=0, at=0, end=1):
        L.share_numbers(cost, groups, share, at, end, out.ctypes.data)
        return out.tolist()

    for cost in (16, 63, 64, 640, 512 * 64 - 1, 512 * 64, 1000003, (1 << 30) + (1 << 28) + 7):
        for groups in (256, 512):
            n = numbers(cost, groups)[0]
            assert n == min(max(cost // 64, 1), groups)
            starts = [numbers(cost, groups, i)[1] for i in range(n + 1)]
            assert starts[0] == 0 and starts[n] == cost and min(np.diff(starts)) >= min(64, cost)
            for i in range(n):
                assert numbers(cost, groups, at=starts[i])[2] == i
                assert numbers(cost, groups, at=starts[i + 1] - 1)[2] == i
                last = min(i + 3, n)
                assert numbers(cost, groups, i, end=starts[last])[3] == last - i
    for first, step, count in ((16, 0, 1), (48, 0, 300), (32, 8, 4000), (1 << 18, 32, 4096)):
        for tile in sorted({0, count // 3, count - 1}):
            lo, hi = (L.cost_before(first, step, count, t) for t in (tile, tile + 1))
            for at in (lo, (lo + hi) // 2, hi - 1):
                assert L.tile_of_cost(first, step, count, at) == tile
    for n in (0, 1, 7, 1 << 24):
        assert L.part_of_tiles(n, 0, 64) == 0 and L.part_of_tiles(n, 64, 64) == n


def test_shares_of_numbers_past_32_bits():
    """What sums of overlapping sequences may wrap to still gives tiles, parts
    and shares that there are."""
    L = lm_attention_kernels.library()
    out = np.zeros(4, np.int32)
    rng = np.random.default_rng(0)
    edges = [-2 ** 31, -2 ** 31 + 1, -1, 0, 1, 31, 2 ** 18, 2 ** 30, 2 ** 31 - 1]
    some = edges + rng.integers(-2 ** 31, 2 ** 31 - 1, 40).tolist()
    for cost in (1, 32, 100, 2 ** 18, 2 ** 31 - 1):
        for at in some:
            for n in (0, 1, 5, 1 << 24):
                assert 0 <= L.part_of_tiles(n, at, cost) <= n
            for groups in (256, 512):
                L.share_numbers(cost, groups, 0, 0, 1, out.ctypes.data)
                n = int(out[0])
                for share in (0, n // 2, n - 1):
                    L.share_numbers(cost, groups, share, 0, at, out.ctypes.data)
                    assert 1 <= out[3] <= n - share
    for first, step, count in ((16, 0, 5), (1 << 18, 0, 1 << 14), (1 << 18, 32, 4096), (1 << 18, 32, 30000)):
        for at in some:
            assert 0 <= L.tile_of_cost(first, step, count, max(at, 0)) < count


def test_lanes_of_a_head():
    """Every head that rotary_qk takes has 65 lanes at most, the last of which
    then has up to 16 elements, none of them rotated."""
    L = lm_attention_kernels.library()
    wide = 0
    for width in range(1, _lib.HV_ROTARY_MAX_WIDTH + 1):
        for pairs in range(width // 2 + 1):
            lanes, of_pairs = L.lanes_of_head(pairs, width), -(-pairs // 8)
            assert lanes <= 65 and lanes * 16 >= width
            if lanes == 65:
                wide += 1
                assert of_pairs <= 64 and 0 < width - 2 * pairs - 16 * (64 - of_pairs) <= 16
    assert wide


# ------------------------------------------------------------------ frequencies

def test_frequencies():
    f = lm.rotary_frequencies(64, 500.0)
    want = [500.0 ** (-2 * i / 64) for i in range(32)]
    assert f.dtype == torch.float32 and np.allclose(f, want, rtol=2 ** -23)
    assert np.allclose(lm.rotary_frequencies(64, 500.0, factor=4.0), np.array(want) / 4, rtol=2 ** -23)
    g = lm.rotary_frequencies(64, 500.0, factor=8.0, trained=256, low=1.0, high=4.0)
    for i, w in enumerate(want):
        turns = w * 256 / (2 * math.pi)
        stay = min(max((turns - 1) / 3, 0), 1)
        assert abs(g[i] - w * (stay + (1 - stay) / 8)) <= 2 ** -23 * w
    assert g[0] == f[0] and g[-1] == f[-1] / 8
    assert lm.rotary_frequencies(0).numel() == 0
    for bad in (dict(rotated=3), dict(rotated=-2), dict(rotated=2048), dict(rotated=4, base=0.0),
                dict(rotated=4, factor=0.0), dict(rotated=4, factor=math.inf),
                dict(rotated=4, trained=0), dict(rotated=4, trained=8, low=4.0, high=4.0)):
        with pytest.raises(ValueError):
            lm.rotary_frequencies(**bad)


# ------------------------------------------------------------------ Python refusals

def _refuse(call, values, types):
    for k in values:
        with pytest.raises(ValueError):
            call(**k)
    for k in types:
        with pytest.raises(TypeError):
            call(**k)


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def test_rotary_refusals():
    def call(**k):
        a = dict(q=torch.zeros(3, 4, 16), k=torch.zeros(3, 2, 16), positions=_i32(3),
                 freqs=torch.ones(8))
        a.update(k)
        return lm.rotary_qk(a.pop("q"), a.pop("k"), a.pop("positions"), a.pop("freqs"), **a)

    out = lm.QK(torch.zeros(3, 4, 16), torch.zeros(3, 2, 16))
    w = torch.ones(16)
    _refuse(call, (
        dict(q=torch.zeros(3, 64)), dict(q=torch.zeros(3, 0, 16)), dict(q=torch.zeros(3, 4, 0)),
        dict(q=torch.zeros(3, 4, 1026), k=None), dict(q=torch.zeros(3, 16, 4).transpose(1, 2)),
        dict(q=torch.zeros(3, 1, 16).expand(3, 4, 16)), dict(k=torch.zeros(2, 2, 16)),
        dict(k=torch.zeros(3, 2, 8)), dict(k=torch.zeros(3, 0, 16)), dict(positions=_i32(2)),
        dict(positions=_i32(3, 1)), dict(positions=_i32(6)[::2]), dict(freqs=torch.ones(9)),
        dict(freqs=torch.ones(4, 2)), dict(freqs=torch.ones(8)[::2]), dict(layout="pairs"),
        dict(scale=math.inf), dict(scale=math.nan), dict(q_weight=torch.ones(15)),
        dict(k_weight=torch.ones(32)[::2]), dict(k=None, k_weight=w), dict(k=None, out=out),
        dict(out=lm.QK(torch.zeros(3, 4, 8), out.k)), dict(out=lm.QK(out.q, None)),
        dict(out=lm.QK(torch.zeros(3, 1, 16).expand(3, 4, 16), out.k)),
        dict(live_rows=_i32(2)), dict(),  # not on a GPU
    ), (
        dict(q=np.zeros((3, 4, 16))), dict(q=torch.zeros(3, 4, 16).double()),
        dict(k=torch.zeros(3, 2, 16).half()), dict(positions=torch.zeros(3, dtype=torch.int64)),
        dict(freqs=torch.ones(8).double()), dict(q_weight=w.half()),
        dict(out=lm.QK(out.q.half(), out.k)),
    ))


def test_cache_refusals():
    def cache(**k):
        a = dict(k=torch.zeros(5, 2, 16, 32, dtype=BF), v=torch.zeros(5, 2, 16, 32, dtype=BF))
        a.update(k)
        return lm.KvCache(a.pop("k"), a.pop("v"), **a)

    e = torch.zeros(5, 2, 16, dtype=torch.int8)
    f8 = torch.zeros(5, 2, 16, 32).to(F8)
    _refuse(cache, (
        dict(k=torch.zeros(5, 2, 16, dtype=BF)), dict(v=torch.zeros(5, 2, 16, 40, dtype=BF)),
        dict(k=torch.zeros(5, 2, 32, 16, dtype=BF).transpose(2, 3)), dict(k_exps=e, v_exps=e),
        dict(k=f8, v=f8), dict(k=f8, v=f8, k_exps=e), dict(k=f8, v=f8, k_exps=e, v_exps=e[:4]),
        *(dict(k=torch.zeros(s, dtype=BF), v=torch.zeros(s, dtype=BF)) for s in (
            (0, 2, 16, 32), (5, 0, 16, 32), (5, 2, 24, 32), (5, 2, 8, 32), (1, 1, 8192, 32),
            (5, 2, 16, 36), (5, 2, 16, 0), (5, 2, 16, 264))),
        dict(k=torch.zeros(5, 2, 16, 24).to(F8), v=torch.zeros(5, 2, 16, 24).to(F8), k_exps=e, v_exps=e),
    ), (
        dict(k=np.zeros(3)), dict(k=torch.zeros(5, 2, 16, 32), v=torch.zeros(5, 2, 16, 32)),
        dict(v=torch.zeros(5, 2, 16, 32, dtype=HF)), dict(dtype=HF),
        dict(k=f8, v=f8, k_exps=e, v_exps=e, dtype=torch.float32),
    ))
    c = lm.KvCache.empty(5, 2, 32, page=32, dtype=HF, e4m3=True, device="cpu")
    assert c.k.shape == (5, 2, 32, 32) and c.k.dtype == F8 and c.v_exps.shape == (5, 2, 32)
    assert c.dtype == HF


def _write(**k):
    a = dict(cache=lm.KvCache.empty(5, 2, 32, page=16, device="cpu"),
             k=torch.zeros(3, 2, 32, dtype=BF), v=torch.zeros(3, 2, 32, dtype=BF), table=_i32(3, 2),
             lengths=_i32(3))
    a.update(k)
    return lm.cache_write(a.pop("cache"), a.pop("k"), a.pop("v"), a.pop("table"), a.pop("lengths"), **a)


def test_write_refusals():
    _refuse(_write, (
        dict(k=torch.zeros(3, 3, 32, dtype=BF)), dict(k=torch.zeros(3, 2, 40, dtype=BF)),
        dict(v=torch.zeros(2, 2, 32, dtype=BF)), dict(table=_i32(2, 2)), dict(table=_i32(6)),
        dict(table=_i32(2, 3).t()), dict(lengths=_i32(2)), dict(starts=_i32(3)), dict(starts=_i32(0)),
        dict(starts=_i32(8)[::2]), dict(),  # not on a GPU
    ), (
        dict(cache=torch.zeros(3)), dict(k=torch.zeros(3, 2, 32)), dict(v=torch.zeros(3, 2, 32)),
        dict(table=torch.zeros(3, 2)), dict(lengths=torch.zeros(3, dtype=torch.int64)),
        dict(starts=torch.zeros(4)),
    ))


ROWS_BAD = (dict(most_keys=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf),
            dict(window=-1), dict(window=3, causal=False),
            dict(q=torch.zeros(3, 5, 32, dtype=BF)), dict(q=torch.zeros(3, 4, 36, dtype=BF)),
            dict(q=torch.zeros(3, 4, 40, dtype=BF)), dict(q=torch.zeros(3, 0, 32, dtype=BF)),
            dict(q=torch.zeros(3, 4, 36, dtype=BF)[..., :32]),
            dict(q=torch.zeros(385, dtype=BF)[1:].view(3, 4, 32)),
            dict(out=lm.Attended(torch.zeros(3, 4, 32, dtype=BF), torch.zeros(3, 4))),
            dict(lse=True, out=lm.Attended(torch.zeros(3, 4, 32, dtype=BF), None)),
            dict(lse=True, out=lm.Attended(torch.zeros(3, 4, 32, dtype=BF), torch.zeros(4, 3))),
            dict(out=lm.Attended(torch.zeros(3, 4, 40, dtype=BF), None)),
            dict(out=lm.Attended(torch.zeros(3, 4, 36, dtype=BF)[..., :32], None)))


def test_attention_refusals():
    def call(**k):
        a = dict(q=torch.zeros(3, 4, 32, dtype=BF), k=torch.zeros(3, 2, 32, dtype=BF),
                 v=torch.zeros(3, 2, 32, dtype=BF), starts=_i32(2))
        a.update(k)
        return lm.attention(a.pop("q"), a.pop("k"), a.pop("v"), a.pop("starts"), **a)

    kv5 = torch.zeros(5, 2, 32, dtype=BF)
    _refuse(call, ROWS_BAD + (
        dict(k=kv5, v=kv5), dict(k=kv5), dict(k_starts=_i32(3)), dict(starts=_i32(0)),
        dict(starts=_i32(4)[::2]), dict(k=torch.zeros(3, 2, 36, dtype=BF)[..., :32]),
        dict(v=torch.zeros(193, dtype=BF)[1:].view(3, 2, 32)),
        dict(k=torch.zeros(3, 0, 32, dtype=BF), v=torch.zeros(3, 0, 32, dtype=BF)),
        dict(k=torch.zeros(3, 2, 264, dtype=BF), v=torch.zeros(3, 2, 264, dtype=BF),
             q=torch.zeros(3, 4, 264, dtype=BF)), dict(),  # not on a GPU
    ), (
        dict(q=torch.zeros(3, 4, 32)), dict(q=[1]), dict(k=torch.zeros(3, 2, 32, dtype=HF)),
        dict(v=torch.zeros(3, 2, 32, dtype=HF)), dict(starts=None), dict(starts=torch.zeros(2)),
        dict(k_starts=torch.zeros(2)), dict(out=lm.Attended(torch.zeros(3, 4, 32), None)),
    ))


def test_paged_refusals():
    def call(**k):
        a = dict(q=torch.zeros(3, 4, 32, dtype=BF),
                 cache=lm.KvCache.empty(5, 2, 32, page=16, device="cpu"), table=_i32(3, 2),
                 lengths=_i32(3))
        a.update(k)
        return lm.paged_attention(a.pop("q"), a.pop("cache"), a.pop("table"), a.pop("lengths"), **a)

    _refuse(call, ROWS_BAD + (
        dict(table=_i32(2, 2)), dict(lengths=_i32(2)), dict(starts=_i32(3)), dict(starts=_i32(0)),
        dict(),  # not on a GPU
    ), (
        dict(cache=3), dict(q=torch.zeros(3, 4, 32, dtype=HF)), dict(q=torch.zeros(3, 4, 32)),
        dict(table=torch.zeros(3, 2)), dict(lengths=torch.zeros(3)), dict(starts=torch.zeros(4)),
    ))


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


PTR = 4096  # never read: every call is refused, or has no rows


def _check(L, call, opcode, dimension, address):
    for cls, cases in ((_lib.HV_ERR_OPCODE, opcode), (_lib.HV_ERR_DIMENSION, dimension),
                       (_lib.HV_ERR_ADDRESS, address)):
        for k in cases:
            _refused(L, call(**k), cls)
    assert call(rows=0) == _lib.HV_OK


@pytest.mark.parametrize("desc", (_lib.RotaryDesc, _lib.CacheWriteDesc, _lib.AttentionDesc,
                                  _lib.PagedAttentionDesc))
def test_packed_descriptors(desc):
    values = [0.5 if t is C.c_float else 3 + i for i, (_, t) in enumerate(desc._fields_)]
    assert _lib.packer(desc)(*values) == bytes(desc(*values))


def test_rotary_c_refusals(library):
    L = library

    def call(**k):
        v = dict(q=PTR, k=PTR, q_out=PTR, k_out=PTR, positions=PTR, freqs=PTR, q_ld=64, q_head_ld=16,
                 k_ld=32, k_head_ld=16, q_out_ld=64, q_out_head_ld=16, k_out_ld=32, k_out_head_ld=16,
                 rows=4, q_heads=4, k_heads=2, width=16, rotated=16, type=_lib.HV_T_BF16, eps=1e-6,
                 scale=1.0)
        v.update(k)
        return L.hv_rotary_qk(C.byref(_lib.RotaryDesc(**v)), None)

    _refused(L, L.hv_rotary_qk(None, None), _lib.HV_ERR_ADDRESS)
    _check(L, call, (dict(type=3), dict(type=-1), dict(layout=2)), (
        dict(rows=-1), dict(rows=1 << 24), dict(q_heads=0), dict(k_heads=-1), dict(q_heads=4097),
        dict(width=0), dict(width=1025), dict(rotated=17), dict(rotated=18), dict(rotated=-2),
        dict(eps=-1.0), dict(eps=math.nan), dict(scale=math.inf), dict(scale=math.nan),
        dict(q_ld=-1), dict(k_out_head_ld=-1)), (
        dict(q=None), dict(k=None), dict(q_out=None), dict(k_out=None), dict(positions=None),
        dict(freqs=None), dict(q=PTR + 1), dict(k_weight=PTR + 1), dict(positions=PTR + 2),
        dict(freqs=PTR + 1)))


CACHE = dict(cache_k=PTR, cache_v=PTR, table=PTR, lengths=PTR, table_ld=4, pages=5, page=16,
             max_pages=4, format=_lib.HV_CACHE_SAME)
CACHE_DIMENSION = (dict(page=8), dict(page=24), dict(page=8192), dict(page=0), dict(page=-16),
                   dict(pages=0), dict(max_pages=-1), dict(table_ld=3), dict(width=0),
                   dict(max_pages=1 << 28, table_ld=1 << 28), dict(max_pages=(1 << 26) + 1, table_ld=1 << 27),
                   dict(width=20), dict(width=264), dict(width=24, format=_lib.HV_CACHE_E4M3))
CACHE_ADDRESS = (dict(cache_k=None), dict(cache_v=None), dict(table=None), dict(lengths=None),
                 dict(format=_lib.HV_CACHE_E4M3), dict(cache_k=PTR + 8), dict(table=PTR + 2),
                 dict(lengths=PTR + 1))


def test_write_c_refusals(library):
    L = library

    def call(**k):
        v = dict(CACHE, k=PTR, v=PTR, starts=PTR, k_ld=64, k_head_ld=32, v_ld=64, v_head_ld=32,
                 rows=4, batch=2, kv_heads=2, width=32, type=_lib.HV_T_BF16)
        v.update(k)
        return L.hv_cache_write(C.byref(_lib.CacheWriteDesc(**v)), None)

    _refused(L, L.hv_cache_write(None, None), _lib.HV_ERR_ADDRESS)
    _check(L, call, (dict(type=0), dict(type=3), dict(format=2)), CACHE_DIMENSION + (
        dict(rows=-1), dict(rows=1 << 24), dict(batch=-1), dict(kv_heads=0), dict(kv_heads=4097),
        dict(rows=1 << 20, kv_heads=65), dict(starts=None), dict(k_ld=-1), dict(v_head_ld=-1)),
        CACHE_ADDRESS + (dict(k=None), dict(v=None), dict(k=PTR + 1), dict(starts=PTR + 2)))
    assert call(batch=0) == _lib.HV_OK
    assert call(max_pages=0) == _lib.HV_OK  # no place for any row


ROWS = dict(q=PTR, out=PTR, starts=PTR, q_ld=128, q_head_ld=32, out_ld=128, out_head_ld=32, rows=4,
            batch=2, heads=4, kv_heads=2, width=32, type=_lib.HV_T_BF16, causal=1, scale=0.1)
ROWS_DIMENSION = (dict(rows=-1), dict(rows=1 << 24), dict(batch=-1), dict(heads=0), dict(heads=3),
                  dict(kv_heads=0), dict(heads=8192), dict(rows=1 << 20, heads=128), dict(width=0),
                  dict(width=20), dict(width=264), dict(window=-1), dict(window=2, causal=0),
                  dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf),
                  dict(q_ld=100), dict(out_head_ld=4), dict(q_ld=-8), dict(most_keys=-1))
ROWS_ADDRESS = (dict(q=None), dict(out=None), dict(q=PTR + 8), dict(out=PTR + 2), dict(lse=PTR + 2),
                dict(starts=PTR + 2))


def test_attention_c_refusals(library):
    L = library

    def call(**k):
        v = dict(ROWS, k=PTR, v=PTR, k_ld=64, k_head_ld=32, v_ld=64, v_head_ld=32, k_rows=4)
        v.update(k)
        if "rows" in k:
            v["k_rows"] = v["rows"]
        return L.hv_attention(C.byref(_lib.AttentionDesc(**v)), None, 0, None)

    _refused(L, L.hv_attention(None, None, 0, None), _lib.HV_ERR_ADDRESS)
    _check(L, call, (dict(type=0), dict(type=3)), ROWS_DIMENSION + (
        dict(k_rows=5), dict(k_rows=-1), dict(k_rows=1 << 24, k_starts=PTR), dict(k_ld=60),
        dict(v_head_ld=-8), dict(k_ld=(1 << 23) + 8), dict(v_ld=(1 << 23) + 8)), ROWS_ADDRESS + (
        dict(k=None), dict(v=None), dict(starts=None), dict(k=PTR + 8), dict(k_starts=PTR + 1)))
    assert call(batch=0) == _lib.HV_OK


def test_paged_c_refusals(library):
    L = library

    def call(**k):
        v = dict(ROWS, **CACHE)
        v.update(k)
        return L.hv_paged_attention(C.byref(_lib.PagedAttentionDesc(**v)), None, 0, None)

    _refused(L, L.hv_paged_attention(None, None, 0, None), _lib.HV_ERR_ADDRESS)
    _check(L, call, (dict(type=0), dict(type=3), dict(format=2)),
           ROWS_DIMENSION + CACHE_DIMENSION + (dict(starts=None),), ROWS_ADDRESS + CACHE_ADDRESS)
    assert call(batch=0) == _lib.HV_OK
