"""The attention operators of heatvit_amd.lm (rotary_qk, cache_write,
attention, paged_attention) against their plain 64-bit forms, at the sizes,
strides, masks, pages and values where they can go wrong, and a run of them
with the norm, the product and the answer."""

import math

import numpy as np
import pytest
import torch

import lm_attention_kernels
import lm_attention_reference as ref

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
HALVES = ("bf16", "f16")


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _bytes(t):
    return t.contiguous().cpu().view(torch.uint8).numpy()


def _dev(t):
    return None if t is None else t.cuda()


def _i32(values):
    return torch.tensor(values, dtype=torch.int32)


# ------------------------------------------------------------------ rotary_qk

def _rotary_inputs(rows, heads, kv, width, rotated, dtype, norm, seed, first=0):
    from heatvit_amd import lm
    g = _gen(seed)
    q = (torch.randn(rows, heads, width, generator=g) * 2).to(dtype)
    k = torch.randn(rows, kv, width, generator=g).to(dtype) if kv else None
    w = [(1 + 0.3 * torch.randn(width, generator=g)).to(dtype) if norm and x is not None else None
         for x in (q, k)]
    p = _i32([first + 3 * i for i in range(rows)])
    return q, k, w, p, lm.rotary_frequencies(rotated, 10000.0)


def _check_rotary(got, q, k, w, p, f, eps, layout, scale):
    for name, x, wt in (("q", q, w[0]), ("k", k, w[1])):
        if x is not None:
            ref.check(getattr(got, name), *ref.rotary(x, wt, p, f, eps, layout, scale), name)


@pytest.mark.parametrize("layout", ("half", "interleaved"))
@pytest.mark.parametrize("norm", (False, True))
@pytest.mark.parametrize("kind", TYPES)
def test_rotary_sizes(kind, norm, layout):
    from heatvit_amd import lm
    for rows, heads, kv, width, rotated in (
            (1, 1, 0, 2, 2), (1, 32, 8, 128, 128), (3, 3, 3, 64, 64), (5, 5, 1, 6, 4),
            (7, 2, 1, 1, 0), (9, 4, 2, 80, 40), (17, 6, 3, 100, 50), (2, 3, 1, 256, 192),
            (4, 2, 2, 30, 30), (33, 8, 2, 96, 18), (2, 1, 1, 1024, 1024), (3, 2, 1, 515, 512),
            (70, 3, 1, 128, 0)):
        x = _rotary_inputs(rows, heads, kv, width, rotated, TYPES[kind], norm, rows + width, 1000)
        q, k, w, p, f = x
        print(f"rotary {kind} {layout} {rows} x {heads}+{kv} x {width}/{rotated}", flush=True)
        got = lm.rotary_qk(q.cuda(), _dev(k), p.cuda(), f.cuda(), q_weight=_dev(w[0]),
                           k_weight=_dev(w[1]), eps=1e-5, layout=layout, scale=1.25)
        _check_rotary(got, q, k, w, p, f, 1e-5, layout, 1.25)


@pytest.mark.parametrize("layout", ("half", "interleaved"))
@pytest.mark.parametrize("norm", (False, True))
@pytest.mark.parametrize("kind", TYPES)
def test_rotary_heads_of_65_lanes(kind, norm, layout):
    """Heads both parts of which end within a lane: all elements count in the
    norm and are written, and nothing else is.  (A lane adds 17 squares in a row
    here, half a step of float32 after the root that the bound's 21 have: the
    mean's and eps' steps are halved by the root too.)"""
    from heatvit_amd import lm
    for width, rotated in ((1024, 2), (1024, 1022), (1011, 2), (1024, 500), (1020, 1002), (1024, 0)):
        assert rotated == 0 or lm_attention_kernels.library().lanes_of_head(rotated // 2, width) == 65
        q, k, w, p, f = _rotary_inputs(5, 3, 2, width, rotated, TYPES[kind], norm, rotated, 77)
        q[1, :, -1], q[2, :, :-1] = 100, 0  # a last element that the norm hangs on
        print(f"rotary {kind} {layout} {width}/{rotated}", flush=True)
        buf = [torch.full((5, n, width + 3), 9.0, dtype=q.dtype, device="cuda") for n in (3, 2)]
        out = lm.QK(*(t[..., 1:1 + width] for t in buf))
        args = dict(q_weight=_dev(w[0]), k_weight=_dev(w[1]), eps=1e-5, layout=layout)
        got = lm.rotary_qk(q.cuda(), k.cuda(), p.cuda(), f.cuda(), out=out, **args)
        _check_rotary(got, q, k, w, p, f, 1e-5, layout, 1.0)
        assert all((t[..., 0] == 9).all() and (t[..., 1 + width:] == 9).all() for t in buf)
        qv, kv = (t.cuda() for t in (q, k))
        lm.rotary_qk(qv, kv, p.cuda(), f.cuda(), out=lm.QK(qv, kv), **args)
        assert torch.equal(qv, got.q) and torch.equal(kv, got.k)


def test_rotary_heads_of_65_lanes_at_the_edges():
    """Squares that leave float32, of such heads' last elements."""
    from heatvit_amd import lm
    q, k, w, p, f = _rotary_inputs(4, 2, 1, 1024, 998, torch.float32, True, 1)
    info = torch.finfo(torch.float32)
    q[0, 0], q[0, 0, -1] = 0, info.max / 4
    q[1, 1] = 0
    q[2, 0], q[2, 0, -1] = 0, info.smallest_normal
    for eps in (1e-6, 0.0):
        with np.errstate(all="ignore"):
            got = lm.rotary_qk(q.cuda(), k.cuda(), p.cuda(), f.cuda(), q_weight=w[0].cuda(),
                               k_weight=w[1].cuda(), eps=eps)
            _check_rotary(got, q, k, w, p, f, eps, "half", 1.0)


@pytest.mark.parametrize("rows", (63, 1025, 5000))
def test_rotary_many_rows(rows):
    from heatvit_amd import lm
    for heads, kv, width, rotated in ((2, 1, 32, 32), (3, 3, 64, 20)):
        q, k, w, p, f = _rotary_inputs(rows, heads, kv, width, rotated, torch.bfloat16, True, rows)
        got = lm.rotary_qk(q.cuda(), k.cuda(), p.cuda(), f.cuda(), q_weight=w[0].cuda(),
                           k_weight=w[1].cuda())
        _check_rotary(got, q, k, w, p, f, 1e-6, "half", 1.0)


def test_rotary_far_positions():
    """Angles of positions up to 2^31 - 1, and before the first, keep what
    float32 would lose."""
    from heatvit_amd import lm
    q, k, _, _, f = _rotary_inputs(8, 2, 1, 64, 64, torch.float32, False, 4)
    p = _i32([0, -1, -1000000, 1 << 20, (1 << 24) + 1, 1000000007, (1 << 31) - 1, -(1 << 31)])
    got = lm.rotary_qk(q.cuda(), k.cuda(), p.cuda(), f.cuda())
    _check_rotary(got, q, k, (None, None), p, f, 1e-6, "half", 1.0)


@pytest.mark.parametrize("kind", TYPES)
def test_rotary_values_at_the_edges(kind):
    """Heads of zeros, of the smallest and of the largest numbers, whose
    squares leave float32, beside ordinary ones; a NaN and an infinity in one
    head of a row."""
    from heatvit_amd import lm
    dtype, info = TYPES[kind], torch.finfo(TYPES[kind])
    q, k, w, p, f = _rotary_inputs(8, 2, 1, 64, 32, dtype, True, 11)
    q[1, 0] = 0
    q[2, 0] = info.smallest_normal
    q[3, 1] = info.max / 4
    q[4, 0, ::7] = -info.max / 8
    q[5, 1, 5] = math.nan
    q[6, 0, 40] = math.inf
    for eps in (1e-6, 0.0):
        with np.errstate(all="ignore"):
            got = lm.rotary_qk(q.cuda(), k.cuda(), p.cuda(), f.cuda(), q_weight=w[0].cuda(),
                               k_weight=w[1].cuda(), eps=eps)
            _check_rotary(got, q, k, w, p, f, eps, "half", 1.0)


@pytest.mark.parametrize("kind", TYPES)
def test_rotary_strides_live_rows_and_in_place(kind):
    """Queries, keys and values side by side in the rows of one product,
    odd starts, in place; rows behind the live ones left alone."""
    from heatvit_amd import lm
    q, k, w, p, f = _rotary_inputs(6, 3, 2, 40, 24, TYPES[kind], True, 3)
    buf = torch.full((6, 7 * 40 + 3), 9.0, dtype=q.dtype, device="cuda")
    qv, kv = buf[:, 1:121].view(6, 3, 40), buf[:, 121:201].view(6, 2, 40)
    qv.copy_(q), kv.copy_(k)
    args = dict(q_weight=w[0].cuda(), k_weight=w[1].cuda(), eps=1e-6)
    got = lm.rotary_qk(qv, kv, p.cuda(), f.cuda(), **args)
    _check_rotary(got, q, k, w, p, f, 1e-6, "half", 1.0)
    live = torch.tensor([4], dtype=torch.int32, device="cuda")
    lm.rotary_qk(qv, kv, p.cuda(), f.cuda(), live_rows=live, out=lm.QK(qv, kv), **args)
    assert torch.equal(qv[:4], got.q[:4]) and torch.equal(kv[:4], got.k[:4])
    assert torch.equal(qv[4:].cpu(), q[4:]) and torch.equal(kv[4:].cpu(), k[4:])
    assert (buf[:, 0] == 9).all() and (buf[:, 201:] == 9).all()
    # heads first in memory
    out = lm.QK(*(torch.empty(t.shape[1], 6, 40, dtype=t.dtype, device="cuda").transpose(0, 1)
                  for t in (q, k)))
    lm.rotary_qk(q.cuda(), k.cuda(), p.cuda(), f.cuda(), out=out, **args)
    assert torch.equal(out.q, got.q) and torch.equal(out.k, got.k)
    assert lm.rotary_qk(q[:0].cuda(), k[:0].cuda(), p[:0].cuda(), f.cuda()).q.shape == (0, 3, 40)


# ------------------------------------------------------------------ caches

class Book:
    """A cache on the CPU and on the GPU, with pages in a shuffled order, its
    unused entries out of range and everything not written NaN."""

    def __init__(self, lengths, kv, width, page, dtype, e4m3, seed, spare=2):
        from heatvit_amd import lm
        self.lengths, self.page, self.dtype, self.e4m3 = list(lengths), page, dtype, e4m3
        counts = [-(-max(n, 0) // page) for n in lengths]
        pages = sum(counts) + spare
        order = torch.randperm(pages, generator=_gen(seed)).tolist()
        most = max([1, *counts]) + 1
        self.table = torch.full((len(counts), most), 2 ** 30, dtype=torch.int32)
        self.table[:, 1::2] = -1
        for b, n in enumerate(counts):
            self.table[b, :n] = _i32(order[:n])
            order = order[n:]
        shape = (pages, kv, page, width)
        if e4m3:
            held = [torch.full(shape, 0x7F, dtype=torch.uint8).view(torch.float8_e4m3fn)
                    for _ in range(2)]
            held += [torch.full(shape[:3], 100, dtype=torch.int8) for _ in range(2)]
        else:
            held = [torch.full(shape, math.nan, dtype=dtype) for _ in range(2)]
        self.cache = lm.KvCache(*(t.cuda() for t in held), dtype=dtype)
        self.k, self.v = ([t.view(torch.uint8).numpy(), None] for t in held[:2])
        if e4m3:
            self.k[1], self.v[1] = held[2].numpy(), held[3].numpy()

    def place(self, b, position):
        return int(self.table[b, position // self.page]), position % self.page

    def put(self, b, position, k, v):
        """A row as the cache holds it: [Hk][D] each."""
        page, at = self.place(b, position)
        for held, x in ((self.k, k), (self.v, v)):
            if self.e4m3:
                q, e = ref.in_e4m3(x)
                held[0][page, :, at], held[1][page, :, at] = q.view(np.uint8).reshape(x.shape), e
            else:
                held[0][page, :, at] = x.contiguous().view(torch.uint8).numpy()

    def same(self):
        for held, got, exps in ((self.k, self.cache.k, self.cache.k_exps),
                                (self.v, self.cache.v, self.cache.v_exps)):
            have, want = _bytes(got), held[0]
            if self.e4m3:  # one NaN: 0x7f with either sign
                nan = (want & 0x7F) == 0x7F
                assert np.array_equal((have & 0x7F) == 0x7F, nan)
                have, want = np.where(nan, 0, have), np.where(nan, 0, want)
                assert np.array_equal(exps.cpu().numpy(), held[1])
            assert np.array_equal(have, want)

    def load(self):
        """What `put` wrote, onto the GPU."""
        for held, to, exps in ((self.k, self.cache.k, self.cache.k_exps),
                               (self.v, self.cache.v, self.cache.v_exps)):
            to.view(torch.uint8).copy_(torch.from_numpy(held[0]))
            if self.e4m3:
                exps.copy_(torch.from_numpy(held[1]))

    def rows(self, b):
        """(k, v) of sequence b, 64 bits, [L][Hk][D]."""
        out = []
        for held in (self.k, self.v):
            rows = []
            for j in range(self.lengths[b]):
                page, at = self.place(b, j)
                x = np.ascontiguousarray(held[0][page, :, at])
                if self.e4m3:
                    rows.append(ref.read_back(x, held[1][page, :, at], self.dtype))
                else:
                    rows.append(torch.from_numpy(x).view(self.dtype).double().numpy())
            out.append(np.stack(rows) if rows else
                       np.zeros((0, self.cache.kv_heads, self.cache.width)))
        return out


def _filled(lengths, kv, width, page, dtype, e4m3, seed):
    book = Book(lengths, kv, width, page, dtype, e4m3, seed)
    g = _gen(seed + 1)
    for b, n in enumerate(lengths):
        for j in range(n):
            k, v = (torch.randn(2, kv, width, generator=g) *
                    torch.exp(torch.randn(2, kv, 1, generator=g))).to(dtype)
            book.put(b, j, k, v)
    book.load()
    return book


@pytest.mark.parametrize("e4m3", (False, True))
@pytest.mark.parametrize("kind", HALVES)
def test_write_sizes(kind, e4m3):
    """New rows of ragged sequences, among them none and all of their keys;
    nothing else changes."""
    from heatvit_amd import lm
    for new, lengths, kv, width, page in (
            ([1], [1], 1, 16, 16), ([1, 1, 1], [5, 16, 17], 2, 64, 16), ([0, 3, 0, 7], [4, 3, 0, 40], 3, 48, 32),
            ([20, 1, 33], [20, 65, 64], 2, 128, 64), ([70, 5], [70, 300], 1, 256, 256),
            ([1] * 70, list(range(1, 71)), 1, 32, 16)):
        book = Book(lengths, kv, width, page, TYPES[kind], e4m3, sum(new))
        g = _gen(width)
        rows = sum(new)
        k, v = (torch.randn(2, rows, kv, width, generator=g) *
                torch.exp(2 * torch.randn(2, rows, kv, 1, generator=g))).to(TYPES[kind])
        starts = [0, *np.cumsum(new).tolist()]
        for b, n in enumerate(new):
            for i in range(n):
                book.put(b, lengths[b] - n + i, k[starts[b] + i], v[starts[b] + i])
        one = all(n == 1 for n in new)
        print(f"write {kind} {e4m3} {new} {width}", flush=True)
        for use in ((False, True) if one else (True,)):
            lm.cache_write(book.cache, k.cuda(), v.cuda(), book.table.cuda(), _i32(lengths).cuda(),
                           starts=_i32(starts).cuda() if use else None)
            book.same()


def test_write_many_sequences():
    """More sequences than are looked through at a time, empty ones among
    them, and rows before the first and behind the last."""
    from heatvit_amd import lm
    new = [(7 * b) % 4 for b in range(700)]
    lengths = [n + b % 5 for b, n in enumerate(new)]
    book = Book(lengths, 1, 16, 16, torch.bfloat16, False, 9)
    starts = (3 + np.cumsum([0, *new])).tolist()
    rows = starts[-1] + 5
    k, v = torch.randn(2, rows, 1, 16, generator=_gen(2)).to(torch.bfloat16)
    for b, n in enumerate(new):
        for i in range(n):
            book.put(b, lengths[b] - n + i, k[starts[b] + i], v[starts[b] + i])
    lm.cache_write(book.cache, k.cuda(), v.cuda(), book.table.cuda(), _i32(lengths).cuda(),
                   starts=_i32(starts).cuda())
    book.same()


def test_write_places_that_are_none():
    """Rows before a sequence's first key, past its table and in pages that the
    cache does not have are not written."""
    from heatvit_amd import lm
    book = Book([40, 2, 20], 2, 16, 16, torch.float16, True, 1)
    k, v = torch.randn(2, 9, 2, 16, generator=_gen(5)).half()
    starts, lengths = [0, 3, 7, 9], [40, 2, 20]
    table = book.table.clone()
    table[0, 2] = book.cache.pages            # keys 32 .. of the first sequence
    for i in (2, 3):                          # four rows, two keys: the first two have no place
        book.put(1, i - 2, k[3 + i], v[3 + i])
    for i in (0, 1):
        book.put(2, 18 + i, k[7 + i], v[7 + i])
    args = book.cache, k.cuda(), v.cuda(), table.cuda()
    lm.cache_write(*args, _i32(lengths).cuda(), starts=_i32(starts).cuda())
    book.same()
    room = table.shape[1] * 16
    for lengths in ([-5, 0, -2 ** 31], [2 ** 31 - 1, room + 4, room + 2]):
        lm.cache_write(*args, _i32(lengths).cuda(), starts=_i32(starts).cuda())
        book.same()


@pytest.mark.parametrize("kind", HALVES)
def test_write_values_at_the_edges(kind):
    """Heads of zeros, tiny and largest values, block borders, infinities and
    NaN; what is read back of finite heads is finite."""
    from heatvit_amd import lm
    dtype, info = TYPES[kind], torch.finfo(TYPES[kind])
    k = torch.zeros(8, 2, 32)
    k[1] = info.smallest_normal
    k[2, 0] = info.max
    k[2, 1, ::3] = -info.max
    k[3, :, 0], k[3, :, 1] = 448.0, 449.0
    k[4] = torch.linspace(-448, 448, 32)
    k[5, 0, 3] = math.inf
    k[6, 1, 4] = math.nan
    k[7] = torch.randn(2, 32, generator=_gen(1))
    k = k.to(dtype)
    book = Book([8], 2, 32, 16, dtype, True, 0)
    for i in range(8):
        book.put(0, i, k[i], -k[i])
    lm.cache_write(book.cache, k.cuda(), -k.cuda(), book.table.cuda(), _i32([8]).cuda(),
                   starts=_i32([0, 8]).cuda())
    book.same()
    back = book.rows(0)[0]
    assert np.isfinite(back[[0, 1, 2, 3, 4, 7]]).all()
    assert np.isnan(back[5, 0, 3]) and np.isnan(back[6, 1, 4])


def test_write_strided_rows():
    from heatvit_amd import lm
    book = Book([3, 2], 2, 40, 16, torch.bfloat16, False, 3)
    buf = torch.randn(5, 5 * 40 + 1, generator=_gen(8)).to(torch.bfloat16)
    k, v = buf[:, 1:81].view(5, 2, 40), buf[:, 121:201].view(5, 2, 40)
    for i in range(5):
        b, j = (0, i) if i < 3 else (1, i - 3)
        book.put(b, j, k[i], v[i])
    dev = buf.cuda()
    table = torch.zeros(2, 9, dtype=torch.int32, device="cuda")[:, :book.table.shape[1]]
    table.copy_(book.table)
    lm.cache_write(book.cache, dev[:, 1:81].view(5, 2, 40), dev[:, 121:201].view(5, 2, 40), table,
                   _i32([3, 2]).cuda(), starts=_i32([0, 3, 5]).cuda())
    book.same()


# ------------------------------------------------------------------ attention

def _packed(new, heads, kv, width, dtype, seed, keys=None):
    g = _gen(seed)
    rows, k_rows = sum(new), sum(new if keys is None else keys)
    q = (torch.randn(rows, heads, width, generator=g) * 1.5).to(dtype)
    k = torch.randn(k_rows, kv, width, generator=g).to(dtype)
    v = (torch.randn(k_rows, kv, width, generator=g) + 0.5).to(dtype)
    return q, k, v


def _starts(new, first=0):
    return [first, *(first + np.cumsum(new)).tolist()]


def _check_attention(got, q, parts, starts, scale, causal, window, dtype, what):
    """parts[b]: (k, v) of sequence b in 64 bits."""
    for b, (k, v) in enumerate(parts):
        at = slice(starts[b], starts[b + 1])
        want = ref.attend(q[at].double().numpy(), k, v, scale, causal, window, dtype)
        ref.check(got.out[at], want[0], want[1], f"{what} sequence {b}")
        if got.lse is not None:
            ref.check(got.lse[at], want[2], want[3], f"{what} lse of sequence {b}")


def _run_attention(new, heads, kv, width, kind, causal, window, seed=0, keys=None, scale=None,
                   lse=True):
    from heatvit_amd import lm
    dtype = TYPES[kind]
    q, k, v = _packed(new, heads, kv, width, dtype, seed, keys)
    starts, ks = _starts(new), _starts(new if keys is None else keys)
    what = f"attention {kind} {new} {keys} {heads}/{kv} x {width} causal {causal} window {window}"
    print(what, flush=True)
    got = lm.attention(q.cuda(), k.cuda(), v.cuda(), _i32(starts).cuda(),
                       k_starts=None if keys is None else _i32(ks).cuda(), causal=causal,
                       window=window, lse=lse, scale=scale)
    parts = [(k[ks[b]:ks[b + 1]].double().numpy(), v[ks[b]:ks[b + 1]].double().numpy())
             for b in range(len(new))]
    _check_attention(got, q, parts, starts, scale or 1 / math.sqrt(width), causal, window, dtype, what)


@pytest.mark.parametrize("width", (8, 16, 40, 64, 72, 96, 128, 136, 192, 256))
@pytest.mark.parametrize("kind", HALVES)
def test_attention_widths(kind, width):
    _run_attention([70, 1, 5], 4, 2, width, kind, True, 0, width)
    _run_attention([33, 2], 3, 1, width, kind, False, 0, width + 1)


@pytest.mark.parametrize("causal", (True, False))
@pytest.mark.parametrize("width", (64, 128, 256))
@pytest.mark.parametrize("kind", HALVES)
def test_attention_lengths(kind, width, causal):
    for new, heads, kv in (([1], 1, 1), ([2, 1, 1], 2, 1), ([31, 32, 33], 2, 2), ([63, 0, 64, 65], 1, 1),
                           ([127, 128, 129], 2, 1), ([0, 255, 0], 1, 1), ([257], 2, 1),
                           ([197, 197], 3, 3), ([300, 1], 8, 1), ([23], 20, 4)):
        _run_attention(new, heads, kv, width, kind, causal, 0, sum(new))


@pytest.mark.parametrize("kind", HALVES)
def test_attention_windows(kind):
    for window in (1, 2, 31, 64, 65, 100, 129, 1000):
        _run_attention([150, 3, 200], 2, 1, 64, kind, True, window, window)
        _run_attention([130], 4, 1, 128, kind, True, window, window)


@pytest.mark.parametrize("kind", HALVES)
def test_attention_other_keys(kind):
    """Keys of their own offsets: more and fewer than rows (whose first rows
    then see nothing), none at all."""
    for causal in (True, False):
        for new, keys in (([5, 40, 3], [70, 8, 0]), ([1, 1], [300, 1]), ([130], [65]), ([4], [1000])):
            _run_attention(new, 4, 2, 64, kind, causal, 0, 5, keys)
    _run_attention([20, 5], 2, 1, 128, kind, True, 7, 5, [200, 3])


def test_attention_many_sequences():
    """More sequences than a workgroup has threads, empty ones among them."""
    _run_attention([(5 * b) % 7 for b in range(1200)], 1, 1, 16, "bf16", True, 0)
    _run_attention([1] * 600, 4, 2, 64, "f16", True, 0)


@pytest.mark.parametrize("kind", HALVES)
def test_attention_scores(kind):
    """Flat scores, one key far above the others, scores far below zero, and a
    largest score that rises from tile to tile."""
    from heatvit_amd import lm
    dtype = TYPES[kind]
    for form in ("flat", "peak", "low", "rising", "falling"):
        q, k, v = _packed([300], 2, 1, 64, dtype, 7)
        ramp = torch.arange(300) / 300
        if form == "flat":
            k[:] = 0
        elif form == "peak":
            k[123] = 30 * torch.sign(q[200, 0].float()).to(dtype)
        elif form == "low":
            q[..., 0], k[..., 0] = 60, -60
        else:
            q[..., 0] = 40
            k[..., 0] = (40 * (ramp if form == "rising" else 1 - ramp))[:, None].to(dtype)
        got = lm.attention(q.cuda(), k.cuda(), v.cuda(), _i32([0, 300]).cuda(), lse=True)
        _check_attention(got, q, [(k.double().numpy(), v.double().numpy())], [0, 300], 0.125, True, 0,
                         dtype, f"{kind} {form}")


@pytest.mark.parametrize("rows", (1, 40))
@pytest.mark.parametrize("below", (20, 24, 26, 28))
@pytest.mark.parametrize("kind", HALVES)
def test_attention_many_small_terms_beside_a_large_one(kind, below, rows, monkeypatch):
    """One key far above 1000 others, whose values alone count as its own is
    zero.  (A term 2^-below of the largest is rounded relative to itself or, in
    float16, by half of its smallest step at most, which is 2^-25 where the
    largest term is 2^7 or more: 2^-32 of that.  The results are normal numbers.)"""
    from heatvit_amd import lm
    monkeypatch.setitem(ref.TINY, torch.float16, 2.0 ** -32)
    dtype, width, keys, g = TYPES[kind], 64, 1001, _gen(3)
    # (whole: a share without the large key would have a reference of its own)
    assert lm_attention_kernels.kernel_of(rows, 1, 1, 1, width, keys) == ("few" if rows == 1 else "tiles")
    for at in (0, 500, 1000):
        q, k = torch.ones(rows, 1, width, dtype=dtype), torch.zeros(keys, 1, width)
        k[:, 0, :4] = torch.randn(keys, 4, generator=g) / 16
        k[at] = below * math.log(2) / 8
        v = 100 * (1 + torch.rand(keys, 1, width, generator=g))
        v[at] = 0
        k, v = k.to(dtype), v.to(dtype)
        got = lm.attention(q.cuda(), k.cuda(), v.cuda(), _i32([0, rows]).cuda(),
                           k_starts=_i32([0, keys]).cuda(), causal=False, lse=True)
        assert (got.out[..., 0] >= 2.0 ** -14).all()
        _check_attention(got, q, [(k.double().numpy(), v.double().numpy())], [0, rows], 0.125, False, 0,
                         dtype, f"{kind} 2^-{below} at {at}")


@pytest.mark.parametrize("width", (64, 128))
@pytest.mark.parametrize("kind", HALVES)
def test_attention_leaves_out_what_is_not_seen(kind, width):
    """NaN and infinities in keys and values of rows behind, of other
    sequences and before the window change no bit of a row; a row that
    sees one is NaN where the formula is."""
    from heatvit_amd import lm
    dtype = TYPES[kind]
    new, heads, kv = [90, 150, 40], 4, 2
    starts = _starts(new, 3)
    q, k, v = _packed([starts[-1] + 6], heads, kv, width, dtype, 21)
    dev = [t.cuda() for t in (q, k, v)]
    s = _i32(starts).cuda()
    for window in (0, 20):
        clean = lm.attention(*dev, s, window=window, lse=True)
        for at, value in ((2, math.nan), (starts[3], math.inf), (starts[1] + 70, math.nan),
                          (starts[1] + 100, math.inf), (starts[2] + 39, -math.inf)):
            for which in (1, 2):
                x = [t.clone() for t in dev]
                x[which][at] = value
                got = lm.attention(*x, s, window=window, lse=True)
                touched = torch.zeros(len(q), dtype=torch.bool)
                b = next((b for b in range(3) if starts[b] <= at < starts[b + 1]), None)
                if b is not None:
                    touched[at:starts[b + 1] if not window else min(at + window, starts[b + 1])] = True
                live = torch.zeros_like(touched)
                live[starts[0]:starts[3]] = True
                same = (live & ~touched).cuda()
                assert torch.equal(got.out[same], clean.out[same]), (at, which)
                assert torch.equal(got.lse[same], clean.lse[same]), (at, which)
                if b is not None and value != value:
                    assert got.out[(live & touched).cuda()].isnan().any(-1).all()


def test_attention_rows_outside_and_bad_offsets():
    """Rows outside all sequences, and every row where the offsets run
    backwards or leave the tensors, are left as they were."""
    from heatvit_amd import lm
    q, k, v = (t.cuda() for t in _packed([40], 2, 1, 64, torch.bfloat16, 2))
    for starts in ([5, 12, 12, 30], [0], [7, 7], [30, 20, 10], [-5, 8], [35, 60], [-2 ** 31, -1]):
        out = lm.Attended(torch.full_like(q, 7.0), torch.full((40, 2), 7.0, device="cuda"))
        lm.attention(q, k, v, _i32(starts).cuda(), lse=True, out=out)
        covered = torch.zeros(40, dtype=torch.bool)
        for a, b in zip(starts, starts[1:]):
            covered[max(a, 0):max(min(b, 40), 0)] = True
        assert (out.out[~covered] == 7).all() and (out.lse[~covered] == 7).all()
        assert out.out[covered.cuda()].isfinite().all()
        assert not covered.any() or (out.out[covered.cuda()] != 7).any()
    assert lm.attention(q[:0], k[:0], v[:0], _i32([0, 0]).cuda()).out.shape == (0, 2, 64)


@pytest.mark.parametrize("kind", HALVES)
def test_attention_strides(kind):
    """Queries, keys and values side by side in one product's rows, heads first
    in memory, an output with a gap."""
    from heatvit_amd import lm
    dtype = TYPES[kind]
    new, heads, kv, width = [60, 9], 4, 2, 64
    q, k, v = _packed(new, heads, kv, width, dtype, 4)
    s = _i32(_starts(new)).cuda()
    want = lm.attention(q.cuda(), k.cuda(), v.cuda(), s, lse=True)
    rows = torch.cat([t.flatten(1) for t in (q, k, v)], 1).cuda()
    qs, ks, vs = (rows[:, a:b].unflatten(1, (-1, width)) for a, b in ((0, 256), (256, 384), (384, 512)))
    buf = torch.full((69, 4, 72), 5.0, dtype=dtype, device="cuda")
    got = lm.attention(qs, ks, vs, s, lse=True,
                       out=lm.Attended(buf[..., :64], torch.empty(69, 4, device="cuda")))
    assert torch.equal(got.out, want.out) and torch.equal(got.lse, want.lse)
    assert (buf[..., 64:] == 5).all()
    got = lm.attention(*(t.cuda().transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)), s)
    assert torch.equal(got.out, want.out)


# ------------------------------------------------------------------ paged_attention

def _run_paged(new, lengths, heads, kv, width, page, kind, e4m3, window=0, causal=True, seed=0,
               starts=True, lse=True):
    from heatvit_amd import lm
    dtype = TYPES[kind]
    book = _filled(lengths, kv, width, page, dtype, e4m3, seed)
    q = (torch.randn(sum(new), heads, width, generator=_gen(seed)) * 1.5).to(dtype)
    what = f"paged {kind} {e4m3} {new} over {lengths} {heads}/{kv} x {width} page {page} " \
           f"window {window} causal {causal}"
    print(what, flush=True)
    at = _starts(new)
    got = lm.paged_attention(q.cuda(), book.cache, book.table.cuda(), _i32(lengths).cuda(),
                             starts=_i32(at).cuda() if starts else None, causal=causal,
                             window=window, lse=lse)
    _check_attention(got, q, [book.rows(b) for b in range(len(new))], at, 1 / math.sqrt(width), causal,
                     window, dtype, what)


@pytest.mark.parametrize("e4m3", (False, True))
@pytest.mark.parametrize("kind", HALVES)
def test_paged_single_rows(kind, e4m3):
    for lengths, heads, kv, width, page in (
            ([1], 1, 1, 16, 16), ([2, 0, 15, 16, 17], 4, 1, 64, 16), ([63, 64, 65, 300], 8, 2, 128, 64),
            ([257, 700], 20, 4, 128, 32), ([33, 90], 3, 3, 80, 16), ([129, 5], 16, 1, 256, 128),
            ([1500], 40, 2, 48, 256), ([31, 32, 33], 6, 6, 192, 16)):
        _run_paged([1] * len(lengths), lengths, heads, kv, width, page, kind, e4m3, starts=False)


@pytest.mark.parametrize("e4m3", (False, True))
@pytest.mark.parametrize("kind", HALVES)
def test_paged_chunks(kind, e4m3):
    for new, lengths, heads, kv, width, page in (
            ([3, 1, 0, 5], [3, 70, 9, 64], 4, 2, 64, 16), ([40, 7], [200, 7], 8, 2, 128, 64),
            ([130], [131], 2, 1, 128, 32), ([9, 20], [4, 300], 4, 4, 96, 16), ([65, 1], [500, 90], 3, 1, 256, 64),
            ([300], [900], 2, 2, 64, 128)):
        _run_paged(new, lengths, heads, kv, width, page, kind, e4m3, seed=1)
    _run_paged([30, 4], [100, 90], 4, 2, 64, 16, kind, e4m3, window=17)
    _run_paged([1, 1], [500, 60], 4, 2, 128, 16, kind, e4m3, window=50)
    _run_paged([30, 4], [100, 90], 4, 2, 64, 16, kind, e4m3, causal=False)


@pytest.mark.parametrize("kind", HALVES)
def test_paged_long_axes(kind):
    """Few rows over long axes, whose parts are joined, beside short ones."""
    _run_paged([1], [5000], 4, 1, 64, 64, kind, False, starts=False)
    _run_paged([1, 1, 1], [3000, 1, 700], 2, 2, 32, 16, kind, True, starts=False)
    _run_paged([6, 2], [4000, 300], 4, 2, 64, 64, kind, False, seed=3)
    _run_paged([1, 1], [4000, 0], 2, 1, 64, 32, kind, False, window=1500, seed=4)


@pytest.mark.parametrize("e4m3", (False, True))
def test_paged_bad_pages(e4m3):
    """A page outside the cache among those a sequence reads, or keys past its
    table, make its rows NaN; the other sequences are as without."""
    from heatvit_amd import lm
    book = _filled([100, 50, 70], 2, 64, 16, torch.bfloat16, e4m3, 6)
    for new in ([1, 1, 1], [5, 3, 40]):
        q = torch.randn(sum(new), 4, 64, generator=_gen(1)).to(torch.bfloat16).cuda()
        at = _starts(new)
        s = _i32(at).cuda()
        lengths = _i32(book.lengths).cuda()
        clean = lm.paged_attention(q, book.cache, book.table.cuda(), lengths, starts=s, lse=True)
        assert clean.out.isfinite().all() and clean.lse.isfinite().all()
        for page in (-1, book.cache.pages, 2 ** 31 - 1, -2 ** 31):
            table = book.table.clone()
            table[1, 2] = page
            got = lm.paged_attention(q, book.cache, table.cuda(), lengths, starts=s, lse=True)
            for b in (0, 2):
                assert torch.equal(got.out[at[b]:at[b + 1]], clean.out[at[b]:at[b + 1]])
                assert torch.equal(got.lse[at[b]:at[b + 1]], clean.lse[at[b]:at[b + 1]])
            assert got.out[at[1]:at[2]].isnan().all() and got.lse[at[1]:at[2]].isnan().all()
        room = book.table.shape[1] * 16
        for length in (room + 1, 2 ** 31 - 1):
            got = lm.paged_attention(q, book.cache, book.table.cuda(), _i32([100, length, 70]).cuda(),
                                     starts=s, lse=True)
            assert got.out[at[1]:at[2]].isnan().all() and got.lse[at[1]:at[2]].isnan().all()
            assert torch.equal(got.out[at[2]:], clean.out[at[2]:])
        got = lm.paged_attention(q, book.cache, book.table.cuda(), _i32([100, -7, 70]).cuda(), starts=s,
                                 lse=True)
        assert (got.out[at[1]:at[2]] == 0).all() and (got.lse[at[1]:at[2]] == -math.inf).all()


@pytest.mark.parametrize("e4m3", (False, True))
@pytest.mark.parametrize("page", (16, 32, 64))
def test_paged_pages_before_a_window(page, e4m3):
    """Pages that lie before what any row sees may be gone: the same bits. The
    first page that a row does see may not."""
    from heatvit_amd import lm
    for new, lengths, width, window, kernel in (
            ([1], [1000], 64, 80, "few"), ([1, 1], [1000, 333], 128, 17, "few"),
            ([1, 1], [2500, 71], 64, 1500, "few in shares"), ([6], [2613], 128, 2200, "few in shares"),
            ([70, 40], [301, 290], 64, 101, "tiles"), ([33], [455], 256, 60, "tiles"),
            ([70], [2601], 64, 933, "tiles in shares"), ([40, 60], [2601, 2222], 128, 700, "tiles in shares")):
        book = _filled(lengths, 2, width, page, torch.bfloat16, e4m3, 5)
        assert lm_attention_kernels.kernel_of(sum(new), len(new), 4, 2, width,
                                              book.table.shape[1] * page) == kernel
        print(f"pages of {page} before a window: {new} of {lengths}, {width}, {window}", flush=True)
        q = torch.randn(sum(new), 4, width, generator=_gen(1)).to(torch.bfloat16).cuda()
        args = dict(starts=_i32(_starts(new)).cuda(), window=window, lse=True)
        n = _i32(lengths).cuda()
        clean = lm.paged_attention(q, book.cache, book.table.cuda(), n, **args)
        assert clean.out.isfinite().all() and clean.lse.isfinite().all()
        table = book.table.clone()
        first = [max(length - rows + 1 - window, 0) // page for length, rows in zip(lengths, new)]
        for b, count in enumerate(first):
            table[b, :count] = _i32([(-1, 2 ** 30, -2 ** 31)[i % 3] for i in range(count)])
        got = lm.paged_attention(q, book.cache, table.cuda(), n, **args)
        assert torch.equal(got.out, clean.out) and torch.equal(got.lse, clean.lse)
        table[0, first[0]] = -1
        got = lm.paged_attention(q, book.cache, table.cuda(), n, **args)
        assert got.out[0].isnan().all() and got.lse[0].isnan().all()


def test_paged_smallest_exponent():
    """Heads of the smallest exponent, as zeros have, beside ordinary ones."""
    from heatvit_amd import lm
    book = Book([40], 1, 64, 16, torch.bfloat16, True, 0)
    g = _gen(3)
    for j in range(40):
        k, v = torch.randn(2, 1, 64, generator=g).to(torch.bfloat16)
        if j % 3 == 0:
            k, v = k * 0, v * 0
        if j % 3 == 1:
            k, v = k * 2.0 ** -125, v * 2.0 ** -125
        book.put(0, j, k, v)
    book.load()
    q = torch.randn(1, 4, 64, generator=g).to(torch.bfloat16)
    got = lm.paged_attention(q.cuda(), book.cache, book.table.cuda(), _i32([40]).cuda(), lse=True)
    _check_attention(got, q, [book.rows(0)], [0, 1], 0.125, True, 0, torch.bfloat16, "exponents")


@pytest.mark.parametrize("kind", HALVES)
@pytest.mark.parametrize("new", ([1, 1], [70, 3]))
def test_paged_exponent_that_is_none(kind, new):
    """An exponent of -128 is NaN for the rows that see it, zeros among its
    elements too, and leaves no trace in the others."""
    from heatvit_amd import lm
    book = _filled([200, 90], 2, 64, 16, TYPES[kind], True, 4)
    q = torch.randn(sum(new), 4, 64, generator=_gen(1)).to(TYPES[kind]).cuda()
    args = book.table.cuda(), _i32([200, 90]).cuda()
    starts = _i32(_starts(new)).cuda()
    clean = lm.paged_attention(q, book.cache, *args, starts=starts, lse=True)
    at = 199 - new[0] // 2
    page, i = book.place(0, at)
    sees = (torch.arange(sum(new)) + 200 - new[0] >= at) & (torch.arange(sum(new)) < new[0])
    assert sees.any() and not sees.all()
    for values, exps in ((book.cache.k, book.cache.k_exps), (book.cache.v, book.cache.v_exps)):
        old = values[page, 1, i].clone(), exps[page, 1, i].clone()
        values.view(torch.uint8)[page, 1, i, ::2] = 0
        exps[page, 1, i] = -128
        got = lm.paged_attention(q, book.cache, *args, starts=starts, lse=True)
        values[page, 1, i], exps[page, 1, i] = old
        assert torch.equal(got.out[:, :2], clean.out[:, :2])  # of the other head of keys
        assert torch.equal(got.out[~sees], clean.out[~sees]) and torch.equal(got.lse[~sees], clean.lse[~sees])
        assert got.out[sees][:, 2:].isnan().all()


@pytest.mark.parametrize("e4m3", (False, True))
def test_paged_far_pages(e4m3):
    """Pages whose elements lie past 2^32, written and read."""
    from heatvit_amd import lm
    pages, kv, width, page = (1 << 31) // (2 * 128 * 64) * 5, 2, 128, 64
    shape = (pages, kv, page, width)
    held = torch.float8_e4m3fn if e4m3 else torch.bfloat16
    t = [torch.empty(shape, dtype=held, device="cuda") for _ in range(2)]
    if e4m3:
        t += [torch.empty(shape[:3], dtype=torch.int8, device="cuda") for _ in range(2)]
    assert t[0].numel() > 1 << 32
    far = lm.KvCache(*t, dtype=torch.bfloat16)
    near = lm.KvCache.empty(4, kv, width, page=page, e4m3=e4m3)
    k, v = torch.randn(2, 150, kv, width, generator=_gen(1)).to(torch.bfloat16).cuda()
    q = torch.randn(3, 4, width, generator=_gen(2)).to(torch.bfloat16).cuda()
    s, n = _i32([0, 150]).cuda(), _i32([150]).cuda()
    got = []
    for cache, table in ((far, [pages - 1, 0, pages - 7]), (near, [2, 0, 3])):
        table = _i32([table]).cuda()
        lm.cache_write(cache, k, v, table, n, starts=s)
        got.append(lm.paged_attention(q, cache, table, n, starts=_i32([0, 3]).cuda(), lse=True))
        got.append(lm.paged_attention(q[:1], cache, table, n, lse=True))
    for a, b in ((got[0], got[2]), (got[1], got[3])):
        assert a.out.isfinite().all()
        assert torch.equal(a.out, b.out) and torch.equal(a.lse, b.lse)


# ------------------------------------------------------------------ shares of the work

def _room(lengths, page):
    return (max(-(-n // page) for n in lengths) + 1) * page


@pytest.mark.parametrize("e4m3", (False, True))
@pytest.mark.parametrize("kind", HALVES)
def test_paged_tiles_in_shares(kind, e4m3):
    """Tiles whose keys are cut into shares: one sequence, a few of very
    different lengths (none and one key among them), windows, wide heads."""
    for new, lengths, heads, kv, width, page, window, causal in (
            ([40], [3000], 4, 1, 64, 64, 0, True), ([130, 20, 1, 0], [2500, 20, 1, 900], 4, 2, 128, 16, 0, True),
            ([64], [2600], 2, 2, 96, 128, 0, False), ([150], [2500], 3, 1, 64, 16, 700, True),
            ([33], [2200], 4, 4, 256, 64, 0, True), ([60, 60], [1900, 2100], 2, 1, 32, 32, 0, True)):
        assert lm_attention_kernels.kernel_of(sum(new), len(new), heads, kv, width,
                                              _room(lengths, page)) == "tiles in shares"
        _run_paged(new, lengths, heads, kv, width, page, kind, e4m3, window, causal, seed=8)


@pytest.mark.parametrize("kind", HALVES)
def test_paged_few_rows_in_shares(kind):
    """Few rows in shares beyond a workgroup's threads of sequences, in groups
    that take two tiles, and whole where sequences are many."""
    lengths = [(37 * b) % 50 for b in range(300)]
    lengths[7], lengths[290] = 2300, 2100
    for lengths, heads, kv, want in ((lengths, 2, 2, "few in shares"), ([900, 30, 2200], 16, 1, "few in shares"),
                                     ([1 + b % 40 for b in range(1200)], 4, 4, "few"),
                                     ([2500, 2], 12, 1, "few in shares")):
        assert lm_attention_kernels.kernel_of(len(lengths), len(lengths), heads, kv, 64,
                                              _room(lengths, 16)) == want
        _run_paged([1] * len(lengths), lengths, heads, kv, 64, 16, kind, False, starts=False, seed=2)


@pytest.mark.parametrize("causal", (True, False))
def test_attention_in_runs(causal):
    """More tiles than the card takes at once, of short sequences (empty ones
    among them) and heads that are no multiple of eight."""
    for new, kv, kind in (([0, 400, 1] * 100, 3, "f16"), ([140 + 3 * (b % 40) for b in range(300)], 2, "bf16")):
        assert lm_attention_kernels.kernel_of(sum(new), len(new), kv, kv, 64, sum(new)) == "tiles"
        assert lm_attention_kernels.library().attention_run(sum(new), len(new), kv, kv, 64, 0) == 2 * kv
        _run_attention(new, kv, kv, 64, kind, causal, 0, 3)


def test_attention_tiles_in_shares():
    """Packed keys of their own, cut into shares."""
    assert lm_attention_kernels.kernel_of(180, 2, 4, 2, 64, 3300) == "tiles in shares"
    _run_attention([100, 80], 4, 2, 64, "bf16", True, 0, 5, [2500, 800])
    _run_attention([100, 80], 4, 2, 128, "f16", False, 0, 5, [2500, 800])
    assert lm_attention_kernels.kernel_of(6, 2, 4, 2, 64, 3300) == "few in shares"
    _run_attention([4, 2], 4, 2, 64, "f16", True, 0, 5, [2500, 800])


@pytest.mark.parametrize("new, lengths", (([1, 1], [300, 2500]), ([3, 2], [2300, 40]), ([90, 45], [700, 2500])))
def test_what_is_said_of_the_longest_sequence(new, lengths):
    """Any number of keys said of the longest sequence gives the result, over a
    cache with a wide table and over packed keys, whole and in shares."""
    from heatvit_amd import lm
    book = _filled(lengths, 2, 64, 64, torch.bfloat16, False, 3)
    q = torch.randn(sum(new), 4, 64, generator=_gen(1)).to(torch.bfloat16)
    at, scale = _starts(new), 0.125
    rows = [book.rows(b) for b in range(2)]
    k, v = (torch.from_numpy(np.concatenate([r[i] for r in rows])).to(torch.bfloat16) for i in range(2))
    table = torch.full((2, 2048), -1, dtype=torch.int32)
    table[:, :book.table.shape[1]] = book.table
    kernels = set()
    for said in (None, 0, 1, max(lengths), 2 ** 31 - 1):
        kernels.add(lm_attention_kernels.kernel_of(sum(new), 2, 4, 2, 64, said or 131072))
        args = dict(most_keys=said, lse=True)
        for got in (lm.paged_attention(q.cuda(), book.cache, table.cuda(), _i32(lengths).cuda(),
                                       starts=_i32(at).cuda(), **args),
                    lm.attention(q.cuda(), k.cuda(), v.cuda(), _i32(at).cuda(),
                                 k_starts=_i32(_starts(lengths)).cuda(), **args)):
            _check_attention(got, q, rows, at, scale, True, 0, torch.bfloat16, f"{new} said {said}")
    assert len(kernels) == 2


@pytest.mark.parametrize("new", ([2, 1], [90, 45]))
def test_shares_leave_out_what_is_not_seen(new):
    """NaN and infinities that a row does not see leave no trace where the keys
    are cut into shares, and a bad page makes its own sequence NaN alone."""
    from heatvit_amd import lm
    lengths, kv = [2500, 800], 2
    book = _filled(lengths, kv, 64, 64, torch.bfloat16, False, 3)
    q = torch.randn(sum(new), 4, 64, generator=_gen(1)).to(torch.bfloat16).cuda()
    assert lm_attention_kernels.kernel_of(sum(new), 2, 4, kv, 64, _room(lengths, 64)).endswith("shares")
    at = _starts(new)
    s, n, table = _i32(at).cuda(), _i32(lengths).cuda(), book.table.cuda()
    for window in (0, 400):
        clean = lm.paged_attention(q, book.cache, table, n, starts=s, window=window, lse=True)
        for position, value in ((2499, math.nan), (2499, math.inf), (50, math.nan), (50, math.inf)):
            for t in (book.cache.k, book.cache.v):
                page, i = book.place(0, position)
                old = t[page, :, i].clone()
                t[page, :, i] = value
                got = lm.paged_attention(q, book.cache, table, n, starts=s, window=window, lse=True)
                t[page, :, i] = old
                rows = torch.arange(sum(new))
                row_at = 2500 - new[0] + rows  # places of the first sequence's rows
                sees = (rows < new[0]) & (position <= row_at) & \
                    ((position > row_at - window) if window else True)
                same = (~sees).cuda()
                assert torch.equal(got.out[same], clean.out[same]), (window, position, value)
                assert torch.equal(got.lse[same], clean.lse[same]), (window, position, value)
                if value != value and sees.any():
                    assert got.out[sees.cuda()].isnan().any(-1).all()
    bad = table.clone()
    bad[0, 20] = book.cache.pages
    clean = lm.paged_attention(q, book.cache, table, n, starts=s, lse=True)
    got = lm.paged_attention(q, book.cache, bad, n, starts=s, lse=True)
    assert got.out[:at[1]].isnan().all() and got.lse[:at[1]].isnan().all()
    assert torch.equal(got.out[at[1]:], clean.out[at[1]:])


@pytest.mark.parametrize("value", (math.nan, math.inf))
@pytest.mark.parametrize("rows, keys, heads, kv, width", ((4096, 4096, 8, 8, 128), (64, 2500, 4, 2, 64),
                                                          (2048, 2048, 4, 4, 64), (700, 3100, 2, 2, 256)))
def test_one_packed_sequence_in_shares_with_a_bad_value(rows, keys, heads, kv, width, value):
    """One element of one value that is no number, where shares of one packed
    sequence hold parts of several tiles: every other element of every row has
    the clean call's bits."""
    from heatvit_amd import lm
    assert lm_attention_kernels.kernel_of(rows, 1, heads, kv, width, keys) == "tiles in shares"
    q, k, v = (t.cuda() for t in _packed([rows], heads, kv, width, torch.bfloat16, 6, [keys]))
    args = dict(k_starts=_i32([0, keys]).cuda(), lse=True)
    starts = _i32([0, rows]).cuda()
    clean = lm.attention(q, k, v, starts, **args)
    row_at = keys - rows + torch.arange(rows, device="cuda")
    for position in (keys - 1, keys - 70, keys - rows // 2, 3):
        x = v.clone()
        x[position, 0, 5] = value
        got = lm.attention(q, k, x, starts, **args)
        touched = torch.zeros(rows, heads, width, dtype=torch.bool, device="cuda")
        touched[row_at >= position, :heads // kv, 5] = True
        assert torch.equal(got.out[~touched], clean.out[~touched]), position
        assert not got.out[touched].isfinite().any(), position
        assert torch.equal(got.lse, clean.lse), position


def test_attention_bad_offsets_in_shares():
    """Offsets that run backwards or leave the tensors where the work is cut
    into shares: nothing outside the rows is written, and the call ends."""
    from heatvit_amd import lm
    q, k, v = (t.cuda() for t in _packed([300], 2, 1, 64, torch.bfloat16, 2, [3000]))
    assert lm_attention_kernels.kernel_of(300, 5, 2, 1, 64, 3000) == "tiles in shares"
    for starts, ks in (([0, 300, 0, 300, 0, 300], [0, 3000, 0, 3000, 0, 3000]),
                       ([2 ** 31 - 1, -2 ** 31, 7, 7, 300, 2 ** 31 - 1], [-5, 9, 4000, 0, 3, 2 ** 31 - 1])):
        out = lm.Attended(torch.full_like(q, 7.0), torch.full((300, 2), 7.0, device="cuda"))
        lm.attention(q, k, v, _i32(starts).cuda(), k_starts=_i32(ks).cuda(), lse=True, out=out)
        torch.cuda.synchronize()
        assert out.out.isfinite().all()


@pytest.mark.parametrize("last", (1, 8128))
def test_attention_overlapping_sequences_in_shares(last):
    """Offsets that run back and forth, of sequences whose cost leaves 32 bits:
    nothing outside their rows is written, and the call ends."""
    from heatvit_amd import lm
    book = _filled([64], 1, 16, 4096, torch.bfloat16, False, 1)
    batch, rows = 2049, 256
    lengths = [2 ** 20] * (batch - 1) + [last]
    assert lm_attention_kernels.kernel_of(300, batch, 1, 1, 16, 2 ** 20) == "few in shares"
    q = torch.randn(300, 1, 16, generator=_gen(2)).to(torch.bfloat16).cuda()
    out = lm.Attended(torch.full_like(q, 7.0), torch.full((300, 1), 7.0, device="cuda"))
    lm.paged_attention(q, book.cache, torch.zeros(batch, 256, dtype=torch.int32, device="cuda"),
                       _i32(lengths).cuda(), starts=_i32([0, rows] * (batch // 2 + 1)).cuda(),
                       causal=False, lse=True, out=out)
    torch.cuda.synchronize()
    assert (out.out[rows:] == 7).all() and (out.lse[rows:] == 7).all()


# ------------------------------------------------------------------ streams, graphs, workspaces

def test_streams_graphs_and_workspaces():
    """A captured step of all four, replayed beside eager calls on other
    inputs; a side stream; a workspace too small refused."""
    from heatvit_amd import _lib, lm
    heads, kv, width = 8, 2, 128
    book = Book([900, 40, 300], kv, width, 64, torch.bfloat16, True, 2)
    lengths = _i32(book.lengths).cuda()
    table = book.table.cuda()
    g = _gen(4)
    old = [torch.randn(1240, kv, width, generator=g).to(torch.bfloat16).cuda() for _ in range(2)]
    lm.cache_write(book.cache, *old, table, lengths, starts=_i32([0, 900, 940, 1240]).cuda())
    q = torch.randn(3, heads, width, generator=g).to(torch.bfloat16).cuda()
    k, v = (torch.randn(3, kv, width, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    positions = lengths - 1
    freqs = lm.rotary_frequencies(width).cuda()
    size = _lib.lib().hv_attention_workspace_bytes(3, 3, heads, kv, width)
    ws = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")

    def step(out):
        r = lm.rotary_qk(q, k, positions, freqs, out=out[0])
        lm.cache_write(book.cache, r.k, v, table, lengths)
        lm.paged_attention(r.q, book.cache, table, lengths, lse=True, out=out[1], workspace=ws)

    def buffers():
        return (lm.QK(torch.empty_like(q), torch.empty_like(k)),
                lm.Attended(torch.empty_like(q), torch.empty(3, heads, device="cuda")))

    eager, held = buffers(), buffers()
    step(eager)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(held)
    for i in range(4):
        q.copy_(torch.randn(3, heads, width, generator=g).to(torch.bfloat16))
        k.copy_(torch.randn(3, kv, width, generator=g).to(torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for pair in held for t in pair]
        step(eager)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, [t for pair in eager for t in pair])), i
    with torch.cuda.stream(side):
        other = lm.paged_attention(eager[0].q, book.cache, table, lengths, lse=True)
    side.synchronize()
    assert torch.equal(other.out, eager[1].out) and torch.equal(other.lse, eager[1].lse)
    if size:
        with pytest.raises(ValueError):
            lm.paged_attention(q, book.cache, table, lengths, workspace=ws[:size - 1])


def test_two_calls_at_once():
    """Calls on two streams, each with its own workspace, give what they give
    alone."""
    from heatvit_amd import lm
    books = [_filled([1300, 200], 2, 64, 64, torch.float16, e, 5 + e) for e in (False, True)]
    lengths = _i32([1300, 200]).cuda()
    q = torch.randn(2, 8, 64, generator=_gen(1)).half().cuda()
    tables = [b.table.cuda() for b in books]
    alone = [lm.paged_attention(q, b.cache, t, lengths) for b, t in zip(books, tables)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(lm.paged_attention(q, books[i].cache, tables[i], lengths))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g.out, alone[i].out) for g in got[i])


def test_same_bits_again():
    """The same call gives the same bits."""
    from heatvit_amd import lm
    book = _filled([2500, 30], 2, 128, 64, torch.bfloat16, True, 1)
    q = torch.randn(2, 16, 128, generator=_gen(1)).to(torch.bfloat16).cuda()
    args = q, book.cache, book.table.cuda(), _i32([2500, 30]).cuda()
    first = lm.paged_attention(*args, lse=True)
    for _ in range(3):
        again = lm.paged_attention(*args, lse=True)
        assert torch.equal(first.out, again.out) and torch.equal(first.lse, again.lse)


@pytest.mark.parametrize("new, lengths", (([1, 1], [300, 90]), ([1, 1], [2500, 90]),
                                          ([90, 45], [300, 90]), ([90, 45], [2500, 90])))
def test_attention_in_place(new, lengths):
    """Results over the queries, of few rows and of tiles, whole and in shares."""
    from heatvit_amd import lm
    book = _filled(lengths, 2, 128, 16, torch.bfloat16, False, 1)
    q = torch.randn(sum(new), 6, 128, generator=_gen(1)).to(torch.bfloat16).cuda()
    args = book.cache, book.table.cuda(), _i32(lengths).cuda()
    starts = _i32(_starts(new)).cuda()
    want = lm.paged_attention(q, *args, starts=starts)
    got = lm.paged_attention(q, *args, starts=starts, out=lm.Attended(q, None))
    assert got.out is q and torch.equal(q, want.out)


# ------------------------------------------------------------------ a run of them

@pytest.mark.parametrize("e4m3", (False, True))
def test_layer(e4m3):
    """Norm, product, rotation, cache, attention, product and answer of two
    prompts and three decoding steps: the decoding's rows are those of the
    whole prompt's attention, and the paged attention of a prompt is the packed
    one where the cache holds 16 bits."""
    from heatvit_amd import lm
    from heatvit_amd.device import DeviceF8Weight
    g = _gen(12)
    heads, kv, width, model = 4, 2, 64, 256
    x = torch.randn(80, model, generator=g).to(torch.bfloat16).cuda()
    norm = torch.ones(model, dtype=torch.bfloat16, device="cuda")
    w = DeviceF8Weight(torch.randn(model, (heads + 2 * kv) * width, generator=g) / 16)
    head = DeviceF8Weight(torch.randn(heads * width, 500, generator=g) / 16)
    ones = torch.ones(width, dtype=torch.bfloat16, device="cuda")
    freqs = lm.rotary_frequencies(width).cuda()
    total, steps = [50, 30], 3

    def qkv(rows, positions):
        r = lm.rms_norm_q8(rows, norm)
        y = lm.gemm_f8(r.q, r.exps, w, row_scale=r.scale)
        q, k, v = (y[:, a * width:b * width].unflatten(1, (-1, width))
                   for a, b in ((0, heads), (heads, heads + kv), (heads + kv, heads + 2 * kv)))
        return *lm.rotary_qk(q, k, positions, freqs, q_weight=ones, k_weight=ones), v

    starts = _starts(total)
    positions = torch.cat([torch.arange(n, dtype=torch.int32) for n in total]).cuda()
    q, k, v = qkv(x, positions)
    whole = lm.attention(q, k, v, _i32(starts).cuda(), lse=True)
    parts = [[t[starts[b]:starts[b + 1]].double().cpu().numpy() for t in (k, v)] for b in range(2)]
    _check_attention(whole, q.cpu(), parts, starts, 0.125, True, 0, torch.bfloat16, "whole")

    cache = lm.KvCache.empty(9, kv, width, page=16, e4m3=e4m3)
    table = _i32([[3, 1, 7, 0], [2, 8, 5, 4]]).cuda()
    first = [n - steps for n in total]
    rows = torch.cat([torch.arange(starts[b], starts[b] + first[b]) for b in range(2)]).cuda()
    s, lengths = _i32(_starts(first)).cuda(), _i32(first).cuda()
    qp, kp, vp = (t[rows].contiguous() for t in (q, k, v))
    lm.cache_write(cache, kp, vp, table, lengths, starts=s)
    prompt = lm.paged_attention(qp, cache, table, lengths, starts=s, lse=True)
    book = [[], []]
    for t, i in ((k, 0), (v, 1)):
        for b in range(2):
            y = t[starts[b]:starts[b + 1]].cpu()
            if e4m3:
                qe, e = ref.in_e4m3(y)
                book[i].append(ref.read_back(qe.reshape(y.shape), e, torch.bfloat16))
            else:
                book[i].append(y.double().numpy())
    at = _starts(first)
    for b in range(2):
        n = first[b]
        want = ref.attend(qp[at[b]:at[b + 1]].double().cpu().numpy(), book[0][b][:n], book[1][b][:n],
                          0.125, True, 0, torch.bfloat16)
        ref.check(prompt.out[at[b]:at[b + 1]], want[0], want[1], "prompt")
    for step in range(steps):
        lengths += 1
        row = torch.tensor([starts[b] + first[b] + step for b in range(2)], device="cuda")
        qn, kn, vn = qkv(x[row], lengths - 1)
        assert torch.equal(kn, k[row]) and torch.equal(vn, v[row])
        lm.cache_write(cache, kn, vn, table, lengths)
        got = lm.paged_attention(qn, cache, table, lengths, lse=True)
        for b in range(2):
            n = first[b] + step + 1
            want = ref.attend(qn[b:b + 1].double().cpu().numpy(), book[0][b][:n], book[1][b][:n], 0.125,
                              True, 0, torch.bfloat16)
            ref.check(got.out[b:b + 1], want[0], want[1], f"step {step}")
            ref.check(got.lse[b:b + 1], want[2], want[3], f"step {step}")
        r = lm.rms_norm_q8(got.out.flatten(1), torch.ones(heads * width, dtype=torch.bfloat16,
                                                         device="cuda"))
        answer = lm.log_probs(lm.gemm_f8(r.q, r.exps, head, row_scale=r.scale), top=3)
        assert answer.top_logp.isfinite().all()
