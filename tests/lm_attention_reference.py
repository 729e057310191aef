"""Plain 64-bit forms of the attention operators (numpy, and torch on the CPU
for the types), and the rounding bounds their results are held to.

U32 and HALF are half a step of float32 and of a type, relative to the value;
TINY is half a step of the type's smallest numbers."""

import numpy as np
import torch

from lm_reference import HALF, U32

TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def rotary(x, weight, positions, freqs, eps, layout, scale):
    """(y, bound) of [T][H][D], 64 bits.

    The norm: a head's squares are added at most 16 in a row and 6 times
    across lanes (22 U32, halved by the root), the mean, eps, the root and the
    division at most 2 U32 each, then two products: 21 U32 relative.  The
    angle's rest of a turn is rounded to float32 (pi U32 at most), its cosine
    and sine are good to 4 U32, the factor rounds once more: 9 U32.  Two
    products and a sum: 3 U32.  The angle in 64 bits is off by 3 * 2^-54 of its
    turns."""
    xd = x.double().numpy()
    rel = 0.0
    if weight is not None:
        xd = xd / np.sqrt(np.square(xd).mean(-1, keepdims=True) + eps) * weight.double().numpy()
        rel = 21 * U32
    n = 2 * len(freqs)
    t = positions.numpy().astype(np.float64)[:, None] * freqs.double().numpy()
    c, s = scale * np.cos(t)[:, None], scale * np.sin(t)[:, None]
    far = (np.abs(t) * 3 * 2.0 ** -53)[:, None] * abs(scale)
    y, bound = xd.copy(), np.abs(xd) * rel
    half = layout == "half"
    ia = slice(0, n // 2) if half else slice(0, n, 2)
    ib = slice(n // 2, n) if half else slice(1, n, 2)
    a, b = xd[..., ia], xd[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    size = (np.abs(a) + np.abs(b)) * (abs(scale) * (rel + 12 * U32) + far)
    bound[..., ia] = bound[..., ib] = size
    return y, bound + HALF[x.dtype] * (np.abs(y) + bound) + TINY[x.dtype]


def head_exps(x):
    """Smallest e >= -127 with max|x| <= 448 * 2^e over the last dimension, NaN
    not counted, an infinity as 2^128."""
    a = np.abs(x.double().numpy())
    a = np.where(np.isnan(a), 0.0, np.where(np.isinf(a), 2.0 ** 128, a)).max(-1)
    e = np.full(a.shape, -127)
    for _ in range(260):
        e = np.where(a > np.ldexp(448.0, e), e + 1, e)
    return e.astype(np.int8)


def in_e4m3(x):
    """(q as uint8, exps) of heads, as the cache holds them."""
    e = head_exps(x)
    v = x.double().numpy()
    top = np.ldexp(240.0, 8 if x.dtype == torch.float16 else 120)
    at_top = (e == (8 if x.dtype == torch.float16 else 120))[..., None]
    v = np.where(at_top & np.isfinite(v), np.clip(v, -top, top), v)
    with np.errstate(all="ignore"):
        v = np.ldexp(v, -e.astype(int)[..., None])
        v = np.where(np.isinf(v), np.nan, v)
    q = torch.from_numpy(v.astype(np.float32)).to(torch.float8_e4m3fn)
    return q.view(torch.uint8).numpy(), e


def read_back(q, exps, dtype):
    """Values of e4m3 bytes with their exponents, rounded to dtype, 64 bits."""
    v = torch.from_numpy(q).view(torch.float8_e4m3fn).double()
    v = v * torch.exp2(torch.from_numpy(exps).double())[..., None]
    return v.to(dtype).double().numpy()


def attend(q, k, v, scale, causal, window, dtype):
    """(out, out bound, lse, lse bound) of one sequence, [n][Hq][D] over
    [L][Hk][D], 64-bit numpy.

    A score is a sum of D exact products in 32 bits (2 U32 an addition, should
    it cut off), scaled and less the largest: ds.  A term p is off by ds +
    4 U32 relative, rounded to the type (HALF relative, TINY of the largest
    term absolute) before it meets v; sums of L terms, and the scaling of what
    was summed before by up to L / 16 new largest scores, cost 3 L U32, the
    division and the joining of parts 16 U32.  out is rounded to the type."""
    n, heads, width = q.shape
    keys, kv = k.shape[:2]
    half, tiny = HALF[dtype], TINY[dtype]
    out, out_bound = np.zeros(q.shape), np.zeros(q.shape)
    lse, lse_bound = np.full((n, heads), -np.inf), np.zeros((n, heads))
    i, j = np.arange(n)[:, None], np.arange(keys)
    last = keys - n + i if causal else np.full_like(i, keys - 1)
    seen = (j <= last) & ((j > last - window) if window else True)
    rows = seen.any(1)
    if not rows.any():
        return out, out_bound, lse, lse_bound
    for h in range(heads):
        kh, vh = k[:, h // (heads // kv)], v[:, h // (heads // kv)]
        for r in np.nonzero(rows)[0]:
            at = seen[r]
            kr, vr, qr = kh[at], vh[at], q[r, h]
            with np.errstate(all="ignore"):
                s = kr @ qr * scale
                size = np.abs(kr) @ np.abs(qr) * scale
                m = s.max()
                p = np.exp(s - m)
                w = p / p.sum()
                o = w @ vr
                rel = size * (width + 4) * 2 * U32 + 4 * U32 * (np.abs(s) + abs(m)) + 8 * U32
                a = w @ np.abs(vr)
                off = (w * rel) @ np.abs(vr) + (w @ rel) * np.abs(o)
                off += (half + (3 * len(s) + 16) * U32) * (a + np.abs(o))
                off += tiny / p.sum() * np.abs(vr).sum(0)
                out[r, h] = o
                out_bound[r, h] = off + half * (np.abs(o) + off) + tiny
                lse[r, h] = m + np.log(p.sum())
                lse_bound[r, h] = w @ rel + (3 * len(s) + 16) * U32 + \
                    8 * U32 * (abs(m) + abs(lse[r, h]) + 1)
    return out, out_bound, lse, lse_bound


def check(got, want, bound, what=""):
    got = got.double().cpu().numpy() if isinstance(got, torch.Tensor) else got
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan), f"{what}: NaN in other places"
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf]), f"{what}: infinities"
    fine = ~nan & ~inf
    off = np.abs(got - want)[fine]
    worst = float((off / np.maximum(bound[fine], 1e-300)).max()) if off.size else 0.0
    assert (off <= bound[fine]).all(), f"{what}: {worst:.3g} times its bound"
    return worst
