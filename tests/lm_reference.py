"""Plain 64-bit forms of the language-model operators (numpy, and torch on the
CPU for the 8-bit types), and the rounding bounds their results are held to.

A rounding is off by at most half a step: U32 = 2^-24 relative in float32,
HALF[t] in an output type."""

import math

import numpy as np
import torch

U32 = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LARGEST = {"e4m3": 448.0, "int8": 127.0}


def block_exps(p, block, largest):
    """Smallest e >= -127 with max|p| <= largest * 2^e, by trying: NaN does
    not count, an infinity gives the exponent of 2^128 (the bits above the
    largest float)."""
    rows, width = p.shape
    block = block or width
    out = np.empty((rows, -(-width // block)), np.int8)
    for b in range(out.shape[1]):
        a = np.abs(p[:, b * block:(b + 1) * block])
        a = np.where(np.isnan(a), 0.0, a).max(1)
        a = np.where(np.isinf(a), 2.0 ** 128, a)
        for r in range(rows):
            e = -127
            if a[r] > 0:
                e = max(-127, math.frexp(a[r])[1] - math.frexp(largest)[1] - 1)
                while a[r] > math.ldexp(largest, e):
                    e += 1
            out[r, b] = e
    return out


def spread(exps, block, width):
    """2^exps for every column."""
    e = np.ldexp(1.0, exps.astype(int))
    return np.repeat(e, block or width, axis=1)[:, :width]


def rms_norm_q8(x, weight, residual, eps, fmt, block):
    """(q as the type it has, exps, scale in 64 bits, residual_out) of CPU
    tensors.  p is the float32 product, as the operator defines it: exact for
    the 16-bit types, rounded once for float32."""
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    p = (h.float() * weight.float()).double().numpy()
    exps = block_exps(p, block, LARGEST[fmt])
    with np.errstate(all="ignore"):
        v = p / spread(exps, block, p.shape[1])
    if fmt == "e4m3":
        v = np.where(np.isinf(v), np.nan, v)
        q = torch.from_numpy(v.astype(np.float32)).to(torch.float8_e4m3fn)
    else:
        with np.errstate(all="ignore"):
            i = np.clip(np.rint(v), -127, 127)
        q = torch.from_numpy(np.where(np.isnan(i), 0, i).astype(np.int8))
    with np.errstate(all="ignore"):
        scale = 1.0 / np.sqrt(np.square(h.double().numpy()).mean(1) + eps)
    return q, exps, scale, (None if residual is None else h)


def scale_bound(width):
    """Relative error of 1 / sqrt(mean + eps): at most width / 64 adds follow
    one another in a thread and 10 join the threads, each U32 of a sum of
    positive terms; the square root halves that; the mean, eps, the root and
    the division round once more each (2 U32 allowed for each)."""
    return (width / 64 + 10) * U32 / 2 + 8 * U32


def gemm_f8(a, a_exps, w, w_exps, row_scale, bias, fast=False):
    """(y, bound without the output's rounding), both 64 bits: at most K + 8
    additions of float32 (2^-23 each, should one cut off instead of rounding)
    of terms whose sizes add up to `size`, then two more roundings.

    fast (16-bit outputs): the 8-bit matrix cores align each product to the
    largest one of its group, of exponent E, and cut it below 2^(E - 13); 2^E
    is at most the largest product of the block, so a block of n terms is off
    by at most n 2^-13 times that, which is at most the largest |a| times the
    largest |w| of the block's row and column."""
    k, n = w.shape
    af = a.double().numpy() * spread(a_exps, 128, k)
    wf = w.double().numpy() * np.repeat(spread(w_exps, 128, n), 128, axis=0)[:k]
    y, size = af @ wf, np.abs(af) @ np.abs(wf)
    if row_scale is not None:
        y, size = y * row_scale[:, None], size * np.abs(row_scale)[:, None]
    if bias is not None:
        y, size = y + bias, size + np.abs(bias)
    bound = size * (k + 8) * 2 * U32
    if fast:
        cut = sum(min(128, k - b) * 2.0 ** -13 * np.abs(af[:, b:b + 128]).max(1)[:, None] *
                  np.abs(wf[b:b + 128]).max(0)[None] for b in range(0, k, 128))
        bound = bound + (cut if row_scale is None else cut * np.abs(row_scale)[:, None])
    return y, bound


def log_probs(x, tokens, scale, top):
    """logits (64-bit numpy) -> dict of 64-bit results and their bounds.

    d = scale (x - max) is rounded twice (2 U32 |d|), its exponential adds
    the exponent's rounding (U32 |d| more) and 4 U32 of its own; a term of S
    is then off by (4 |d| + 4) U32 relative, S by that weighted with p, plus
    one U32 for each of at most V / 64 + 16 additions.  The weighted sum T
    adds another factor d to each term.  `scale` itself is rounded to 32 bits
    (1 U32 |d| more, counted in the four)."""
    with np.errstate(all="ignore"):
        m = x.max(1, keepdims=True)
        d = np.where(np.isneginf(x), -np.inf, (x - m) * scale)
        e = np.exp(d)
        s = e.sum(1, keepdims=True)
        log_s = np.log(s)
        p = e / s
        ad = np.where(p > 0, np.abs(d), 0.0)
        adds = x.shape[1] / 64 + 16
        s_rel = ((p * (4 * ad + 4)).sum(1) + adds) * U32
        t = (p * ad).sum(1)
        out = {"entropy": log_s[:, 0] + t,
               "entropy_bound": s_rel * (1 + t) + ((p * ad * (5 * ad + 6)).sum(1) + adds * t) * U32
               + 4 * U32 * (np.abs(log_s[:, 0]) + t + 1)}
        lp = d - log_s
        lp_bound = np.where(np.isfinite(d), 4 * np.abs(d) * U32, 0) + s_rel[:, None] + \
            2 * U32 * (np.abs(log_s) + np.where(np.isfinite(lp), np.abs(lp), 0)) + U32
    if tokens is not None:
        at = np.clip(tokens, 0, x.shape[1] - 1)
        out["logp"] = np.take_along_axis(lp, at, 1)
        out["logp_bound"] = np.take_along_axis(lp_bound, at, 1)
        out["logp"] = np.where(tokens < 0, 0.0, np.where(tokens >= x.shape[1], np.nan, out["logp"]))
    if top:
        order = np.argsort(-x, axis=1, kind="stable")[:, :top]
        out["top_index"] = order
        out["top_logp"] = np.take_along_axis(lp, order, 1)
        out["top_logp_bound"] = np.take_along_axis(lp_bound, order, 1)
    return out
