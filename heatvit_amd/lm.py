"""Operators of language models on device tensors: the path norm -> product ->
answer of rows of floating-point activations.

  rms_norm_q8   residual addition and root-mean-square norm, output in 8 bits
                with power-of-two scales (e4m3 for gemm_f8, int8)
  gemm_f8       e4m3 rows times a DeviceF8Weight, an exponent for each block
                of 128
  log_probs     log probabilities of given tokens, entropy and the most
                probable tokens, from float or int32 logits

Inputs and results are torch tensors on one GPU; every call only enqueues its
kernels on that GPU's current stream and may be captured into a HIP graph
(with `out=` and `workspace=`, or with the capture's own allocations).
`live_rows`, an int32 tensor of one value on the device, gives the rows that
count; rows behind it are left as they were.  Results that the caller does
not pass in `out` are new tensors.  There is no gradient: the inputs are taken
as they are, and the outputs require none.
"""

import math
from typing import NamedTuple, Optional

import torch

from . import _lib
from .device import F8_BLOCK, DeviceF8Weight

_TYPES = {torch.float32: _lib.HV_T_F32, torch.float16: _lib.HV_T_F16,
          torch.bfloat16: _lib.HV_T_BF16}
_LOGIT_TYPES = {**_TYPES, torch.int32: _lib.HV_T_I32}
_FORMATS = {"e4m3": (_lib.HV_Q_E4M3, torch.float8_e4m3fn), "int8": (_lib.HV_Q_I8, torch.int8)}


class Q8Rows(NamedTuple):
    """q * 2^exps * scale stands for the normalised rows."""
    q: torch.Tensor                    # [R][C] float8_e4m3fn or int8
    exps: torch.Tensor                 # [R][blocks] int8
    scale: torch.Tensor                # [R] float32
    residual: Optional[torch.Tensor]   # [R][C], x + residual


class LogProbs(NamedTuple):
    logp: Optional[torch.Tensor]       # float32, the shape of `tokens`
    entropy: torch.Tensor              # [R] float32
    top_logp: Optional[torch.Tensor]   # [R][top] float32
    top_index: Optional[torch.Tensor]  # [R][top] int32


def _matrix(name, t, dtypes):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} has type {t.dtype}")
    if t.dim() != 2:
        raise ValueError(f"{name} must be [rows][columns]")
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"{name} must have adjacent columns")
    if t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise ValueError(f"the rows of {name} overlap")
    return t


def _given(name, t, shape, dtype, strided=False):
    """A result or vector that the caller passes."""
    if not isinstance(t, torch.Tensor) or t.dtype != dtype:
        raise TypeError(f"{name} must be a tensor of {dtype}")
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must have the shape {list(shape)}")
    if strided:
        _matrix(name, t, (dtype,))
    elif not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t


def _ld(t):
    """Row stride of a matrix; one that has a single row may have any."""
    return t.stride(0) if t.shape[0] > 1 else max(t.shape[1], 1)


def _on(device, **tensors):
    """All tensors on the one GPU `device`."""
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, not on {device}")
    if device.type != "cuda":
        raise ValueError("the inputs must be on a GPU")


def _live(live_rows):
    if live_rows is None:
        return None
    if live_rows.dtype != torch.int32 or live_rows.numel() != 1:
        raise ValueError("live_rows must be an int32 tensor of one value")
    return live_rows.data_ptr()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _call(entry, what, device, *args):
    """The library call, on the device's current stream."""
    if torch.cuda.current_device() == device.index:
        rc = entry(*args, torch.cuda.current_stream().cuda_stream)
    else:
        with torch.cuda.device(device):
            rc = entry(*args, torch.cuda.current_stream().cuda_stream)
    _lib.check(rc, what)


def _workspace(workspace, size, device):
    if workspace is None:
        return torch.empty(size, dtype=torch.uint8, device=device) if size else None
    if workspace.dtype != torch.uint8 or not workspace.is_contiguous() or workspace.numel() < size:
        raise ValueError(f"workspace must be {size} contiguous bytes (uint8)")
    return workspace


def rms_norm_q8(x, weight, *, residual=None, eps=1e-6, fmt="e4m3", block=F8_BLOCK,
                live_rows=None, out=None):
    """h = x + residual (rounded once to x's type), p = weight * h,
    scale = 1 / sqrt(mean(h^2) + eps) of each row, and p in 8 bits: q = p /
    2^exps rounded to nearest even, exps the smallest that holds the block.

    x, residual [R][C] and weight [C] of one type (float32, float16,
    bfloat16); fmt "e4m3" or "int8"; block 128 columns, or 0 for one exponent
    a row.  `out`: the Q8Rows to write; its residual may be `residual` or `x`
    itself.  Returns Q8Rows(q, exps, scale, residual)."""
    _matrix("x", x, _TYPES)
    if fmt not in _FORMATS:
        raise ValueError("fmt must be 'e4m3' or 'int8'")
    if block not in (0, F8_BLOCK):
        raise ValueError("block must be 128, or 0 for one exponent a row")
    rows, width = x.shape
    if not width:
        raise ValueError("x has no columns")
    form, q_type = _FORMATS[fmt]
    blocks = -(-width // F8_BLOCK) if block else 1
    _given("weight", weight, (width,), x.dtype)
    if residual is not None:
        _matrix("residual", residual, (x.dtype,))
        if residual.shape != x.shape:
            raise ValueError("residual must have the shape of x")
    if out is None:
        out = Q8Rows(torch.empty((rows, width), dtype=q_type, device=x.device),
                     torch.empty((rows, blocks), dtype=torch.int8, device=x.device),
                     torch.empty(rows, dtype=torch.float32, device=x.device),
                     None if residual is None else
                     torch.empty((rows, width), dtype=x.dtype, device=x.device))
    else:
        _given("out.q", out.q, (rows, width), q_type, strided=True)
        _given("out.exps", out.exps, (rows, blocks), torch.int8, strided=True)
        _given("out.scale", out.scale, (rows,), torch.float32)
        if (residual is None) != (out.residual is None):
            raise ValueError("out.residual goes with residual")
        if residual is not None:
            _given("out.residual", out.residual, (rows, width), x.dtype, strided=True)
    q, exps, scale, kept = out
    _on(x.device, weight=weight, residual=residual, q=q, exps=exps, scale=scale, kept=kept,
        live_rows=live_rows)
    d = _lib.RmsNormDesc(
        x.data_ptr(), _ptr(residual), weight.data_ptr(), _ptr(kept), q.data_ptr(),
        exps.data_ptr(), scale.data_ptr(), _live(live_rows), _ld(x),
        0 if residual is None else _ld(residual), 0 if kept is None else _ld(kept), _ld(q),
        _ld(exps), rows, width, _TYPES[x.dtype], form, block, eps)
    _call(_lib.lib().hv_rms_norm_q8, "rms_norm_q8", x.device, d)
    return out


def gemm_f8(a, a_exps, w, *, row_scale=None, bias=None, out_dtype=torch.bfloat16, live_rows=None,
            out=None, workspace=None):
    """row_scale[m] * sum_k a[m][k] 2^a_exps[m][k/128] W[k][n] 2^w_exps[k/128][n/128]
    + bias[n], rounded once to out_dtype.  A float32 output is summed in
    float32 from exact products; a 16-bit one on the 8-bit matrix cores, which
    cut a product's bits below 2^-13 of the largest one beside it.

    a [M][K] float8_e4m3fn and a_exps [M][ceil(K/128)] int8 (rms_norm_q8
    writes both, and row_scale); w a DeviceF8Weight [K][N]; row_scale [M] and
    bias [N] float32.  The rows of `a` start at multiples of 16 bytes.
    Returns [M][N] (`out` if given)."""
    if not isinstance(w, DeviceF8Weight):
        raise TypeError("w must be a DeviceF8Weight")
    _matrix("a", a, (torch.float8_e4m3fn,))
    _matrix("a_exps", a_exps, (torch.int8,))
    rows, inner = a.shape
    if inner != w.inner:
        raise ValueError(f"K mismatch: a has {inner}, w has {w.inner}")
    if tuple(a_exps.shape) != (rows, -(-inner // F8_BLOCK)):
        raise ValueError("a_exps must be [M][ceil(K/128)]")
    if out_dtype not in _TYPES:
        raise TypeError(f"out_dtype {out_dtype} is not float32, float16 or bfloat16")
    if row_scale is not None:
        _given("row_scale", row_scale, (rows,), torch.float32)
    if bias is not None:
        _given("bias", bias, (w.width,), torch.float32)
    if out is None:
        out = torch.empty((rows, w.width), dtype=out_dtype, device=a.device)
    else:
        _given("out", out, (rows, w.width), out_dtype, strided=True)
    _on(a.device, a_exps=a_exps, w=w, row_scale=row_scale, bias=bias, out=out,
        live_rows=live_rows, workspace=workspace)
    L = _lib.lib()
    workspace = _workspace(workspace, L.hv_gemm_f8_workspace_bytes(rows, w.width, inner), a.device)
    d = _lib.GemmF8Desc(
        a.data_ptr(), a_exps.data_ptr(), w.packed.data_ptr(), w.exps.data_ptr(), _ptr(row_scale),
        _ptr(bias), out.data_ptr(), _live(live_rows), _ld(a) if rows > 1 else -(-inner // 16) * 16,
        _ld(a_exps), _ld(out), rows, w.width, inner, _TYPES[out_dtype])
    _call(L.hv_gemm_f8, "gemm_f8", a.device, d, _ptr(workspace),
          0 if workspace is None else workspace.numel())
    return out


def log_probs(logits, tokens=None, *, scale_exp=0, temperature=1.0, top=0, live_rows=None,
              out=None, workspace=None):
    """Log probabilities under softmax(logits * 2^scale_exp / temperature).

    logits [R][V] float32, float16, bfloat16, or int32 (the model's, with
    scale_exp LOGIT_SCALE_EXP); tokens (optional) [R] or [R][G] int32: those
    whose log probabilities are asked for; one below 0 gets 0, one of V or
    more NaN.  top <= 64: so many most probable tokens, in order, equal
    logits by the lower index.  Logits of -inf have probability 0; a NaN or
    +inf makes its row's log probabilities and entropy NaN.
    Returns LogProbs(logp, entropy, top_logp, top_index) (`out` if given)."""
    _matrix("logits", logits, _LOGIT_TYPES)
    rows, width = logits.shape
    if not width:
        raise ValueError("logits has no columns")
    top = int(top)
    if not 0 <= top <= min(_lib.HV_LOG_PROBS_MAX_TOP, width):
        raise ValueError(f"top {top} outside [0, {_lib.HV_LOG_PROBS_MAX_TOP}] or over the width")
    if not (temperature > 0 and math.isfinite(temperature)):
        raise ValueError("temperature must be positive and finite")
    scale = math.ldexp(1.0, scale_exp) / temperature
    count = 0
    if tokens is not None:
        if not isinstance(tokens, torch.Tensor) or tokens.dtype != torch.int32:
            raise TypeError("tokens must be an int32 tensor")
        if tokens.dim() not in (1, 2) or tokens.shape[0] != rows or not tokens.is_contiguous():
            raise ValueError("tokens must be contiguous, [R] or [R][G]")
        count = 1 if tokens.dim() == 1 else tokens.shape[1]
    f32 = dict(dtype=torch.float32, device=logits.device)
    if out is None:
        out = LogProbs(None if tokens is None else torch.empty(tokens.shape, **f32),
                       torch.empty(rows, **f32),
                       torch.empty((rows, top), **f32) if top else None,
                       torch.empty((rows, top), dtype=torch.int32, device=logits.device)
                       if top else None)
    else:
        if (tokens is None) != (out.logp is None) or bool(top) != (out.top_logp is not None) or \
                bool(top) != (out.top_index is not None):
            raise ValueError("out.logp goes with tokens, out.top_logp and out.top_index with top")
        if tokens is not None:
            _given("out.logp", out.logp, tuple(tokens.shape), torch.float32)
        _given("out.entropy", out.entropy, (rows,), torch.float32)
        if top:
            _given("out.top_logp", out.top_logp, (rows, top), torch.float32)
            _given("out.top_index", out.top_index, (rows, top), torch.int32)
    _on(logits.device, tokens=tokens, logp=out.logp, entropy=out.entropy, top_logp=out.top_logp,
        top_index=out.top_index, live_rows=live_rows, workspace=workspace)
    L = _lib.lib()
    workspace = _workspace(workspace, L.hv_log_probs_workspace_bytes(rows, width, top),
                           logits.device)
    d = _lib.LogProbsDesc(
        logits.data_ptr(), _ptr(tokens), _ptr(out.logp), out.entropy.data_ptr(),
        _ptr(out.top_logp), _ptr(out.top_index), _live(live_rows), _ld(logits), count, rows,
        width, _LOGIT_TYPES[logits.dtype], count, top, scale)
    _call(L.hv_log_probs, "log_probs", logits.device, d, _ptr(workspace),
          0 if workspace is None else workspace.numel())
    return out
