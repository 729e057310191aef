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
(with `out=` and `workspace=`, or with the capture's own allocations; a
workspace serves one call at a time).
`live_rows`, an int32 tensor of one value on the device, gives the rows that
count; rows behind it are left as they were.  Results that the caller does
not pass in `out` are new tensors.  There is no gradient: the inputs are taken
as they are, and the outputs require none.
"""

import math
import struct
from typing import NamedTuple, Optional

import torch

from . import _lib
from .device import F8_BLOCK, DeviceF8Weight

_TYPES = {torch.float32: _lib.HV_T_F32, torch.float16: _lib.HV_T_F16,
          torch.bfloat16: _lib.HV_T_BF16}
_LOGIT_TYPES = {**_TYPES, torch.int32: _lib.HV_T_I32}
_NORM, _GEMM, _ANSWER = (_lib.packer(d) for d in (_lib.RmsNormDesc, _lib.GemmF8Desc,
                                                  _lib.LogProbsDesc))
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
    """(rows, columns, row stride) of a matrix with adjacent columns."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} has type {t.dtype}")
    if t.dim() != 2:
        raise ValueError(f"{name} must be [rows][columns]")
    rows, columns = t.shape
    ld, step = t.stride()
    if step != 1 and columns > 1:
        raise ValueError(f"{name} must have adjacent columns")
    if rows <= 1:
        ld = columns
    elif ld < columns:
        raise ValueError(f"the rows of {name} overlap")
    return rows, columns, ld


def _given(name, t, shape, dtype):
    """A contiguous vector or result that the caller passes."""
    if not isinstance(t, torch.Tensor) or t.dtype != dtype:
        raise TypeError(f"{name} must be a tensor of {dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} must have the shape {list(shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _given_matrix(name, t, shape, dtype):
    """Row stride of a matrix that the caller passes."""
    if not isinstance(t, torch.Tensor) or t.dtype != dtype:
        raise TypeError(f"{name} must be a tensor of {dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} must have the shape {list(shape)}")
    if t.is_contiguous():  # the strides need not be looked at
        return shape[1]
    return _matrix(name, t, (dtype,))[2]


def _call(entry, what, index, tensors, pack, values, *args):
    """The library call, with the values as its descriptor, on the current
    stream of GPU `index`, where all of the tensors are.  (The stream's handle
    comes from the getter behind torch.cuda.current_stream(), which takes 2.4
    us to wrap it.)"""
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise ValueError(f"{what}: tensors on cuda:{index} and on {t.device}")
    try:
        d = pack(*values)
    except (struct.error, OverflowError) as e:
        raise ValueError(f"{what}: a size or number is out of range ({e})") from None
    if torch.cuda.current_device() == index:
        rc = entry(d, *args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = entry(d, *args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        raise _lib.error(rc, what)


def _live(live_rows):
    if live_rows is None:
        return 0
    if live_rows.dtype != torch.int32 or live_rows.numel() != 1:
        raise ValueError("live_rows must be an int32 tensor of one value")
    return live_rows.data_ptr()


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _workspace(workspace, size, like):
    """(tensor, pointer, bytes)"""
    if workspace is None:
        if not size:
            return None, None, 0
        workspace = like.new_empty(size, dtype=torch.uint8)
    elif workspace.dtype != torch.uint8 or not workspace.is_contiguous() or \
            workspace.numel() < size:
        raise ValueError(f"workspace must be {size} contiguous bytes (uint8)")
    return workspace, workspace.data_ptr(), workspace.numel()


def rms_norm_q8(x, weight, *, residual=None, eps=1e-6, fmt="e4m3", block=F8_BLOCK,
                live_rows=None, out=None):
    """h = x + residual (rounded once to x's type), p = weight * h,
    scale = 1 / sqrt(mean(h^2) + eps) of each row, and p in 8 bits: q = p /
    2^exps rounded to nearest even, exps the smallest that holds the block.

    x, residual [R][C] and weight [C] of one type (float32, float16,
    bfloat16); fmt "e4m3" or "int8"; block 128 columns, or 0 for one exponent
    a row (gemm_f8 takes the first).  A NaN or an infinity is NaN in e4m3; int8
    has the end of its range for an infinity and 0 for NaN, and the row's scale
    is 0 or NaN.  `out`: the Q8Rows to write; its residual may be `residual` or `x`
    itself.  Returns Q8Rows(q, exps, scale, residual)."""
    rows, width, x_ld = _matrix("x", x, _TYPES)
    if fmt not in _FORMATS:
        raise ValueError("fmt must be 'e4m3' or 'int8'")
    if block != 0 and block != F8_BLOCK:
        raise ValueError("block must be 128, or 0 for one exponent a row")
    if not width:
        raise ValueError("x has no columns")
    form, q_type = _FORMATS[fmt]
    blocks = -(-width // F8_BLOCK) if block else 1
    dtype = x.dtype
    _given("weight", weight, (width,), dtype)
    residual_ld = kept_ld = 0
    if residual is not None:
        residual_ld = _given_matrix("residual", residual, x.shape, dtype)
    if out is None:
        q = torch.empty_like(x, dtype=q_type, memory_format=torch.contiguous_format)
        exps = x.new_empty((rows, blocks), dtype=torch.int8)
        scale = x.new_empty(rows, dtype=torch.float32)
        kept, q_ld, exps_ld, kept_ld = None, width, blocks, width
        if residual is not None:
            kept = torch.empty_like(x, memory_format=torch.contiguous_format)
        out = Q8Rows(q, exps, scale, kept)
    else:
        q, exps, scale, kept = out
        q_ld = _given_matrix("out.q", q, x.shape, q_type)
        exps_ld = _given_matrix("out.exps", exps, (rows, blocks), torch.int8)
        _given("out.scale", scale, (rows,), torch.float32)
        if (residual is None) != (kept is None):
            raise ValueError("out.residual goes with residual")
        if kept is not None:
            kept_ld = _given_matrix("out.residual", kept, x.shape, dtype)
    values = (
        x.data_ptr(), _ptr(residual), weight.data_ptr(), _ptr(kept), q.data_ptr(),
        exps.data_ptr(), scale.data_ptr(), _live(live_rows), x_ld, residual_ld, kept_ld, q_ld,
        exps_ld, rows, width, _TYPES[dtype], form, block, eps)
    if not x.is_cuda:
        raise ValueError("the inputs must be on a GPU")
    _call(_lib.lib().hv_rms_norm_q8, "rms_norm_q8", x.get_device(),
          (weight, residual, q, exps, scale, kept, live_rows), _NORM, values)
    return out


def gemm_f8(a, a_exps, w, *, row_scale=None, bias=None, out_dtype=torch.bfloat16, live_rows=None,
            out=None):
    """row_scale[m] * sum_k a[m][k] 2^a_exps[m][k/128] W[k][n] 2^w_exps[k/128][n/128]
    + bias[n], rounded once to out_dtype.  A float32 output is summed in
    float32 from exact products; a 16-bit one on the 8-bit matrix cores, which
    cut a product's bits below 2^-13 of the largest one beside it (1.5e-5 of
    the result's norm on normal values, 1e-4 with a column in each block 64
    times the others: where that counts, ask for float32).

    a [M][K] float8_e4m3fn and a_exps [M][ceil(K/128)] int8 (rms_norm_q8
    writes both, and row_scale) in [-127, 127] (-128 makes the row NaN); w a
    DeviceF8Weight [K][N]; row_scale [M] and bias [N] float32.  The rows of `a`
    start at multiples of 16 bytes.
    Returns [M][N] (`out` if given)."""
    if not isinstance(w, DeviceF8Weight):
        raise TypeError("w must be a DeviceF8Weight")
    rows, inner, lda = _matrix("a", a, (torch.float8_e4m3fn,))
    width = w.width
    if inner != w.inner:
        raise ValueError(f"K mismatch: a has {inner}, w has {w.inner}")
    exps_ld = _given_matrix("a_exps", a_exps, (rows, -(-inner // F8_BLOCK)), torch.int8)
    if out_dtype not in _TYPES:
        raise TypeError(f"out_dtype {out_dtype} is not float32, float16 or bfloat16")
    if row_scale is not None:
        _given("row_scale", row_scale, (rows,), torch.float32)
    if bias is not None:
        _given("bias", bias, (width,), torch.float32)
    if out is None:
        out, ldc = a.new_empty((rows, width), dtype=out_dtype), width
    else:
        ldc = _given_matrix("out", out, (rows, width), out_dtype)
    if not a.is_cuda:
        raise ValueError("the inputs must be on a GPU")
    values = (
        a.data_ptr(), a_exps.data_ptr(), w.packed.data_ptr(), w.exps.data_ptr(), _ptr(row_scale),
        _ptr(bias), out.data_ptr(), _live(live_rows), lda, exps_ld, ldc, rows, width, inner,
        _TYPES[out_dtype])
    _call(_lib.lib().hv_gemm_f8, "gemm_f8", a.get_device(),
          (a_exps, w.packed, row_scale, bias, out, live_rows), _GEMM, values)
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
    rows, width, ld = _matrix("logits", logits, _LOGIT_TYPES)
    if not width:
        raise ValueError("logits has no columns")
    if not 0 <= top <= min(_lib.HV_LOG_PROBS_MAX_TOP, width):
        raise ValueError(f"top {top} outside [0, {_lib.HV_LOG_PROBS_MAX_TOP}] or over the width")
    if not 0 < temperature < math.inf:
        raise ValueError("temperature must be positive and finite")
    try:
        scale = math.ldexp(1.0, scale_exp) / temperature
    except OverflowError:
        raise ValueError(f"2^{scale_exp} / temperature is out of range") from None
    count = 0
    if tokens is not None:
        if not isinstance(tokens, torch.Tensor) or tokens.dtype != torch.int32:
            raise TypeError("tokens must be an int32 tensor")
        if tokens.dim() not in (1, 2) or tokens.shape[0] != rows or not tokens.is_contiguous():
            raise ValueError("tokens must be contiguous, [R] or [R][G]")
        count = 1 if tokens.dim() == 1 else tokens.shape[1]
    if out is None:
        logp = top_logp = top_index = None
        f32 = torch.float32
        if tokens is not None:
            logp = torch.empty_like(tokens, dtype=f32, memory_format=torch.contiguous_format)
        entropy = logits.new_empty(rows, dtype=f32)
        if top:
            top_logp = logits.new_empty((rows, top), dtype=f32)
            top_index = torch.empty_like(top_logp, dtype=torch.int32)
        out = LogProbs(logp, entropy, top_logp, top_index)
    else:
        logp, entropy, top_logp, top_index = out
        if (tokens is None) != (logp is None) or bool(top) != (top_logp is not None) or \
                bool(top) != (top_index is not None):
            raise ValueError("out.logp goes with tokens, out.top_logp and out.top_index with top")
        if tokens is not None:
            _given("out.logp", logp, tokens.shape, torch.float32)
        _given("out.entropy", entropy, (rows,), torch.float32)
        if top:
            _given("out.top_logp", top_logp, (rows, top), torch.float32)
            _given("out.top_index", top_index, (rows, top), torch.int32)
    if not logits.is_cuda:
        raise ValueError("the inputs must be on a GPU")
    L = _lib.lib()
    workspace, ws_at, ws_size = _workspace(
        workspace, L.hv_log_probs_workspace_bytes(rows, width, top), logits)
    values = (
        logits.data_ptr(), _ptr(tokens), _ptr(logp), entropy.data_ptr(), _ptr(top_logp),
        _ptr(top_index), _live(live_rows), ld, count, rows, width, _LOGIT_TYPES[logits.dtype],
        count, top, scale)
    _call(L.hv_log_probs, "log_probs", logits.get_device(),
          (tokens, logp, entropy, top_logp, top_index, live_rows, workspace), _ANSWER,
          values, ws_at, ws_size)
    return out
