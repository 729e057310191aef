"""Operators of language models on device tensors: the path norm -> product ->
attention -> answer of rows of floating-point activations.

  rms_norm_q8      residual addition and root-mean-square norm, output in 8
                   bits with power-of-two scales (e4m3 for gemm_f8, int8)
  gemm_f8          e4m3 rows times a DeviceF8Weight, an exponent for each block
                   of 128
  rotary_qk        norms of the heads of queries and keys and the rotation by
                   their positions
  cache_write      new keys and values into a KvCache, in 16 bits or in e4m3
  attention        attention of packed sequences, grouped heads, causal or not
  paged_attention  attention of new rows over a KvCache
  log_probs        log probabilities of given tokens, entropy and the most
                   probable tokens, from float or int32 logits

Inputs and results are torch tensors on one GPU; every call only enqueues its
kernels on that GPU's current stream and may be captured into a HIP graph
(with `out=` and `workspace=`, or with the capture's own allocations; a
workspace serves one call at a time).
`live_rows`, an int32 tensor of one value on the device, gives the rows that
count; rows behind it are left as they were.  The attention's operators take
int32 offsets of sequences instead (`starts`), and leave rows outside all
sequences as they were.  Results that the caller does
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
_HEAD_TYPES = {torch.float16: _lib.HV_T_F16, torch.bfloat16: _lib.HV_T_BF16}
_NORM, _GEMM, _ANSWER, _ROTARY, _WRITE, _ATTEND, _PAGED = (
    _lib.packer(d) for d in (_lib.RmsNormDesc, _lib.GemmF8Desc, _lib.LogProbsDesc, _lib.RotaryDesc,
                             _lib.CacheWriteDesc, _lib.AttentionDesc, _lib.PagedAttentionDesc))
_LAYOUTS = {"half": _lib.HV_ROTARY_HALF, "interleaved": _lib.HV_ROTARY_INTERLEAVED}
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


# ------------------------------------------------------------------ attention

class QK(NamedTuple):
    q: torch.Tensor                    # [T][Hq][D]
    k: Optional[torch.Tensor]          # [T][Hk][D]


class Attended(NamedTuple):
    out: torch.Tensor                  # [T][Hq][D]
    lse: Optional[torch.Tensor]        # [T][Hq] float32


def _heads(name, t, dtypes):
    """(rows, heads, width, row stride, head stride) of [rows][heads][width]
    whose heads' elements are adjacent and whose heads do not overlap."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} has type {t.dtype}")
    if t.dim() != 3:
        raise ValueError(f"{name} must be [rows][heads][width]")
    rows, heads, width = t.shape
    ld, head_ld, step = t.stride()
    if t.is_contiguous():
        return rows, heads, width, heads * width, width
    if step != 1 and width > 1:
        raise ValueError(f"the elements of {name}'s heads must be adjacent")
    if heads <= 1:
        head_ld = width
    if rows <= 1:
        ld = max(1, heads - 1) * head_ld + width
    inner, outer, count = (head_ld, ld, heads) if head_ld <= ld else (ld, head_ld, rows)
    if rows and heads and (inner < width or outer < (count - 1) * inner + width):
        raise ValueError(f"the heads of {name} overlap")
    return rows, heads, width, ld, head_ld


def _heads_like(name, t, shape, dtype):
    """(row stride, head stride) of a result that the caller passes."""
    if not isinstance(t, torch.Tensor) or t.dtype != dtype:
        raise TypeError(f"{name} must be a tensor of {dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} must have the shape {list(shape)}")
    return _heads(name, t, (dtype,))[3:]


def _ints(name, t, shape):
    """An int32 vector of the call; a length of None is any."""
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32:
        raise TypeError(f"{name} must be an int32 tensor")
    if t.dim() != 1 or (shape is not None and t.shape[0] != shape):
        raise ValueError(f"{name} must be a vector" +
                         ("" if shape is None else f" of {shape}"))
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _batch(starts, rows, batch=None):
    """Sequences of packed rows: as many as the offsets say."""
    if starts is None:
        return rows if batch is None else batch
    _ints("starts", starts, None if batch is None else batch + 1)
    if not starts.shape[0]:
        raise ValueError("starts must hold one offset more than there are sequences")
    return starts.shape[0] - 1


def rotary_frequencies(rotated, base=10000.0, *, factor=1.0, trained=None, low=1.0, high=4.0):
    """float32 frequencies (radians a position) of rotated / 2 pairs,
    base^(-2 i / rotated), for rotary_qk.

    factor > 1 stretches them for contexts longer than the `trained` positions
    of the model: without `trained` all are divided by it; with it those that
    turn fewer than `low` times within the trained positions are, those that
    turn more than `high` times stay, and in between the share that stays grows
    evenly with the turns."""
    if rotated < 0 or rotated % 2 or rotated > _lib.HV_ROTARY_MAX_WIDTH:
        raise ValueError(f"rotated {rotated} must be even, up to {_lib.HV_ROTARY_MAX_WIDTH}")
    if not 0 < base < math.inf or not 0 < factor < math.inf:
        raise ValueError("base and factor must be positive and finite")
    f = base ** (torch.arange(0, rotated, 2, dtype=torch.float64) / -max(rotated, 1))
    if trained is None:
        return (f / factor).float()
    if not trained > 0 or not 0 <= low < high < math.inf:
        raise ValueError("trained must be positive, and 0 <= low < high")
    stays = ((f * trained / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
    return (f * (stays + (1 - stays) / factor)).float()


def rotary_qk(q, k, positions, freqs, *, q_weight=None, k_weight=None, eps=1e-6, layout="half",
              scale=1.0, live_rows=None, out=None):
    """y = x / sqrt(mean(x^2) + eps) * weight of each head of q and of k (y = x
    without a weight), and the pairs (a, b) of y's first 2 len(freqs) elements
    turned by t = position * freqs[pair]: scale * (a cos t - b sin t, a sin t +
    b cos t), in float32 (the angle in float64), rounded once to q's type.

    q [T][Hq][D] and k [T][Hk][D] (or None) of one type (float32, float16,
    bfloat16), D <= 1024; positions [T] int32; freqs [R/2] float32 (see
    rotary_frequencies), R <= D; q_weight, k_weight [D] of q's type.  layout
    "half": pair i is elements i and R/2 + i; "interleaved": 2 i and 2 i + 1.
    `out`: the QK to write, its tensors q and k themselves if wanted (or apart
    from both).  Returns QK(q, k)."""
    rows, q_heads, width, q_ld, q_head_ld = _heads("q", q, _TYPES)
    dtype = q.dtype
    if not 1 <= width <= _lib.HV_ROTARY_MAX_WIDTH or not q_heads:
        raise ValueError(f"q must have heads of 1 to {_lib.HV_ROTARY_MAX_WIDTH} elements")
    k_heads = k_ld = k_head_ld = k_out_ld = k_out_head_ld = 0
    if k is not None:
        k_rows, k_heads, k_width, k_ld, k_head_ld = _heads("k", k, (dtype,))
        if k_rows != rows or k_width != width or not k_heads:
            raise ValueError(f"k must be [{rows}][heads][{width}]")
    _ints("positions", positions, rows)
    if not isinstance(freqs, torch.Tensor) or freqs.dtype != torch.float32:
        raise TypeError("freqs must be a float32 tensor")
    if freqs.dim() != 1 or not freqs.is_contiguous() or 2 * freqs.shape[0] > width:
        raise ValueError(f"freqs must be contiguous, [R/2] with R at most {width}")
    if layout not in _LAYOUTS:
        raise ValueError("layout must be 'half' or 'interleaved'")
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    if k is None and k_weight is not None:
        raise ValueError("k_weight goes with k")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None:
            _given(name, w, (width,), dtype)
    if out is None:
        out = QK(torch.empty_like(q, memory_format=torch.contiguous_format), None if k is None else
                 torch.empty_like(k, memory_format=torch.contiguous_format))
        q_out_ld, q_out_head_ld = q_heads * width, width
        k_out_ld, k_out_head_ld = k_heads * width, width
    else:
        if (k is None) != (out[1] is None):
            raise ValueError("out.k goes with k")
        q_out_ld, q_out_head_ld = _heads_like("out.q", out[0], q.shape, dtype)
        if k is not None:
            k_out_ld, k_out_head_ld = _heads_like("out.k", out[1], k.shape, dtype)
    if not q.is_cuda:
        raise ValueError("the inputs must be on a GPU")
    values = (
        q.data_ptr(), _ptr(k), _ptr(q_weight), _ptr(k_weight), out[0].data_ptr(), _ptr(out[1]),
        positions.data_ptr(), freqs.data_ptr(), _live(live_rows), q_ld, q_head_ld, k_ld, k_head_ld,
        q_out_ld, q_out_head_ld, k_out_ld, k_out_head_ld, rows, q_heads, k_heads, width,
        2 * freqs.shape[0], _TYPES[dtype], _LAYOUTS[layout], eps, scale, 0)
    _call(_lib.lib().hv_rotary_qk, "rotary_qk", q.get_device(),
          (k, q_weight, k_weight, out[0], out[1], positions, freqs, live_rows), _ROTARY, values)
    return out


class KvCache:
    """Pages of keys and values: k and v [pages][kv_heads][page][D] of float16
    or bfloat16, or of float8_e4m3fn with k_exps and v_exps [pages][kv_heads]
    [page] int8 (value * 2^exps, rounded to `dtype` where it is read; -128 is
    NaN).  page is a power of two from 16 to 4096, D a multiple of 8 (e4m3: 16) up
    to 256.

    The tensors are the caller's and are written in place; KvCache.empty
    makes them."""

    def __init__(self, k, v, k_exps=None, v_exps=None, *, dtype=None):
        for name, t in (("k", k), ("v", v)):
            if not isinstance(t, torch.Tensor):
                raise TypeError(f"{name} must be a torch tensor")
            if t.dim() != 4 or not t.is_contiguous() or t.shape != k.shape:
                raise ValueError("k and v must be contiguous [pages][kv_heads][page][D], alike")
        q8 = k.dtype == torch.float8_e4m3fn
        dtype = dtype or (torch.bfloat16 if q8 else k.dtype)
        if dtype not in _HEAD_TYPES or v.dtype != k.dtype or (not q8 and k.dtype != dtype):
            raise TypeError(f"a cache of {k.dtype} and {v.dtype} for heads of {dtype}")
        pages, heads, page, width = k.shape
        if not pages or not heads:
            raise ValueError("a cache needs a page and a head")
        if not _lib.HV_CACHE_MIN_PAGE <= page <= _lib.HV_CACHE_MAX_PAGE or page & (page - 1):
            raise ValueError(f"page {page} is no power of two from {_lib.HV_CACHE_MIN_PAGE} to "
                             f"{_lib.HV_CACHE_MAX_PAGE}")
        unit = 16 if q8 else 8
        if not unit <= width <= _lib.HV_ATTENTION_MAX_WIDTH or width % unit:
            raise ValueError(f"heads of {width} are no multiple of {unit} up to "
                             f"{_lib.HV_ATTENTION_MAX_WIDTH}")
        if (k_exps is None) != (v_exps is None) or q8 != (k_exps is not None):
            raise ValueError("k_exps and v_exps go with e4m3")
        if q8:
            _given("k_exps", k_exps, (pages, heads, page), torch.int8)
            _given("v_exps", v_exps, (pages, heads, page), torch.int8)
        if len({t.device for t in (k, v, k_exps, v_exps) if t is not None}) != 1:
            raise ValueError("the tensors of a cache must be on one device")
        self.k, self.v, self.k_exps, self.v_exps, self.dtype = k, v, k_exps, v_exps, dtype
        self.pages, self.kv_heads, self.page, self.width = pages, heads, page, width
        self._format = _lib.HV_CACHE_E4M3 if q8 else _lib.HV_CACHE_SAME

    @classmethod
    def empty(cls, pages, kv_heads, width, *, page=64, dtype=torch.bfloat16, e4m3=False,
              device="cuda"):
        shape = (pages, kv_heads, page, width)
        held = torch.float8_e4m3fn if e4m3 else dtype
        tensors = [torch.zeros(shape, dtype=held, device=device) for _ in range(2)]
        if e4m3:
            tensors += [torch.zeros(shape[:3], dtype=torch.int8, device=device) for _ in range(2)]
        return cls(*tensors, dtype=dtype)

    def _values(self, table, lengths, batch):
        """The descriptor's fields, and the tensors to look at."""
        if not isinstance(table, torch.Tensor) or table.dtype != torch.int32:
            raise TypeError("table must be an int32 tensor")
        if table.dim() != 2 or table.shape[0] != batch:
            raise ValueError(f"table must be [{batch}][pages of a sequence]")
        _, most, table_ld = _matrix("table", table, (torch.int32,))
        _ints("lengths", lengths, batch)
        values = (self.k.data_ptr(), self.v.data_ptr(), _ptr(self.k_exps), _ptr(self.v_exps),
                  table.data_ptr(), lengths.data_ptr(), table_ld, self.pages, self.page, most,
                  self._format)
        return values, (self.k, table, lengths)


def cache_write(cache, k, v, table, lengths, *, starts=None):
    """New keys and values into a KvCache: rows starts[b] .. starts[b+1] - 1 of
    k and v are the last keys of sequence b, which has lengths[b] with them, key
    j in page table[b][j / page].  Without `starts` each sequence has one row.

    k, v [T][Hk][D] of the cache's dtype; table [B][pages] int32, lengths [B]
    and starts [B + 1] int32, all on the device.  In e4m3 each head of a row
    gets the smallest exponent that holds it (with an infinity, which is read back
    as NaN, the largest).  A row is not written where its
    place lies before the first key, past the table or in a page that the
    cache does not have.  Sequences that share a page must not both write it."""
    if not isinstance(cache, KvCache):
        raise TypeError("cache must be a KvCache")
    rows, heads, width, k_ld, k_head_ld = _heads("k", k, (cache.dtype,))
    if heads != cache.kv_heads or width != cache.width:
        raise ValueError(f"k must be [rows][{cache.kv_heads}][{cache.width}]")
    v_ld, v_head_ld = _heads_like("v", v, k.shape, cache.dtype)
    batch = _batch(starts, rows)
    values, tensors = cache._values(table, lengths, batch)
    if not k.is_cuda:
        raise ValueError("the inputs must be on a GPU")
    values += (k.data_ptr(), v.data_ptr(), _ptr(starts), k_ld, k_head_ld, v_ld, v_head_ld, rows,
               batch, heads, width, _HEAD_TYPES[cache.dtype], 0)
    _call(_lib.lib().hv_cache_write, "cache_write", k.get_device(), (v, starts, *tensors), _WRITE,
          values)


def _aligned(name, t, *lds):
    if t.data_ptr() % 16 or any(ld % 8 for ld in lds):
        raise ValueError(f"the heads of {name} must start at multiples of 16 bytes")


def _attention_rows(q, kv_heads, starts, batch, scale, causal, window, most_keys, lse, out):
    """The descriptor's fields of the rows, the result and the tensors to look at."""
    rows, heads, width, q_ld, q_head_ld = _heads("q", q, _HEAD_TYPES)
    if not 8 <= width <= _lib.HV_ATTENTION_MAX_WIDTH or width % 8:
        raise ValueError(f"heads of {width} are no multiple of 8 up to "
                         f"{_lib.HV_ATTENTION_MAX_WIDTH}")
    if not heads or not kv_heads or heads % kv_heads:
        raise ValueError(f"{heads} heads of queries for {kv_heads} of keys")
    if scale is None:
        scale = 1.0 / math.sqrt(width)
    if not 0 < scale <= 1e30:
        raise ValueError("scale must lie in (0, 1e30]")
    if window < 0 or (window and not causal):
        raise ValueError("window must not be negative, and goes with causal")
    if most_keys is None:
        most_keys = 0
    elif most_keys < 0:
        raise ValueError("most_keys must not be negative")
    _aligned("q", q, q_ld, q_head_ld)
    if out is None:
        out = Attended(torch.empty_like(q, memory_format=torch.contiguous_format),
                       q.new_empty((rows, heads), dtype=torch.float32) if lse else None)
        out_ld, out_head_ld = heads * width, width
    else:
        if bool(lse) != (out[1] is not None):
            raise ValueError("out.lse goes with lse")
        out_ld, out_head_ld = _heads_like("out.out", out[0], q.shape, q.dtype)
        _aligned("out.out", out[0], out_ld, out_head_ld)
        if lse:
            _given("out.lse", out[1], (rows, heads), torch.float32)
    values = (q.data_ptr(), out[0].data_ptr(), _ptr(out[1]), _ptr(starts), q_ld, q_head_ld, out_ld,
              out_head_ld, rows, batch, heads, kv_heads, width, _HEAD_TYPES[q.dtype], bool(causal),
              window, scale, most_keys)
    return values, Attended(*out), (out[0], out[1], starts)


def attention(q, k, v, starts, *, k_starts=None, scale=None, causal=True, window=0, most_keys=None,
              lse=False, out=None, workspace=None):
    """Attention of packed sequences: rows starts[b] .. starts[b+1] - 1 of q over
    rows k_starts[b] .. k_starts[b+1] - 1 of k and v (without k_starts, of starts).

    q [T][Hq][D], k and v [S][Hk][D] of float16 or bfloat16, Hq a multiple of Hk
    (head h reads head h / (Hq / Hk)), D a multiple of 8 up to 256, heads at
    multiples of 16 bytes; starts, k_starts [B + 1] int32 on the device.  scale: 1 /
    sqrt(D) if None.  causal: the last row of a sequence sees all of its keys, each
    row before it one less; window > 0: the last `window` of those. A row that sees
    nothing gets zeros (and -inf in lse); what a row does not see leaves no trace in
    it.  Sequences may be empty; offsets that leave the tensors are taken at their
    ends, and where sequences overlap, rows of any of the call's hold any values.
    most_keys: about as many keys as the longest sequence has, where the program
    knows it (else twice the mean is taken): it says whether the work of few long
    sequences is cut into shares, and so no more than roundings.  `out`: the
    Attended to write, its tensor q itself if wanted, and apart from k and v.
    Returns Attended(out, lse), lse [T][Hq] the logarithm of the sum of exponentials
    where asked for."""
    if not isinstance(k, torch.Tensor) or not isinstance(q, torch.Tensor):
        raise TypeError("q and k must be torch tensors")
    if q.dtype not in _HEAD_TYPES:
        raise TypeError(f"q has type {q.dtype}")
    k_rows, kv_heads, width, k_ld, k_head_ld = _heads("k", k, (q.dtype,))
    v_ld, v_head_ld = _heads_like("v", v, k.shape, q.dtype)
    if starts is None:
        raise TypeError("starts must be an int32 tensor")
    batch = _batch(starts, 0)
    if k_starts is not None:
        _ints("k_starts", k_starts, batch + 1)
    values, out, tensors = _attention_rows(q, kv_heads, starts, batch, scale, causal, window,
                                           most_keys, lse, out)
    if q.shape[2] != width or (k_starts is None and k_rows != q.shape[0]):
        raise ValueError(f"k of {list(k.shape)} does not go with q of {list(q.shape)}")
    _aligned("k", k, k_ld, k_head_ld)
    _aligned("v", v, v_ld, v_head_ld)
    if not q.is_cuda:
        raise ValueError("the inputs must be on a GPU")
    values += (k.data_ptr(), v.data_ptr(), _ptr(k_starts), k_ld, k_head_ld, v_ld, v_head_ld,
               k_rows, 0)
    _attend(_lib.lib().hv_attention, "attention", q, (k, v, k_starts, *tensors), _ATTEND, values,
            batch, kv_heads, workspace)
    return out


def paged_attention(q, cache, table, lengths, *, starts=None, scale=None, causal=True, window=0,
                    most_keys=None, lse=False, out=None, workspace=None):
    """Attention of new rows over a KvCache that holds their keys already
    (cache_write): rows starts[b] .. starts[b+1] - 1 of q (without `starts` row b)
    over the lengths[b] keys of sequence b, key j in page table[b][j / page].

    q [T][Hq][D] of the cache's dtype; the rest as in attention, but without
    most_keys a sequence is taken to be as long as the table has room for: pass it
    where the table is much wider than the sequences are long (in a captured graph,
    for the lengths that it will be replayed with).  A sequence whose table has no
    room for its keys gets NaN, and so does a row that sees a page that the cache
    does not have (and perhaps others of its sequence); table entries of pages that
    no row sees, as those that a window has left behind, may be anything."""
    if not isinstance(cache, KvCache):
        raise TypeError("cache must be a KvCache")
    if not isinstance(q, torch.Tensor) or q.dtype != cache.dtype:
        raise TypeError(f"q must be a tensor of {cache.dtype}")
    batch = _batch(starts, q.shape[0] if q.dim() else 0)
    values, out, tensors = _attention_rows(q, cache.kv_heads, starts, batch, scale, causal, window,
                                           most_keys, lse, out)
    if q.shape[2] != cache.width:
        raise ValueError(f"q must be [rows][heads][{cache.width}]")
    more, held = cache._values(table, lengths, batch)
    if not q.is_cuda:
        raise ValueError("the inputs must be on a GPU")
    _attend(_lib.lib().hv_paged_attention, "paged_attention", q, (*tensors, *held), _PAGED,
            values + more, batch, cache.kv_heads, workspace)
    return out


def _attend(entry, what, q, tensors, pack, values, batch, kv_heads, workspace):
    rows, heads, width = q.shape
    size = _lib.lib().hv_attention_workspace_bytes(rows, batch, heads, kv_heads, width)
    workspace, ws_at, ws_size = _workspace(workspace, size, q)
    _call(entry, what, q.get_device(), (*tensors, workspace), pack, values, ws_at, ws_size)
