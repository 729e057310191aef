"""Timing cases of the language-model operators on one MI355X.

Three operators that follow one another at the end of a language model's step
(the first two in each of its linear layers):

  norm     root-mean-square norm with the residual's addition, its output in 8
           bits with power-of-two scales (heatvit_amd.lm.rms_norm_q8)
  product  matrix product of e4m3 rows and weights with an exponent for each
           block of 128 (heatvit_amd.lm.gemm_f8)
  answer   log probabilities of given tokens, entropy and the most probable
           tokens (heatvit_amd.lm.log_probs)

With `own` false a pass is the plain form in elementary torch operations.
"""

import math

import torch

own = False

BLOCK = 128                 # columns that share an exponent
LARGEST = {"e4m3": 448.0, "int8": 127.0}
MIN_EXP = -127
EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32,
         "int32": torch.int32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4, "int32": 4}
LOGIT_EXP = -14             # exponent of the classifier's int32 logits

# What a drawn case may cost at most: the largest listed ones.
NORM_VALUES = 16384 * 8192
PRODUCT_MACS = 8192 ** 3
PRODUCT_VALUES = 50432 * 768
ANSWER_BYTES = 2048 * 131072 * 2


def listed():
    return [
        # one token of a decoding step
        {"name": "norm_token", "op": "norm", "rows": 1, "width": 4096, "type": "bf16",
         "format": "e4m3", "block": BLOCK, "residual": True},
        # the rows of a few packed sequences, a width that ends inside a block
        {"name": "norm_ragged", "op": "norm", "rows": 1003, "width": 1000, "type": "f32",
         "format": "e4m3", "block": BLOCK, "residual": False},
        # rows for the int8 product: one exponent a row
        {"name": "norm_int8_rows", "op": "norm", "rows": 4096, "width": 5120, "type": "f16",
         "format": "int8", "block": 0, "residual": True},
        # a long prompt
        {"name": "norm_prompt", "op": "norm", "rows": 16384, "width": 8192, "type": "bf16",
         "format": "e4m3", "block": BLOCK, "residual": True},
        # one token of a decoding step
        {"name": "product_token", "op": "product", "rows": 1, "inner": 4096, "width": 4096,
         "type": "bf16", "row_scale": True, "bias": False},
        # a decoding step of a small batch, into a wide layer
        {"name": "product_batch", "op": "product", "rows": 48, "inner": 4096, "width": 14336,
         "type": "bf16", "row_scale": True, "bias": False},
        # the tokens of 256 images into the model's hidden layer (inner size ends inside a block)
        {"name": "product_images", "op": "product", "rows": 50432, "inner": 192, "width": 768,
         "type": "bf16", "row_scale": False, "bias": True},
        # the logits of a ragged batch, in 32 bits
        {"name": "product_logits", "op": "product", "rows": 333, "inner": 2048, "width": 32001,
         "type": "f32", "row_scale": True, "bias": False},
        # a long prompt through a square layer
        {"name": "product_prompt", "op": "product", "rows": 8192, "inner": 8192, "width": 8192,
         "type": "bf16", "row_scale": True, "bias": False},
        # the classifier's int32 logits of one benchmark batch, with the five best classes
        {"name": "answer_images", "op": "answer", "rows": 256, "width": 1000, "type": "int32",
         "tokens": 1, "top": 5, "masked": False},
        # one token of a decoding step over a large vocabulary, with alternatives
        {"name": "answer_token", "op": "answer", "rows": 1, "width": 131072, "type": "bf16",
         "tokens": 1, "top": 20, "masked": False},
        # scoring a prompt: every position's next token
        {"name": "answer_prompt", "op": "answer", "rows": 2048, "width": 131072, "type": "bf16",
         "tokens": 1, "top": 5, "masked": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm", "product", "answer"))
    if op == "norm":
        width = _log_int(rng, 64, 16384)
        if rng.random() < 0.5:
            width = -(-width // 64) * 64
        rows = _log_int(rng, 1, min(65536, NORM_VALUES // width))
        form = rng.choice(("e4m3", "e4m3", "int8"))
        return {"op": op, "rows": rows, "width": width, "type": rng.choice(("bf16", "f16", "f32")),
                "format": form, "block": rng.choice((BLOCK, 0)), "residual": rng.random() < 0.7}
    if op == "product":
        inner = -(-_log_int(rng, 128, 8192) // 16) * 16
        width = _log_int(rng, 128, 16384)
        rows = _log_int(rng, 1, min(16384, PRODUCT_MACS // (inner * width),
                                    PRODUCT_VALUES // width))
        return {"op": op, "rows": rows, "inner": inner, "width": width,
                "type": rng.choice(("bf16", "f16", "f32")), "row_scale": rng.random() < 0.5,
                "bias": rng.random() < 0.5}
    kind = rng.choice(("bf16", "f16", "f32", "int32"))
    width = _log_int(rng, 1000, 262144)
    rows = _log_int(rng, 1, min(4096, ANSWER_BYTES // (SIZE[kind] * width)))
    return {"op": op, "rows": rows, "width": width, "type": kind, "tokens": rng.randint(1, 4),
            "top": rng.randint(0, 32), "masked": kind != "int32" and rng.random() < 0.3}


# ------------------------------------------------------------------ inputs

def _exps(p, block, largest):
    """Smallest e with max|p| <= largest * 2^e over each block of p's columns."""
    rows, width = p.shape
    block = block or width
    blocks = -(-width // block)
    a = torch.nn.functional.pad(p.abs(), (0, blocks * block - width))
    a = a.view(rows, blocks, block).amax(-1)
    m, k = torch.frexp(a)
    top = math.frexp(largest)
    e = k - top[1] + (m > top[0])
    return torch.where(a > 0, e.clamp(min=MIN_EXP), MIN_EXP).to(torch.int8)


def _spread(e, block, width):
    """2^e for every column."""
    s = torch.exp2(e.double())
    return s.repeat_interleave(block or width, dim=1)[:, :width]


def _quantised(p, block, form):
    e = _exps(p, block, LARGEST[form])
    q = (p * _spread(-e.int(), block, p.shape[1])).float()
    q = q.to(torch.float8_e4m3fn) if form == "e4m3" else torch.round(q).to(torch.int8)
    return q, e


def _activations(rows, width, gen):
    """Rows of a residual stream: normal values, some channels much larger."""
    dev = gen.device
    channel = torch.exp(torch.randn(width, device=dev, generator=gen) * 0.7)
    return torch.randn(rows, width, device=dev, generator=gen) * channel


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, rows, width = case["op"], case["rows"], case["width"]
    state = {"case": case}
    if op == "norm":
        dt = TYPES[case["type"]]
        state["x"] = _activations(rows, width, gen).to(dt)
        state["residual"] = ((4.0 * _activations(rows, width, gen)).to(dt) if case["residual"]
                             else None)
        state["weight"] = (1.0 + 0.2 * torch.randn(width, device="cuda", generator=gen)).to(dt)
    elif op == "product":
        inner = case["inner"]
        state["a"], state["a_exps"] = _quantised(_activations(rows, inner, gen), BLOCK, "e4m3")
        w = torch.randn(inner, width, device="cuda", generator=gen) / math.sqrt(inner)
        ki, ni = -(-inner // BLOCK), -(-width // BLOCK)
        flat = torch.nn.functional.pad(w, (0, ni * BLOCK - width, 0, ki * BLOCK - inner))
        flat = flat.view(ki, BLOCK, ni, BLOCK).permute(0, 2, 1, 3).reshape(ki * ni, BLOCK * BLOCK)
        w_exps = _exps(flat, 0, LARGEST["e4m3"]).view(ki, ni)
        w8 = (w * _weight_scale(-w_exps.int(), inner, width)).to(torch.float8_e4m3fn)
        state["row_scale"] = (torch.rand(rows, device="cuda", generator=gen) + 0.5
                              if case["row_scale"] else None)
        state["bias"] = (torch.randn(width, device="cuda", generator=gen) if case["bias"]
                         else None)
        state["w"], state["w_exps"] = w8, w_exps
        if own:  # a program lays its weights out once
            from heatvit_amd.device import DeviceF8Weight
            state["weight"] = DeviceF8Weight(w8, w_exps)
    else:
        kind = case["type"]
        x = torch.randn(rows, width, device="cuda", generator=gen) * 2.5
        # a few candidates stand out in each row
        at = torch.randint(0, width, (rows, 8), device="cuda", generator=gen)
        x.scatter_(1, at, torch.rand(rows, 8, device="cuda", generator=gen) * 8 + 6)
        if case["masked"]:  # tokens that a grammar forbids
            x.masked_fill_(torch.rand(1, width, device="cuda", generator=gen) < 0.2, -math.inf)
        if kind == "int32":
            x = torch.round(x * 2.0 ** -LOGIT_EXP)
        state["logits"] = x.to(TYPES[kind])
        tokens = torch.randint(0, width, (rows, case["tokens"]), device="cuda", generator=gen)
        tokens[:, 0] = at[:, 0]
        state["tokens"] = tokens.to(torch.int32)
        state["scale_exp"] = LOGIT_EXP if kind == "int32" else 0
    return state


# ------------------------------------------------------------------ one pass

def run(state):
    case = state["case"]
    if case["op"] == "norm":
        return _run_norm(state, case)
    if case["op"] == "product":
        return _run_product(state, case)
    return _run_answer(state, case)


def _run_norm(state, case):
    if own:
        from heatvit_amd import lm
        r = lm.rms_norm_q8(state["x"], state["weight"], residual=state["residual"], eps=EPS,
                           fmt=case["format"], block=case["block"])
        out = {"q": r.q, "exps": r.exps, "scale": r.scale}
        if case["residual"]:
            out["residual"] = r.residual
        return out
    h = state["x"]
    if case["residual"]:
        h = (h.float() + state["residual"].float()).to(h.dtype)
    hf = h.float()
    p = hf * state["weight"].float()
    e = _exps(p, case["block"], LARGEST[case["format"]])
    q = p * _spread(-e.int(), case["block"], case["width"]).float()
    q = q.to(torch.float8_e4m3fn) if case["format"] == "e4m3" else torch.round(q).to(torch.int8)
    out = {"q": q, "exps": e, "scale": torch.rsqrt((hf * hf).mean(-1) + EPS)}
    if case["residual"]:
        out["residual"] = h
    return out


def _weight_scale(e, inner, width):
    """2^e of a weight's 128 x 128 blocks, for every element."""
    s = torch.exp2(e.double()).float()
    return s.repeat_interleave(BLOCK, 0)[:inner].repeat_interleave(BLOCK, 1)[:, :width]


def _run_product(state, case):
    dt = TYPES[case["type"]]
    if own:
        from heatvit_amd import lm
        return lm.gemm_f8(state["a"], state["a_exps"], state["weight"], row_scale=state["row_scale"],
                          bias=state["bias"], out_dtype=dt)
    inner, width = case["inner"], case["width"]
    a = state["a"].float() * _spread(state["a_exps"], BLOCK, inner).float()
    w = state["w"].float() * _weight_scale(state["w_exps"], inner, width)
    y = a @ w
    if case["row_scale"]:
        y = y * state["row_scale"][:, None]
    if case["bias"]:
        y = y + state["bias"]
    return y.to(dt)


def _ordered(x):
    """64-bit keys whose order is the value's, equal values by the lower index."""
    if x.dtype == torch.int32:
        v = x.long()
    else:
        b = (x.float() + 0.0).view(torch.int32)  # one zero
        v = torch.where(b < 0, b ^ 0x7FFFFFFF, b).long()
    return v * (1 << 32) - torch.arange(x.shape[1], device=x.device)


def _run_answer(state, case):
    logits, tokens, top = state["logits"], state["tokens"], case["top"]
    if own:
        from heatvit_amd import lm
        r = lm.log_probs(logits, tokens, scale_exp=state["scale_exp"], top=top)
        out = {"logp": r.logp, "entropy": r.entropy}
        if top:
            out["top_logp"], out["top_index"] = r.top_logp, r.top_index
        return out
    # int32 logits less their maximum are exact in 64 bits only
    x = logits.double() if logits.dtype == torch.int32 else logits.float()
    x = x * 2.0 ** state["scale_exp"]
    d = x - x.amax(-1, keepdim=True)
    e = torch.exp(d)
    total = e.sum(-1)
    log_total = torch.log(total)
    weighted = torch.where(e > 0, e * d, 0.0).sum(-1)
    out = {"logp": (d.gather(1, tokens.long()) - log_total[:, None]).float(),
           "entropy": (log_total - weighted / total).float()}
    if top:
        at = torch.topk(_ordered(logits), top).indices
        out["top_logp"] = (d.gather(1, at) - log_total[:, None]).float()
        out["top_index"] = at.to(torch.int32)
    return out


# ------------------------------------------------------------------ what it costs and gives

def work(case):
    rows, width, s = case["rows"], case["width"], SIZE[case["type"]]
    if case["op"] == "norm":
        blocks = -(-width // (case["block"] or width))
        streams = 3 if case["residual"] else 1
        return {"bytes": rows * width * (s * streams + 1) + rows * (blocks + 4) + width * s,
                "flops": 6 * rows * width}
    if case["op"] == "product":
        inner = case["inner"]
        ki, ni = -(-inner // BLOCK), -(-width // BLOCK)
        extra = 4 * rows * case["row_scale"] + 4 * width * case["bias"]
        return {"bytes": rows * (inner + ki) + inner * width + ki * ni + rows * width * s + extra,
                "flops": 2 * rows * inner * width}
    return {"bytes": rows * width * s + rows * (8 * case["tokens"] + 4 + 8 * case["top"]),
            "flops": 8 * rows * width}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "norm":
        h = state["x"].double()
        given = None
        if case["residual"]:
            given = h + state["residual"].double()
            h = given.to(state["x"].dtype).double()  # the residual that is kept
        p = h * state["weight"].double()
        e = _exps(p.float(), case["block"], LARGEST[case["format"]])
        q = p * _spread(-e.int(), case["block"], case["width"])
        out = {"q": q if case["format"] == "e4m3" else None, "exps": None,
               "scale": 1.0 / torch.sqrt(h.square().mean(-1) + EPS)}
        if case["residual"]:
            out["residual"] = given
        return out
    if case["op"] == "product":
        inner, width = case["inner"], case["width"]
        w = state["w"].double() * _weight_scale(state["w_exps"], inner, width).double()
        y = (state["a"].double() * _spread(state["a_exps"], BLOCK, inner)) @ w
        if case["row_scale"]:
            y *= state["row_scale"].double()[:, None]
        if case["bias"]:
            y += state["bias"].double()
        return y
    x = state["logits"].double() * 2.0 ** state["scale_exp"]
    log_p = x - torch.logsumexp(x, -1, keepdim=True)
    p = torch.exp(log_p)
    out = {"logp": log_p.gather(1, state["tokens"].long()),
           "entropy": -torch.where(p > 0, p * log_p, 0.0).sum(-1)}
    if case["top"]:
        out["top_logp"], out["top_index"] = torch.topk(log_p, case["top"]).values, None
    return out
