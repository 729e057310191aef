"""Timing cases of a language model's attention on one MI355X: what lies between
the product that makes queries, keys and values and the one behind the attention.

  rotary  norms of queries and keys for each head with the rotation by their
          positions in the same pass (heatvit_amd.lm.rotary_qk)
  write   keys and values into the pages of a cache, in 16 bits or in e4m3 with
          a power-of-two scale for each head of each token
          (heatvit_amd.lm.cache_write)
  prompt  attention over packed sequences with grouped heads
          (heatvit_amd.lm.attention)
  chunk   attention of one or more new tokens of each sequence over such a cache
          (heatvit_amd.lm.paged_attention)

With `own` false a pass is the plain form in elementary torch operations.
"""

import math
import random

import torch

own = False

LARGEST = 448.0     # of e4m3
MIN_EXP = -127
EPS = 1e-6
BASE = 10000.0
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}

# What a drawn case may cost at most: the largest listed ones.
ROTARY_VALUES = 16384 * 40 * 128
WRITE_VALUES = 16384 * 8 * 128
SCORES = 8 * 32 * 4000 * 4000          # of the plain form, padded to the longest
PAIRS = 32 * 8192 * 8192 * 128 // 2    # visible pairs by head width
CACHE_VALUES = 64 * 1700 * 8 * 128     # of keys, as of values


def listed():
    return [
        # one token of a decoding step
        {"name": "rotary_token", "op": "rotary", "rows": 1, "heads": 32, "kv_heads": 8,
         "width": 128, "rotated": 128, "type": "bf16", "layout": "half", "norm": True,
         "factor": 1.0, "far": 8192},
        # packed sequences: part of an odd head rotated, positions far behind, in 32 bits
        {"name": "rotary_ragged", "op": "rotary", "rows": 1003, "heads": 20, "kv_heads": 20,
         "width": 100, "rotated": 50, "type": "f32", "layout": "interleaved", "norm": False,
         "factor": 4.0, "far": 1000000},
        # a long prompt
        {"name": "rotary_prompt", "op": "rotary", "rows": 16384, "heads": 32, "kv_heads": 8,
         "width": 128, "rotated": 128, "type": "bf16", "layout": "half", "norm": True,
         "factor": 8.0, "far": 131072},
        # the new tokens of a decoding step of a batch
        {"name": "write_step", "op": "write", "sequences": 64, "tokens": 1, "keys": 4096,
         "ragged": True, "kv_heads": 8, "width": 128, "type": "bf16", "format": "e4m3",
         "page": 64},
        # a long prompt
        {"name": "write_prompt", "op": "write", "sequences": 4, "tokens": 4096, "keys": 4096,
         "ragged": False, "kv_heads": 8, "width": 128, "type": "bf16", "format": "e4m3",
         "page": 64},
        # the tokens of one benchmark batch of images, every token seeing every other
        {"name": "prompt_images", "op": "prompt", "sequences": 256, "tokens": 197,
         "ragged": False, "heads": 3, "kv_heads": 3, "width": 64, "type": "f16",
         "causal": False, "window": 0, "lse": False},
        # prompts of very different lengths in one call
        {"name": "prompt_ragged", "op": "prompt", "sequences": 8, "tokens": 4000,
         "ragged": True, "heads": 32, "kv_heads": 8, "width": 128, "type": "bf16",
         "causal": True, "window": 0, "lse": True},
        # a long prompt
        {"name": "prompt_long", "op": "prompt", "sequences": 1, "tokens": 8192,
         "ragged": False, "heads": 32, "kv_heads": 8, "width": 128, "type": "bf16",
         "causal": True, "window": 0, "lse": False},
        # a decoding step of a few short sequences, small pages, a head to itself
        {"name": "chunk_step", "op": "chunk", "sequences": 8, "tokens": 1, "keys": 1000,
         "ragged": True, "heads": 16, "kv_heads": 16, "width": 64, "type": "f16",
         "format": "same", "page": 16, "window": 0, "lse": False},
        # a decoding step of a batch over a large cache
        {"name": "chunk_batch", "op": "chunk", "sequences": 64, "tokens": 1, "keys": 16384,
         "ragged": True, "heads": 32, "kv_heads": 8, "width": 128, "type": "bf16",
         "format": "same", "page": 64, "window": 0, "lse": False},
        # one token over a long cache in 8 bits
        {"name": "chunk_token", "op": "chunk", "sequences": 1, "tokens": 1, "keys": 32768,
         "ragged": False, "heads": 32, "kv_heads": 8, "width": 128, "type": "bf16",
         "format": "e4m3", "page": 64, "window": 0, "lse": False},
        # the next pieces of a few prompts over what the cache holds of them, in 8 bits
        {"name": "chunk_prompt", "op": "chunk", "sequences": 4, "tokens": 512, "keys": 16384,
         "ragged": True, "heads": 32, "kv_heads": 8, "width": 128, "type": "bf16",
         "format": "e4m3", "page": 64, "window": 0, "lse": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def _heads(rng, most):
    kv = rng.choice((1, 2, 3, 4, 8, 12, 16))
    return min(kv * rng.choice((1, 1, 2, 4, 5, 8)), max(most // kv, 1) * kv), kv


def draw(rng):
    op = rng.choice(("rotary", "write", "prompt", "chunk"))
    if op == "rotary":
        heads, kv = _heads(rng, 64)
        width = 2 * _log_int(rng, 16, 128)
        rotated = rng.choice((width, width, 2 * rng.randint(1, width // 2)))
        return {"op": op, "rows": _log_int(rng, 1, min(32768, ROTARY_VALUES // ((heads + kv) * width))),
                "heads": heads, "kv_heads": kv, "width": width, "rotated": rotated,
                "type": rng.choice(("bf16", "f16", "f32")),
                "layout": rng.choice(("half", "interleaved")), "norm": rng.random() < 0.5,
                "factor": rng.choice((1.0, 4.0, 32.0)), "far": _log_int(rng, 1000, 1000000)}
    width = 16 * _log_int(rng, 2, 16)
    if op == "write":
        _, kv = _heads(rng, 64)
        sequences = _log_int(rng, 1, 256)
        most = max(1, WRITE_VALUES // (sequences * kv * width))
        tokens = _log_int(rng, 1, min(8192, most))
        return {"op": op, "sequences": sequences, "tokens": tokens,
                "keys": tokens + rng.randint(0, min(4096, 8 * most)), "ragged": rng.random() < 0.6,
                "kv_heads": kv, "width": width, "type": rng.choice(("bf16", "f16")),
                "format": rng.choice(("same", "e4m3")), "page": rng.choice((16, 32, 64, 128, 256))}
    heads, kv = _heads(rng, 64)
    sequences = _log_int(rng, 1, 128)
    common = {"op": op, "sequences": sequences, "ragged": rng.random() < 0.6, "heads": heads,
              "kv_heads": kv, "width": width, "type": rng.choice(("bf16", "f16")),
              "lse": rng.random() < 0.3}
    window = rng.choice((0, 0, 0, rng.randint(1, 1500)))
    if op == "prompt":
        most = math.isqrt(min(SCORES // (sequences * heads), PAIRS // (sequences * heads * width)))
        causal = rng.random() < 0.8
        return {**common, "tokens": _log_int(rng, 1, min(8192, most)), "causal": causal,
                "window": window if causal else 0}
    keys = _log_int(rng, 16, min(65536, max(16, CACHE_VALUES // (sequences * kv * width))))
    most = min(PAIRS // (keys * sequences * heads * width), SCORES // (keys * sequences * heads))
    tokens = rng.choice((1, _log_int(rng, 1, max(1, min(2048, keys, most)))))
    return {**common, "tokens": tokens, "keys": keys, "window": window,
            "format": rng.choice(("same", "e4m3")), "page": rng.choice((16, 32, 64, 128, 256))}


# ------------------------------------------------------------------ inputs

def _spread(largest, count, ragged):
    """`count` lengths up to `largest`: all the same, or even over their logarithm."""
    if not ragged:
        return [largest] * count
    return [max(1, int(round(largest ** ((i + 1) / count)))) for i in range(count)]


def _lengths(case, seed=0):
    """(new tokens, keys) of every sequence, in the order that the seed gives."""
    count, ragged = case["sequences"], case["ragged"]
    new = _spread(case["tokens"], count, ragged)
    keys = [max(n, k) for n, k in zip(new, _spread(case["keys"], count, ragged))] \
        if "keys" in case else new
    order = list(range(count))
    random.Random(seed).shuffle(order)
    return [new[i] for i in order], [keys[i] for i in order]


def _starts(lengths):
    s = [0]
    for n in lengths:
        s.append(s[-1] + n)
    return torch.tensor(s, dtype=torch.int32, device="cuda")


def _row_exps(x):
    """Smallest e >= -127 with max|x| <= 448 2^e of each row (last dimension)."""
    a = x.abs().amax(-1)
    m, k = torch.frexp(a)
    top = math.frexp(LARGEST)
    return torch.where(a > 0, (k - top[1] + (m > top[0])).clamp(min=MIN_EXP), MIN_EXP).to(torch.int8)


def _scale(exps):
    return torch.exp2(exps.double())[..., None]


def _in_8_bits(x):
    e = _row_exps(x)
    return (x.float() * _scale(-e.int()).float()).to(torch.float8_e4m3fn), e


def _heads_of(shape, dtype, gen):
    """Values of heads, some channels larger than others."""
    channel = torch.exp(0.4 * torch.randn(shape[-1], device="cuda", generator=gen))
    channel /= channel.square().mean().sqrt()
    return (torch.randn(shape, device="cuda", generator=gen) * channel).to(dtype)


def _cache(state, case, lengths, gen):
    """Pages of keys and values, and which pages each sequence has."""
    page, kv, width = case["page"], case["kv_heads"], case["width"]
    counts = [-(-n // page) for n in lengths]
    pages = sum(counts) + 2
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    table = torch.full((len(counts), max(counts)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = order[at:at + n]
        at += n
    state["table"] = table
    state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for name in ("k", "v"):
        x = _heads_of((pages, kv, page, width), TYPES[case["type"]], gen)
        exps = None
        if case["format"] == "e4m3":
            x, exps = _in_8_bits(x)
        state["cache_" + name], state["cache_" + name + "_exps"] = x, exps
    if own:  # the handle that a program keeps
        from heatvit_amd import lm
        state["cache"] = lm.KvCache(state["cache_k"], state["cache_v"], state["cache_k_exps"],
                                    state["cache_v_exps"], dtype=TYPES[case["type"]])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, dt, width = case["op"], TYPES[case["type"]], case["width"]
    state = {"case": case}
    if op == "rotary":
        rows, half = case["rows"], case["rotated"] // 2
        state["q"] = _heads_of((rows, case["heads"], width), dt, gen)
        state["k"] = _heads_of((rows, case["kv_heads"], width), dt, gen)
        first = random.Random(seed).randint(0, case["far"])
        state["positions"] = torch.arange(first, first + rows, dtype=torch.int32, device="cuda")
        # long contexts: the slow half of the frequencies slowed down further
        i = torch.arange(half, dtype=torch.float64)
        f = BASE ** (-i / half)
        state["freqs"] = torch.where(2 * i < half, f, f / case["factor"]).float().cuda()
        state["scale"] = 1.0 + 0.1 * math.log(case["factor"])
        for name in ("q_weight", "k_weight"):
            state[name] = ((1.0 + 0.2 * torch.randn(width, device="cuda", generator=gen)).to(dt)
                           if case["norm"] else None)
        return state
    new, keys = _lengths(case, seed)
    rows = sum(new)
    state["starts"] = _starts(new)
    if op == "write":
        state["k"] = _heads_of((rows, case["kv_heads"], width), dt, gen)
        state["v"] = _heads_of((rows, case["kv_heads"], width), dt, gen)
        _cache(state, case, keys, gen)
        return state
    state["most"] = max(new), max(keys)  # the program knows its longest sequence
    state["q"] = _heads_of((rows, case["heads"], width), dt, gen)
    if op == "prompt":
        state["k"] = _heads_of((rows, case["kv_heads"], width), dt, gen)
        state["v"] = _heads_of((rows, case["kv_heads"], width), dt, gen)
    else:
        _cache(state, case, keys, gen)
    return state


# ------------------------------------------------------------------ one pass

def run(state):
    case = state["case"]
    return {"rotary": _run_rotary, "write": _run_write, "prompt": _run_prompt,
            "chunk": _run_chunk}[case["op"]](state, case)


def _run_rotary(state, case):
    if own:
        from heatvit_amd import lm
        r = lm.rotary_qk(state["q"], state["k"], state["positions"], state["freqs"],
                         q_weight=state["q_weight"], k_weight=state["k_weight"], eps=EPS,
                         layout=case["layout"], scale=state["scale"])
        return {"q": r.q, "k": r.k}
    angle = state["positions"].double()[:, None] * state["freqs"].double()
    cos = (torch.cos(angle) * state["scale"]).float()[:, None]
    sin = (torch.sin(angle) * state["scale"]).float()[:, None]
    return {"q": _rotated(state["q"], state["q_weight"], cos, sin, case),
            "k": _rotated(state["k"], state["k_weight"], cos, sin, case)}


def _rotated(x, weight, cos, sin, case):
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * weight.float()
    n = case["rotated"]
    if case["layout"] == "half":
        a, b = y[..., :n // 2], y[..., n // 2:n]
        r = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    else:
        a, b = y[..., 0:n:2], y[..., 1:n:2]
        r = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    return torch.cat((r, y[..., n:]), -1).to(x.dtype)


def _rows_of(starts, rows):
    """(sequence, place in it) of every packed row."""
    at = torch.arange(rows, device="cuda")
    b = torch.searchsorted(starts, at, right=True) - 1
    return b, at - starts.long()[b]


def _run_write(state, case):
    out = {}
    if own:
        from heatvit_amd import lm
        lm.cache_write(state["cache"], state["k"], state["v"], state["table"], state["lengths"],
                       starts=state["starts"])
    else:
        rows, page, starts = state["k"].shape[0], case["page"], state["starts"].long()
        b, i = _rows_of(state["starts"], rows)
        position = state["lengths"].long()[b] - (starts[1:] - starts[:-1])[b] + i
        at = state["table"].long()[b, position // page], slice(None), position % page
        for name in ("k", "v"):
            cache, exps = state["cache_" + name], state["cache_" + name + "_exps"]
            x = state[name]
            if exps is not None:
                x, exps[at] = _in_8_bits(x)
                x, cache = x.view(torch.uint8), cache.view(torch.uint8)
            cache[at] = x
    for name in ("k", "v"):
        out[name], out[name + "_exps"] = state["cache_" + name], state["cache_" + name + "_exps"]
    return out


def _run_prompt(state, case):
    if own:
        from heatvit_amd import lm
        r = lm.attention(state["q"], state["k"], state["v"], state["starts"],
                         causal=case["causal"], window=case["window"], lse=case["lse"])
        return _answer(r.out, r.lse, case)
    starts = state["starts"].long()
    n = starts[1:] - starts[:-1]
    at = torch.arange(state["most"][1], device="cuda").minimum(n[:, None] - 1) + starts[:-1, None]
    return _attended(state, case, state["k"].float()[at], state["v"].float()[at], n)


def _run_chunk(state, case):
    if own:
        from heatvit_amd import lm
        r = lm.paged_attention(state["q"], state["cache"], state["table"], state["lengths"],
                               starts=state["starts"], window=case["window"], lse=case["lse"])
        return _answer(r.out, r.lse, case)
    return _attended(state, case, _gathered(state, case, "k"), _gathered(state, case, "v"),
                     state["lengths"].long())


def _gathered(state, case, name):
    """[sequence][key][head][width] of a cache, in 32 bits."""
    cache, exps = state["cache_" + name], state["cache_" + name + "_exps"]
    table = state["table"].long().clamp(min=0)
    if exps is None:
        x = cache[table].float()
    else:
        x = cache.view(torch.uint8)[table].view(torch.float8_e4m3fn).float()
        x *= _scale(exps[table].int()).float()
    b, pages, heads, page, width = x.shape
    return x.transpose(2, 3).reshape(b, pages * page, heads, width)[:, :state["most"][1]]


def _attended(state, case, k, v, keys):
    """The attention of rows padded to the longest sequence."""
    q, starts = state["q"], state["starts"].long()
    n = starts[1:] - starts[:-1]
    count, most, kv, width = len(n), state["most"][0], case["kv_heads"], case["width"]
    group = case["heads"] // kv
    i = torch.arange(most, device="cuda")
    padded = q.float()[i.minimum(n[:, None] - 1) + starts[:-1, None]]
    padded = padded.view(count, most, kv, group, width).permute(0, 2, 3, 1, 4)
    j = torch.arange(k.shape[1], device="cuda")
    last = (keys - n)[:, None] + i if case.get("causal", True) else (keys - 1)[:, None] + 0 * i
    last = last.minimum((keys - 1)[:, None])
    seen = j <= last[..., None]
    if case["window"]:
        seen &= j > last[..., None] - case["window"]
    s = padded.reshape(count, kv, group * most, width) @ k.permute(0, 2, 3, 1).contiguous()
    s = s.view(count, kv, group, most, -1).mul_(1.0 / math.sqrt(width))
    s.masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    s.sub_(top).exp_()
    total = s.sum(-1)
    o = s.view(count, kv, group * most, -1) @ v.transpose(1, 2).contiguous()
    o = o.view(count, kv, group, most, width) / total[..., None]
    b, i = _rows_of(state["starts"], len(q))
    out = o.permute(0, 3, 1, 2, 4).reshape(count, most, kv * group, width)[b, i].to(q.dtype)
    lse = (top[..., 0] + torch.log(total)).permute(0, 3, 1, 2).reshape(count, most, -1)[b, i]
    return _answer(out, lse, case)


def _answer(out, lse, case):
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}


# ------------------------------------------------------------------ what it costs and gives

def work(case):
    s, width = SIZE[case["type"]], case["width"]
    if case["op"] == "rotary":
        heads, rows = case["heads"] + case["kv_heads"], case["rows"]
        return {"bytes": rows * (2 * heads * width * s + 4) + 2 * case["rotated"] +
                (2 * width * s if case["norm"] else 0),
                "flops": rows * heads * (3 * case["rotated"] + (4 * width if case["norm"] else 0))}
    new, keys = _lengths(case)
    kv, rows = case["kv_heads"], sum(new)
    held = width + 1 if case.get("format") == "e4m3" else width * s
    if case["op"] == "write":
        return {"bytes": 2 * rows * kv * (width * s + held), "flops": 4 * rows * kv * width}
    window, seen, read = case["window"], 0, 0
    for n, k in zip(new, keys):
        if case.get("causal", True):
            # row i sees k - n + i + 1 keys, at most the window
            full = k - n
            short = n if not window else max(0, min(n, window - full))
            seen += short * full + short * (short + 1) // 2 + (n - short) * window
            read += min(k, window + n - 1) if window else k
        else:
            seen += n * k
            read += k
    return {"bytes": rows * case["heads"] * (2 * width * s + 4 * case["lse"]) +
            2 * read * kv * held, "flops": 4 * seen * case["heads"] * width}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rotary":
        turn = torch.polar(torch.full_like(state["freqs"], state["scale"]).double() *
                           torch.ones_like(state["positions"]).double()[:, None],
                           state["positions"].double()[:, None] * state["freqs"].double())
        out = {}
        for name in ("q", "k"):
            y, n = state[name].double(), case["rotated"]
            if case["norm"]:
                y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + EPS)
                y = y * state[name + "_weight"].double()
            if case["layout"] == "half":
                z = torch.complex(y[..., :n // 2].clone(), y[..., n // 2:n].clone())
            else:
                z = torch.view_as_complex(y[..., :n].reshape(*y.shape[:2], n // 2, 2).contiguous())
            z = z * turn[:, None]
            pairs = torch.cat((z.real, z.imag), -1) if case["layout"] == "half" else \
                torch.view_as_real(z).flatten(-2)
            out[name] = torch.cat((pairs, y[..., n:]), -1)
        return out
    new, keys = _lengths(case, seed)
    if case["op"] == "write":
        out = {}
        for name in ("k", "v"):
            cache, exps = state["cache_" + name].double(), state["cache_" + name + "_exps"]
            row = 0
            for b, (n, k) in enumerate(zip(new, keys)):
                x = state[name][row:row + n].double()
                if exps is not None:
                    x = x * _scale(-_row_exps(x).int())
                place = torch.arange(k - n, k, device="cuda")
                cache[state["table"][b].long()[place // case["page"]], :,
                      place % case["page"]] = x
                row += n
            out[name], out[name + "_exps"] = cache, None
        return out
    out, lse, row = [], [], 0
    group, scale = case["heads"] // case["kv_heads"], 1.0 / math.sqrt(case["width"])
    if sum(n * k for n, k in zip(new, keys)) * case["heads"] > 1 << 33:
        return None
    for b, (n, k) in enumerate(zip(new, keys)):
        if case["op"] == "prompt":
            both = [state[name][row:row + n].double() for name in ("k", "v")]
        else:
            at = state["table"][b, :-(-k // case["page"])].long()
            both = []
            for name in ("k", "v"):
                x, exps = state["cache_" + name], state["cache_" + name + "_exps"]
                x = torch.stack([x[p] for p in at.tolist()]).double()
                if exps is not None:
                    x = x * _scale(exps[at].int())
                both.append(x.transpose(1, 2).flatten(0, 1)[:k])
        place = torch.arange(k, device="cuda")
        me = torch.arange(k - n, k, device="cuda")[:, None]
        seen = torch.ones(n, k, dtype=torch.bool, device="cuda")
        if case.get("causal", True):
            seen = place <= me
            if case["window"]:
                seen &= place > me - case["window"]
        o, l = [], []
        for h in range(case["heads"]):
            s = state["q"][row:row + n, h].double() @ both[0][:, h // group].t().contiguous()
            s = torch.where(seen, s * scale, -math.inf)
            l.append(torch.logsumexp(s, -1))
            o.append(torch.softmax(s, -1) @ both[1][:, h // group])
        out.append(torch.stack(o, 1))
        lse.append(torch.stack(l, 1))
        row += n
    return _answer(torch.cat(out), torch.cat(lse), case)
