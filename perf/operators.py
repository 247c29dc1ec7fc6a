"""What the decoding operators compute, in plain torch, and the calls that
reach the framework's kernels for them.

Three operators, as a program uses them one after the other behind a prefill:

* ``rotary``: rotary positions of queries and keys (``Rotary``), forward and
  backward;
* ``cache``: keys and values quantised into a paged cache as they are
  written, and read back (``KvCache.write`` / ``KvCache.read``);
* ``tree``: attention of the newest tokens -- one per sequence, or a tree of
  drafted ones -- over that cache (``tree_attention``).

A case says which operator, its sizes and its types.  ``run`` makes the plain
computation where ``own`` is false and the framework's call where it is true.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
SMALLEST_SCALE = 2.0 ** -96


# ---- cases -----------------------------------------------------------------------------------------


def _rotary(name, **kw):
    return dict({"name": name, "op": "rotary", "b": 1, "t": 1, "hq": 32, "hkv": 8, "d": 128, "r": 128, "far": 131072, "layout": "half",
                 "scaling": "none", "type": "bf16", "grad": False}, **kw)


def _cache(name, **kw):
    return dict({"name": name, "op": "cache", "b": 1, "t": 1, "hkv": 8, "d": 128, "page": 16, "fmt": "int8", "type": "bf16", "start": 0}, **kw)


def _tree(name, **kw):
    return dict({"name": name, "op": "tree", "b": 1, "t": 1, "ctx": 1024, "hq": 32, "hkv": 8, "d": 128, "page": 16, "fmt": "bf16",
                 "bias": False, "mask": "none"}, **kw)


def listed():
    return [
        # one decoding step of 64 sequences: the latency of a call
        _rotary("rotary_decode_64", b=64, scaling="llama3"),
        # a prefill chunk of a long context behind 98304 earlier tokens
        _rotary("rotary_prefill_32k", t=32768, scaling="yarn"),
        # a training step: forward and gradient, half of each head rotated, in 32 bits, odd length
        _rotary("rotary_train_4097", b=2, t=4097, d=128, r=64, layout="interleaved", type="f32", far=4097, grad=True),
        # one decoding step of 64 sequences goes into the cache
        _cache("cache_append_64", b=64, start=4095),
        # a block of 16384 tokens and one more go into the cache after their prefill
        _cache("cache_prefill_16385", t=16385, fmt="e4m3", page=64),
        # three prompts of a model with 64-wide heads, from 32-bit projections
        _cache("cache_prompts_f32", b=3, t=1000, hkv=4, d=64, type="f32", start=77),
        # one user's next token after a short prompt: latency
        _tree("tree_decode_1k", ctx=1000),
        # a server's step: 64 sequences of up to 8192 tokens in 8 bits
        _tree("tree_decode_64x8k", b=64, ctx=8191, fmt="int8"),
        # one user's next token at the full context
        _tree("tree_decode_128k", ctx=131071, fmt="e4m3", page=64),
        # drafted trees of 13 tokens for 16 sequences
        _tree("tree_draft_16x13", b=16, t=13, ctx=4001, fmt="int8", mask="tree"),
        # a wide tree of 64 drafted tokens at the full context, unquantised
        _tree("tree_wide_128k", t=64, ctx=131072, page=64, mask="tree"),
        # after the DCC-KV layer: seven compact blocks of 1024 keys with their logit bias and a local block, a chain of 8
        _tree("tree_compact_7x1k", t=8, ctx=7 * 1024 + 16384, bias=True),
    ]


def _size(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng: random.Random):
    op = rng.choice(["rotary", "cache", "tree", "tree"])
    d = rng.choice([64, 96, 128, 128])
    hkv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 8])
    if op == "rotary":
        grad = rng.random() < 0.4
        b = _size(rng, 1, 64)
        t = _size(rng, 1, max(1, 16384 // b))
        return dict(_rotary("", b=b, t=t, hq=hkv * group, hkv=hkv, d=d, r=rng.choice([d, d, d // 2]), far=max(t, _size(rng, 1024, 1 << 20)),
                            layout=rng.choice(["half", "interleaved"]), scaling=rng.choice(["none", "linear", "ntk", "yarn", "llama3"]),
                            type=rng.choice(["bf16", "f32"]), grad=grad))
    if op == "cache":
        b = _size(rng, 1, 128)
        return _cache("", b=b, t=_size(rng, 1, max(1, 16384 // b)), hkv=hkv, d=d, page=rng.choice([8, 16, 32, 64, 128]),
                      fmt=rng.choice(["int8", "e4m3", "bf16"]), type=rng.choice(["bf16", "bf16", "f32"]), start=rng.randrange(0, 5000))
    b = _size(rng, 1, 64)
    t = rng.choice([1, 1, _size(rng, 2, 64)])
    most = 131072 * 2048 // (b * max(2048, t * hkv * group))
    return _tree("", b=b, t=t, ctx=_size(rng, 64, max(64, most)), hq=hkv * group, hkv=hkv, d=d, page=rng.choice([8, 16, 32, 64, 128]),
                 fmt=rng.choice(["bf16", "int8", "e4m3"]), bias=rng.random() < 0.25, mask="tree" if t > 1 and rng.random() < 0.7 else "none")


def _lengths(case):
    """The tokens of each sequence before the newest: from half of ``ctx`` (rounded down) to all of it."""
    b, ctx = case["b"], case["ctx"]
    return [ctx - (i * (ctx - ctx // 2)) // max(1, b - 1) if b > 1 else ctx for i in range(b)]


# ---- inputs ----------------------------------------------------------------------------------------


def _values(g, shape, dtype):
    """Keys or values as a model has them: normal, with four channels eight times as large."""
    x = torch.randn(*shape, generator=g, device=DEV)
    x[..., torch.randperm(shape[-1], generator=g, device=DEV)[:4]] *= 8
    return x.to(dtype)


def _scaling(case):
    return {"none": None,
            "linear": {"rope_type": "linear", "factor": 4.0},
            "ntk": {"rope_type": "ntk", "factor": 4.0},
            "yarn": {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 8192, "beta_fast": 32.0, "beta_slow": 1.0},
            "llama3": {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
                       "original_max_position_embeddings": 8192}}[case["scaling"]]


THETA = 500000.0


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": case}
    if case["op"] == "rotary":
        b, t, dt = case["b"], case["t"], TYPES[case["type"]]
        s["q"] = torch.randn(b, case["hq"], t, case["d"], generator=g, device=DEV).to(dt).requires_grad_(case["grad"])
        s["k"] = _values(g, (b, case["hkv"], t, case["d"]), dt).requires_grad_(case["grad"])
        first = torch.randint(0, case["far"] - t + 1, (b, 1), generator=g, device=DEV)
        s["positions"] = first + torch.arange(t, device=DEV)
        if case["grad"]:
            s["gq"], s["gk"] = (torch.randn(x.shape, generator=g, device=DEV).to(dt) for x in (s["q"], s["k"]))
        if own:  # the handle that a program keeps
            import dcc_kv_b200 as dk
            s["rotary"] = dk.Rotary(case["d"], rotary_dim=case["r"], theta=THETA, layout=case["layout"], scaling=_scaling(case))
        return s
    h, d, page, b = case["hkv"], case["d"], case["page"], case["b"]
    tokens = case["t"] + (case["start"] if case["op"] == "cache" else case["ctx"])
    per = -(-tokens // page)
    s["page_table"] = torch.randperm(b * per, generator=g, device=DEV).to(torch.int32).view(b, per)
    n = b * per
    if case["op"] == "cache":
        dt = TYPES[case["type"]]
        s["k"], s["v"] = (_values(g, (b, h, case["t"], d), dt) for _ in range(2))
        s["start"] = torch.full((b,), case["start"], dtype=torch.int32, device=DEV)
        code = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn, "bf16": torch.bfloat16}[case["fmt"]]
        s["pages"] = {x: torch.zeros(n, h, page, d, dtype=torch.int8 if case["fmt"] == "e4m3" else code, device=DEV).view(code) for x in "kv"}
        if case["fmt"] != "bf16":
            s["pages"].update({x + "_scale": torch.zeros(n, h, page, device=DEV) for x in "kv"})
    else:
        s["q"] = torch.randn(b, case["hq"], case["t"], d, generator=g, device=DEV).to(torch.bfloat16)
        s["pages"] = {}
        for x in "kv":
            codes, scale = _quantise(_values(g, (n, h, page, d), torch.bfloat16), case["fmt"])
            s["pages"][x] = codes
            if scale is not None:
                s["pages"][x + "_scale"] = scale
            del codes, scale
        if case["bias"]:
            s["pages"]["logit_bias"] = torch.randn(n, h, page, generator=g, device=DEV)
        s["context_lens"] = torch.tensor(_lengths(case), dtype=torch.int32, device=DEV)
        s["tree"] = None
        if case["mask"] == "tree":
            r, t = random.Random(seed), case["t"]
            sees = [[False] * t for _ in range(t)]
            for i in range(t):
                parent = r.randrange(-1, i) if i else -1
                sees[i] = list(sees[parent]) if parent >= 0 else [False] * t
                sees[i][i] = True
            s["tree"] = torch.tensor(sees, device=DEV)
    if own:
        import dcc_kv_b200 as dk
        s["cache"] = dk.KvCache(**s["pages"])
    return s


# ---- plain forms -----------------------------------------------------------------------------------


def _frequencies(case):
    """Radians per position of each pair, and the factor on the result."""
    r, scaling = case["r"], _scaling(case) or {"rope_type": "none"}
    i = torch.arange(r // 2, dtype=torch.float64, device=DEV)
    kind, factor = scaling["rope_type"], scaling.get("factor", 1.0)
    f = THETA ** (-2.0 * i / r)
    if kind == "linear":
        return f / factor, 1.0
    if kind == "ntk":  # the base grows so that the slowest pair is slowed by the factor
        return (THETA * factor ** (r / (r - 2.0))) ** (-2.0 * i / r), 1.0
    if kind == "yarn":  # pairs that turn often keep their speed, those that turn less than once are slowed
        turns = [r * math.log(scaling["original_max_position_embeddings"] / (2 * math.pi * scaling[x])) / (2 * math.log(THETA)) for x in ("beta_fast", "beta_slow")]
        low, high = max(math.floor(turns[0]), 0), min(math.ceil(turns[1]), r - 1)
        slowed = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
        return f / factor * slowed + f * (1 - slowed), 0.1 * math.log(factor) + 1.0
    if kind == "llama3":  # by wavelength: short ones keep their speed, long ones are slowed, a ramp between
        n = scaling["original_max_position_embeddings"] * f / (2 * math.pi)
        kept = ((n - scaling["low_freq_factor"]) / (scaling["high_freq_factor"] - scaling["low_freq_factor"])).clamp(0, 1)
        return f / factor * (1 - kept) + f * kept, 1.0
    return f, 1.0


def _rotate(x, cos, sin, case):
    r = case["r"]
    x = x.float()
    if case["layout"] == "half":
        a, b = x[..., : r // 2], x[..., r // 2: r]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([y, x[..., r:]], -1)


def _plain_rotary(s):
    case = s["case"]
    f, m = _frequencies(case)
    angle = s["positions"].double()[:, None, :, None] * f
    cos, sin = (torch.cos(angle) * m).float(), (torch.sin(angle) * m).float()
    dt = s["q"].dtype
    with torch.no_grad():
        out = [_rotate(s[x], cos, sin, case).to(dt) for x in "qk"]
        if case["grad"]:
            out += [_rotate(s[x], cos, -sin, case).to(dt) for x in ("gq", "gk")]
    return out


def _quantise(x, fmt):
    """Codes and scales of rows (the last axis)."""
    if fmt == "bf16":
        return x.to(torch.bfloat16), None
    x = x.float()
    top = x.abs().amax(-1).double()  # the divisions in 64 bits: a quotient next to a tie has to fall to its own side
    if fmt == "int8":
        scale = (top / 127).float().clamp_min(SMALLEST_SCALE)
        return torch.round(x / scale.double()[..., None]).clamp(-127, 127).to(torch.int8), scale
    f, e = torch.frexp(top / 448)  # f 2^e with 1/2 <= f < 1: the smallest power of two that takes the largest value to 448 or less
    scale = torch.exp2((e - (f == 0.5).to(e.dtype)).double()).float().clamp_min(SMALLEST_SCALE)
    return (x / scale[..., None]).to(torch.float8_e4m3fn), scale


def _values_of(codes, scale):
    return codes.float() if scale is None else codes.float() * scale[..., None]


def _gather(pages, table):
    """The pages [n, H, P, ...] of each sequence as [B, H, tokens, ...]."""
    x = pages.view(torch.int8)[table.long()].view(pages.dtype) if pages.dtype == torch.float8_e4m3fn else pages[table.long()]
    return x.transpose(1, 2).flatten(2, 3)


def _plain_cache(s):
    case, p = s["case"], s["pages"]
    t, page = case["t"], case["page"]
    at = s["start"].long()[:, None] + torch.arange(t, device=DEV)
    ids, row = s["page_table"].long().gather(1, at // page), at % page
    out = []
    for x in "kv":
        codes, scale = _quantise(s[x], case["fmt"])
        to = p[x].view(torch.int8) if case["fmt"] == "e4m3" else p[x]
        to[ids, :, row] = (codes.view(torch.int8) if case["fmt"] == "e4m3" else codes).transpose(1, 2)
        back = to[ids, :, row].view(p[x].dtype)
        if scale is not None:
            p[x + "_scale"][ids, :, row] = scale.transpose(1, 2)
            scale = p[x + "_scale"][ids, :, row]
        out.append(_values_of(back, scale).transpose(1, 2).to(torch.bfloat16))
    return out + [p[x + "_scale"] for x in "kv" if case["fmt"] != "bf16"]


def _seen(s, tokens):
    """[B, T, tokens]: which cached tokens each of the newest sees."""
    t, ctx = s["case"]["t"], s["context_lens"].long()[:, None, None]
    j = torch.arange(tokens, device=DEV) - ctx
    tree = s["tree"] if s["tree"] is not None else torch.ones(t, t, dtype=torch.bool, device=DEV).tril()
    new = tree[torch.arange(t, device=DEV)[None, :, None], j.clamp(0, t - 1)]
    return (j < 0) | ((j < t) & new)


def _plain_tree(s):
    case, p = s["case"], s["pages"]
    b, t, hq, h, d = (case[x] for x in ("b", "t", "hq", "hkv", "d"))
    k, v = (_gather(p[x], s["page_table"]).float() for x in "kv")
    if "k_scale" in p:
        k *= _gather(p["k_scale"], s["page_table"]).float()[..., None]
        v *= _gather(p["v_scale"], s["page_table"]).float()[..., None]
    q = s["q"].float().view(b, h, hq // h * t, d)  # query heads g of a KV head, one after the other
    x = (q * d ** -0.5) @ k.transpose(-1, -2)
    if "logit_bias" in p:
        x += _gather(p["logit_bias"], s["page_table"]).float()[:, :, None]
    x = x.view(b, h, hq // h, t, -1)
    x.masked_fill_(~_seen(s, x.shape[-1])[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x = torch.exp(x - top)
    total = x.sum(-1, keepdim=True)
    o = (x.view(b, h, hq // h * t, -1) @ v).view(b, h, hq // h, t, d) / total
    return o.view(b, hq, t, d), (top + torch.log(total)).view(b, hq, t)


# ---- one pass --------------------------------------------------------------------------------------


def run(s):
    case = s["case"]
    if case["op"] == "rotary":
        if not own:
            return _plain_rotary(s)
        out = s["rotary"](s["q"], s["positions"], s["k"])
        return [*out, *torch.autograd.grad(out, (s["q"], s["k"]), (s["gq"], s["gk"]))] if case["grad"] else list(out)
    if case["op"] == "cache":
        if not own:
            return _plain_cache(s)
        s["cache"].write(s["k"], s["v"], s["page_table"], s["start"])
        out = list(s["cache"].read(s["page_table"], s["start"], case["t"], dtype=torch.bfloat16))
        return out + [s["pages"][x + "_scale"] for x in "kv" if case["fmt"] != "bf16"]
    if not own:
        o, lse = _plain_tree(s)
        return [o.to(torch.bfloat16), lse]
    import dcc_kv_b200 as dk
    return list(dk.tree_attention(s["q"], s["cache"], s["page_table"], s["context_lens"], tree=s["tree"]))


def work(case):
    size = {"bf16": 2, "f32": 4, "int8": 1, "e4m3": 1}
    b, t, h, d = (case[x] for x in ("b", "t", "hkv", "d"))
    if case["op"] == "rotary":
        n = b * t * (case["hq"] + h)
        passes = 2 if case["grad"] else 1
        return {"bytes": passes * (2 * n * d * size[case["type"]] + 8 * b * t), "flops": passes * 3 * n * case["r"]}
    scale = 4 if case["fmt"] in ("int8", "e4m3") else 0
    if case["op"] == "cache":  # in, to the cache, from the cache, out
        rows = 2 * b * t * h
        return {"bytes": rows * (d * size[case["type"]] + 2 * (d * size[case["fmt"]] + scale) + 2 * d), "flops": 4 * rows * d}
    tokens = sum(_lengths(case)) + b * t
    row = 2 * (d * size[case["fmt"]] + scale) + (4 if case["bias"] else 0)
    return {"bytes": tokens * h * row + b * t * case["hq"] * (4 * d + 4), "flops": 4 * tokens * t * case["hq"] * d}


# ---- the definition in 64 bits ---------------------------------------------------------------------


def _exact_frequencies(case):
    r, kind = case["r"], case["scaling"]
    f = [math.exp(-2 * i / r * math.log(THETA)) for i in range(r // 2)]
    if kind == "linear":
        return [x / 4 for x in f], 1.0
    if kind == "ntk":
        return [x * 4 ** (-2 * i / (r - 2)) for i, x in enumerate(f)], 1.0
    if kind == "llama3":
        out = []
        for x in f:
            wave = 2 * math.pi / x
            w = 0.0 if wave > 8192 / 1 else 1.0 if wave < 8192 / 4 else (8192 / wave - 1) / (4 - 1)
            out.append((1 - w) * x / 8 + w * x)
        return out, 1.0
    if kind == "yarn":
        at = lambda turns: r * math.log(8192 / (turns * 2 * math.pi)) / (2 * math.log(THETA))  # noqa: E731
        low, high = max(math.floor(at(32)), 0), min(math.ceil(at(1)), r - 1)
        w = [min(1.0, max(0.0, (i - low) / (high - low))) for i in range(r // 2)]
        return [x * (1 - y) + x / 16 * y for x, y in zip(f, w)], 0.1 * math.log(16) + 1
    return f, 1.0


def _rows(pages, ids):
    """[H, tokens, ...] of one sequence's pages."""
    x = pages.view(torch.int8)[ids].view(pages.dtype) if pages.dtype == torch.float8_e4m3fn else pages[ids]
    return torch.cat(list(x.double()), 1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":  # complex numbers: a pair is turned by e^(i angle)
        f, m = _exact_frequencies(case)
        f = torch.tensor(f, dtype=torch.float64, device=DEV)
        turn = torch.polar(torch.full((), m, dtype=torch.float64, device=DEV).expand(case["b"], case["t"], case["r"] // 2).contiguous(),
                           s["positions"].double()[..., None] * f)[:, None]

        def turned(x, by):
            x, r, half = x.detach().double(), case["r"], case["layout"] == "half"
            pair = x[..., :r].unflatten(-1, (2, r // 2) if half else (r // 2, 2)).movedim(-2 if half else -1, 0)
            z = torch.complex(pair[0], pair[1]) * by
            y = torch.stack([z.real, z.imag], -2 if half else -1).flatten(-2)
            return torch.cat([y, x[..., r:]], -1)

        out = [turned(s[x], turn) for x in "qk"]
        return out + [turned(s[x], turn.conj()) for x in ("gq", "gk")] if case["grad"] else out
    if case["op"] == "cache":
        out, scales = [], []
        start, t, page, fmt = case["start"], case["t"], case["page"], case["fmt"]
        for x in "kv":
            y = s[x].double()
            if fmt == "bf16":
                out.append(y.bfloat16().double())
                continue
            top = y.abs().amax(-1, keepdim=True)
            if fmt == "int8":
                scale = (top / 127).float().double().clamp_min(SMALLEST_SCALE)
                out.append(torch.round(y / scale).clamp(-127, 127) * scale)
            else:
                scale = torch.exp2(torch.ceil(torch.log2(top / 448)))
                scale = torch.where(448 * scale < top, 2 * scale, torch.where(224 * scale >= top, scale / 2, scale)).clamp_min(SMALLEST_SCALE)
                z = y / scale
                step = torch.exp2((torch.frexp(z)[1].clamp_min(-5) - 4).double())  # four digits, subnormal below 2^-6
                out.append(torch.round(z / step) * step * scale)
            pool = torch.zeros(s["pages"][x + "_scale"].shape, dtype=torch.float64, device=DEV)
            for b in range(case["b"]):
                at = torch.arange(start, start + t, device=DEV)
                pool[s["page_table"][b].long()[at // page], :, at % page] = scale[b, :, :, 0].T
            scales.append(pool)
        return out + scales
    # tree: sequence by sequence, query head by query head
    p, g, t = s["pages"], case["hq"] // case["hkv"], case["t"]
    o = torch.empty(case["b"], case["hq"], t, case["d"], dtype=torch.float64, device=DEV)
    lse = torch.empty(case["b"], case["hq"], t, dtype=torch.float64, device=DEV)
    for b, n in enumerate(_lengths(case)):
        ids = s["page_table"][b].long()
        rows = {x: _rows(y, ids)[:, : n + t] for x, y in p.items()}
        kv = [rows[x] * rows[x + "_scale"][..., None] if x + "_scale" in rows else rows[x] for x in "kv"]
        hidden = torch.zeros(t, n + t, dtype=torch.float64, device=DEV)
        sees = s["tree"] if s["tree"] is not None else torch.ones(t, t, dtype=torch.bool, device=DEV).tril()
        hidden[:, n:].masked_fill_(~sees, -math.inf)
        for h in range(case["hq"]):
            x = s["q"][b, h].double() @ kv[0][h // g].T / math.sqrt(case["d"]) + hidden
            if "logit_bias" in rows:
                x += rows["logit_bias"][h // g]
            lse[b, h] = torch.logsumexp(x, -1)
            o[b, h] = torch.softmax(x, -1) @ kv[1][h // g]
    return [o, lse]
