"""64-bit statements of the decoding operators, for their tests."""
from __future__ import annotations

import math

import torch

F32 = 2.0 ** -24   # half a step
BF16 = 2.0 ** -8
SMALLEST = 2.0 ** -96


def rotate(x, positions, freqs, magnitude, layout, inverse=False):
    """x [B, H, T, d] float64, positions [B, T]; a pair as a complex number times e^(i angle)."""
    r = 2 * len(freqs)
    angle = positions.double()[:, None, :, None] * torch.tensor(freqs, dtype=torch.float64, device=x.device)
    turn = torch.polar(torch.full_like(angle, magnitude), -angle if inverse else angle)
    half = layout == "half"
    pair = x[..., :r].unflatten(-1, (2, r // 2) if half else (r // 2, 2)).movedim(-2 if half else -1, 0)
    z = torch.complex(pair[0].contiguous(), pair[1].contiguous()) * turn
    y = torch.stack([z.real, z.imag], -2 if half else -1).flatten(-2)
    return torch.cat([y, x[..., r:]], -1)


def quantise(x, fmt):
    """Codes (float64) and scales (float64, each a float32 number) of rows."""
    x = x.double()
    if fmt in ("bf16", "f32"):
        return x.to(torch.bfloat16 if fmt == "bf16" else torch.float32).double(), None
    top = x.abs().amax(-1, keepdim=True)
    if fmt == "int8":
        scale = (top / 127).float().double().clamp_min(SMALLEST)
        return torch.round(x / scale).clamp(-127, 127), scale[..., 0]
    scale = torch.exp2(torch.ceil(torch.log2(top / 448))).clamp_min(SMALLEST)
    scale = torch.where(448 * scale < top, 2 * scale, torch.where((224 * scale >= top) & (scale > SMALLEST), scale / 2, scale))
    z = x / scale
    step = torch.exp2((torch.frexp(z)[1].clamp_min(-5) - 4).double())
    return torch.round(z / step) * step, scale[..., 0]


def cached(cache, page_table, b, n):
    """(k, v [H, n, d], bias [H, n] or None) of positions 0..n of sequence b, float64;
    a position without a page has NaN keys (and must not be asked for)."""
    P = cache.page_size
    ids = page_table[b].long()
    pos = torch.arange(n, device=ids.device)
    page = ids[pos // P]
    out = []
    for code, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        c = code.float().double()[page, :, pos % P].transpose(0, 1)
        if scale is not None:
            c = c * scale.double()[page, :, pos % P].transpose(0, 1)[..., None]
        out.append(c)
    bias = None if cache.logit_bias is None else cache.logit_bias.double()[page, :, pos % P].transpose(0, 1)
    return out[0], out[1], bias


def tree(q, cache, page_table, ctx, counts=None, mask=None, scale=None, seen_pos=None):
    """(o, lse, a, ex): the output and its log-sum-exp, softmax(x) |v| and the
    largest sum |q||k| scale of a row's keys, for tolerances.  float64."""
    B, HQ, T, d = q.shape
    g = HQ // cache.n_kv_heads
    dev = q.device
    o = torch.zeros(B, HQ, T, d, dtype=torch.float64, device=dev)
    a = torch.zeros_like(o)
    lse = torch.full((B, HQ, T), -math.inf, dtype=torch.float64, device=dev)
    ex = torch.zeros(B, HQ, T, dtype=torch.float64, device=dev)
    scale = d ** -0.5 if scale is None else scale
    for b in range(B):
        n = T if counts is None else int(counts[b])
        c = int(ctx[b])
        if n == 0:
            continue
        k, v, bias = cached(cache, page_table, b, c + n)
        m = torch.ones(T, T, dtype=torch.bool, device=dev).tril() if mask is None else (mask if mask.dim() == 2 else mask[b])
        sees = torch.cat([torch.ones(n, c, dtype=torch.bool, device=dev), m[:n, :n]], 1)
        if seen_pos is not None:
            sees = sees & seen_pos[b][: c + n]
        for h in range(HQ):
            kk, vv = k[h // g], v[h // g]
            qq = q[b, h, :n].double()
            x = qq @ kk.T * scale
            if bias is not None:
                x = x + bias[h // g]
            x = x.masked_fill(~sees, -math.inf)
            some = sees.any(1)
            top = x.amax(1, keepdim=True)
            e = torch.where(sees, torch.exp(x - torch.where(some[:, None], top, torch.zeros_like(top))), torch.zeros_like(x))
            l = e.sum(1, keepdim=True)
            p = e / torch.where(l == 0, torch.ones_like(l), l)
            vz = torch.where(sees.any(0)[:, None], vv, torch.zeros_like(vv))
            o[b, h, :n] = p @ vz
            a[b, h, :n] = p @ vz.abs()
            if cache.v_scale is not None and q.dtype == torch.bfloat16:
                # p times the V scale is held in fp16, in units of at most the row's
                # largest such product: below 2^-14 of the unit half a step is 2^-25 of
                # it whatever p is, and a key adds that times its code.  (2^-17 here:
                # the tolerance takes 2^-8 of a.)
                ids = page_table[b].long()
                pos = torch.arange(c + n, device=dev)
                s = cache.v_scale.double()[ids[pos // cache.page_size], h // g, pos % cache.page_size]
                code = torch.where(s > 0, vz.abs().T / torch.where(s > 0, s, torch.ones_like(s)), torch.zeros_like(s))
                a[b, h, :n] += 2.0 ** -17 * (p * torch.nan_to_num(s)).amax(1, keepdim=True) * torch.nan_to_num(code).sum(1)
            lse[b, h, :n] = torch.where(some, top[:, 0] + torch.log(l[:, 0]), torch.full_like(l[:, 0], -math.inf))
            ex[b, h, :n] = (qq.abs() @ kk.abs().T * abs(scale)).masked_fill(~sees, 0.).amax(1)
    return o, lse, a, ex


def tree_tolerances(o, lse, a, ex, d, keys, dtype):
    """A logit is a sum of d exact products in 32 bits: off by (d + 4) 2^-24 ex
    at most, and so is ln p; exponentials, their sum over the keys and the
    weighted sum add (keys + 16) 2^-24 and, in the SFU's 2^x, 2^-21.  In
    bf16 each p is held to half a step and the result is rounded once."""
    dx = (d + 4) * F32 * ex + 2.0 ** -21
    rel = 2 * dx[..., None] + (keys + 16) * F32
    to = rel * a + F32 * o.abs()
    if dtype == torch.bfloat16:
        to = to + BF16 * a + BF16 * o.abs() + 1e-30
    return to, dx + (keys + 16) * F32 + 4 * F32 * torch.nan_to_num(lse.abs(), posinf=0.0)


def tree_close(got, want, d, keys):
    """Assert (o, lse) against tree()'s answer."""
    o, lse = got
    wo, wl, a, ex = want
    to, tl = tree_tolerances(wo, wl, a, ex, d, keys, o.dtype)
    assert torch.isfinite(o).all()
    off = (o.double() - wo).abs() - to
    assert off.max() <= 0, f"output off by {(o.double() - wo).abs().max():.3e}, {off.max():.3e} over its bound"
    none = torch.isinf(wl)
    assert torch.equal(torch.isinf(lse) & (lse < 0), none)
    assert (o[none] == 0).all()
    off = ((lse.double() - wl).abs() - tl)[~none]
    assert off.numel() == 0 or off.max() <= 0, f"lse over its bound by {off.max():.3e}"
