"""Decoding behind the prefill on the GPU: rotary positions, the quantised
paged cache and the attention of the newest tokens over it, against their
definitions in 64 bits (decode_ref.py, where the tolerances are derived)."""
from __future__ import annotations

import math
import random

import pytest
import torch

import dcc_kv_b200 as dk
import decode_ref as ref

from gpu_util import assert_no_device_timeouts, dev

pytestmark = pytest.mark.gpu

SCALINGS = [None,
            {"rope_type": "linear", "factor": 4.0},
            {"rope_type": "ntk", "factor": 2.5},
            {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096},
            {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
             "original_max_position_embeddings": 8192}]


def within(got, want, bound):
    """got within bound of want everywhere, with a short message."""
    over = float(((got.double() - want).abs() - bound).max()) if got.numel() else 0.0
    assert over <= 0, f"{over:.3e} over its bound"


def gen(seed):
    return torch.Generator(device=dev()).manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=dev()).to(dtype)


# ---- rotary ----------------------------------------------------------------------------------------


def rotary_bound(x, want, magnitude, dtype):
    """Sine and cosine: 2^-22 absolute (an angle within 2^-23 of a turn's
    fraction, and their own rounding), times magnitude; the two products and
    their sum three half steps; the result one half step of its type.
    In 64 bits the angle itself is what rounds: f, the product position * f
    (and f / 2 pi and its product on the kernel's side) are each off by 2^-53
    of an angle below 2^20, six such roundings in both sides together, and an
    angle's error moves a sine or cosine by as much: 2 * 6 * 2^-33."""
    if dtype == torch.float64:
        return 12 * 2.0 ** -33 * magnitude * x.abs().amax() + 0 * want
    to = magnitude * x.abs().amax(-1, keepdim=True) * (2 * 2.0 ** -22 + 6 * ref.F32)
    return to + (ref.BF16 if dtype == torch.bfloat16 else ref.F32) * want.abs()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("b,t,hq,hkv,d,r,scaling", [
    (1, 1, 4, 1, 64, 64, 0), (3, 5, 8, 2, 128, 128, 1), (2, 33, 3, 3, 96, 48, 2), (1, 257, 2, 1, 20, 10, 3),
    (1, 130, 32, 8, 128, 64, 4), (2, 7, 1, 1, 2, 2, 0), (1, 9, 2, 2, 40, 24, 0), (1, 3, 2, 1, 256, 256, 1)])
def test_rotary_against_64_bits(dtype, layout, b, t, hq, hkv, d, r, scaling):
    g = gen(1)
    q, k = randn(g, b, hq, t, d, dtype=dtype), randn(g, b, hkv, t, d, dtype=dtype)
    far = torch.randint(0, 1 << 20, (b, t), generator=g, device=dev())
    rot = dk.Rotary(d, rotary_dim=r, theta=500000.0, layout=layout, scaling=SCALINGS[scaling])
    for pos in (far, far.int(), far[0]):
        out = rot(q, pos, k)
        p2 = pos.expand(b, t) if pos.dim() == 1 else pos
        for x, y in zip((q, k), out):
            want = ref.rotate(x.double(), p2, rot.frequencies, rot.magnitude, layout)
            assert y.dtype == dtype and y.shape == x.shape
            within(y, want, rotary_bound(x.double(), want, rot.magnitude, dtype))
            assert torch.equal(y[..., r:], x[..., r:])
    assert torch.equal(rot(q, far), rot(q, far, k)[0])


def test_rotary_strides_inplace_and_empty():
    g = gen(2)
    rot = dk.Rotary(128, rotary_dim=64)
    pos = torch.arange(40, device=dev()) + 100000
    full = randn(g, 2, 40, 6, 130, dtype=torch.bfloat16)
    x = full[:, :, :, 1:129].transpose(1, 2)          # token-major, rows that are not 16-byte aligned
    want = rot(x.contiguous(), pos)
    assert torch.equal(rot(x, pos), want)
    aligned = randn(g, 2, 40, 6, 128, dtype=torch.bfloat16).transpose(1, 2)
    want2 = rot(aligned.contiguous(), pos)
    assert torch.equal(rot(aligned, pos), want2)
    e = aligned[:1].expand(2, 6, 40, 128)             # a broadcast batch
    assert torch.equal(rot(e, pos), rot(e.contiguous(), pos))
    with pytest.raises(ValueError, match="expanded"):
        rot(e, pos, inplace=True)
    before = full.clone()
    got = rot(x, pos, inplace=True)
    assert got.data_ptr() == x.data_ptr() and torch.equal(x, want)
    assert torch.equal(full[..., [0, 129]], before[..., [0, 129]])
    assert rot(x[:, :, :0], pos[:0]).shape == (2, 6, 0, 128)
    assert rot(x[:0], pos).shape == (0, 6, 40, 128)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_gradient(layout):
    g = gen(3)
    rot = dk.Rotary(24, rotary_dim=16, layout=layout, scaling=SCALINGS[3])
    pos = torch.randint(0, 100000, (2, 5), generator=g, device=dev())
    q = randn(g, 2, 3, 5, 24, dtype=torch.float64).requires_grad_()
    k = randn(g, 2, 1, 5, 24, dtype=torch.float64).requires_grad_()
    assert torch.autograd.gradcheck(lambda a, b: rot(a, pos, b), (q, k))
    assert torch.autograd.gradgradcheck(lambda a, b: rot(a, pos, b), (q, k))
    # the formula: the transpose of the map is the map with the angles negated
    gq, gk = randn(g, *q.shape, dtype=torch.float64), randn(g, *k.shape, dtype=torch.float64)
    dq, dk_ = torch.autograd.grad(rot(q, pos, k), (q, k), (gq, gk))
    for grad, got in ((gq, dq), (gk, dk_)):
        want = ref.rotate(grad, pos, rot.frequencies, rot.magnitude, layout, inverse=True)
        within(got, want, 12 * 2.0 ** -36 * rot.magnitude * grad.abs().max())   # angles below 2^17, see rotary_bound
    # one of two, a broadcast leaf, a broadcast gradient
    (only,) = torch.autograd.grad(rot(q.detach(), pos, k)[1].sum(), k)
    ones = ref.rotate(torch.ones_like(k), pos, rot.frequencies, rot.magnitude, layout, inverse=True)
    within(only, ones, 12 * 2.0 ** -36 * rot.magnitude)
    leaf = randn(g, 1, 3, 1, 24, dtype=torch.float64).requires_grad_()
    (gl,) = torch.autograd.grad(rot(leaf.expand(2, 3, 5, 24), pos), leaf, gq)
    want = ref.rotate(gq, pos, rot.frequencies, rot.magnitude, layout, inverse=True).sum((0, 2), keepdim=True)
    within(gl, want, 10 * 12 * 2.0 ** -36 * rot.magnitude * gq.abs().max())   # ten summands
    with pytest.raises(ValueError, match="gradient"):
        rot(q, pos, inplace=True)


def test_rotary_forward_and_backward_in_a_graph():
    g = gen(4)
    rot = dk.Rotary(64)
    pos = torch.zeros(1, 8, dtype=torch.int64, device=dev())
    q = randn(g, 1, 4, 8, 64).requires_grad_()
    gq = randn(g, 1, 4, 8, 64)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        rot(q, pos)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = rot(q, pos)
        (dq,) = torch.autograd.grad(y, q, gq)
    for first in (0, 77777):
        pos.copy_(torch.arange(first, first + 8)[None])
        graph.replay()
        y2 = rot(q, pos)
        assert torch.equal(y, y2)
        assert torch.equal(dq, torch.autograd.grad(y2, q, gq)[0])


# ---- cache -----------------------------------------------------------------------------------------


def make_table(g, b, per, n_pages):
    return torch.randperm(n_pages, generator=g, device=dev())[: b * per].to(torch.int32).view(b, per).contiguous()


@pytest.mark.parametrize("fmt", ["int8", "e4m3", "bf16", "f32"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("b,t,h,d,page", [(1, 1, 1, 128, 16), (3, 37, 2, 64, 8), (2, 130, 4, 96, 64), (1, 300, 1, 128, 1),
                                          (2, 19, 3, 7, 5), (1, 50, 2, 40, 33), (1, 0, 1, 64, 16)])
def test_cache_write_and_read(fmt, dtype, b, t, h, d, page):
    g = gen(5)
    k, v = randn(g, b, h, t, d, dtype=dtype) * 3, randn(g, b, h, t, d, dtype=dtype)
    k, v = k.to(dtype), v.to(dtype)
    if t > 4:
        k[:, :, 1] = 0
        k[:, :, 2] *= 1e-30
        v[:, :, 3] *= 1e30
        v[:, :, 4, : d // 2] = 0
    start = torch.tensor([0, 5, 23][:b], dtype=torch.int32, device=dev())
    per = -(-(t + 23) // page) + 1
    n_pages = b * per + 3
    table = make_table(g, b, per, n_pages)
    cache = dk.KvCache.empty(n_pages, page, h, d, fmt, logit_bias=True, device=dev())
    bias = randn(g, b, h, t)
    cache.write(k, v, table, start, logit_bias=bias)
    for out_dtype in (torch.bfloat16, torch.float32):
        rk, rv, rb = cache.read(table, start, t, dtype=out_dtype, logit_bias=True)
        assert torch.equal(rb, bias)
        for x, y in ((k, rk), (v, rv)):
            codes, scale = ref.quantise(x, fmt)
            # code * scale in 64 bits is exact; the read rounds it to 32 bits (at once for bf16: then to bf16)
            want = (codes if scale is None else codes * scale[..., None]).float().to(out_dtype)
            assert torch.equal(y, want)
    # nothing else was touched
    total = cache.k.float().abs().sum(-1) + (cache.k_scale if cache.k_scale is not None else 0)
    written = torch.zeros(n_pages, page, dtype=torch.bool, device=dev())
    for s in range(b):
        pos = torch.arange(t, device=dev()) + int(start[s])
        written[table[s].long()[pos // page], pos % page] = True
    assert (total.sum(1)[~written] == 0).all()


def test_int8_ties_go_to_even_by_the_exact_quotient():
    """Rows whose quotients are exact ties and their neighbours in bfloat16 and float32."""
    top = torch.tensor([127.0, 127 * 2.0 ** -40, 127 * 3.0, 254.0 * 1.25], device=dev())
    n = torch.arange(-127, 127, device=dev()) + 0.5
    x = (n[None] * (top / 127)[:, None]).float()
    x = torch.cat([x, torch.nextafter(x, torch.full_like(x, 1e9)), torch.nextafter(x, torch.full_like(x, -1e9))], 0)
    x = torch.cat([x, x[:, :2]], 1)
    x[:, -1] = top.repeat(3)
    for d in (128, 127):
        rows = torch.cat([x[:, i: i + d - 1] for i in (0, 64, 127)], 0)
        rows = torch.cat([rows, top.repeat(9)[:, None]], 1)[None, None]      # each with its largest value
        cache = dk.KvCache.empty(8, 16, 1, d, "int8", device=dev())
        table = torch.arange(8, dtype=torch.int32, device=dev())[None]
        cache.write(rows, -rows, table, 0)
        codes, scale = ref.quantise(rows, "int8")
        got = cache.k.permute(1, 0, 2, 3).reshape(1, 128, d)[:, : rows.shape[2]]
        assert torch.equal(got.double(), codes[0])
        assert torch.equal(cache.v.permute(1, 0, 2, 3).reshape(1, 128, d)[:, : rows.shape[2]], -got)


def test_cache_rows_that_are_not_finite():
    g = gen(6)
    for fmt in ("int8", "e4m3"):
        x = randn(g, 1, 1, 5, 64)
        x[0, 0, 1, 3], x[0, 0, 2, 63], x[0, 0, 3, 0] = math.nan, math.inf, -math.inf
        cache = dk.KvCache.empty(1, 16, 1, 64, fmt, device=dev())
        table = torch.zeros(1, 1, dtype=torch.int32, device=dev())
        cache.write(x, x, table, 0)
        k, v = cache.read(table, 0, 5, dtype=torch.float32)
        bad = torch.tensor([False, True, True, True, False], device=dev())
        assert torch.isnan(k[0, 0][bad]).all() and torch.isfinite(k[0, 0][~bad]).all()
        assert torch.equal(torch.isnan(v), torch.isnan(k))


def test_cache_skips_what_has_no_page():
    g = gen(7)
    cache = dk.KvCache.empty(4, 4, 2, 64, "int8", device=dev())
    table = torch.tensor([[0, -1, 7], [3, 1, 2147483647]], dtype=torch.int32, device=dev())
    k = randn(g, 2, 2, 20, 64)
    start = torch.tensor([-3, 2], dtype=torch.int32, device=dev())
    counts = torch.tensor([20, 5], dtype=torch.int32, device=dev())
    cache.write(k, k, table, start, counts)
    rk, _ = cache.read(table, start, 20, counts=counts, dtype=torch.float32)
    live0 = torch.tensor([0 <= t - 3 < 4 for t in range(20)], device=dev())
    live1 = torch.tensor([t < 5 for t in range(20)], device=dev())    # positions 2..6: pages 3 and 1
    for s, live in ((0, live0), (1, live1)):
        assert (rk[s][:, ~live] == 0).all()
        codes, scale = ref.quantise(k[s][:, live], "int8")
        assert torch.equal(rk[s][:, live], (codes * scale[..., None]).float())
    assert (cache.k_scale[2] == 0).all()


def test_cache_strides():
    g = gen(8)
    base = randn(g, 2, 30, 4, 131, dtype=torch.bfloat16)
    table = make_table(g, 2, 4, 8)
    for view in (base[..., :128], base[..., 1:129]):
        k = view.transpose(1, 2)                      # token-major; aligned and not
        a, b = (dk.KvCache.empty(8, 16, 4, 128, "e4m3", device=dev()) for _ in range(2))
        a.write(k, k, table, 3)
        b.write(k.contiguous(), k.contiguous(), table, 3)
        assert torch.equal(a.k.view(torch.uint8), b.k.view(torch.uint8)) and torch.equal(a.v_scale, b.v_scale)


# ---- tree attention --------------------------------------------------------------------------------


def filled(g, fmt, b, h, d, page, tokens, bias=False, outliers=True):
    """A cache with `tokens` positions of each of b sequences in random pages."""
    per = max(1, -(-tokens // page))
    n = b * per + 2
    table = make_table(g, b, per, n)
    cache = dk.KvCache.empty(n, page, h, d, fmt, logit_bias=bias, device=dev())
    k, v = randn(g, b, h, tokens, d), randn(g, b, h, tokens, d)
    if outliers:
        k[..., : max(1, d // 32)] *= 8
    cache.write(k, v, table, 0, logit_bias=randn(g, b, h, tokens) * 2 if bias else None)
    return cache, table


def random_tree(r, t):
    return dk.tree_mask([r.randrange(-1, i) if i else -1 for i in range(t)])


def lens(*x):
    return torch.tensor(x, dtype=torch.int32, device=dev())


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3", "f32"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("b,t,hq,hkv,d,page,ctx,bias", [
    (1, 1, 1, 1, 128, 16, 0, False), (2, 1, 8, 2, 64, 16, 127, True), (3, 1, 32, 8, 128, 64, 1000, False),
    (2, 5, 4, 4, 96, 8, 250, True), (1, 13, 32, 8, 128, 16, 700, False), (2, 64, 8, 1, 128, 128, 513, False),
    (1, 33, 16, 2, 64, 7, 129, True), (2, 3, 6, 3, 20, 16, 40, False), (1, 200, 4, 1, 128, 64, 60, False),
    (1, 2, 2, 2, 16, 1, 300, False)])
def test_tree_attention_against_64_bits(fmt, dtype, b, t, hq, hkv, d, page, ctx, bias):
    g, r = gen(9), random.Random(9)
    cache, table = filled(g, fmt, b, hkv, d, page, ctx + t, bias)
    q = randn(g, b, hq, t, d, dtype=dtype)
    at = lens(*[ctx - (i * ctx) // (b + 1) for i in range(b)])
    for mask in (None, random_tree(r, t).to(dev()), torch.stack([random_tree(r, t) for _ in range(b)]).to(dev())):
        got = dk.tree_attention(q, cache, table, at, tree=mask)
        ref.tree_close(got, ref.tree(q, cache, table, at, mask=mask), d, ctx + t)
    assert_no_device_timeouts()


def test_tree_masks_that_leave_rows_empty_and_padded_batches():
    g = gen(10)
    for fmt, dtype in (("bf16", torch.bfloat16), ("int8", torch.bfloat16), ("f32", torch.float32)):
        cache, table = filled(g, fmt, 4, 2, 128, 16, 300)
        q = randn(g, 4, 8, 9, 128, dtype=dtype)
        mask = torch.rand(4, 9, 9, generator=g, device=dev()) < 0.4
        mask[:, 3] = False
        ctx, counts = lens(0, 130, 0, 291), lens(9, 0, 4, 7)
        got = dk.tree_attention(q, cache, table, ctx, counts=counts, tree=mask)
        want = ref.tree(q, cache, table, ctx, counts=counts, mask=mask)
        assert torch.isinf(want[1][0, :, 3]).all()
        ref.tree_close(got, want, 128, 300)
        # lengths outside what they may be count as the nearest that may
        odd = dk.tree_attention(q, cache, table, lens(-5, 130, 0, 291), counts=lens(100, -1, 4, 7), tree=mask)
        assert torch.equal(odd[0], got[0]) and torch.equal(odd[1], got[1])
        none = dk.tree_attention(q, cache, table, lens(0, 0, 0, 0), counts=lens(0, 0, 0, 0))
        assert (none[0] == 0).all() and torch.isinf(none[1]).all()


@pytest.mark.parametrize("fmt,dtype", [("bf16", torch.bfloat16), ("e4m3", torch.bfloat16), ("f32", torch.float32)])
def test_tree_what_is_hidden_does_not_matter(fmt, dtype):
    """NaN and infinities in stale rows, behind the sequence and in drafted keys that a row does not see."""
    g = gen(11)
    cache, table = filled(g, fmt, 1, 2, 64, 16, 200)
    q = randn(g, 1, 4, 6, 64, dtype=dtype)
    ctx = lens(140)
    mask = torch.eye(6, dtype=torch.bool, device=dev())
    want = dk.tree_attention(q, cache, table, ctx, tree=mask)
    poison = torch.full((1, 2, 54, 64), math.nan, device=dev())
    poison[:, :, ::2, 0] = math.inf
    cache.write(poison, poison, table, 146)             # behind the last newest token
    got = dk.tree_attention(q, cache, table, ctx, tree=mask)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for x in (math.nan, math.inf, -math.inf):
        cache.write(torch.zeros(1, 2, 1, 64, device=dev()), torch.full((1, 2, 1, 64), x, device=dev()), table, 142)
        got = dk.tree_attention(q, cache, table, ctx, tree=mask)
        keep = torch.tensor([0, 1, 3, 4, 5], device=dev())
        assert torch.equal(got[0][:, :, keep], want[0][:, :, keep])
        assert not torch.isfinite(got[0][:, :, 2]).any()
        assert torch.equal(got[1][:, :, keep], want[1][:, :, keep])
    cache.write(torch.full((1, 2, 1, 64), math.nan, device=dev()), torch.zeros(1, 2, 1, 64, device=dev()), table, 142)
    got = dk.tree_attention(q, cache, table, ctx, tree=mask)
    assert torch.equal(got[0][:, :, keep], want[0][:, :, keep]) and torch.isnan(got[0][:, :, 2]).all()


@pytest.mark.parametrize("fmt,dtype", [("bf16", torch.bfloat16), ("int8", torch.bfloat16), ("f32", torch.float32)])
def test_tree_biases_at_the_ends_of_their_type(fmt, dtype):
    g = gen(12)
    lowest = torch.finfo(torch.float32).min
    cache, table = filled(g, fmt, 1, 1, 64, 16, 400, bias=True)
    q = randn(g, 1, 2, 1, 64, dtype=dtype)
    k, v, b = cache.read(table, 0, 400, dtype=torch.float32, logit_bias=True)
    # half of the keys hidden by the lowest value: as if they were not there
    b[:, :, ::2] = lowest
    cache.write(k, v, table, 0, logit_bias=b)
    ref.tree_close(dk.tree_attention(q, cache, table, lens(399)), ref.tree(q, cache, table, lens(399)), 64, 400)
    b[:, :, ::2] = -math.inf
    cache.write(k, v, table, 0, logit_bias=b)
    seen = torch.arange(400, device=dev())[None] % 2 == 1
    zero_b = torch.nan_to_num(b, neginf=0.0)
    got = dk.tree_attention(q, cache, table, lens(399))
    cache.write(k, v, table, 0, logit_bias=zero_b)
    ref.tree_close(got, ref.tree(q, cache, table, lens(399), seen_pos=seen), 64, 400)
    # every key at the lowest value: all alike
    b[:] = lowest
    cache.write(k, v, table, 0, logit_bias=b)
    o, lse = dk.tree_attention(q, cache, table, lens(399))
    want = ref.cached(cache, table, 0, 400)[1].mean(1)
    a = ref.cached(cache, table, 0, 400)[1].abs().mean(1)
    tol = (420 * ref.F32 + 2.0 ** -20) * a + (2 * ref.BF16 * a if dtype == torch.bfloat16 else 0)
    within(o[0, :, 0], want.repeat_interleave(2, 0), tol.repeat_interleave(2, 0))
    assert (lse == lowest).all()
    # every key at -inf: nothing is seen
    b[:] = -math.inf
    cache.write(k, v, table, 0, logit_bias=b)
    o, lse = dk.tree_attention(q, cache, table, lens(399))
    assert (o == 0).all() and torch.isinf(lse).all()


def test_tree_positions_without_a_page_are_not_seen():
    g = gen(13)
    for fmt, dtype in (("bf16", torch.bfloat16), ("int8", torch.bfloat16), ("f32", torch.float32)):
        cache, table = filled(g, fmt, 2, 2, 128, 16, 256)
        q = randn(g, 2, 4, 3, 128, dtype=dtype)
        bad = table.clone()
        bad[0, 2], bad[0, 9], bad[1, 0] = -1, cache.n_pages, 2147483647
        seen = torch.ones(2, 256, dtype=torch.bool, device=dev())
        seen[0, 32:48] = seen[0, 144:160] = seen[1, 0:16] = False
        ctx = lens(253, 201)
        got = dk.tree_attention(q, cache, bad, ctx)
        ref.tree_close(got, ref.tree(q, cache, table, ctx, seen_pos=seen), 128, 256)
        # a context behind the end of the table: only what the table holds
        short = dk.tree_attention(q, cache, table[:, :3].contiguous(), lens(100, 48))
        seen[:] = False
        seen[:, :48] = True
        ref.tree_close(short, ref.tree(q, cache, table, lens(100, 48), seen_pos=seen), 128, 256)


def test_tree_strides_and_scale():
    g = gen(14)
    cache, table = filled(g, "int8", 2, 2, 128, 16, 300)
    full = randn(g, 2, 5, 8, 130, dtype=torch.bfloat16)
    mask = torch.rand(5, 10, generator=g, device=dev()) < 0.5
    for q in (full[..., :128].transpose(1, 2), full[..., 1:129].transpose(1, 2)):
        a = dk.tree_attention(q, cache, table, lens(200, 33), tree=mask[:, ::2], scale=0.25)
        ref.tree_close(a, ref.tree(q, cache, table, lens(200, 33), mask=mask[:, ::2], scale=0.25), 128, 300)
    wide = torch.cat([table, table], 1)[:, : table.shape[1]]           # a row stride of its own
    b = dk.tree_attention(q.contiguous(), cache, wide, lens(200, 33), tree=mask[:, ::2].contiguous(), scale=0.25)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_tree_attention_is_repeatable_and_runs_in_a_graph():
    g = gen(15)
    cache, table = filled(g, "e4m3", 3, 4, 128, 32, 2000)
    q = randn(g, 3, 16, 4, 128, dtype=torch.bfloat16)
    ctx = lens(5, 5, 5)
    first = dk.tree_attention(q, cache, table, ctx)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lse = dk.tree_attention(q, cache, table, ctx)
    with torch.cuda.graph(other, pool=graph.pool()):
        o2, lse2 = dk.tree_attention(q, cache, table, ctx)
    for at in ((5, 5, 5), (1996, 0, 700), (127, 128, 1500)):
        ctx.copy_(lens(*at))
        graph.replay()
        eager = dk.tree_attention(q, cache, table, ctx)
        assert torch.equal(o, eager[0]) and torch.equal(lse, eager[1])
        other.replay()
        assert torch.equal(o2, eager[0]) and torch.equal(lse2, eager[1])
        ref.tree_close(eager, ref.tree(q, cache, table, ctx), 128, 2000)
    ctx.copy_(lens(5, 5, 5))
    assert torch.equal(dk.tree_attention(q, cache, table, ctx)[0], first[0])


def test_tree_on_two_streams_at_once():
    g = gen(16)
    cache, table = filled(g, "int8", 2, 2, 128, 16, 3000)
    qs = [randn(g, 2, 8, 3, 128, dtype=torch.bfloat16) for _ in range(4)]
    want = [dk.tree_attention(q, cache, table, lens(2990, 1000)) for q in qs]
    ctx = lens(2990, 1000)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i, q in enumerate(qs):
        with torch.cuda.stream(streams[i % 2]):
            got.append(dk.tree_attention(q, cache, table, ctx))
    torch.cuda.synchronize()
    for x, y in zip(got, want):
        assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])


def test_tree_many_sequences():
    """More sequences than a block has threads, most of them empty."""
    g = gen(17)
    n = 1500
    cache, table = filled(g, "bf16", n, 1, 64, 16, 40)
    q = randn(g, n, 2, 1, 64, dtype=torch.bfloat16)
    r = random.Random(3)
    ctx = torch.tensor([r.randrange(0, 40) for _ in range(n)], dtype=torch.int32, device=dev())
    counts = torch.tensor([int(r.random() < 0.3) for _ in range(n)], dtype=torch.int32, device=dev())
    ref.tree_close(dk.tree_attention(q, cache, table, ctx, counts=counts),
                   ref.tree(q, cache, table, ctx, counts=counts), 64, 41)


# ---- together --------------------------------------------------------------------------------------


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
def test_decoding_steps(fmt):
    """Rotary positions, the cache and the attention, one token after the other, against 64 bits on what the cache holds."""
    g = gen(18)
    b, hq, hkv, d, prompt = 2, 8, 2, 128, 190
    rot = dk.Rotary(d, theta=500000.0, scaling=SCALINGS[4])
    cache = dk.KvCache.empty(40, 16, hkv, d, fmt, device=dev())
    table = make_table(g, b, 16, 40)
    pos = torch.arange(prompt, device=dev())
    k, v = randn(g, b, hkv, prompt, d, dtype=torch.bfloat16), randn(g, b, hkv, prompt, d, dtype=torch.bfloat16)
    cache.write(rot(k, pos), v, table, 0)
    ctx = lens(prompt, prompt)
    for step in range(4):
        q, k, v = (randn(g, b, h, 1, d, dtype=torch.bfloat16) for h in (hq, hkv, hkv))
        q, k = rot(q, ctx[:, None], k)
        cache.write(k, v, table, ctx)
        got = dk.tree_attention(q, cache, table, ctx)
        ref.tree_close(got, ref.tree(q, cache, table, ctx), d, prompt + 4)
        kept = cache.read(table, ctx, 1, dtype=torch.float32)[0]
        codes, scale = ref.quantise(k, fmt)
        assert torch.equal(kept, (codes if scale is None else codes * scale[..., None]).float())
        ctx += 1
    # a tree of drafted tokens, then the accepted path alone as a chain: the same rows
    parents = [-1, 0, 0, 1, 2, 4]
    q, k, v = (randn(g, b, h, 6, d, dtype=torch.bfloat16) for h in (hq, hkv, hkv))
    cache.write(k, v, table, ctx)
    tree = dk.tree_attention(q, cache, table, ctx, tree=dk.tree_mask(parents).to(dev()))
    path = torch.tensor([0, 2, 4, 5], device=dev())
    cache.write(k[:, :, path], v[:, :, path], table, ctx)
    chain = dk.tree_attention(q[:, :, path], cache, table, ctx)
    want = ref.tree(q[:, :, path], cache, table, ctx)
    ref.tree_close(chain, want, d, prompt + 12)
    ref.tree_close((tree[0][:, :, path], tree[1][:, :, path]), want, d, prompt + 12)


def test_decoding_behind_the_layer():
    """The last block's compact and local keys in a cache: the attention of new tokens over it is the attention over
    the layer's own segments."""
    from dcc_kv_b200.workloads import layer_inputs
    nb, length, hq, hkv, d = 3, 256, 8, 2, 128
    q, k, v = layer_inputs(nb, length, hq, hkv, d, device="cuda", first_seed=3)
    layer = dk.DccKvSyncLayer(nb, length, hq, hkv, d, 64, window=64)
    layer(q, k, v)
    cache = dk.KvCache.empty(30, 16, hkv, d, "bf16", logit_bias=True, device=dev())
    table = make_table(gen(19), 1, 26, 30)
    n = layer.write_cache(cache, table, 2, k, v)
    assert n == 2 * 64 + length
    g = gen(20)
    nq, nk, nv = (randn(g, 1, h, 5, d, dtype=torch.bfloat16) for h in (hq, hkv, hkv))
    cache.write(nk, nv, table, n)
    ctx = lens(n)
    o, lse = dk.tree_attention(nq, cache, table, ctx)
    ref.tree_close((o, lse), ref.tree(nq, cache, table, ctx), d, n + 5)
    old = [(k[2], v[2], None), (layer.ck[2], layer.cv[2], layer.cb[2])]
    o1, l1 = dk.attention(nq[0], old)
    o2, l2 = dk.attention(nq[0], [(nk[0], nv[0], None)], causal=True)
    both, bl = dk.merge_lse([o1, o2], [l1, l2])
    wo, wl, a, _ = ref.tree(nq, cache, table, ctx)
    # three bf16 roundings on the way of the layer's kernels
    within(both, wo[0], 4 * ref.BF16 * (a[0] + wo[0].abs()))
    assert (bl.double() - wl[0]).abs().max() < 1e-3
    # and the cache gives back what the layer built
    rk, rv, rb = cache.read(table, 0, 128, logit_bias=True)
    assert torch.equal(rk[0], layer.ck[2]) and torch.equal(rv[0], layer.cv[2]) and torch.equal(rb[0], layer.cb[2])
    with pytest.raises(ValueError, match="logit bias"):
        layer.write_cache(dk.KvCache.empty(30, 16, hkv, d, "bf16", device=dev()), table, 2, k, v)
    with pytest.raises(ValueError, match="page table"):
        layer.write_cache(cache, table[:, :4], 2, k, v)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_on_a_device_that_is_not_the_current_one():
    d1 = torch.device("cuda", 1)
    x = torch.randn(1, 2, 3, 64, device=d1)
    pos = torch.arange(3, device=d1)
    rot = dk.Rotary(64)
    assert torch.allclose(rot(x, pos).cpu(), rot(x.to(dev()), pos.to(dev())).cpu())
    table = torch.zeros(1, 1, dtype=torch.int32, device=d1)
    cache = dk.KvCache.empty(1, 16, 2, 64, "int8", device=d1)
    cache.write(x, x, table, 0)
    o, _ = dk.tree_attention(x.bfloat16(), cache, table, torch.zeros(1, dtype=torch.int32, device=d1))
    assert o.device == d1 and torch.isfinite(o).all()
