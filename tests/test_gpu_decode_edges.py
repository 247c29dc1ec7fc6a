"""Decoding operators on the GPU at the edges of what they take: other streams,
values that are not finite or of extreme size, masks, pools that a caller
filled, and waits that ran out."""
from __future__ import annotations

import math

import pytest
import torch

import dcc_kv_b200 as dk
import decode_ref as ref

from gpu_util import assert_no_device_timeouts, dev
from test_gpu_decode import filled, gen, lens, randn, within

pytestmark = pytest.mark.gpu

# newest tokens, query heads of a KV head: both sides of every rule on rows
ROWS = [(1, 4), (6, 2), (20, 4), (70, 2), (70, 4)]


def packed(g, fmt, b, d, n, k, v, bias=None, page=16):
    """b sequences that read the same n cached tokens (one KV head): one sequence
    is whole in a CTA when b is large."""
    per = -(-n // page)
    cache = dk.KvCache.empty(per, page, 1, d, fmt, logit_bias=bias is not None, device=dev())
    table = torch.arange(per, dtype=torch.int32, device=dev())[None]
    cache.write(k, v, table, 0, logit_bias=bias)
    return cache, table.expand(b, per)


def test_hand_over_on_another_stream_behind_a_host_forward():
    """The compact keys are still being built on the layer's own stream when write_cache is called."""
    from dcc_kv_b200.workloads import layer_inputs
    nb, length, hq, hkv, d = 4, 2048, 8, 2, 128
    layer = dk.DccKvSyncLayer(nb, length, hq, hkv, d, 256, window=64)
    cache = dk.KvCache.empty(300, 16, hkv, d, "bf16", logit_bias=True, device=dev())
    table = torch.arange(300, dtype=torch.int32, device=dev())[None]
    other = torch.cuda.Stream()
    for seed in (3, 4, 3):
        q, k, v = (x.pin_memory() for x in layer_inputs(nb, length, hq, hkv, d, device="cpu", first_seed=seed))
        kd, vd = k.cuda(), v.cuda()
        torch.cuda.synchronize()
        layer(q, k, v)
        with torch.cuda.stream(other):
            layer.write_cache(cache, table, nb - 1, kd, vd)
        torch.cuda.synchronize()
        rk, rv, rb = cache.read(table, 0, layer.total[nb - 1], logit_bias=True)
        for got, want in ((rk, layer.ck), (rv, layer.cv), (rb, layer.cb)):
            assert torch.equal(got[0], want[nb - 1])


# ---- rotary ------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("t", [1, 5, 300])
def test_rotary_of_queries_with_another_last_stride(dtype, t):
    """The copy that is made of them must live until the launch, beside results and copies of its size."""
    g = gen(44)
    rot = dk.Rotary(64)
    pos = torch.arange(t, device=dev()) + 5000
    for _ in range(8):
        q = randn(g, 64, 2, 3, t, dtype=dtype).permute(1, 2, 3, 0)
        for k in (randn(g, 2, 3, t, 64, dtype=dtype), randn(g, 64, 2, 3, t, dtype=dtype).permute(1, 2, 3, 0)):
            a, b = rot(q, pos, k)
            assert torch.equal(a, rot(q.contiguous(), pos)) and torch.equal(b, rot(k.contiguous(), pos))


# ---- attention: values that are not finite -----------------------------------------------------------


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3", "f32"])
@pytest.mark.parametrize("t,group", ROWS)
@pytest.mark.parametrize("at", [0, 300, 777])
def test_a_nan_value_makes_the_rows_that_see_it_nan(fmt, t, group, at):
    """One column of it in the types without a scale; the log-sum-exp is that of the keys."""
    g = gen(31)
    cache, table = filled(g, fmt, 1, 2, 64, 16, 900 + t, outliers=False)
    q = randn(g, 1, 2 * group, t, 64, dtype=torch.bfloat16)
    want = dk.tree_attention(q, cache, table, lens(900))
    k, v = cache.read(table, lens(at), 1, dtype=torch.float32)
    v[..., 5] = math.nan
    cache.write(k, v, table, at)
    o, lse = dk.tree_attention(q, cache, table, lens(900))
    hit = torch.ones(64, dtype=torch.bool, device=dev())
    if fmt in ("bf16", "f32"):
        hit[:] = False
        hit[5] = True
    assert torch.isnan(o[..., hit]).all()
    assert torch.equal(o[..., ~hit], want[0][..., ~hit])
    # the row's max may be up to 2^-100 lower and is then a number below 128: half a step of it and one of the difference
    within(lse, want[1].double(), 2.0 ** -17 * (1 + want[1].double().abs()))


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3", "f32"])
@pytest.mark.parametrize("t,group", ROWS)
@pytest.mark.parametrize("at", [40, 130, 300, 777])
@pytest.mark.parametrize("b", [1, 160])
def test_a_nan_value_counts_however_small_its_weight(fmt, t, group, at, b):
    """Its weight underflows beside keys e^1600 ahead, in the same tile or in another one, of the same CTA or not."""
    g = gen(32)
    n = 900
    k, v = torch.zeros(1, 1, n, 64, device=dev()), randn(g, 1, 1, n, 64)
    k[..., 0] = -800.0
    top = 512 if at != 777 else 16
    k[:, :, top: top + 16, 0] = 800.0
    v[:, :, at] = math.nan
    cache, table = packed(g, fmt, b, 64, n, k, v)
    q = torch.zeros(b, group, t, 64, dtype=torch.bfloat16, device=dev())
    q[..., 0] = 1
    o, lse = dk.tree_attention(q, cache, table, lens(*[n - t] * b), scale=1.0)
    assert torch.isnan(o).all()
    assert torch.isfinite(lse).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,group", ROWS[1:])
@pytest.mark.parametrize("ctx,d", [(140, 64), (1000, 128), (129, 48)])
def test_nan_codes_of_a_pool_filled_elsewhere(dtype, t, group, ctx, d):
    """e4m3 has a NaN code, which write() never leaves: the newest rows that do not see it are unaffected."""
    g = gen(38)
    cache, table = filled(g, "e4m3", 1, 2, d, 16, ctx + t)
    q = randn(g, 1, 2 * group, t, d, dtype=dtype)
    mask = torch.eye(t, dtype=torch.bool, device=dev())
    want = dk.tree_attention(q, cache, table, lens(ctx), tree=mask)
    codes = cache.v.view(torch.uint8)
    for at in (2, t - 1):
        page, off = int(table[0, (ctx + at) // 16]), (ctx + at) % 16
        keep = torch.tensor([i for i in range(t) if i != at], device=dev())
        old = codes[page, :, off].clone()
        for code, col in ((0x7f, 0), (0xff, 7), (0x7f, d - 1)):
            codes[page, :, off, col] = code
            got = dk.tree_attention(q, cache, table, lens(ctx), tree=mask)
            assert torch.equal(got[0][:, :, keep], want[0][:, :, keep])
            assert torch.equal(got[1][:, :, keep], want[1][:, :, keep])
            assert torch.isnan(got[0][:, :, at, col]).all()
            codes[page, :, off] = old


# ---- attention: values of extreme size beside 8-bit codes, whose weights carry the V scale in fp16 ------


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("group", [2, 40, 140])
@pytest.mark.parametrize("b", [1, 160])
@pytest.mark.parametrize("size", [1e-6, 1.0, 1e8])
@pytest.mark.parametrize("low", [torch.finfo(torch.float32).min, -1e30])
def test_biases_at_the_lowest_value_beside_values_of_any_size(fmt, group, b, size, low):
    """All keys alike: the mean of the values, although a logarithm of the V scale is lost beside such scores."""
    g = gen(33)
    n = 400
    k, v = (randn(g, 1, 1, n, 64) for _ in range(2))
    cache, table = packed(g, fmt, b, 64, n, k, v * size, bias=torch.full((1, 1, n), low, device=dev()))
    q = randn(g, b, group, 1, 64, dtype=torch.bfloat16)
    o, lse = dk.tree_attention(q, cache, table, lens(*[n - 1] * b))
    vv = ref.cached(cache, table, 0, n)[1]
    want, a = vv.mean(1), vv.abs().mean(1)
    # the sum and the quotient in 32 bits; the weight's rounding and the result's
    bound = ((n + 20) * ref.F32 + 2.0 ** -20) * a + 2 * ref.BF16 * a
    within(o[:, :, 0], want.expand(b, group, 64), bound.expand(b, group, 64))
    assert torch.isfinite(lse).all()


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("t,group", ROWS)
@pytest.mark.parametrize("b", [1, 160])
@pytest.mark.parametrize("low", [torch.finfo(torch.float32).min, -1e9, -1e8, -3e7, -1e4])
@pytest.mark.parametrize("written", [True, False])
def test_padding_of_zeros_hidden_by_a_large_bias(fmt, t, group, b, low, written):
    """Padded keys whose values are zeros (or were never written: scale 0), whole tiles and single ones."""
    g = gen(43)
    n = 900
    pad = torch.zeros(n, dtype=torch.bool, device=dev())
    pad[:200] = pad[300:433] = pad[512:640] = pad[700:860:2] = True
    k, v, bias = randn(g, 1, 1, n, 64), randn(g, 1, 1, n, 64) * 2.0 ** 12, randn(g, 1, 1, n)
    v[:, :, pad] = 0
    bias[:, :, pad] = low
    cache, table = packed(g, fmt, b, 64, n, k, v, bias=bias)
    if not written and cache.v_scale is not None:
        cache.v_scale.view(-1)[:n][pad] = 0
    q = randn(g, 1, group, t, 64, dtype=torch.bfloat16)
    o, lse = dk.tree_attention(q.expand(b, group, t, 64), cache, table, lens(*[n - t] * b))
    want = ref.tree(q, cache, table, lens(n - t))
    for s in (0, b // 2, b - 1):
        ref.tree_close((o[s: s + 1], lse[s: s + 1]), want, 64, n)
    # only padding is seen: zeros, and the log-sum-exp of the padding
    o, lse = dk.tree_attention(q.expand(b, group, t, 64), cache, table, lens(*[100] * b))
    assert (o == 0).all() and torch.isfinite(lse).all()
    within(lse, torch.full_like(lse, low).double(), 2.0 ** -23 * abs(low) + 100.0)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("t,group", ROWS)
@pytest.mark.parametrize("b", [1, 160])
@pytest.mark.parametrize("size", [2.0 ** 122, 2.0 ** -90])
def test_values_at_the_ends_of_their_type(fmt, t, group, b, size):
    g = gen(34)
    n = 700
    k, v = randn(g, 1, 1, n, 64) * 4, randn(g, 1, 1, n, 64)
    v[:, :, ::7] *= 2.0 ** -20
    cache, table = packed(g, fmt, b, 64, n, k, v * size)
    q = randn(g, 1, group, t, 64, dtype=torch.bfloat16)
    o, lse = dk.tree_attention(q.expand(b, group, t, 64), cache, table, lens(*[n - t] * b))
    want = ref.tree(q, cache, table, lens(n - t))
    for i in (0, b // 2, b - 1):
        ref.tree_close((o[i: i + 1], lse[i: i + 1]), want, 64, n)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("group", [1, 40, 140])
def test_many_small_weights_add_up(fmt, group):
    """One key ahead of 262143 others that weigh 2^-26.3 of it each: 0.3 % in all, in columns of their own.
    fp16 holds each to 2^-25 / 64 of the largest weight at worst."""
    b, n = 200, 262144
    k, v = torch.zeros(1, 1, n, 64, device=dev()), torch.zeros(1, 1, n, 64, device=dev())
    k[..., 0], k[:, :, 0, 0] = 1, -1
    v[..., 1], v[:, :, 0, 1], v[:, :, 0, 0] = 1, 0, 1
    cache, table = packed(gen(35), fmt, b, 64, n, k, v, page=64)
    q = torch.zeros(1, group, 1, 64, dtype=torch.bfloat16, device=dev())
    q[..., 0] = -1
    scale = 13.15 * math.log(2)
    o, _ = dk.tree_attention(q.expand(b, group, 1, 64), cache, table, lens(*[n - 1] * b), scale=scale)
    kk, vv, _ = ref.cached(cache, table, 0, n)
    p = torch.softmax(q[0, :, 0].double() @ kk[0].T * scale, -1)
    want, a = p @ vv[0], p @ vv[0].abs()
    # logits below 2^5 in 32 bits, twice; exponential and sum in 32 bits; the result's rounding
    bound = (2 * 32 * 4 * ref.F32 + 2.0 ** -20) * a + ref.BF16 * want.abs() + n * 2.0 ** -31
    assert (want[:, 1] > 20 * n * 2.0 ** -31).all()
    within(o[:, :, 0], want.expand(b, group, 64), bound.expand(b, group, 64))


# ---- attention: masks, for every number of rows at which another kernel takes the call --------------------


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3", "f32"])
@pytest.mark.parametrize("t,group", ROWS[1:])
@pytest.mark.parametrize("ctx", [140, 1000])
def test_hidden_values_do_not_matter_for_any_number_of_rows(fmt, t, group, ctx):
    """Rows behind the sequence, and drafted keys and values that a row does not see, in every kernel."""
    g = gen(39)
    hkv = 2
    total = ctx + t + 54
    cache, table = filled(g, fmt, 1, hkv, 64, 16, total)
    q = randn(g, 1, hkv * group, t, 64, dtype=torch.bfloat16)
    mask = torch.eye(t, dtype=torch.bool, device=dev())
    want = dk.tree_attention(q, cache, table, lens(ctx), tree=mask)
    ref.tree_close(want, ref.tree(q, cache, table, lens(ctx), mask=mask), 64, ctx + t)
    poison = torch.full((1, hkv, 54, 64), math.nan, device=dev())
    poison[:, :, ::2, 0] = math.inf
    cache.write(poison, poison, table, ctx + t)
    got = dk.tree_attention(q, cache, table, lens(ctx), tree=mask)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for j in (2, t - 1):
        keep = torch.tensor([i for i in range(t) if i != j], device=dev())
        k0, v0 = cache.read(table, lens(ctx + j), 1, dtype=torch.float32)
        for x in (math.nan, math.inf, -math.inf):
            cache.write(torch.zeros(1, hkv, 1, 64, device=dev()), torch.full((1, hkv, 1, 64), x, device=dev()), table, ctx + j)
            got = dk.tree_attention(q, cache, table, lens(ctx), tree=mask)
            assert torch.equal(got[0][:, :, keep], want[0][:, :, keep])
            assert not torch.isfinite(got[0][:, :, j]).any()
            assert torch.equal(got[1][:, :, keep], want[1][:, :, keep])
        cache.write(torch.full((1, hkv, 1, 64), math.nan, device=dev()), torch.zeros(1, hkv, 1, 64, device=dev()), table, ctx + j)
        got = dk.tree_attention(q, cache, table, lens(ctx), tree=mask)
        assert torch.equal(got[0][:, :, keep], want[0][:, :, keep]) and torch.isnan(got[0][:, :, j]).all()
        cache.write(k0, v0, table, ctx + j)
    assert_no_device_timeouts()


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("t,group", [(1, 20), (1, 70), (1, 140), (1, 280)])
def test_hidden_by_bias_for_any_number_of_rows(fmt, t, group):
    """Single keys, whole tiles and all of them hidden by -inf or by the type's lowest value."""
    g = gen(40)
    lowest = torch.finfo(torch.float32).min
    n = 900
    cache, table = filled(g, fmt, 1, 1, 64, 16, n, bias=True)
    q = randn(g, 1, group, 1, 64, dtype=torch.bfloat16)
    k, v, b = cache.read(table, 0, n, dtype=torch.float32, logit_bias=True)
    keep = b.clone()
    at = lens(n - 1)
    b[:, :, ::2] = lowest
    cache.write(k, v, table, 0, logit_bias=b)
    ref.tree_close(dk.tree_attention(q, cache, table, at), ref.tree(q, cache, table, at), 64, n)
    b[:, :, ::2] = -math.inf
    cache.write(k, v, table, 0, logit_bias=b)
    seen = torch.arange(n, device=dev())[None] % 2 == 1
    got = dk.tree_attention(q, cache, table, at)
    cache.write(k, v, table, 0, logit_bias=torch.nan_to_num(b, neginf=0.0))
    ref.tree_close(got, ref.tree(q, cache, table, at, seen_pos=seen), 64, n)
    # only the first tiles hidden, or only the last
    for lo, hi in ((0, 300), (128, 256), (600, n)):
        for x in (lowest, -math.inf):
            b = keep.clone()
            b[:, :, lo:hi] = x
            cache.write(k, v, table, 0, logit_bias=b)
            got = dk.tree_attention(q, cache, table, at)
            cache.write(k, v, table, 0, logit_bias=torch.nan_to_num(b, neginf=0.0))
            s = torch.ones(1, n, dtype=torch.bool, device=dev())
            if x == -math.inf:
                s[:, lo:hi] = False
            ref.tree_close(got, ref.tree(q, cache, table, at, seen_pos=s), 64, n)
    b[:] = lowest
    cache.write(k, v, table, 0, logit_bias=b)
    o, lse = dk.tree_attention(q, cache, table, at)
    vv = ref.cached(cache, table, 0, n)[1]
    want, a = vv.mean(1), vv.abs().mean(1)
    within(o[0, :, 0], want.expand(group, 64), ((n + 20) * ref.F32 + 2.0 ** -20) * a + 2 * ref.BF16 * a)
    assert (lse == lowest).all()
    b[:] = -math.inf
    cache.write(k, v, table, 0, logit_bias=b)
    o, lse = dk.tree_attention(q, cache, table, at)
    assert (o == 0).all() and torch.isinf(lse).all()


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("t,group", ROWS)
@pytest.mark.parametrize("page", [16, 64, 24])
def test_positions_without_a_page_for_any_number_of_rows(fmt, t, group, page):
    g = gen(41)
    n = 1200
    cache, table = filled(g, fmt, 2, 2, 128, page, n)
    per = table.shape[1]
    q = randn(g, 2, 2 * group, t, 128, dtype=torch.bfloat16)
    bad = table.clone()
    bad[0, 2], bad[0, 9], bad[1, 0], bad[1, 5:8] = -1, cache.n_pages, 2147483647, -2147483648
    seen = torch.ones(2, per * page, dtype=torch.bool, device=dev())
    for s, i in ((0, 2), (0, 9), (1, 0), (1, 5), (1, 6), (1, 7)):
        seen[s, i * page: (i + 1) * page] = False
    ctx = lens(n - t, 701)
    got = dk.tree_attention(q, cache, bad, ctx)
    ref.tree_close(got, ref.tree(q, cache, table, ctx, seen_pos=seen), 128, n)
    m = 3 * page
    short = dk.tree_attention(q, cache, table[:, :3].contiguous(), lens(100, 48))
    seen[:] = False
    seen[:, :m] = True
    ref.tree_close(short, ref.tree(q, cache, table, lens(100, 48), seen_pos=seen), 128, n)


@pytest.mark.parametrize("fmt,dtype", [("bf16", torch.bfloat16), ("int8", torch.bfloat16), ("e4m3", torch.bfloat16), ("f32", torch.float32)])
@pytest.mark.parametrize("t,group,b", [(4096, 8, 1), (1200, 16, 2)])
@pytest.mark.parametrize("masked", [False, True])
def test_more_row_tiles_than_a_grid_holds(fmt, dtype, t, group, b, masked):
    """A prompt at once: every CTA takes several tiles of rows, one after the other."""
    g = gen(42)
    cache, table = filled(g, fmt, b, 1, 64, 16, 300 + t)
    q = randn(g, b, group, t, 64, dtype=dtype)
    mask = (torch.rand(t, t, generator=g, device=dev()) < 0.5) if masked else None
    at = lens(*[300, 77][:b])
    got = dk.tree_attention(q, cache, table, at, tree=mask)
    ref.tree_close(got, ref.tree(q, cache, table, at, mask=mask), 64, 300 + t)
    cache.check()


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3", "f32"])
def test_pools_whose_offsets_pass_32_bits(fmt):
    """Pages at the end of a pool of more than 2^32 elements hold, and give, what those of a small pool do."""
    g = gen(45)
    h, d, page, per = 8, 128, 16, 40
    n_pages = 2 ** 32 // (h * d * page) + 2 * per
    tables = [torch.arange(n, dtype=torch.int32, device=dev()).flip(0).view(2, per) for n in (2 * per,)]
    tables.append(tables[0] + (n_pages - 2 * per))
    caches = [dk.KvCache.empty(n, page, h, d, fmt, device=dev()) for n in (2 * per, n_pages)]
    k, v = randn(g, 2, h, 600, d), randn(g, 2, h, 600, d)
    q = randn(g, 2, 4 * h, 20, d, dtype=torch.bfloat16)
    got = []
    for cache, table in zip(caches, tables):
        cache.write(k, v, table, lens(0, 20))
        got.append([*cache.read(table, lens(0, 20), 600, dtype=torch.float32),
                    *dk.tree_attention(q[:, :, :1], cache, table, lens(599, 300)),
                    *dk.tree_attention(q, cache, table, lens(580, 300)),
                    *dk.tree_attention(q[:, :, :2].float(), cache, table, lens(580, 300))])
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_rotary_of_more_than_32_bits_of_bytes():
    rot = dk.Rotary(128)
    t = 2 ** 19 + 33
    x = torch.empty(1, 34, t, 128, dtype=torch.bfloat16, device=dev()).normal_(generator=gen(46))
    pos = torch.arange(t, device=dev())
    y = rot(x, pos)
    for cut in (slice(0, 7), slice(t - 7, t)):
        assert torch.equal(y[:, :, cut], rot(x[:, :, cut].contiguous(), pos[cut]))


# ---- together ----------------------------------------------------------------------------------------


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
def test_a_decoding_step_as_a_graph(fmt):
    """Rotary positions, cache write and attention captured once; lengths and tokens change under the replays."""
    g = gen(47)
    b, hq, hkv, d = 3, 8, 2, 128
    rot = dk.Rotary(d, theta=500000.0)
    caches = [dk.KvCache.empty(60, 16, hkv, d, fmt, device=dev()) for _ in range(2)]
    table = torch.randperm(60, generator=g, device=dev())[:45].to(torch.int32).view(b, 15)
    k, v = (randn(g, b, hkv, 200, d, dtype=torch.bfloat16) for _ in range(2))
    for cache in caches:
        cache.write(k, v, table, 0)
    x = [randn(g, b, h, 1, d, dtype=torch.bfloat16) for h in (hq, hkv, hkv)]
    at = lens(200, 128, 77)

    def step(cache):
        q, k = rot(x[0], at[:, None], x[1])
        cache.write(k, x[2], table, at)
        return dk.tree_attention(q, cache, table, at)

    graph = torch.cuda.CUDAGraph()
    step(caches[0])
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        o, lse = step(caches[0])
    for _ in range(5):
        for t in x:
            t.normal_(generator=g)
        graph.replay()
        want = step(caches[1])
        assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
        at += 1
    for a, c in zip(caches[0].read(table, 0, 240), caches[1].read(table, 0, 240)):
        assert torch.equal(a, c)
    caches[0].check()


# ---- waits that run out ------------------------------------------------------------------------------


def test_a_wait_that_ran_out_reaches_a_program_that_only_decodes():
    """An mbarrier nothing arrives at, 10 ms limit, no fault: the next call raises, the one after it is right again."""
    from dcc_kv_b200 import _lib as L
    g = gen(36)
    cache, table = filled(g, "bf16", 1, 2, 64, 16, 400)
    q = randn(g, 1, 8, 20, 64, dtype=torch.bfloat16)
    want = dk.tree_attention(q, cache, table, lens(300))
    cache.check()
    for _ in range(2):
        L.check(L.lib().dcc_debug_expire_wait(10_000_000, L.stream_ptr(dev())), "debug_expire_wait")
        torch.cuda.synchronize()
        with pytest.raises(L.DccError) as err:
            dk.tree_attention(q, cache, table, lens(300))
        assert err.value.status == L.DCC_ERR_TIMEOUT
        got = dk.tree_attention(q, cache, table, lens(300))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    L.check(L.lib().dcc_debug_expire_wait(10_000_000, L.stream_ptr(dev())), "debug_expire_wait")
    with pytest.raises(L.DccError) as err:
        cache.check()
    assert err.value.status == L.DCC_ERR_TIMEOUT
    cache.check()
    got = dk.tree_attention(q, cache, table, lens(300))   # check() has reported and cleared it
    assert torch.equal(got[0], want[0])


def test_error_report_refusals():
    from dcc_kv_b200 import _lib as L
    word = torch.zeros(1, dtype=torch.int32)
    assert L.lib().dcc_device_error_report(word.data_ptr()) in (L.DCC_ERR_INVALID_ARGUMENT, L.DCC_ERR_CUDA)
    assert L.lib().dcc_device_error_report(word.cuda().data_ptr()) == L.DCC_ERR_INVALID_ARGUMENT


def test_first_call_inside_a_capture():
    """A process whose first attention is captured: nothing that a capture forbids is done."""
    from dcc_kv_b200 import _lib as L
    g = gen(37)
    cache, table = filled(g, "int8", 1, 2, 64, 16, 400)
    q, at = randn(g, 1, 8, 20, 64, dtype=torch.bfloat16), lens(300)
    torch.cuda.synchronize()
    saved = dict(L._reports)
    L._reports.clear()
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o, lse = dk.tree_attention(q, cache, table, at)
        assert not L._reports
    finally:
        L._reports.update(saved)
    graph.replay()
    want = dk.tree_attention(q, cache, table, at)
    assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
    cache.check()
