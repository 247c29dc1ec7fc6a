"""Tree attention where spans hold many key tiles and many pieces, for the row
counts, page sizes and magnitudes at which its kernels change what they do."""
import random

import pytest
import torch

import decode_ref as ref
import dcc_kv_b200 as dk
from gpu_util import assert_no_device_timeouts
from test_gpu_decode import filled, gen, lens, randn, random_tree

pytestmark = pytest.mark.gpu


def check(q, cache, table, at, most, **kw):
    got = dk.tree_attention(q, cache, table, at, tree=kw.get("mask"))
    torch.cuda.synchronize()
    assert_no_device_timeouts()
    ref.tree_close(got, ref.tree(q, cache, table, at, **kw), q.shape[3], most)
    again = dk.tree_attention(q, cache, table, at, tree=kw.get("mask"))
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("b,t,hq,hkv,d,page,ctx,bias", [
    (3, 1, 4, 1, 128, 16, 40000, False), (5, 1, 32, 8, 128, 64, 9000, False), (2, 3, 16, 4, 64, 16, 30000, True),
    (4, 8, 32, 8, 128, 16, 6000, False), (3, 13, 32, 8, 128, 16, 7000, True), (2, 64, 8, 4, 128, 64, 20000, False),
    (1, 64, 32, 8, 128, 64, 40000, False), (2, 70, 16, 4, 64, 8, 9000, True), (40, 20, 8, 4, 128, 16, 700, False),
    (1, 300, 4, 1, 96, 32, 30000, False)])
def test_long_spans(fmt, b, t, hq, hkv, d, page, ctx, bias):
    """Sequences of different lengths, several tiles and pieces a CTA, under a random tree."""
    g, r = gen(5), random.Random(1)
    cache, table = filled(g, fmt, b, hkv, d, page, ctx + t, bias)
    q = randn(g, b, hq, t, d, dtype=torch.bfloat16)
    at = lens(*[ctx - (i * ctx) // (b + 1) for i in range(b)])
    check(q, cache, table, at, ctx + t, mask=random_tree(r, t).cuda() if t > 1 else None)


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("rows", [7, 8, 9, 16, 17, 32, 33, 127, 128, 129, 255, 256, 257])
def test_row_counts_at_which_the_kernel_changes(fmt, rows):
    g = gen(rows)
    cache, table = filled(g, fmt, 2, 1, 128, 24, 1500 + rows, False)
    q = randn(g, 2, 1, rows, 128, dtype=torch.bfloat16)
    check(q, cache, table, lens(1500, 129), 1500 + rows)


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("t", [1, 4, 33])
@pytest.mark.parametrize("page", [8, 24, 40, 136])
def test_pages_that_end_inside_a_tile(fmt, t, page):
    """Also lengths that end on, before and behind the ends of tiles and pages."""
    g = gen(page)
    at = [0, 127 - t if t < 127 else 0, 128, 255, 256, 257, page - 1, page, 1000]
    cache, table = filled(g, fmt, len(at), 2, 64, page, 1000 + t, True)
    q = randn(g, len(at), 8, t, 64, dtype=torch.bfloat16)
    check(q, cache, table, lens(*at), 1000 + t)


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("t", [1, 4, 9])
@pytest.mark.parametrize("up", [-60, 60])
def test_magnitudes(fmt, t, up):
    """Queries of 2^up beside keys of 2^-up; values of 2^-up too, of rows whose
    sizes differ by 2^20.  Powers of two change no rounding of the formula."""
    g = gen(up + 100)
    b, hkv, d, page, n = 2, 2, 128, 16, 900
    per = -(-(n + t) // page)
    cache = dk.KvCache.empty(b * per, page, hkv, d, fmt, device="cuda")
    table = torch.arange(b * per, dtype=torch.int32, device="cuda").view(b, per)
    k = randn(g, b, hkv, n + t, d, dtype=torch.bfloat16) * 2.0 ** -up
    v = randn(g, b, hkv, n + t, d, dtype=torch.bfloat16) * 2.0 ** -up
    v[:, :, ::3] *= 2.0 ** -20
    cache.write(k, v, table, lens(0, 0))
    q = randn(g, b, 8, t, d, dtype=torch.bfloat16) * 2.0 ** up
    check(q, cache, table, lens(n, 77), n + t)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("t", [1, 4, 9])
def test_rows_that_were_never_written_are_zeros(fmt, t):
    """A fresh pool has codes and scales of 0: such keys have logit 0 and value 0."""
    g = gen(3)
    cache = dk.KvCache.empty(40, 16, 2, 128, fmt, device="cuda")
    table = torch.arange(40, dtype=torch.int32, device="cuda").view(1, 40)
    k, v = (randn(g, 1, 2, 200, 128, dtype=torch.bfloat16) for _ in range(2))
    cache.write(k, v, table, lens(100))
    q = randn(g, 1, 8, t, 128, dtype=torch.bfloat16)
    check(q, cache, table, lens(500), 500 + t)


@pytest.mark.parametrize("fmt", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("t", [1, 4, 9, 40])
@pytest.mark.parametrize("d", [16, 32, 48, 80, 112])
def test_head_dims(fmt, t, d):
    g = gen(d)
    cache, table = filled(g, fmt, 2, 2, d, 16, 300 + t, False)
    q = randn(g, 2, 8, t, d, dtype=torch.bfloat16)
    check(q, cache, table, lens(300, 65), 300 + t)


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("t", [1, 40])
def test_pool_or_table_without_pages(fmt, t):
    for pages, width in ((0, 3), (4, 0), (0, 0)):
        cache = dk.KvCache.empty(pages, 16, 2, 64, fmt, device="cuda")
        table = torch.zeros(2, width, dtype=torch.int32, device="cuda")
        o, lse = dk.tree_attention(torch.ones(2, 4, t, 64, dtype=torch.bfloat16, device="cuda"), cache, table, lens(20, 0))
        assert (o == 0).all() and (lse == -float("inf")).all()
        cache.write(torch.ones(2, 2, t, 64, device="cuda"), torch.ones(2, 2, t, 64, device="cuda"), table, 0)
        k, v = cache.read(table, 0, t)
        assert (k == 0).all() == (v == 0).all()
        if width == 0 or pages == 0:
            assert (k == 0).all()
