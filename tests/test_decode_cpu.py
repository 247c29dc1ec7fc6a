"""The decoding operators without a GPU: their host arithmetic, and what they
refuse before anything is launched."""
from __future__ import annotations

import copy
import ctypes as C
import math

import pytest
import torch

import dcc_kv_b200 as dk
from dcc_kv_b200 import _lib as L


def test_struct_layouts():
    for cls in (L.dcc_rotary_tensor, L.dcc_kv_pages, L.dcc_kv_tokens, L.dcc_tree_query):
        assert L.lib().dcc_struct_size(cls.__name__.encode()) == C.sizeof(cls), cls.__name__


def test_frequencies():
    f, m = dk.rotary_frequencies(8, 10000.0)
    assert m == 1.0 and f == pytest.approx([1.0, 0.1, 0.01, 0.001], rel=1e-15)
    assert dk.rotary_frequencies(8, 10000.0, {"rope_type": "default"}) == (f, 1.0)
    lin, _ = dk.rotary_frequencies(8, 10000.0, {"rope_type": "linear", "factor": 4})
    assert lin == pytest.approx([x / 4 for x in f], rel=1e-15)
    ntk, _ = dk.rotary_frequencies(8, 10000.0, {"type": "ntk", "factor": 4})
    assert ntk[0] == 1.0 and ntk[-1] == pytest.approx(f[-1] / 4, rel=1e-12)


@pytest.mark.parametrize("kind,extra", [("llama3", {"low_freq_factor": 1.0, "high_freq_factor": 4.0}), ("yarn", {}),
                                        ("yarn", {"beta_fast": 16.0, "beta_slow": 2.0, "attention_factor": 1.5})])
def test_frequencies_agree_with_transformers(kind, extra):
    pytest.importorskip("transformers")
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    scaling = {"rope_type": kind, "factor": 8.0, "original_max_position_embeddings": 8192, "rope_theta": 500000.0, **extra}
    cfg = LlamaConfig(hidden_size=4096, num_attention_heads=32, max_position_embeddings=65536, rope_theta=500000.0,
                      rope_scaling=dict(scaling), rope_parameters=dict(scaling))
    want, magnitude = ROPE_INIT_FUNCTIONS[kind](cfg, "cpu")
    f, m = dk.rotary_frequencies(128, 500000.0, scaling)
    assert m == pytest.approx(magnitude, rel=1e-7)
    assert torch.tensor(f, dtype=torch.float64) == pytest.approx(want.double(), rel=1e-5)   # theirs are 32-bit


def test_rotary_refusals():
    for bad in (dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=130), dict(layout="other"), dict(theta=1.0),
                dict(scaling={"rope_type": "other"}), dict(scaling={"rope_type": "linear"}),
                dict(scaling={"rope_type": "linear", "factor": -1.0}), dict(scaling={"rope_type": "yarn", "factor": 4.0}),
                dict(rotary_dim=2, scaling={"rope_type": "ntk", "factor": 4.0}),
                dict(scaling={"rope_type": "llama3", "factor": 8, "low_freq_factor": 4, "high_freq_factor": 4,
                              "original_max_position_embeddings": 8192})):
        with pytest.raises(ValueError):
            dk.Rotary(128, **bad)
    with pytest.raises(ValueError):
        dk.Rotary(512)
    rot = dk.Rotary(64)
    x, pos = torch.zeros(2, 4, 3, 64), torch.arange(3)
    for q, p, k in ((x[..., :32], pos, None), (x[0], pos, None), (x, pos.float(), None), (x, pos[:2], None),
                    (x, pos[None], None), (x, pos, x[:1]), (x, pos, x[:, :, :2]), (x, pos, x.double()),
                    (x.half(), pos, None)):
        with pytest.raises(ValueError):
            rot(q, p, k)
    with pytest.raises(ValueError, match="CUDA"):
        rot(x, pos)


def test_tree_mask():
    m = dk.tree_mask([-1, 0, 0, 2, -1])
    assert m.int().tolist() == [[1, 0, 0, 0, 0], [1, 1, 0, 0, 0], [1, 0, 1, 0, 0], [1, 0, 1, 1, 0], [0, 0, 0, 0, 1]]
    assert dk.tree_mask([]).shape == (0, 0)
    for bad in ([0], [-1, 1], [-2], [-1, 5]):
        with pytest.raises(ValueError):
            dk.tree_mask(bad)


def cache(fmt="int8", **kw):
    return dk.KvCache.empty(4, 16, 2, 64, fmt, device="cpu", **kw)


def test_cache_refusals():
    for bad in ((4, 0, 2, 64, "int8"), (4, 16, 0, 64, "int8"), (4, 16, 2, 129, "int8"), (4, 16, 2, 0, "int8"),
                (4, 16, 2, 64, "int4"), (-1, 16, 2, 64, "int8")):
        with pytest.raises(ValueError):
            dk.KvCache.empty(*bad, device="cpu")
    c = cache()
    with pytest.raises(ValueError):
        dk.KvCache(c.k, c.v)                                  # int8 without scales
    with pytest.raises(ValueError):
        dk.KvCache(c.k.float(), c.v.float(), c.k_scale, c.v_scale)
    with pytest.raises(ValueError):
        dk.KvCache(c.k, c.v[:2], c.k_scale, c.v_scale)
    with pytest.raises(ValueError):
        dk.KvCache(c.k, c.v, c.k_scale.double(), c.v_scale)
    with pytest.raises(ValueError):
        dk.KvCache(c.k, c.v, c.k_scale, c.v_scale, c.k_scale[:, :1])
    with pytest.raises(ValueError):
        dk.KvCache(c.k.transpose(0, 1).contiguous().transpose(0, 1), c.v, c.k_scale, c.v_scale)
    assert (c.n_pages, c.page_size, c.n_kv_heads, c.head_dim) == (4, 16, 2, 64)
    k, table = torch.zeros(1, 2, 3, 64), torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        c.write(k, k, table, 0)
    with pytest.raises(ValueError, match="CUDA"):
        c.read(table, 0, 3)
    for bad in (k[0], k[:, :1], k[..., :32], k.double(), k.half()):
        with pytest.raises(ValueError):
            c.write(bad, bad, table, 0)
    with pytest.raises(ValueError):
        c.write(k, k.bfloat16(), table, 0)
    with pytest.raises(ValueError):
        c.read(table, 0, 3, dtype=torch.float64)
    with pytest.raises(ValueError):
        c.read(table, 0, -1)


def test_index_tensor_refusals():
    from dcc_kv_b200.kv_cache import check_table
    c, table, one = cache(), torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    check_table(c, 2, page_table=table, start=one, counts=None)
    for bad in (table.long(), table[0], table[:1], table.T.contiguous().T):
        with pytest.raises(ValueError):
            check_table(c, 2, page_table=bad, start=one)
    for bad in (one.long(), one[:1], one[None], torch.zeros(4, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError):
            check_table(c, 2, page_table=table, start=bad)


def test_tree_attention_refusals():
    c, table, ctx = cache(), torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    q = torch.zeros(1, 4, 3, 64)
    for bad in (q[0], q[..., :32], q.double(), q.half(), q[:, :3], q[:, :0]):
        with pytest.raises(ValueError):
            dk.tree_attention(bad, c, table, ctx)
    for bad in (torch.ones(3, 3), torch.ones(2, 2, dtype=torch.bool), torch.ones(2, 3, 3, dtype=torch.bool)):
        with pytest.raises(ValueError):
            dk.tree_attention(q, c, table, ctx, tree=bad)
    with pytest.raises(ValueError, match="CUDA"):
        dk.tree_attention(q, c, table, ctx)


def test_c_entries_refuse_before_a_device_is_touched():
    lib = L.lib()
    turns = (C.c_double * 4)(1, 1, 1, 1)
    one = (L.dcc_rotary_tensor * 1)()
    one[0] = (256, 256, 8, 8, 8, 8, 8, 8, 1)

    def rotary(tensors=one, n=1, pos=256, b=1, t=1, d=8, freqs=4, tr=turns, layout=0, dtype=1):
        return lib.dcc_rotary(tensors, n, pos, 1, 0, 1, b, t, d, freqs, tr, 1.0, layout, 0, dtype, None)

    assert rotary(n=0) == rotary(n=3) == rotary(tensors=None) == rotary(tr=None) == L.DCC_ERR_INVALID_ARGUMENT
    assert rotary(layout=2) == rotary(pos=None) == rotary(b=-1) == L.DCC_ERR_INVALID_ARGUMENT
    assert rotary(freqs=5) == rotary(freqs=0) == L.DCC_ERR_UNSUPPORTED
    assert rotary(dtype=9) == L.DCC_ERR_DTYPE
    assert rotary(b=0) == rotary(t=0) == L.DCC_OK

    pages = L.dcc_kv_pages(256, 256, 256, 256, None, 4, 16, 2, 64, L.DCC_KV_INT8)
    tok = L.dcc_kv_tokens(256, 256, None, 0, 0, 64, 0, 0, 64, 0, 0, 256, None, 256, 4, 3, 1, 4)
    for fn in (lib.dcc_kv_cache_write, lib.dcc_kv_cache_read):
        assert fn(None, tok, 1, None) == fn(pages, None, 1, None) == L.DCC_ERR_INVALID_ARGUMENT
        assert fn(pages, tok, L.DCC_F64, None) == L.DCC_ERR_DTYPE
        for key, value, status in (("format", 9, L.DCC_ERR_DTYPE), ("head_dim", 129, L.DCC_ERR_UNSUPPORTED),
                                   ("page_size", 0, L.DCC_ERR_INVALID_ARGUMENT), ("k_scale", None, L.DCC_ERR_INVALID_ARGUMENT)):
            bad = L.dcc_kv_pages.from_buffer_copy(pages)
            setattr(bad, key, value)
            assert fn(bad, tok, 1, None) == status, key
        for key, value in (("T", -1), ("n_seqs", -1), ("k", None), ("start", None), ("page_table", None)):
            bad = L.dcc_kv_tokens.from_buffer_copy(tok)
            setattr(bad, key, value)
            assert fn(pages, bad, 1, None) == L.DCC_ERR_INVALID_ARGUMENT, key
    biased = L.dcc_kv_tokens.from_buffer_copy(tok)
    biased.bias = 256
    assert lib.dcc_kv_cache_write(pages, biased, 1, None) == L.DCC_ERR_INVALID_ARGUMENT

    query = L.dcc_tree_query(256, 256, None, 0, 0, 64, 0, 0, 64, 256, None, None, 0, 256, 4, 3, 1, 4, 4, 0)
    need = lib.dcc_tree_attention_workspace_bytes(pages, query, 1)
    assert need > 0

    def tree(q=query, c=pages, dtype=1, ws=256, n=need):
        return lib.dcc_tree_attention(c, q, 0.125, dtype, ws, n, None)

    assert tree(q=None) == tree(c=None) == L.DCC_ERR_INVALID_ARGUMENT
    assert tree(dtype=L.DCC_F64) == L.DCC_ERR_DTYPE
    assert tree(n=need - 1) == tree(ws=None) == L.DCC_ERR_WORKSPACE
    for key, value, status in (("n_q_heads", 3, L.DCC_ERR_INVALID_ARGUMENT), ("T", 4097, L.DCC_ERR_UNSUPPORTED),
                               ("T", -1, L.DCC_ERR_INVALID_ARGUMENT), ("context", None, L.DCC_ERR_INVALID_ARGUMENT),
                               ("page_table", None, L.DCC_ERR_INVALID_ARGUMENT), ("q", None, L.DCC_ERR_INVALID_ARGUMENT)):
        bad = L.dcc_tree_query.from_buffer_copy(query)
        setattr(bad, key, value)
        assert tree(q=bad) == status, key
    empty = L.dcc_tree_query.from_buffer_copy(query)
    empty.T = 0
    assert tree(q=empty, ws=None, n=0) == L.DCC_OK
    assert math.isfinite(need)


def test_a_copied_cache_points_at_its_own_tensors():
    cache = dk.KvCache.empty(2, 8, 1, 16, device="cpu")
    other = copy.deepcopy(cache)
    assert other.k.data_ptr() != cache.k.data_ptr()
    assert other._pages.k == other.k.data_ptr() and other._pages.v_scale == other.v_scale.data_ptr()
