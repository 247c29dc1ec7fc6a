"""What stands around the launches of the paged cache, without a GPU."""
from __future__ import annotations

import pytest
import torch

import dcc_kv_b200 as dk
from dcc_kv_b200 import _lib as L


class NoLaunch:
    """The library without its launches."""

    def __getattr__(self, name):
        return lambda *args: L.DCC_OK


@pytest.fixture
def no_launch(monkeypatch):
    monkeypatch.setattr(L, "lib", lambda: NoLaunch())
    monkeypatch.setattr(L, "require_cuda", lambda *tensors: None)
    monkeypatch.setattr(L, "stream_ptr", lambda device: 0)
    monkeypatch.setattr(L, "on_device", lambda device: torch.no_grad())


@pytest.mark.parametrize("fmt", ["int8", "f32"])
def test_a_write_is_seen_by_a_backward_that_saved_the_pool(no_launch, fmt):
    cache = dk.KvCache.empty(4, 16, 2, 64, fmt, logit_bias=True, device="cpu")
    k, table = torch.zeros(1, 2, 3, 64), torch.zeros(1, 2, dtype=torch.int32)
    pools = [x for x in (cache.k, cache.v, cache.k_scale, cache.v_scale, cache.logit_bias) if x is not None]
    before = [x._version for x in pools]
    w = torch.ones((), requires_grad=True)
    y = (w * cache.logit_bias).sum()
    cache.read(table, torch.zeros(1, dtype=torch.int32), 3)
    assert [x._version for x in pools] == before
    cache.write(k, k, table, 0)
    assert all(x._version > n for x, n in zip(pools, before))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_a_workspace_that_is_not_aligned_is_refused():
    lib = L.lib()
    pages = L.dcc_kv_pages(256, 256, 256, 256, None, 4, 16, 2, 64, L.DCC_KV_INT8)
    query = L.dcc_tree_query(256, 256, None, 0, 0, 64, 0, 0, 64, 256, None, None, 0, 256, 4, 3, 1, 4, 4, 0)
    need = lib.dcc_tree_attention_workspace_bytes(pages, query, L.DCC_BF16)
    for at in (257, 264, 4096 + 4):
        assert lib.dcc_tree_attention(pages, query, 0.125, L.DCC_BF16, at, need + 16, None) == L.DCC_ERR_INVALID_ARGUMENT
        assert b"aligned" in lib.dcc_last_error()
