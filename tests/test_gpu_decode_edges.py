"""Decoding operators on the GPU at the edges of what they take: other streams,
values that are not finite or of extreme size, masks, pools that a caller
filled, and waits that ran out."""
from __future__ import annotations

import pytest
import torch

import dcc_kv_b200 as dk

from gpu_util import dev

pytestmark = pytest.mark.gpu


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
