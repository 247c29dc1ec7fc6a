"""Rotary positions without a GPU: the scalings' keys, and what autograd sees."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import dcc_kv_b200 as dk
import decode_ref as ref
from dcc_kv_b200 import _lib as L


@pytest.mark.parametrize("theta,n,extra", [
    (150000.0, 4096, {"factor": 32.0, "truncate": False}), (150000.0, 4096, {"factor": 32.0, "truncate": True}),
    (10000.0, 4096, {"factor": 40.0, "mscale": 1.0, "mscale_all_dim": 1.0}),
    (10000.0, 4096, {"factor": 40.0, "mscale": 0.707, "mscale_all_dim": 1.2}),
    (10000.0, 4096, {"factor": 40.0, "mscale": 0.707}), (10000.0, 4096, {"factor": 40.0, "mscale_all_dim": 1.0}),
    (10000.0, 4096, {"factor": 40.0, "mscale": 1.0, "mscale_all_dim": 1.0, "attention_factor": 1.25}),
    (10000.0, 4096, {"factor": 40.0, "mscale": 0.0, "mscale_all_dim": 1.0}),
    (1000000.0, 32768, {"factor": 4.0, "beta_fast": 32.0, "beta_slow": 1.0, "truncate": False})])
def test_every_yarn_key_agrees_with_transformers(theta, n, extra):
    pytest.importorskip("transformers")
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    scaling = {"rope_type": "yarn", "original_max_position_embeddings": n, "rope_theta": theta, **extra}
    cfg = LlamaConfig(hidden_size=64 * 32, num_attention_heads=32, max_position_embeddings=int(n * extra["factor"]),
                      rope_theta=theta, rope_scaling=dict(scaling), rope_parameters=dict(scaling))
    want, magnitude = ROPE_INIT_FUNCTIONS["yarn"](cfg, "cpu")
    for given in (theta, None):
        f, m = dk.rotary_frequencies(64, given, scaling)
        assert m == pytest.approx(magnitude, rel=1e-7)
        assert torch.tensor(f, dtype=torch.float64) == pytest.approx(want.double(), rel=1e-5)   # theirs are 32-bit
    rot = dk.Rotary(64, scaling=scaling)
    assert rot.theta == theta and rot.magnitude == m and rot.frequencies == f


def test_scaling_keys_that_would_be_dropped_are_refused():
    base = {"factor": 4.0, "original_max_position_embeddings": 4096}
    llama = {"low_freq_factor": 1.0, "high_freq_factor": 4.0}
    for bad in ({"rope_type": "linear", "factor": 4.0, "mscale": 1.0}, {"rope_type": "yarn", "beta": 3.0, **base},
                {"rope_type": "ntk", "factor": 4.0, "alpha": 1000}, {"rope_type": "llama3", "truncate": False, **llama, **base},
                {"rope_type": "default", "factor": 4.0}, {"factor": 4.0}, {"rope_type": "linear", "factor": None},
                {"rope_type": "yarn", "attention_factor": 0.0, **base}, {"rope_type": "default", "mrope_section": [16, 24, 24]}):
        with pytest.raises(ValueError, match="rotary scaling"):
            dk.Rotary(128, scaling=bad)
    with pytest.raises(ValueError, match="rope_theta"):
        dk.Rotary(128, theta=500000.0, scaling={"rope_type": "linear", "factor": 4.0, "rope_theta": 10000.0})
    with pytest.raises(ValueError, match="exceed 1"):
        dk.Rotary(128, scaling={"rope_type": "default", "rope_theta": 0.5})
    with pytest.raises(ValueError, match="partial_rotary_factor"):
        dk.Rotary(128, rotary_dim=32, scaling={"rope_type": "default", "partial_rotary_factor": 0.5})
    rot = dk.Rotary(128, scaling={"rope_type": "default", "partial_rotary_factor": 0.5, "rope_theta": 50000, "factor": None})
    assert rot.rotary_dim == 64 and rot.theta == 50000.0 and len(rot.frequencies) == 32
    assert dk.Rotary(128).theta == 10000.0
    assert dk.Rotary(128, scaling={"type": "linear", **base}).frequencies[0] == 0.25


@pytest.fixture
def on_the_cpu(monkeypatch):
    """The launch replaced by its definition, so that what stands around it runs without a GPU."""
    def run(self, xs, positions, inverse, outs=None):
        p = positions.expand(xs[0].shape[0], -1) if positions.dim() == 1 else positions
        ys = [ref.rotate(x.detach().double(), p, self.frequencies, self.magnitude, self.layout, inverse).to(x.dtype) for x in xs]
        if outs is not None:
            for o, y in zip(outs, ys):
                o.detach().numpy()[...] = y.numpy()   # past autograd, as a launch
        return ys if outs is None else list(outs)
    monkeypatch.setattr(dk.Rotary, "_run", run)
    monkeypatch.setattr(L, "require_cuda", lambda *tensors: None)


def test_forward_mode_tangents(on_the_cpu):
    rot, pos = dk.Rotary(16, rotary_dim=8), torch.arange(3) + 1000
    q, tq = torch.randn(2, 2, 4, 3, 16, dtype=torch.float64)
    k, tk = torch.randn(2, 2, 1, 3, 16, dtype=torch.float64)
    with forward_ad.dual_level():
        a, b = rot(forward_ad.make_dual(q, tq), pos, forward_ad.make_dual(k, tk))
        for y, x, t in ((a, q, tq), (b, k, tk)):
            got = forward_ad.unpack_dual(y)
            assert torch.equal(got.primal, rot(x, pos)) and torch.equal(got.tangent, rot(t, pos))
        a, b = rot(q, pos, forward_ad.make_dual(k, tk))          # one of two
        assert forward_ad.unpack_dual(a).tangent is None or not forward_ad.unpack_dual(a).tangent.any()
        assert torch.equal(forward_ad.unpack_dual(b).tangent, rot(tk, pos))
        assert torch.equal(forward_ad.unpack_dual(rot(forward_ad.make_dual(q, tq), pos)).tangent, rot(tq, pos))
        with torch.no_grad(), pytest.raises(ValueError, match="gradient"):
            rot(forward_ad.make_dual(q, tq), pos, inplace=True)
    assert torch.autograd.gradcheck(lambda x, y: rot(x, pos, y), (q.requires_grad_(), k.requires_grad_()),
                                    check_forward_ad=True, check_backward_ad=True)
    assert torch.autograd.gradgradcheck(lambda x, y: rot(x, pos, y), (q, k), check_fwd_over_rev=True)


def test_inplace_is_seen_by_a_backward_that_saved_the_tensor(on_the_cpu):
    rot, pos = dk.Rotary(16), torch.arange(3)
    w = torch.randn(2, 2, 3, 16, requires_grad=True)
    q, k = torch.randn(2, 2, 2, 3, 16)
    for saved in (q, k):
        y = (w * saved).sum()
        rot(q, pos, k, inplace=True)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    y = (w * q).sum()
    rot(q, pos)
    y.backward()
    with torch.inference_mode():
        rot(torch.randn(1, 1, 3, 16), pos, inplace=True)


def test_rows_that_overlap(monkeypatch):
    """Views whose rows lie one element apart: the result has rows of its own."""
    called = []

    class Library:
        def dcc_rotary(self, arr, n, *rest):
            called.extend((t.y_seq_stride, t.y_head_stride, t.y_row_stride) for t in arr)
            return L.DCC_OK

    monkeypatch.setattr(L, "lib", Library)
    monkeypatch.setattr(L, "require_cuda", lambda *tensors: None)
    monkeypatch.setattr(L, "stream_ptr", lambda device: 0)
    monkeypatch.setattr(L, "on_device", lambda device: torch.no_grad())
    base = torch.zeros(4096)
    rot = dk.Rotary(64)
    for shape, strides in (((1, 3, 5, 64), (0, 70, 1, 1)), ((2, 3, 4, 64), (1000, 100, 1, 1)), ((2, 3, 5, 64), (1, 64, 2, 1)),
                           ((2, 3, 5, 64), (0, 0, 0, 1))):
        y = rot(torch.as_strided(base, shape, strides), torch.arange(shape[2]))
        assert y.shape == shape and y.stride(3) == 1 and called[-1] == y.stride()[:3]
        steps = sorted((s, n) for s, n in zip(y.stride(), shape) if n > 1)
        assert all(s >= n0 * s0 for (s0, n0), (s, _) in zip(steps, steps[1:]))
    x = torch.zeros(2, 5, 3, 64).transpose(1, 2)       # ordinary views keep the order of their axes
    assert rot(x, torch.arange(5)).stride() == x.stride()


def test_inplace_refuses_what_overlaps_itself(on_the_cpu):
    base, rot = torch.zeros(4096), dk.Rotary(64)
    for shape, strides in (((1, 3, 5, 64), (0, 70, 1, 1)), ((2, 3, 4, 64), (1000, 100, 32, 1)), ((2, 3, 5, 64), (320, 320, 64, 1)),
                           ((2, 3, 5, 64), (0, 320, 64, 1)), ((1, 1, 2, 64), (0, 0, 63, 1))):
        with pytest.raises(ValueError, match="overlap"):
            rot(torch.as_strided(base, shape, strides), torch.arange(shape[2]), inplace=True)
    for shape, strides in (((1, 3, 5, 64), (0, 400, 64, 1)), ((2, 3, 5, 64), (64, 640, 128, 1)), ((2, 1, 0, 64), (0, 0, 0, 1)),
                           ((2, 3, 4, 64), (768, 64, 192, 1))):
        x = torch.as_strided(base, shape, strides)
        assert rot(x, torch.arange(shape[2]), inplace=True) is x


def test_copies_of_strided_inputs_live_until_the_launch(monkeypatch):
    """Of queries with another last stride a copy is made; the results of the keys must not take its place."""
    import ctypes as C
    seen = []

    class Library:
        def dcc_rotary(self, arr, n, *rest):
            seen.append([torch.frombuffer(bytearray(C.string_at(t.x, 4 * 64 * 5)), dtype=torch.float32) for t in arr])
            for t in arr:  # what a launch does at once on the CPU
                C.memset(t.y, 0, 4 * 64 * 5)
            return L.DCC_OK

    monkeypatch.setattr(L, "lib", Library)
    monkeypatch.setattr(L, "require_cuda", lambda *tensors: None)
    monkeypatch.setattr(L, "stream_ptr", lambda device: 0)
    monkeypatch.setattr(L, "on_device", lambda device: torch.no_grad())
    real = torch.empty_like
    monkeypatch.setattr(torch, "empty_like", lambda x, **kw: real(x, **kw).fill_(-1))
    rot = dk.Rotary(64)
    for _ in range(8):
        q, k = (torch.randn(64, 1, 1, 5).permute(1, 2, 3, 0) for _ in range(2))
        rot(q, torch.arange(5), k)
        for got, x in zip(seen[-1], (q, k)):
            assert torch.equal(got, x.flatten())
