"""Rotary positions of queries and keys (GPU), with their gradient.

The layer takes queries and keys whose positions are already applied
(hf_attention.py); a program that decodes over a :class:`~dcc_kv_b200.KvCache`
applies them itself, before the keys are written.  One launch turns queries
and keys together:

    rotary = Rotary(128, theta=500000.0, scaling={"rope_type": "llama3", ...})
    q, k = rotary(q, positions, k)
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Mapping, Optional, Tuple, Union

import torch
from torch.autograd import forward_ad

from . import _lib as L

_LAYOUTS = {"half": L.DCC_ROTARY_HALF, "interleaved": L.DCC_ROTARY_INTERLEAVED}


# what each kind of scaling reads; the first ones may stand beside any of them
_KEYS = {"": ("rope_type", "type", "rope_theta", "partial_rotary_factor", "original_max_position_embeddings"),
         "default": (), "linear": ("factor",), "ntk": ("factor",),
         # ("finetuned" says how a model was made, not how it turns)
         "yarn": ("factor", "beta_fast", "beta_slow", "truncate", "attention_factor", "mscale", "mscale_all_dim", "finetuned"),
         "llama3": ("factor", "low_freq_factor", "high_freq_factor")}


def _need(scaling: Mapping, key: str) -> float:
    if scaling.get(key) is None:
        raise ValueError(f"rotary scaling {_kind(scaling)!r} needs {key!r}")
    value = float(scaling[key])
    if not value > 0:
        raise ValueError(f"rotary scaling: {key} must be positive, got {scaling[key]}")
    return value


def _kind(scaling: Mapping) -> str:
    kind = scaling.get("rope_type", scaling.get("type")) or "default"
    if kind not in _KEYS or kind == "":
        raise ValueError(f"unknown rotary scaling {kind!r}; use linear, ntk, yarn or llama3")
    return kind


def _theta(theta: Optional[float], scaling: Optional[Mapping]) -> float:
    """``theta``, or the one that stands in ``scaling``, or 10000."""
    own = None if scaling is None else scaling.get("rope_theta")
    if theta is not None and own is not None and float(own) != float(theta):
        raise ValueError(f"rotary scaling holds rope_theta {own}, theta is {theta}")
    theta = float(theta if theta is not None else own if own is not None else 10000.0)
    if not theta > 1:
        raise ValueError(f"theta must exceed 1, got {theta}")
    return theta


def rotary_frequencies(rotary_dim: int, theta: Optional[float] = None,
                       scaling: Optional[Mapping] = None) -> Tuple[list, float]:
    """Radians per position of each of the ``rotary_dim // 2`` pairs, and the
    magnitude that multiplies the rotated part.  f_i = theta^(-2i / rotary_dim),
    changed for long contexts by ``scaling`` (keys as in a transformers
    ``rope_scaling``; a key that its kind does not read is refused):

    * ``linear``: f / factor (positions interpolated);
    * ``ntk``: the base grows to theta * factor^(r / (r - 2)), which slows the
      slowest pair by the factor and leaves the fastest;
    * ``yarn``: pairs that turn more than ``beta_fast`` (32) times over
      ``original_max_position_embeddings`` keep f, those under ``beta_slow`` (1)
      get f / factor, a linear ramp over the pair index between (from and to
      whole indices unless ``truncate`` is false); magnitude
      ``attention_factor``, else with a(m) = 0.1 m ln(factor) + 1 (1 for a
      factor up to 1) a(``mscale``) / a(``mscale_all_dim``) where both are
      given and not 0, else a(1);
    * ``llama3``: pairs with more than ``high_freq_factor`` turns keep f, those
      under ``low_freq_factor`` get f / factor, a linear ramp over the turns
      between.

    Without ``theta`` the ``rope_theta`` of ``scaling`` holds, else 10000."""
    r = rotary_dim
    theta = _theta(theta, scaling)
    f = [theta ** (-2.0 * i / r) for i in range(r // 2)]
    if scaling is None:
        return f, 1.0
    kind = _kind(scaling)
    unknown = [k for k, x in scaling.items() if x is not None and k not in _KEYS[""] and k not in _KEYS[kind]]
    if unknown:
        raise ValueError(f"rotary scaling {kind!r} does not read {', '.join(map(repr, unknown))}")
    if kind == "default":
        return f, 1.0
    if kind == "linear":
        factor = _need(scaling, "factor")
        return [x / factor for x in f], 1.0
    if kind == "ntk":
        factor = _need(scaling, "factor")
        if r <= 2:
            raise ValueError("rotary scaling 'ntk' needs more than one pair")
        base = theta * factor ** (r / (r - 2.0))
        return [base ** (-2.0 * i / r) for i in range(r // 2)], 1.0
    if kind == "yarn":
        factor, n = _need(scaling, "factor"), _need(scaling, "original_max_position_embeddings")
        fast, slow = float(scaling.get("beta_fast") or 32.0), float(scaling.get("beta_slow") or 1.0)

        def pair_with(turns: float) -> float:
            return r * math.log(n / (2.0 * math.pi * turns)) / (2.0 * math.log(theta))

        def growth(m: float) -> float:
            return 0.1 * m * math.log(factor) + 1.0 if factor > 1 else 1.0

        low, high = pair_with(fast), pair_with(slow)
        if scaling.get("truncate") is None or scaling["truncate"]:
            low, high = math.floor(low), math.ceil(high)
        low, high = max(low, 0), min(high, r - 1)
        width = max(high - low, 1e-3)
        slowed = [min(max((i - low) / width, 0.0), 1.0) for i in range(r // 2)]
        if scaling.get("attention_factor") is not None:
            magnitude = _need(scaling, "attention_factor")
        elif scaling.get("mscale") and scaling.get("mscale_all_dim"):
            magnitude = growth(float(scaling["mscale"])) / growth(float(scaling["mscale_all_dim"]))
        else:
            magnitude = growth(1.0)
        return [x / factor * s + x * (1.0 - s) for x, s in zip(f, slowed)], magnitude
    factor, n = _need(scaling, "factor"), _need(scaling, "original_max_position_embeddings")
    low, high = _need(scaling, "low_freq_factor"), _need(scaling, "high_freq_factor")
    if not high > low:
        raise ValueError("rotary scaling 'llama3': high_freq_factor must exceed low_freq_factor")
    out = []
    for x in f:
        kept = min(max((n * x / (2.0 * math.pi) - low) / (high - low), 0.0), 1.0)
        out.append(x / factor * (1.0 - kept) + x * kept)
    return out, 1.0


class Rotary:
    """Rotary positions of one kind of head: pairs (i, i + r/2) of the first
    r = ``rotary_dim`` elements (``layout="half"``) or (2i, 2i + 1)
    (``"interleaved"``); the rest of the head is passed through.  See
    :func:`rotary_frequencies` for ``theta`` and ``scaling``; a
    ``partial_rotary_factor`` of the latter is r / ``head_dim``."""

    def __init__(self, head_dim: int, rotary_dim: Optional[int] = None, theta: Optional[float] = None,
                 layout: str = "half", scaling: Optional[Mapping] = None):
        part = None if scaling is None else scaling.get("partial_rotary_factor")
        if part is not None:
            part = int(head_dim * part)
            if rotary_dim not in (None, part):
                raise ValueError(f"rotary scaling holds partial_rotary_factor {scaling['partial_rotary_factor']}, "
                                 f"rotary_dim is {rotary_dim} of {head_dim}")
        r = rotary_dim if rotary_dim is not None else part if part is not None else head_dim
        if r < 2 or r % 2 or r > head_dim:
            raise ValueError(f"rotary_dim must be even and within the head of {head_dim}, got {r}")
        if r > 256:
            raise ValueError(f"rotary_dim up to 256 is supported, got {r}")
        if layout not in _LAYOUTS:
            raise ValueError(f"layout must be 'half' or 'interleaved', got {layout!r}")
        self.head_dim, self.rotary_dim, self.theta, self.layout = head_dim, r, _theta(theta, scaling), layout
        self.frequencies, self.magnitude = rotary_frequencies(r, self.theta, scaling)
        self._turns = (C.c_double * (r // 2))(*[f / (2.0 * math.pi) for f in self.frequencies])

    def _check(self, x: torch.Tensor, positions: torch.Tensor, first: torch.Tensor, name: str) -> None:
        if x.dim() != 4 or x.shape[-1] != self.head_dim:
            raise ValueError(f"{name} must be [batch, heads, tokens, {self.head_dim}], got {tuple(x.shape)}")
        if x.shape[0] != first.shape[0] or x.shape[2] != first.shape[2]:
            raise ValueError(f"{name} {tuple(x.shape)} and q {tuple(first.shape)} differ in batch or tokens")
        if x.dtype != first.dtype:
            raise ValueError(f"{name} is {x.dtype}, q is {first.dtype}")

    def _run(self, xs, positions: torch.Tensor, inverse: bool, outs=None):
        dev = xs[0].device
        b, _, t, d = xs[0].shape
        arr = (L.dcc_rotary_tensor * len(xs))()
        ys, held = [], []  # held: copies that the launch reads stay until it is made
        for i, x in enumerate(xs):
            sx = x.stride()
            if sx[3] != 1 and d > 1:
                x = x.contiguous()
                held.append(x)
                sx = x.stride()
            if outs is not None:
                y, sy = outs[i], sx
            else:
                y = torch.empty_like(x)  # keeps the order of the axes, but not always a unit last stride of rows that overlap
                sy = y.stride()
                if sy[3] != 1:
                    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
                    sy = y.stride()
            arr[i] = (x.data_ptr(), y.data_ptr(), *sx[:3], *sy[:3], x.shape[1])
            ys.append(y)
        code = L.dtype_code(xs[0])
        ps = positions.stride() if positions.dim() == 2 else (0, positions.stride(0))
        with L.on_device(dev):
            L.check(L.lib().dcc_rotary(arr, len(xs), positions.data_ptr(), positions.dtype == torch.int64,
                                       ps[0], ps[1], b, t, d, self.rotary_dim // 2, self._turns, self.magnitude,
                                       _LAYOUTS[self.layout], inverse, code, L.stream_ptr(dev)), "rotary")
        return ys

    def __call__(self, q: torch.Tensor, positions: torch.Tensor, k: Optional[torch.Tensor] = None,
                 inplace: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
        """q [B, H_q, T, d] and, optionally, k [B, H_kv, T, d] (float32,
        float64 or bfloat16, any strides); positions [T] or [B, T], int32 or
        int64.  Returns the rotated q, or (q, k).  Differentiable in q and k.
        ``inplace`` writes over q and k (no gradient)."""
        self._check(q, positions, q, "q")
        if k is not None:
            self._check(k, positions, q, "k")
        if positions.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"positions must be int32 or int64, got {positions.dtype}")
        if positions.shape not in ((q.shape[2],), (q.shape[0], q.shape[2])):
            raise ValueError(f"positions must be [{q.shape[2]}] or [{q.shape[0]}, {q.shape[2]}], "
                             f"got {tuple(positions.shape)}")
        L.dtype_code(q)
        L.require_cuda(q, positions, k)
        L.same_device(q.device, positions=positions, k=k)
        xs = (q,) if k is None else (q, k)
        if inplace:
            if _differentiated(xs):
                raise ValueError("inplace rotary positions have no gradient; run without inplace")
            for x in xs:
                if x.stride(3) != 1 or _overlaps(x):
                    raise ValueError("inplace needs tensors with unit last stride that are not expanded and do not overlap themselves")
            ys = self._run(xs, positions, False, outs=xs)
            L.written(*xs)
        else:
            ys = self._map(xs, positions, False)
        return ys[0] if k is None else (ys[0], ys[1])

    def _map(self, xs, positions: torch.Tensor, inverse: bool):
        if _differentiated(xs):
            return _RotaryFunction.apply(self, positions, inverse, *xs)
        return self._run(xs, positions, inverse)


def _overlaps(x: torch.Tensor) -> bool:
    """Two indices of x may be one element: an axis steps by no more than what the axes below it span."""
    span = 0
    for stride, n in sorted((s, n) for s, n in zip(x.stride(), x.shape) if n > 1):
        if stride <= span:
            return x.numel() > 0
        span += stride * (n - 1)
    return False


def _differentiated(xs) -> bool:
    """Autograd follows what happens to one of them, in reverse or forward mode."""
    if torch.is_grad_enabled():
        for x in xs:
            if x.requires_grad:
                return True
    if forward_ad._current_level < 0:  # outside of every dual_level()
        return False
    return any(forward_ad.unpack_dual(x).tangent is not None for x in xs)


class _RotaryFunction(torch.autograd.Function):
    """The map is linear: it is its own derivative, and its gradient is the map
    with the angles negated."""

    @staticmethod
    def forward(ctx, rotary: Rotary, positions: torch.Tensor, inverse: bool, *xs):
        ctx.rotary, ctx.inverse = rotary, inverse
        ctx.save_for_backward(positions)
        ctx.save_for_forward(positions)
        return tuple(rotary._run(xs, positions, inverse))

    @staticmethod
    def jvp(ctx, _rotary, _positions, _inverse, *tangents):
        (positions,) = ctx.saved_tensors
        ys = iter(ctx.rotary._map([t for t in tangents if t is not None], positions, ctx.inverse))
        return tuple(None if t is None else next(ys) for t in tangents)

    @staticmethod
    def backward(ctx, *grads):
        (positions,) = ctx.saved_tensors
        wanted = [i for i in range(len(grads)) if ctx.needs_input_grad[3 + i]]
        out = [None] * len(grads)
        if wanted:
            for i, y in zip(wanted, ctx.rotary._map([grads[i] for i in wanted], positions, not ctx.inverse)):
                out[i] = y
        return (None, None, None, *out)
