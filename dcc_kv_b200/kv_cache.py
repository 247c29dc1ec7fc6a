"""A paged KV cache that is quantised as it is written (GPU).

What decoding needs behind the prefill: the keys and values of every earlier
token -- or, behind :class:`~dcc_kv_b200.DccKvSyncLayer`, the compact blocks with
their logit bias and the local block (``DccKvSyncLayer.write_cache``) -- read
again for every new token by :func:`~dcc_kv_b200.tree_attention`.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple, Union

import torch

from . import _lib as L

_FORMATS = {torch.bfloat16: L.DCC_KV_BF16, torch.float32: L.DCC_KV_F32, torch.int8: L.DCC_KV_INT8,
            torch.float8_e4m3fn: L.DCC_KV_E4M3}
_NAMES = {"bf16": torch.bfloat16, "f32": torch.float32, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
_SCALED = (torch.int8, torch.float8_e4m3fn)


@dataclass(frozen=True)
class KvCache:
    """Pages of ``page_size`` tokens of every KV head.  ``k``, ``v``
    [n_pages, H_kv, page_size, d] hold codes; int8 and e4m3 codes have one
    float32 scale per token and KV head in ``k_scale``, ``v_scale``
    [n_pages, H_kv, page_size] (value = code * scale, scale >= 0).  ``logit_bias``, of the
    scales' shape, is added to the logits of a key, as for compact keys.
    Which pages a sequence owns is the caller's: every call takes a page table
    [B, max_pages] (int32), position p of a sequence being row p % page_size
    of its page p // page_size."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: Optional[torch.Tensor] = None
    v_scale: Optional[torch.Tensor] = None
    logit_bias: Optional[torch.Tensor] = None

    def __post_init__(self):
        k = self.k
        if k.dim() != 4 or self.v.shape != k.shape:
            raise ValueError("k and v must be [n_pages, H_kv, page_size, d], with one shape")
        if k.dtype not in _FORMATS or self.v.dtype != k.dtype:
            raise ValueError(f"k and v must share a dtype of bfloat16, float32, int8 or float8_e4m3fn; got {k.dtype}, "
                             f"{self.v.dtype}")
        if not 1 <= k.shape[3] <= 128 or k.shape[2] < 1 or k.shape[1] < 1:
            raise ValueError("need a page_size and KV heads of at least 1 and a head_dim in [1, 128]; "
                             f"got k {tuple(k.shape)}")
        scaled = k.dtype in _SCALED
        for name, t in (("k_scale", self.k_scale), ("v_scale", self.v_scale), ("logit_bias", self.logit_bias)):
            if name != "logit_bias" and (t is not None) != scaled:
                raise ValueError(f"{name} comes with int8 and float8_e4m3fn codes, and only with them")
            if t is not None and (t.dtype != torch.float32 or t.shape != k.shape[:3]):
                raise ValueError(f"{name} must be float32 {tuple(k.shape[:3])}")
        for t in (k, self.v, self.k_scale, self.v_scale, self.logit_bias):
            if t is not None and (t.device != k.device or not t.is_contiguous()):
                raise ValueError("the tensors of a cache must be contiguous and on one device")

    @property
    def _pages(self) -> L.dcc_kv_pages:
        """The C struct: its sizes are made once, its pointers are those of now."""
        k, p = self.k, self.__dict__.get("_struct")
        if p is None:
            p = L.dcc_kv_pages(None, None, None, None, None, k.shape[0], k.shape[2], k.shape[1], k.shape[3],
                               _FORMATS[k.dtype])
            object.__setattr__(self, "_struct", p)
        p.k, p.v = k.data_ptr(), self.v.data_ptr()
        if self.k_scale is not None:
            p.k_scale, p.v_scale = self.k_scale.data_ptr(), self.v_scale.data_ptr()
        if self.logit_bias is not None:
            p.bias = self.logit_bias.data_ptr()
        return p

    def __getstate__(self):
        return {name: x for name, x in self.__dict__.items() if name != "_struct"}

    @classmethod
    def empty(cls, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int, fmt: str = "int8",
              logit_bias: bool = False, device: Union[str, torch.device] = "cuda") -> "KvCache":
        """A cache without tokens.  ``fmt``: "int8", "e4m3", "bf16" or "f32"."""
        if fmt not in _NAMES:
            raise ValueError(f"fmt must be one of {', '.join(_NAMES)}, got {fmt!r}")
        if n_pages < 0:
            raise ValueError("n_pages must not be negative")
        dt, shape = _NAMES[fmt], (n_pages, n_kv_heads, page_size, head_dim)

        def side(wanted):
            return torch.zeros(shape[:3], dtype=torch.float32, device=device) if wanted else None

        return cls(torch.zeros(shape, dtype=dt, device=device), torch.zeros(shape, dtype=dt, device=device),
                   side(dt in _SCALED), side(dt in _SCALED), side(logit_bias))

    @property
    def n_pages(self) -> int:
        return self.k.shape[0]

    @property
    def n_kv_heads(self) -> int:
        return self.k.shape[1]

    @property
    def page_size(self) -> int:
        return self.k.shape[2]

    @property
    def head_dim(self) -> int:
        return self.k.shape[3]

    @property
    def device(self) -> torch.device:
        return self.k.device

    def _tokens(self, k, v, bias, page_table, start, counts, b: int, t: int) -> L.dcc_kv_tokens:
        check_table(self, b, page_table=page_table, start=start, counts=counts)
        s = bias.stride() if bias is not None else (0, 0)
        return L.dcc_kv_tokens(k.data_ptr(), v.data_ptr(), L.ptr(bias), *k.stride()[:3], *v.stride()[:3], s[0], s[1],
                               start.data_ptr(), L.ptr(counts), page_table.data_ptr(), page_table.stride(0), t, b,
                               page_table.shape[1])

    def write(self, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor,
              start: Union[int, torch.Tensor], counts: Optional[torch.Tensor] = None,
              logit_bias: Optional[torch.Tensor] = None) -> None:
        """Tokens t < counts[s] (all, without ``counts``) of k, v
        [B, H_kv, T, d] (bfloat16 or float32, any strides) to positions
        start[s] + t of sequence s.  ``start`` [B] int32, or one int for all;
        ``counts`` [B] int32; ``logit_bias`` [B, H_kv, T] float32 (zeros when
        the cache has a bias and none is given).  Tokens without a page --
        a position below zero or behind the table, a page number outside the
        cache -- are skipped.  The positions written by one call must lie in
        different rows: two sequences that share a page are read together, not
        written together."""
        b, t = self._check_rows(k, v)
        L.require_cuda(k, v, page_table)
        if k.stride(3) != 1:
            k = k.contiguous()
        if v.stride(3) != 1:
            v = v.contiguous()
        if logit_bias is not None:
            if self.logit_bias is None:
                raise ValueError("this cache holds no logit bias; make it with logit_bias=True")
            if logit_bias.shape != k.shape[:3] or logit_bias.dtype != torch.float32:
                raise ValueError(f"logit_bias must be float32 {tuple(k.shape[:3])}")
            L.same_device(self.device, logit_bias=logit_bias)
            logit_bias = logit_bias.contiguous() if logit_bias.stride(2) != 1 else logit_bias
        dev = self.k.device
        L.same_device(dev, k=k, v=v)
        with L.on_device(dev):
            start = self._start(start, b)
            tok = self._tokens(k, v, logit_bias, page_table, start, counts, b, t)
            L.check(L.lib().dcc_kv_cache_write(self._pages, tok, L.dtype_code(k), L.stream_ptr(dev)), "kv_cache_write")
        L.written(self.k, self.v, self.k_scale, self.v_scale, self.logit_bias)

    def read(self, page_table: torch.Tensor, start: Union[int, torch.Tensor], length: int,
             counts: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.bfloat16,
             logit_bias: bool = False) -> Tuple[torch.Tensor, ...]:
        """The values (code * scale in float32, then rounded to ``dtype``,
        bfloat16 or float32) of positions start[s] .. start[s] + length: (k, v)
        [B, H_kv, length, d], and the logit bias [B, H_kv, length] when asked
        for.  Zeros where a sequence has no page and behind counts[s]."""
        if dtype not in (torch.bfloat16, torch.float32):
            raise ValueError(f"the cache is read as bfloat16 or float32, got {dtype}")
        if length < 0:
            raise ValueError("length must not be negative")
        L.require_cuda(self.k, page_table)
        with L.on_device(self.device):
            b = page_table.shape[0]
            shape = (b, self.n_kv_heads, length, self.head_dim)
            k = torch.empty(shape, dtype=dtype, device=self.device)
            v = torch.empty(shape, dtype=dtype, device=self.device)
            bias = torch.empty(shape[:3], dtype=torch.float32, device=self.device) if logit_bias else None
            tok = self._tokens(k, v, bias, page_table, self._start(start, b), counts, b, length)
            L.check(L.lib().dcc_kv_cache_read(self._pages, tok, L.dtype_code(k), L.stream_ptr(self.device)),
                    "kv_cache_read")
        return (k, v, bias) if logit_bias else (k, v)

    def check(self) -> None:
        """Synchronises the device and raises ``DccError(DCC_ERR_TIMEOUT)`` if a
        bounded device wait of any :func:`~dcc_kv_b200.tree_attention` on it so
        far gave up (each call also reports the ones before it)."""
        L.require_cuda(self.k)
        L.check_give_ups(self.device, "tree_attention")

    def _check_rows(self, k: torch.Tensor, v: torch.Tensor) -> Tuple[int, int]:
        if k.dim() != 4 or k.shape[1] != self.n_kv_heads or k.shape[3] != self.head_dim or v.shape != k.shape:
            raise ValueError(f"k and v must be [B, {self.n_kv_heads}, T, {self.head_dim}]; got {tuple(k.shape)}, "
                             f"{tuple(v.shape)}")
        if k.dtype != v.dtype or k.dtype not in (torch.bfloat16, torch.float32):
            raise ValueError(f"k and v must share bfloat16 or float32; got {k.dtype}, {v.dtype}")
        return k.shape[0], k.shape[2]

    def _start(self, start: Union[int, torch.Tensor], b: int) -> torch.Tensor:
        if isinstance(start, int):
            return torch.full((b,), start, dtype=torch.int32, device=self.device)
        return start


def check_table(cache: KvCache, b: int, page_table: torch.Tensor, **per_seq: Optional[torch.Tensor]) -> None:
    """The index tensors that go with a cache: page_table [b, max_pages] and
    one value per sequence, all int32 on the cache's device."""
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[0] != b:
        raise ValueError(f"page_table must be int32 [{b}, max_pages]; got {page_table.dtype} {tuple(page_table.shape)}")
    if page_table.shape[1] > 1 and page_table.stride(1) != 1:
        raise ValueError("page_table rows must be contiguous")
    dev = cache.device
    if page_table.device != dev:
        raise ValueError(f"page_table is on {page_table.device}, the cache on {dev}")
    for name, t in per_seq.items():
        if t is None:
            continue
        if t.dtype != torch.int32 or t.shape != (b,) or (b > 1 and t.stride(0) != 1):
            raise ValueError(f"{name} must be contiguous int32 [{b}]; got {t.dtype} {tuple(t.shape)}")
        if t.device != dev:
            raise ValueError(f"{name} is on {t.device}, the cache on {dev}")
