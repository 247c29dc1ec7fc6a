"""Attention of the newest tokens over a paged cache (GPU): one token per
sequence (decoding), a chain of them, or a tree of drafted tokens.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence, Tuple

import torch

from . import _lib as L
from .kv_cache import KvCache, check_table


def tree_mask(parents: Sequence[int]) -> torch.Tensor:
    """[T, T] bool (CPU): which drafted tokens each one sees -- itself, its
    parent, its parent's parent and so on.  ``parents[t]`` < t is the token
    that t continues, -1 the cached context."""
    n = len(parents)
    sees = torch.zeros(n, n, dtype=torch.bool)
    for t, parent in enumerate(parents):
        if not -1 <= parent < t:
            raise ValueError(f"parents[{t}] must be in [-1, {t}), got {parent}")
        if parent >= 0:
            sees[t] = sees[parent]
        sees[t, t] = True
    return sees


def _misaligned(q: torch.Tensor) -> bool:
    """Rows of a bfloat16 tensor that do not start on 16-byte boundaries (the tensor-core kernel needs them)."""
    sb, sh, st, _ = q.stride()
    return (q.data_ptr() & 15) != 0 or ((sb | sh | st) & 7) != 0


def tree_attention(q: torch.Tensor, cache: KvCache, page_table: torch.Tensor, context_lens: torch.Tensor,
                   counts: Optional[torch.Tensor] = None, tree: Optional[torch.Tensor] = None,
                   scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """q [B, H_q, T, d] (bfloat16 or float32, any strides): the T newest tokens
    of each sequence, whose keys and values stand in the cache at positions
    context_lens[s] + t, behind the context_lens[s] earlier ones.  Token t sees
    the whole context and the newest tokens i with tree[t, i]
    (``tree`` [T, T] or [B, T, T] bool; without it i <= t, a chain).  With
    ``counts`` [B] only the first counts[s] of the T tokens exist.  Query head h
    reads KV head h // (H_q // H_kv); the cache's logit bias is added to the
    logits; ``scale`` defaults to 1 / sqrt(d).

    Returns (O [B, H_q, T, d] in q's dtype, LSE [B, H_q, T] float32), without
    gradients, as :func:`~dcc_kv_b200.attention` does:
    :func:`~dcc_kv_b200.merge_lse` joins it with attention over other keys.  A row that sees nothing, and the rows
    behind counts[s], give O = 0 and LSE = -inf.

    Waits inside the kernels are bounded: one that gave up leaves the call's
    output invalid and is reported by the next call on the device, or by
    ``cache.check()``, as ``DccError(DCC_ERR_TIMEOUT)``."""
    if q.dim() != 4 or q.shape[3] != cache.head_dim:
        raise ValueError(f"q must be [B, H_q, T, {cache.head_dim}], got {tuple(q.shape)}")
    b, hq, t, d = q.shape
    if q.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"q must be bfloat16 or float32, got {q.dtype}")
    if hq < 1 or hq % cache.n_kv_heads:
        raise ValueError(f"{hq} query heads are not a multiple of {cache.n_kv_heads} KV heads")
    tree_ptr, tree_stride = None, 0
    if tree is not None:
        if tree.dtype != torch.bool or tree.shape not in ((t, t), (b, t, t)):
            raise ValueError(f"tree must be bool [{t}, {t}] or [{b}, {t}, {t}]; got {tree.dtype} {tuple(tree.shape)}")
        tree = tree.contiguous()
        tree_ptr, tree_stride = tree.data_ptr(), t * t if tree.dim() == 3 else 0
    dev = cache.device
    L.require_cuda(q, cache.k, page_table)
    check_table(cache, b, page_table=page_table, context_lens=context_lens, counts=counts)
    L.same_device(dev, q=q, tree=tree)
    if (q.stride(3) != 1 and d > 1) or (q.dtype == torch.bfloat16 and _misaligned(q)):
        q = q.clone(memory_format=torch.contiguous_format)
    code = L.dtype_code(q)
    with L.on_device(dev):
        L.poll_give_ups(dev)
        o = torch.empty(b, hq, t, d, dtype=q.dtype, device=dev)
        lse = torch.empty(b, hq, t, dtype=torch.float32, device=dev)
        query = L.dcc_tree_query(q.data_ptr(), o.data_ptr(), lse.data_ptr(), *q.stride()[:3], *o.stride()[:3],
                                 context_lens.data_ptr(), L.ptr(counts), tree_ptr, tree_stride,
                                 page_table.data_ptr(), page_table.stride(0), t, b, hq, page_table.shape[1], 0)
        lib, pages = L.lib(), cache._pages
        ws = L.workspace(lib.dcc_tree_attention_workspace_bytes(pages, query, code), dev)
        L.check(lib.dcc_tree_attention(pages, query, 1.0 / math.sqrt(d) if scale is None else scale, code,
                                       ws.data_ptr(), ws.numel(), L.stream_ptr(dev)), "tree_attention")
    return o, lse
