"""Attention of drafted token trees over a paged cache: the verify (and, with one node, the decode)
step's attention.

* ``tree_layout(parents, ...)`` -- masks, positions and cache slots of the nodes of drafted trees;
* ``tree_attention(q, k_cache, v_cache, ...)`` -- the attention itself (csrc/tree_attn.cu).

No counterpart in the reference's operator modules, whose server does these steps elsewhere.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import check, ptr
from .rotary import _TYPES, _heads, _index, cache_args
from .w8a16_gemv import PDL, _stream, _workspace

MAX_NODES = 64
_PARTIALS: dict = {}


def _partials(ws) -> torch.Tensor:
    """The attention scratch beside a scratch slot's workspace (made at the slot's first call)."""
    t = _PARTIALS.get(id(ws))
    if t is None:
        n = ctypes.c_int64()
        check(_lib.lib().fnx_tree_attention_workspace_floats(ctypes.byref(n)), "tree_attention")
        t = torch.empty(n.value, dtype=torch.float32, device=ws.device)
        _PARTIALS[id(ws)] = t  # workspaces live as long as the process
    return t


def _page_table(page_table: torch.Tensor, batch: int, device) -> None:
    if page_table.dim() != 2 or page_table.shape[0] != batch or page_table.dtype != torch.int32 or \
            page_table.device != device or (page_table.stride(1) != 1 and page_table.shape[1] > 1):
        raise ValueError(f"page_table must be a row-contiguous int32 [{batch}, pages] tensor on {device}")


def tree_layout(
    parents: torch.Tensor,
    node_offsets: torch.Tensor,
    context_lens: torch.Tensor,
    page_table: torch.Tensor,
    page_size: int,
    num_pages: int,
    pdl: Optional[bool] = None,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(tree_mask, positions, slots), int64 [nodes] each, of the drafted trees of a batch.

    parents int32 [nodes]: each node's parent as an index within its request (below its own), -1 for
    a root; node_offsets int32 [batch + 1]; context_lens int32 [batch]; page_table int32 [batch,
    pages].  Bit j of a node's mask is set where it sees node j: itself and its ancestors.  Its
    position is the context length plus its depth, its slot that of the context's length plus its
    index."""
    if not parents.is_cuda:
        raise ValueError("tree_layout needs CUDA tensors")
    dev, N, B = parents.device, parents.shape[0], context_lens.shape[0]
    _index(parents, "parents", N, torch.int32, dev)
    _index(node_offsets, "node_offsets", B + 1, torch.int32, dev)
    _index(context_lens, "context_lens", B, torch.int32, dev)
    _page_table(page_table, B, dev)
    out = torch.empty((3, N), dtype=torch.int64, device=dev)
    rc = _lib.lib().fnx_tree_layout(
        ptr(parents), ptr(node_offsets), ptr(context_lens), ptr(page_table), page_table.stride(0),
        page_table.shape[1], int(num_pages), int(page_size), B, N, ptr(out[0]), ptr(out[1]), ptr(out[2]),
        ptr(_workspace(dev).error_flag), int(PDL if pdl is None else pdl), _stream(parents))
    check(rc, "tree_layout")
    return out[0], out[1], out[2]


def tree_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    context_lens: torch.Tensor,
    node_offsets: torch.Tensor,
    tree_mask: Optional[torch.Tensor] = None,
    max_nodes: int = MAX_NODES,
    max_context: Optional[int] = None,
    scale: Optional[float] = None,
    out: Optional[torch.Tensor] = None,
    lse: Optional[torch.Tensor] = None,
    pdl: Optional[bool] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """q [nodes, q_heads, dim] bf16 or fp16, dim 64, 128 or 256; caches [pages, page_size, kv_heads,
    dim] of q's type; page_table int32 [batch, pages], context_lens int32 [batch], node_offsets int32
    [batch + 1]; tree_mask int64 [nodes] (None: chains).  Request b's nodes are rows node_offsets[b] ..
    node_offsets[b + 1] - 1 of q, at most ``max_nodes`` (<= 64); their keys and values are already in
    the cache, at places context_lens[b] + index.

    Node i attends the context and the drafted tokens whose bit is set in tree_mask[i].  Returns
    (out [nodes, q_heads, dim], lse fp32 [nodes, q_heads]), lse being the natural logarithm of the
    sum of exp(scale q k) (scale: dim ** -0.5 unless given); a row that sees nothing gives 0 and -inf.
    ``max_context`` bounds context_lens (default: what the page table holds).  Lengths are read on the
    device, so a captured call follows them; lengths beyond the bounds and pages outside the cache are
    reported by ``check_device_errors``."""
    if q.dim() != 3:
        raise ValueError(f"q must be [nodes, heads, dim], got {tuple(q.shape)}")
    if q.dtype not in _TYPES:
        raise NotImplementedError(f"tree_attention: bf16 or fp16, got {q.dtype}")
    if not q.is_cuda:
        raise ValueError("tree_attention needs CUDA tensors")
    N, Hq, D = q.shape
    dev, B = q.device, context_lens.shape[0]
    _heads(q, "q", N, D, q)
    ks, vs = cache_args(k_cache, v_cache)
    pages, page_size, Hk, Dk = k_cache.shape
    if Dk != D or k_cache.dtype != q.dtype or k_cache.device != dev or v_cache.device != dev:
        raise ValueError(f"caches must be [pages, page_size, kv_heads, {D}] {q.dtype} tensors on {dev}")
    if Hk < 1 or Hq % Hk:
        raise ValueError(f"{Hq} query heads must be a multiple of {Hk} kv heads")
    _index(context_lens, "context_lens", B, torch.int32, dev)
    _index(node_offsets, "node_offsets", B + 1, torch.int32, dev)
    _page_table(page_table, B, dev)
    if tree_mask is not None:
        _index(tree_mask, "tree_mask", N, torch.int64, dev)
    if out is None:
        out = torch.empty((N, Hq, D), dtype=q.dtype, device=dev)
    else:
        _heads(out, "out", N, D, q)
        if out.shape[1] != Hq:
            raise ValueError(f"out must have q's {Hq} heads")
    if lse is None:
        lse = torch.empty((N, Hq), dtype=torch.float32, device=dev)
    elif tuple(lse.shape) != (N, Hq) or lse.dtype != torch.float32 or lse.device != dev or \
            not lse.is_contiguous():
        raise ValueError(f"lse must be a contiguous fp32 [{N}, {Hq}] tensor on {dev}")
    ws = _workspace(dev)
    rc = _lib.lib().fnx_tree_attention(
        ptr(q), q.stride(0), q.stride(1), ptr(k_cache), ks, ptr(v_cache), vs, pages, page_size,
        ptr(page_table), page_table.stride(0), page_table.shape[1], ptr(context_lens), ptr(node_offsets),
        ptr(tree_mask), ptr(out), out.stride(0), out.stride(1), ptr(lse), B, N, Hq, Hk, D, int(max_nodes),
        page_table.shape[1] * page_size if max_context is None else int(max_context),
        D ** -0.5 if scale is None else float(scale), _TYPES[q.dtype], ptr(_partials(ws)),
        ptr(ws.error_flag), int(PDL if pdl is None else pdl), _stream(q))
    check(rc, "tree_attention")
    return out, lse
