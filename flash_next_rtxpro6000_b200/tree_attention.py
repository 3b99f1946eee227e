"""Attention of drafted token trees over a paged cache: the verify (and, with one node, the decode)
step's attention.

* ``tree_layout(parents, ...)`` -- masks, positions and cache slots of the nodes of drafted trees;
* ``tree_attention(q, k_cache, v_cache, ...)`` -- the attention itself (csrc/tree_attn.cu).

No counterpart in the reference's operator modules, whose server does these steps elsewhere.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .w8a16_gemv import PDL, _flag, _scratch

MAX_NODES = 64


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
    index.  Nodes of no request (ahead of node_offsets[0], from node_offsets[batch] on) get mask 0,
    position 0 and slot -1, so a captured step may be replayed with fewer nodes."""
    return _lib.ops().tree_layout(parents, node_offsets, context_lens, page_table, page_size, num_pages,
                                  _flag(parents), PDL if pdl is None else pdl)


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
    sum of exp(scale q k) (scale: dim ** -0.5 unless given, positive); a row that sees nothing gives 0 and -inf.
    ``max_context`` bounds context_lens (default: what the page table holds).  The form of the kernel is
    chosen by these bounds, so bounds near the real lengths are faster: one token over 1,000 keys takes
    11.8 us with its own and 15.0 with 262,080; 24 requests of up to 9 nodes and 6,000 keys 104 us with a
    max_nodes of 9 and 115 with 64; long contexts and wide trees lose at most 2 %.  Lengths are read on the
    device, so a captured call follows them; lengths beyond the bounds and pages outside the cache are
    reported by ``check_device_errors``.  Rows of no request, and those of one with lengths beyond the
    bounds, give 0 and -inf."""
    flag, partials, _ = _scratch(q)
    return _lib.ops().tree_attention(q, k_cache, v_cache, page_table, context_lens, node_offsets, tree_mask,
                                     max_nodes, max_context, scale, out, lse, partials, flag,
                                     PDL if pdl is None else pdl)
