"""The 8-bit paged cache of a decode, verify or prompt step, and the attention that reads it.

* ``rotary_append8(q, k, v, ...)`` -- rotary positions on queries and keys, keys and values stored as
  e4m3 with a scale for each block of tokens and kv head, in one launch (csrc/append8.cu);
* ``tree_attention8(q, k_cache, v_cache, k_scale, v_scale, ...)`` -- attention of drafted token trees
  over that cache (csrc/tree_attn8.cu).

The cache is a pair of float8_e4m3fn tensors [pages, page_size, kv_heads, dim] with fp32 scales
[pages, page_size / block, kv_heads]: an element is its e4m3 value times its block's scale.  Blocks
are 16, 32 or 64 tokens, pages whole numbers of blocks, dim 64, 128 or 256.  Against a 16-bit cache it
holds twice the tokens and the attention reads half of the bytes.

No counterpart in the reference's operator modules, whose server does these steps elsewhere.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .tree_attention import MAX_NODES
from .w8a16_gemv import PDL, _flag, _scratch


def rotary_append8(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    positions: torch.Tensor,
    context_lens: torch.Tensor,
    node_offsets: torch.Tensor,
    page_table: torch.Tensor,
    table: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    interleaved: bool = False,
    out: Optional[torch.Tensor] = None,
    pdl: Optional[bool] = None,
) -> torch.Tensor:
    """q [T, q_heads, dim], k and v [T, kv_heads, dim], bf16 or fp16 (views of one projection's rows
    are fine); positions int64 [T]; context_lens int32 [batch], node_offsets int32 [batch + 1],
    page_table int32 [batch, pages]; table fp32 [P, rotated] from ``rotary_table``; the cache as the
    module's documentation says.

    Rotates the first ``rotated`` elements of each query and key head as ``rotary_append`` does and
    returns the queries (in ``out``, which may be q).  Request b's tokens, rows node_offsets[b] ..
    node_offsets[b + 1] - 1 (any number: nodes of a tree, a prompt chunk), are stored at places
    context_lens[b] + index.  A block that gets tokens takes the smallest power of two as its scale by which
    its new elements divided fit into e4m3 (at most 448), at least 2^-40, and at least its old scale where
    tokens of the context stay in it; these take the new scale too.  What lies in a block behind the context
    when the call begins does not count.  So drafts that are refused later leave nothing behind but their scale in
    the block that they shared with the context: its tokens keep what they lost to it (elements below 2^-6 of the
    scale are rounded to multiples of 2^-9 of it), and the block's next tokens take at least that scale.  Infinite
    elements and NaN are stored as NaN and do not count.

    Rows of no request are rotated and not stored.  Positions outside the table, lengths that contradict
    each other or the page table, and pages outside the cache are reported by ``check_device_errors``;
    nothing is stored for the latter two.  No block may get tokens of two requests in one call: a request that
    shares pages with another one needs the page that it appends to for itself."""
    return _lib.ops().rotary_append8(q, k, v, positions, context_lens, node_offsets, page_table, table, k_cache,
                                     v_cache, k_scale, v_scale, interleaved, out, _flag(q),
                                     PDL if pdl is None else pdl)


def tree_attention8(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
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
    """``tree_attention`` (its arguments, results and errors) over an 8-bit cache: q bf16 or fp16, keys and
    values e4m3 with the scales of their blocks.

    Scales outside [2^-40, 2^120] or NaN, which ``rotary_append8`` does not write, are reported by
    ``check_device_errors`` and count as 2^-40; others need not be powers of two.  The scales of the values that a
    row sees should lie within a factor of 2^60 of each other.  Weights are rounded to fp16 for the second product,
    whatever q's type.  The cache takes half of a 16-bit one's memory; the time is about the same, since the chain of
    a tile's scores and weights bounds both."""
    flag, partials, _ = _scratch(q)
    return _lib.ops().tree_attention8(q, k_cache, v_cache, k_scale, v_scale, page_table, context_lens, node_offsets,
                                      tree_mask, max_nodes, max_context, scale, out, lse, partials, flag,
                                      PDL if pdl is None else pdl)
