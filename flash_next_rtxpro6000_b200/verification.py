"""The end of a verify step: which drafted tokens stand, and their keys and values moved behind the
context.

* ``verify_tokens(target_probs, draft_probs, ...)`` -- the accepted path of each drafted tree and the
  token after it, from given random numbers (csrc/verify.cu);
* ``compact_nodes(k_cache, v_cache, ...)`` -- the path's keys and values moved to the places that
  follow the context, in all layers (csrc/compact.cu).

``sampling.token_probs`` makes the probabilities.  No counterpart in the reference's operator modules,
whose server does these steps elsewhere.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .tree_attention import MAX_NODES
from .w8a16_gemv import PDL, _flag


def verify_tokens(
    target_probs: torch.Tensor,
    draft_probs: Optional[torch.Tensor],
    tokens: torch.Tensor,
    parents: torch.Tensor,
    node_offsets: torch.Tensor,
    node_uniforms: torch.Tensor,
    draw_uniforms: torch.Tensor,
    max_nodes: int = MAX_NODES,
    pdl: Optional[bool] = None,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(path int32 [batch, max_nodes], accepted int32 [batch], next_tokens int64 [batch]).

    target_probs fp32 [nodes, V]: row i is the target's distribution of the token after node i;
    draft_probs (like it, or None): row i the distribution from which node i's children were drawn,
    independently of each other (rows of nodes without children are not read).  None: children were
    chosen, not drawn, as by a greedy drafter.  tokens int64 [nodes] and parents int32 [nodes] as for
    ``tree_layout``: node 0 of a request is its last token and starts the path.  node_uniforms fp32
    [nodes] and draw_uniforms fp32 [batch] are random numbers in [0, 1).  At most 64 nodes a request
    and V at most 2^21.

    From the path's end on, its children are asked in order: with r = p (the target's row) and S = 1 at
    first, token x is accepted where u q(x) < r(x) / S, and its node becomes the path's end; otherwise r
    becomes max(r / S - q, 0) and S its sum (without draft_probs: accepted where u S < r(x), otherwise x
    leaves r and S).  A refusal that would leave nothing leaves r and S as they are.  The next token is drawn
    from r, in the order of tokens, by draw_uniforms.  So the accepted tokens and the next one have the
    target's distribution whatever the drafter's is.  ``path`` has the accepted nodes' indices, node 0 first,
    then -1.  Sums are of whole numbers: results are the same bit for bit from call to call.

    A request without nodes accepts 0 and gives -1; one whose row at the path's end is zeros (nothing of 2^-52
    or more) gives -1.  Parents that are not earlier nodes (those nodes are never asked), tokens outside the
    vocabulary (refused), lengths outside the bounds and rows that are no distributions but sum to 64 or more (both
    as without nodes) are reported by ``check_device_errors``."""
    return _lib.ops().verify_tokens(target_probs, draft_probs, tokens, parents, node_offsets, node_uniforms,
                                    draw_uniforms, max_nodes, _flag(target_probs), PDL if pdl is None else pdl)


def compact_nodes(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    context_lens: torch.Tensor,
    path: torch.Tensor,
    accepted: torch.Tensor,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
    pdl: Optional[bool] = None,
) -> torch.Tensor:
    """The contexts' new lengths, int32 [batch]: context_lens + accepted.

    For d < accepted[b], what lies at place context_lens[b] + path[b, d] of request b goes to place
    context_lens[b] + d, as if everything were read first; ``path`` (int32 [batch, nodes <= 64]) and
    ``accepted`` (int32 [batch]) as ``verify_tokens`` gives them, rising from 0 on.  Caches [pages,
    page_size, kv_heads, dim], or [layers, pages, page_size, kv_heads, dim] for all layers in one launch:
    bf16 or fp16, or float8_e4m3fn with k_scale and v_scale ([layers,] pages, page_size / block,
    kv_heads) as of ``rotary_append8``.  There a block's scale becomes the largest of those of the tokens that
    come to it and, where tokens of the context stay in it, its own; elements whose scale changes are rounded
    again (exact for powers of two, but for elements 2^14 below their block's largest).  It does not fall again: tokens
    keep the scale that refused drafts brought to their block (``rotary_append8``).

    Paths that do not rise or reach past the pages, and pages outside the cache, are reported by
    ``check_device_errors``; such a request is left as it was.  No page may be moved in for two requests."""
    return _lib.ops().compact_nodes(k_cache, v_cache, page_table, context_lens, path, accepted, k_scale, v_scale,
                                    _flag(k_cache), PDL if pdl is None else pdl)
