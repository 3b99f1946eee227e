"""Sampling from the lm_head's logits with temperature, top-k, top-p and min-p, from given random
numbers (csrc/sample.cu).

``sample_tokens`` stands where the greedy argmax of ``w8a16_gemv`` or ``draft_topk1_postprocess``
would: one token per row of logits, for every node of a verify pass in one launch.  ``token_probs`` gives
the probabilities that it draws from, which ``verify_tokens`` takes.  No counterpart in the reference's
operator modules.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .w8a16_gemv import PDL


def sample_tokens(
    logits: torch.Tensor,
    uniforms: torch.Tensor,
    temperature: Optional[torch.Tensor] = None,
    top_k: Optional[torch.Tensor] = None,
    top_p: Optional[torch.Tensor] = None,
    min_p: Optional[torch.Tensor] = None,
    pdl: Optional[bool] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """(tokens int64 [M], probs fp32 [M]) of logits [M, V] (fp32, bf16 or fp16, rows contiguous, V at
    most 2^21).

    uniforms fp32 [M] in [0, 1); temperature, top_p, min_p fp32 [M], top_k int32 [M], each None for
    off.  In the order of falling logits (lower token first on ties) top-k keeps ``top_k`` tokens,
    top-p the shortest prefix whose probability reaches ``top_p`` of those, min-p the tokens with at
    least ``min_p`` of the largest probability; the token drawn is the one at which the running
    probability passes ``uniforms`` of what is kept, and ``probs`` is its probability there.
    Temperature 0 draws the first token; top_k < 1, top_p >= 1 and min_p <= 0 keep everything.  NaN
    logits count as -inf; a row of nothing else gives token -1 and probability 0.  Weights are whole
    numbers, so results are the same bit for bit from call to call."""
    return _lib.ops().sample_tokens(logits, uniforms, temperature, top_k, top_p, min_p,
                                    PDL if pdl is None else pdl)


def token_probs(
    logits: torch.Tensor,
    temperature: Optional[torch.Tensor] = None,
    top_k: Optional[torch.Tensor] = None,
    top_p: Optional[torch.Tensor] = None,
    min_p: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    pdl: Optional[bool] = None,
) -> torch.Tensor:
    """fp32 [M, V] (in ``out``, which must not overlap logits): the probabilities from which ``sample_tokens``
    draws with the same arguments -- each kept token's weight over that of all kept tokens, 0 for the others.
    Temperature 0 gives 1 to the first token; a row without a logit above -inf is zeros."""
    return _lib.ops().token_probs(logits, temperature, top_k, top_p, min_p, out, PDL if pdl is None else pdl)
