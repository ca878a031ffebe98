"""The check of drafted tokens on the B200 (``include/b200_verify.h``): the end of a
speculative decoding step, between the target's logits and ``b200_cache_accept``."""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from .paged_cache import _call


def b200_verify_drafts(logits: torch.Tensor, tokens: torch.Tensor, uniforms: torch.Tensor,
                       draft_probs: Optional[torch.Tensor] = None,
                       parents: Optional[torch.Tensor] = None,
                       draft_lens: Optional[torch.Tensor] = None, temperature: float = 1.0
                       ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Which drafted tokens the target keeps, and the token that follows them.

    ``tokens`` ``[B, T]`` (int64 or int32) are drafted nodes: node 0 is the root, the last
    token that is already decided (its id is not read); node ``i`` follows ``parents[b, i] <
    i`` (int32 ``[T]`` or ``[B, T]``; without it a chain; -1: not looked at).  ``logits`` ``[B, T,
    V]`` (bfloat16, float16 or float32) are the target's after each node, ``p = softmax(logits /
    temperature)``; at temperature 0 all weight lies on the largest logit, the first of equal
    ones.  ``draft_probs`` ``[B, T - 1, V]`` are the distributions ``q`` that each node's children
    were drawn from; without them, and at temperature 0, a draft counts as certain (``q`` is 1 at
    its token).  ``draft_lens`` int32 ``[B]``: nodes of each sequence, all ``T`` without it.

    From the root on, a node's children are asked in order: child ``c`` is kept where
    ``uniforms[b, c] * q(token) < p(token)``, and the path goes on from it; else ``p`` becomes
    ``max(p - q, 0)``, normalised, for the next child.  Where none is kept the path ends and
    the next token is the first ``v`` whose cumulated ``p`` is past ``uniforms[b, 0]``.  With
    ``uniforms`` (float32 ``[B, T]``) in [0, 1) the tokens are distributed as the target's own.

    Returns ``paths`` int32 ``[B, T]`` (the nodes kept, the root first, then -1), ``counts`` int32
    ``[B]``, as ``b200_cache_accept`` takes them, and the next tokens int64 ``[B]`` (-1 for a
    sequence without nodes, and where the path ends at a row that is no distribution: a NaN or
    +infinity, or nothing above -infinity).  Launched on the current stream; no call waits for
    the host.  A token or parent out of range is reported like every device error of this package.
    Inference only."""
    return _call("verify_drafts", logits.device, logits, tokens, uniforms, draft_probs, parents,
                 draft_lens, float(temperature))
