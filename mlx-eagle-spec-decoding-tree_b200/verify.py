"""Verification of drafted tokens against the target's probabilities, from given random numbers.

``SpecDecoder`` grows a tree of the draft's likeliest tokens and draws its own random numbers.  A chain of tokens that were *drawn* from a draft
distribution is verified by the ratio of the two probabilities; done here for a batch of requests in one launch, from distributions in
whatever way they were made (temperature, top-k, penalties) and random numbers that the caller holds.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib


def verify_tokens(draft_tokens: torch.Tensor, target_probs: torch.Tensor, uniforms: torch.Tensor, *, draft_probs: Optional[torch.Tensor] = None,
                  draft_lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(tokens (B, K + 1) int32, accepted (B,) int32)``: of each request the drafted tokens that stand, one token more, then -1.

    Token ``i`` of ``draft_tokens (B, K)`` int32 stands while ``uniforms[i] * q_i(x_i) < p_i(x_i)`` and those before it do, ``p`` =
    ``target_probs (B, K + 1, V)``, ``q`` = ``draft_probs (B, K, V)`` (None: the drafts were not drawn, ``q`` is 1 at them).  The token behind the ``n`` that
    stand is drawn by ``uniforms[K]`` from ``max(p_n - q_n, 0)``, or from ``p_n`` if all stand: the lowest ``j`` whose sum of weights ``0 .. j`` exceeds
    ``uniforms[K]`` times the sum of all.  With ``uniforms (B, K + 1)`` float32 independent in [0, 1) and rows that sum to one the tokens are distributed as
    drawn from the target.  ``draft_lengths (B,)`` int32 says how many drafts a request has (None: ``K``); the row of ``p`` behind the last of them is used.

    Distributions are float32, float16 or bfloat16, both of one type, any strides but a contiguous last dimension.  Rows of another sum
    are taken as they are: the draw goes by its weights' sum, whether a draft stands does not.
    Products, differences and sums are in 64 bits.  A drafted token outside the vocabulary is refused; where ``p_n - q_n`` leaves nothing, the
    token is drawn from ``p_n``, and where that is empty it is 0.  ``K`` at most 1024."""
    both = _lib.ops().verify_tokens(draft_tokens, target_probs, uniforms, draft_probs, draft_lengths)
    if both is not None:
        return both
    _lib.require_tensor("target_probs", target_probs, tuple(_lib.DTYPES), (None, None, None), packed=False)
    B, rows, V = target_probs.shape
    K = rows - 1
    if K < 0 or K > 1024 or V < 1 or V > 1 << 30 or B > 65535:
        raise _lib.B200Error("target_probs must be (requests, drafts + 1, vocabulary): at most 65535, 1024 drafts, 2^30")
    _lib.require_tensor("draft_tokens", draft_tokens, (torch.int32,), (B, K), target_probs, packed=False)
    _lib.require_tensor("uniforms", uniforms, (torch.float32,), (B, K + 1), target_probs, packed=False)
    if draft_probs is not None:
        _lib.require_tensor("draft_probs", draft_probs, (target_probs.dtype,), (B, K, V), target_probs, packed=False)
    if draft_lengths is not None:
        _lib.require_tensor("draft_lengths", draft_lengths, (torch.int32,), (B,), target_probs)
    tokens = torch.empty(B, K + 1, dtype=torch.int32, device=target_probs.device)
    accepted = torch.empty(B, dtype=torch.int32, device=target_probs.device)
    with _lib.on_device(target_probs):
        rc = _lib.lib().b200_verify_tokens(
            _lib.ptr(draft_tokens), draft_tokens.stride(0), _lib.ptr(target_probs), target_probs.stride(0), target_probs.stride(1),
            _lib.ptr(draft_probs), 0 if draft_probs is None else draft_probs.stride(0), 0 if draft_probs is None else draft_probs.stride(1),
            _lib.ptr(uniforms), uniforms.stride(0), _lib.ptr(draft_lengths), _lib.DTYPES[target_probs.dtype], B, K, V, _lib.ptr(tokens),
            _lib.ptr(accepted), _lib.stream_ptr(target_probs.device))
    _lib.check(rc, "b200_verify_tokens")
    return tokens, accepted
