"""Verification of drafted tokens: which of them the target keeps, and the next token.

No reference counterpart. Speculative decoding: a cheaper model drafts tokens, the
target computes all of them in one step, and random numbers decide so that what
comes out has the target's distribution. The outputs are what
:func:`morphottention_amd.morpho_cache_compact`, ``MorphoCache.accept`` and
``MorphoLoop.accept`` take.
"""

from __future__ import annotations

import torch

from ._ops import add_op_namespace_prefix, ops


@torch.library.register_fake(add_op_namespace_prefix("verify_drafts"))
def _verify_drafts_fake(logits, tokens, uniform, tree, new_lens, draft_logits, temperature):
    B, n, _V = logits.shape
    return [logits.new_empty((B, n), dtype=torch.int32), logits.new_empty((B,), dtype=torch.int32),
            logits.new_empty((B,), dtype=torch.int64)]


def morpho_verify_drafts(logits: torch.Tensor, tokens: torch.Tensor, uniform: torch.Tensor, *,
                         tree: torch.Tensor | None = None, new_lens: torch.Tensor | None = None,
                         draft_logits: torch.Tensor | None = None,
                         temperature: float = 1.0) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Which tokens of a step are kept, and the token behind them.

    Token 0 of a sequence is decided (the token that the step before gave), the
    others are drafts. With p and q the softmax over ``temperature`` of the target's
    and the drafter's logits behind the token at hand, r = p and Z = 1, the drafts
    behind it are asked in ascending order: draft t is kept if ``uniform q(t) Z <
    r(t)``, and is then the token at hand; else r becomes ``max(r / Z - q, 0)`` and Z
    its sum. When none is left, the next token is the first one whose running sum
    of r passes ``uniform Z``. All sums are in 64 bits: the same inputs give the same
    tokens as any other 64-bit evaluation, up to rounding at a border (2^-45 or so,
    over the part of the row that the drafts turned down have left).

    :param logits: the target's ``[B, n, vocab]``, ``n <= 64``, float16, bfloat16 or
        float32; row i is the one behind token i. Contiguous along the vocabulary, of
        any other strides. NaN and -inf have no chance.
    :param tokens: int64 ``[B, n]``.
    :param uniform: float32 ``[B, n]``, random numbers in [0, 1): number i decides on
        draft i, number 0 draws the next token.
    :param tree: int64 ``[B, n]`` as in :func:`morphottention_amd.morpho_cache_attention`:
        token i was drafted behind that of the highest bit below i. A chain if not given.
    :param new_lens: int32 ``[B]``, tokens of each sequence where not all have ``n``;
        0: padding.
    :param draft_logits: ``[B, n - 1, vocab]`` of the type of ``logits``: row i are those
        that the drafts behind token i were drawn from at ``temperature``,
        independently of each other. Not given: the drafts were not drawn but
        chosen (q is 1 at the draft).
    :param temperature: 1e-4 to 1e4; or 0: a draft is kept if it is the target's best
        token (of equal ones the lowest), which is also the next one at the end.
    :returns: ``keep`` int32 ``[B, n]``, the places of the kept tokens, 0 first, ascending,
        then -1; ``keep_lens`` int32 ``[B]``, how many; ``token`` int64 ``[B]``, the next
        token, -1 for padding or where a row has no token with a chance.
    """
    detached = None if draft_logits is None else draft_logits.detach()
    keep, keep_lens, token = ops.verify_drafts(logits.detach(), tokens, uniform, tree, new_lens, detached, temperature)
    return keep, keep_lens, token
