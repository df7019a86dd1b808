"""Log probabilities of given tokens under rows of vocabulary logits, the entropy of each row and its most probable tokens.

    z = logits / temperature      logprob = z[id] - logsumexp(z)      entropy = logsumexp(z) - sum_j softmax(z)_j z_j

What scoring and training on rollouts needs behind the head (policy ratio, entropy bonus, their gradient), and what a
server returns beside sampled tokens.  The logits are read once, and read and written once by the backward pass; no
probabilities are stored.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from ..tmix.wkv7 import _extension


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor             # float32, the shape of token_ids
    entropy: torch.Tensor              # float32, the shape of token_ids
    top_ids: torch.Tensor | None       # int64 [..., top_k], most probable first; None when top_k is 0
    top_logprobs: torch.Tensor | None  # float32 [..., top_k]


def rl_infctx_head_token_logprobs(logits: torch.Tensor, token_ids: torch.Tensor, *, temperature: float = 1.0,
                                  top_k: int = 0, ignore_index: int = -100) -> TokenLogprobs:
    """Returns ``TokenLogprobs(logprobs, entropy, top_ids, top_logprobs)``; differentiable in ``logits`` through the first
    two (once; the top alternatives carry no gradient).

    ``logits`` is ``[..., V]`` bfloat16, float16 or float32 with unit stride along V and rows that at most two strides
    describe (so ``logits[:, :-1]`` needs no copy); ``token_ids`` int64 or int32 of shape ``[...]``; ``temperature`` 1e-30 to
    1e30; ``top_k`` 0 to 32.
    Equal logits rank by their ids, lowest first, and NaN ranks above all.  A row whose id is ``ignore_index`` is left
    out: logprob, entropy and gradient 0, top ids -1, top logprobs -inf.  Any other id outside the vocabulary makes that
    row's logprob and gradient NaN.  Masked logits may be -inf or the type's lowest value; in a row of -inf alone every
    logprob is -inf, entropy and gradient are 0.  A NaN or +inf makes its row's results NaN.

    The same call twice gives the same bits, and no row's values touch another's.  But few rows are divided among several CTAs,
    which add up in another order: a row's float results may differ in their last bits between batches of other sizes (above and
    below 128 and 256 rows, for wide vocabularies) and between rows at other alignments (odd vocabularies).  A policy ratio
    between differently batched passes is 1 up to that.

    Errors: ``TypeError`` for wrong types, ``ValueError`` for wrong shapes, layouts and values, before any launch."""
    return TokenLogprobs(*_extension().head_token_logprobs(logits, token_ids, temperature, top_k, ignore_index))


__all__ = ["TokenLogprobs", "rl_infctx_head_token_logprobs"]
