"""Gated scan: the elementwise sibling of the WKV7 recurrence, one fp32 number of state per (sequence, channel).

    h_t = rho_t * h_{t-1} + i_t * x_t        y_t = h_t

``decay_mode`` is WKV7's: "logits" (``rho = exp(-e^{-1/2} * sigmoid(logit + bias))``) or "retention" (``rho`` itself).
``input_mode`` says what enters the state: "unit" (``i_t = 1``) or "complement" (``i_t = 1 - rho_t``, an exponential
moving average with a data-dependent rate).  Tokens are bfloat16, float16 or float32; the state is float32.

A retention is a number in [0, 1].  An infinity or NaN among a channel's inputs or in its state (or a state that overflows)
leaves the channel infinite or NaN from that token to the end of its sequence; from logits it is NaN where ``rho * inf`` would
have kept an infinity.  Earlier tokens, other channels and other sequences are as they would be without it.

The same call twice gives the same bits.  Which kernel and how many CTAs share a sequence follows from the shape of the whole
batch, so a sequence's results may differ in their last bits between batches.

* :func:`infer_tmix_gated_scan_fp32io16_forward_varlen` serves packed sequences (decode steps and prompts of any length)
  in place on a state pool, with the metadata ticket of the WKV7 operators: one ticket serves both in a step.
* :func:`pretrain_tmix_gated_scan_fp32io16` is differentiable, over dense or packed rows, with an initial state that
  takes a gradient and a final state that gives one.

Errors: ``TypeError`` for wrong types, ``ValueError`` for wrong shapes, layouts and values, before any launch; invalid
metadata raises ``RuntimeError`` where it is validated on the host, as for the WKV7 operators.
"""

from __future__ import annotations

import torch

from ..wkv7 import _extension, prepare_tmix_wkv7_recurrent_metadata
from .pretrain import pretrain_tmix_gated_scan_fp32io16


def infer_tmix_gated_scan_fp32io16_forward_varlen(
        x: torch.Tensor, decay_logits: torch.Tensor, *, state_pool: torch.Tensor, cu_seqlens: torch.Tensor,
        state_indices: torch.Tensor, decay_bias: torch.Tensor | None = None, max_seqlen: int | None = None,
        validated_metadata: object | None = None, decay_mode: str = "logits",
        input_mode: str = "unit") -> torch.Tensor:
    """Packed gated scan, in place on ``state_pool`` at ``state_indices``; returns y.

    ``x`` and ``decay_logits`` are ``[total_tokens, C]`` (rows may lie apart, as in a slice of a wider projection),
    ``state_pool`` float32 ``[slots, C]``, ``decay_bias`` ``[C]`` (logits mode only).  Metadata, tickets, CUDA-graph use and
    the fail-closed rules are those of the WKV7 operators: without ``validated_metadata`` the metadata is checked on the
    host (one sync); with a capacity ticket nothing synchronises, rows behind the last active sequence are left as they
    were allocated, and invalid metadata fills y with NaN and leaves the pool untouched.  No gradients: for those there is
    the training form."""
    native = _extension()
    longest = -1 if max_seqlen is None else max_seqlen
    if validated_metadata is None:
        native.check_tmix_gated_scan_fp32(cu_seqlens, state_indices, state_pool, x, decay_logits, decay_bias, None, longest,
                                          decay_mode, input_mode)
        validated_metadata = prepare_tmix_wkv7_recurrent_metadata(
            cu_seqlens, state_indices, total_tokens=x.shape[0], state_pool_size=state_pool.shape[0],
            max_seqlen=max_seqlen)
    return native.tmix_gated_scan_fp32(cu_seqlens, state_indices, state_pool, x, decay_logits, decay_bias,
                                       validated_metadata, longest, decay_mode, input_mode)


__all__ = ["infer_tmix_gated_scan_fp32io16_forward_varlen", "pretrain_tmix_gated_scan_fp32io16"]
