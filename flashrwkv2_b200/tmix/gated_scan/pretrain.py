"""Training form of the gated scan (see the package docstring); its autograd node lives in the native module."""

from __future__ import annotations

import torch

from ..wkv7 import _extension


def pretrain_tmix_gated_scan_fp32io16(
        x: torch.Tensor, decay_logits: torch.Tensor, *, initial_state: torch.Tensor | None = None,
        cu_seqlens: torch.Tensor | None = None, decay_mode: str = "logits",
        input_mode: str = "unit") -> tuple[torch.Tensor, torch.Tensor]:
    """Differentiable gated scan; returns ``(y, final_state)``.

    ``x`` and ``decay_logits`` are dense ``[B, T, C]``, or packed ``[total_tokens, C]`` with ``cu_seqlens`` (int32 ``[N+1]``,
    non-empty sequences).  ``initial_state`` is float32 ``[B or N, C]`` (zeros when None), ``final_state`` the same shape.
    Gradients reach ``x``, ``decay_logits`` (the retention in that mode) and ``initial_state``, through y and through the
    final state.  Rows may lie apart (a slice of a wider projection) at one regular distance.  ``cu_seqlens`` is validated
    on the device without a sync: bad bounds make every output NaN.  The backward pass can be captured into a CUDA graph
    together with its forward pass, as torch asks for it: after a warm-up on a side stream, and with no other autograd
    graph of the same leaves alive.  It is differentiable once."""
    return _extension().pretrain_tmix_gated_scan(x, decay_logits, initial_state, cu_seqlens, decay_mode, input_mode)


__all__ = ["pretrain_tmix_gated_scan_fp32io16"]
