"""Training form of the gated scan: forward with saved tile states, and backward (see the package docstring)."""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from ..wkv7 import _extension


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, decay_logits, initial_state, cu_seqlens, decay_mode, input_mode):
        y, final_state, boundary, bounds, status = _extension().pretrain_tmix_gated_scan_forward(
            x, decay_logits, initial_state, cu_seqlens, decay_mode, input_mode)
        ctx.save_for_backward(x, decay_logits, initial_state, bounds, status, boundary)
        ctx.modes = decay_mode, input_mode
        ctx.set_materialize_grads(False)
        return y, final_state

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output, grad_final):
        x, decay_logits, initial_state, bounds, status, boundary = ctx.saved_tensors
        grad_output = torch.zeros_like(x, memory_format=torch.contiguous_format) if grad_output is None else grad_output.contiguous()
        if grad_final is not None:
            grad_final = grad_final.contiguous()
        dx, ddecay, dinitial = _extension().pretrain_tmix_gated_scan_backward(
            x, decay_logits, initial_state, bounds, status, boundary, grad_output, grad_final, *ctx.modes)
        return dx, ddecay, dinitial, None, None, None


def pretrain_tmix_gated_scan_fp32io16(
        x: torch.Tensor, decay_logits: torch.Tensor, *, initial_state: torch.Tensor | None = None,
        cu_seqlens: torch.Tensor | None = None, decay_mode: str = "logits",
        input_mode: str = "unit") -> tuple[torch.Tensor, torch.Tensor]:
    """Differentiable gated scan; returns ``(y, final_state)``.

    ``x`` and ``decay_logits`` are dense ``[B, T, C]``, or packed ``[total_tokens, C]`` with ``cu_seqlens`` (int32 ``[N+1]``,
    non-empty sequences).  ``initial_state`` is float32 ``[B or N, C]`` (zeros when None), ``final_state`` the same shape.
    Gradients reach ``x``, ``decay_logits`` (the retention in that mode) and ``initial_state``, through y and through the
    final state.  ``cu_seqlens`` is validated on the device without a sync: bad bounds make every output NaN.  The backward
    pass can be captured into a CUDA graph together with its forward pass; it is differentiable once."""
    return _GatedScan.apply(x, decay_logits, initial_state, cu_seqlens, decay_mode, input_mode)


__all__ = ["pretrain_tmix_gated_scan_fp32io16"]
