"""GPU parity of the gated scan where rows begin at addresses that are aligned to nothing, and sequences are long enough for whole
tiles of 256 tokens: their 16-byte pieces are copied, shifted and stored without bounds checks.

Expectation and bounds: oracle.gated_scan_oracle in float64."""

from __future__ import annotations

import math

import pytest
import torch

from test_gated_scan_gpu import case, check_serve, check_train

pytestmark = pytest.mark.gpu

DEV = "cuda"

# one sequence on a cluster of two and of five CTAs; so many channels by sequences that one CTA walks each; tiles that begin at odd rows
SHAPES = [([300], 33), ([1100], 33), ([300] * 16, 1003), ([1100], 1003), ([3, 300, 1, 517], 33)]


def rows_of(c, sliced):
    """x and decay on the GPU, whole or as column slices of one tensor with NaN around them."""
    width = c["x"].shape[1]
    if not sliced:
        return c["x"].to(DEV), c["decay"].to(DEV)
    wide = torch.full((c["x"].shape[0], 2 * width + 4), math.nan, dtype=c["x"].dtype)
    wide[:, 1:1 + width], wide[:, 2 + width:2 + 2 * width] = c["x"], c["decay"]
    wide = wide.to(DEV)
    return wide[:, 1:1 + width], wide[:, 2 + width:2 + 2 * width]


@pytest.mark.parametrize("sliced", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("lengths,channels", SHAPES)
@pytest.mark.parametrize("decay_mode,input_mode", [("logits", "complement"), ("retention", "unit")])
def test_whole_tiles_at_odd_addresses(decay_mode, input_mode, lengths, channels, dtype, sliced):
    from flashrwkv2_b200 import infer_tmix_gated_scan_fp32io16_forward_varlen, pretrain_tmix_gated_scan_fp32io16

    c = case(lengths, channels, dtype, decay_mode, seed=40)
    n = len(lengths)
    g = torch.Generator().manual_seed(41)
    initial, dfinal = (torch.randn(n, channels, generator=g) for _ in range(2))
    dy = torch.randn(c["x"].shape, generator=g).to(dtype)
    x, decay = rows_of(c, sliced)
    pool = c["pool"].to(DEV)
    y = infer_tmix_gated_scan_fp32io16_forward_varlen(x, decay, state_pool=pool, cu_seqlens=c["cu"].to(DEV),
                                                      state_indices=c["slots"].to(DEV), decay_mode=decay_mode, input_mode=input_mode)
    check_serve(c, y.cpu(), pool.cpu(), decay_mode, input_mode)

    x, decay, h0 = x.detach().requires_grad_(), decay.detach().requires_grad_(), initial.to(DEV).requires_grad_()
    assert not sliced or x.stride(0) % 2 == 0 and x.data_ptr() % 16 != 0
    y, final = pretrain_tmix_gated_scan_fp32io16(x, decay, initial_state=h0, cu_seqlens=c["cu"].to(DEV), decay_mode=decay_mode,
                                                 input_mode=input_mode)
    got = torch.autograd.grad((y, final), (x, decay, h0), (dy.to(DEV), dfinal.to(DEV)))
    check_train(c, [t.detach().cpu() for t in (y, final, *got)], initial, dy, dfinal, decay_mode, input_mode)
