"""CPU checks of the gated scan's refusals that Python makes."""

from __future__ import annotations

import pytest
import torch


@pytest.mark.parametrize("max_seqlen", [0, -3, True, 2.5, "4"])
def test_a_longest_length_that_is_none(monkeypatch, max_seqlen):
    import flashrwkv2_b200 as pkg
    from flashrwkv2_b200 import _C_sm100

    monkeypatch.setattr(pkg, "_C", _C_sm100)
    x = torch.zeros(5, 6)
    for ticket in (None, object()):
        with pytest.raises(ValueError, match="max_seqlen must be a positive integer"):
            pkg.infer_tmix_gated_scan_fp32io16_forward_varlen(
                x, x, state_pool=torch.zeros(3, 6), cu_seqlens=torch.tensor([0, 2, 5], dtype=torch.int32),
                state_indices=torch.tensor([2, 0], dtype=torch.int32), max_seqlen=max_seqlen, validated_metadata=ticket)
