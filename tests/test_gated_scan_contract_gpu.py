"""GPU checks of what the gated scan's entry points promise beside their values: tickets, refusals, bad numbers."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import gated_scan_oracle as oracle

pytestmark = pytest.mark.gpu

DEV = "cuda"


def operators():
    import flashrwkv2_b200 as pkg

    return (pkg.infer_tmix_gated_scan_fp32io16_forward_varlen, pkg.pretrain_tmix_gated_scan_fp32io16,
            pkg.prepare_tmix_wkv7_recurrent_metadata)


def int32(*values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("tokens", [1, 3, 40])
def test_a_ticket_with_room_for_more_sequences_than_tokens(tokens):
    """Sequence and token capacity are independent, as for WKV7: what is not active is not looked at."""
    serve, _, prepare = operators()
    sequences, channels = 50, 72
    g = torch.Generator().manual_seed(tokens)
    x, decay = (torch.randn(tokens, channels, generator=g).to(torch.bfloat16) for _ in range(2))
    pool = torch.randn(sequences, channels, generator=g)
    for lengths in ([1], [1] * tokens, [tokens]):
        total, n = sum(lengths), len(lengths)
        cu = int32(*torch.tensor([0] + lengths).cumsum(0).tolist(), *[-5] * (sequences - n))
        slots = int32(*range(7, 7 + n), *[-5] * (sequences - n))
        ticket = prepare(cu, slots, state_pool_size=sequences, token_capacity=tokens, sequence_capacity=sequences,
                         max_seqlen_capacity=tokens, num_active_tokens=int32(total), num_active_sequences=int32(n))
        got_pool = pool.to(DEV)
        y = serve(x.to(DEV), decay.to(DEV), state_pool=got_pool, cu_seqlens=cu, state_indices=slots, validated_metadata=ticket)
        at = 0
        for i, length in enumerate(lengths):
            want = oracle.forward(x[at:at + length], decay[at:at + length], None, pool[7 + i], "logits", "unit")
            off = want["off"] + oracle.half_step(torch.bfloat16, want["y"]) + want["off"] * 2.0 ** -8
            assert bool(((y[at:at + length].cpu().double() - want["y"]).abs() <= off).all())
            assert bool(((got_pool[7 + i].cpu().double() - want["final"]).abs() <= want["final_off"] + 2.0 ** -24 * want["final"].abs()).all())
            at += length
        rest = [i for i in range(sequences) if not 7 <= i < 7 + n]
        assert torch.equal(got_pool.cpu()[rest], pool[rest])
