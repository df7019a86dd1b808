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


def serving_call(**changes):
    g = torch.Generator().manual_seed(0)
    args = dict(x=torch.randn(5, 6, generator=g).to(DEV), decay_logits=torch.randn(5, 6, generator=g).to(DEV),
                state_pool=torch.ones(3, 6, device=DEV), cu_seqlens=int32(0, 2, 5), state_indices=int32(2, 0))
    args.update(changes)
    return args


@pytest.mark.parametrize("changes,error,text", [
    (dict(x=lambda: torch.zeros((), device=DEV)), ValueError, "packed shape"),
    (dict(x=lambda: torch.zeros(5, 6, dtype=torch.float64, device=DEV)), TypeError, "bfloat16, float16 or float32"),
    (dict(decay_logits=lambda: torch.zeros(5, 6, device=DEV, dtype=torch.bfloat16)), TypeError, "x's dtype"),
    (dict(state_pool=lambda: torch.zeros((), device=DEV)), ValueError, "state_pool must have shape"),
    (dict(state_pool=lambda: torch.zeros(3, 6)), ValueError, "share x's device"),
    (dict(cu_seqlens=lambda: int32(0, 2, 5).long()), TypeError, "int32"),
    (dict(cu_seqlens=lambda: int32(0, 2, 5).cpu()), ValueError, "share x's device"),
    (dict(cu_seqlens=lambda: int32(0, 5)), ValueError, "cu_seqlens must have shape"),
    (dict(cu_seqlens=lambda: None), TypeError, "incompatible function arguments"),
    # with metadata that would be refused as well: what can be said without it comes first
    (dict(cu_seqlens=lambda: int32(0, 5, 2), decay_mode=lambda: "exp"), ValueError, "decay_mode"),
    (dict(state_indices=lambda: int32(9, 9), decay_bias=lambda: torch.zeros(5, device=DEV)), ValueError, "decay_bias"),
    # and metadata that is refused where it is validated
    (dict(cu_seqlens=lambda: int32(0, 5, 2)), RuntimeError, "query_start_loc"),
    (dict(state_indices=lambda: int32(9, 0)), RuntimeError, "state_indices"),
])
def test_refusals_on_the_gpu_come_before_the_metadata(changes, error, text):
    serve, _, _ = operators()
    args = serving_call(**{k: v() for k, v in changes.items()})
    with pytest.raises(error, match=text):
        serve(**args)
    if "state_pool" not in changes:
        assert bool((args["state_pool"] == 1).all())


@pytest.mark.parametrize("poison", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("lengths", [[20, 900, 30], [3, 10, 2]])
@pytest.mark.parametrize("decay_mode,input_mode", [("logits", "unit"), ("logits", "complement"), ("retention", "unit")])
def test_where_a_bad_number_reaches(decay_mode, input_mode, lengths, poison):
    """From its token to the end of its sequence, in its channel; every other number keeps its bits, gradients among them."""
    serve, train, _ = operators()
    channels, total, n = 40, sum(lengths), len(lengths)
    g = torch.Generator().manual_seed(7)
    x = torch.randn(total, channels, generator=g)
    decay = torch.randn(total, channels, generator=g)
    if decay_mode == "retention":
        decay = torch.sigmoid(decay)
    pool, dy = torch.randn(n, channels, generator=g), torch.randn(total, channels, generator=g).to(DEV)
    cu = torch.tensor([0] + lengths).cumsum(0)
    first, last = int(cu[1]), int(cu[2])
    at = first + lengths[1] // 2

    def both(x, pool):
        state = pool.to(DEV)
        y = serve(x.to(DEV), decay.to(DEV), state_pool=state, cu_seqlens=int32(*cu.tolist()), state_indices=int32(*range(n)),
                  decay_mode=decay_mode, input_mode=input_mode)
        leaves = [t.to(DEV).requires_grad_() for t in (x, decay, pool)]
        rows, final = train(*leaves[:2], initial_state=leaves[2], cu_seqlens=int32(*cu.tolist()), decay_mode=decay_mode,
                            input_mode=input_mode)
        grads = torch.autograd.grad((rows, final), leaves, (dy, torch.ones_like(final)))
        return [t.detach().cpu() for t in (y, state, rows, final, *grads)]

    clean = both(x, pool)
    x, pool = x.clone(), pool.clone()
    x[at, 7] = poison    # an input in the middle of the second sequence
    pool[1, 9] = poison  # and its state
    bad = both(x, pool)
    rows_hit = torch.zeros(total, channels, dtype=torch.bool)
    rows_hit[at:last, 7] = rows_hit[first:last, 9] = True
    state_hit = torch.zeros(n, channels, dtype=torch.bool)
    state_hit[1, [7, 9]] = True
    for k, hit in ((0, rows_hit), (1, state_hit), (2, rows_hit), (3, state_hit)):
        assert not torch.isfinite(bad[k][hit]).any() and torch.equal(bad[k][~hit], clean[k][~hit]), k
    # x enters no gradient but the decay's, there from its own token on (complement) or from the next
    assert torch.equal(bad[4], clean[4]) and torch.equal(bad[6], clean[6])
    assert torch.equal(bad[5][~rows_hit], clean[5][~rows_hit])
