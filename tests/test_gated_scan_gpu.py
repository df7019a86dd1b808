"""GPU parity of the gated scan: in-place serving operator, training forward and backward.

Expectation: oracle.gated_scan_oracle in float64, which also gives the bound of fp32 arithmetic for every element; a rounded
output may differ by that and half a step of its type."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import gated_scan_oracle as oracle

pytestmark = pytest.mark.gpu

DEV = "cuda"
MODES = [(d, i) for d in ("logits", "retention") for i in ("unit", "complement")]
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def case(lengths, channels, dtype, decay_mode, seed=0, spare=2, slow=False):
    g = torch.Generator().manual_seed(seed + 1000 * len(lengths) + channels)
    total, n = sum(lengths), len(lengths)
    x = torch.randn(total, channels, generator=g).to(dtype)
    if decay_mode == "logits":
        decay = ((6 if slow else 2) * torch.randn(total, channels, generator=g) - (6 if slow else 1)).to(dtype)
    else:
        decay = (torch.rand(total, channels, generator=g) ** (0.02 if slow else 0.5)).to(dtype)
    pool = torch.randn(n + spare, channels, generator=g)
    slots = torch.randperm(n + spare, generator=g)[:n].to(torch.int32)
    cu = torch.tensor([0] + lengths).cumsum(0).to(torch.int32)
    return dict(x=x, decay=decay, pool=pool, slots=slots, cu=cu, lengths=lengths,
                bias=(0.5 * torch.randn(channels, generator=g)).to(dtype))


def serve(c, decay_mode, input_mode, bias=False, pool=None, **more):
    from flashrwkv2_b200 import infer_tmix_gated_scan_fp32io16_forward_varlen as op

    pool = c["pool"].to(DEV) if pool is None else pool
    y = op(c["x"].to(DEV), c["decay"].to(DEV), state_pool=pool, cu_seqlens=c["cu"].to(DEV),
           state_indices=c["slots"].to(DEV), decay_bias=c["bias"].to(DEV) if bias else None, decay_mode=decay_mode,
           input_mode=input_mode, **more)
    torch.cuda.synchronize()
    return y.cpu(), pool.cpu()


def close(got, want, off, dtype, what):
    allowed = off + oracle.half_step(dtype, want) + off * torch.finfo(dtype).eps
    excess = (got.double() - want).abs() - allowed
    assert torch.isfinite(got.double()).all(), what
    assert float(excess.max()) <= 0, (what, float(excess.max()), int(excess.argmax()))


def check_serve(c, y, pool, decay_mode, input_mode, bias=False):
    dtype = c["x"].dtype
    untouched = torch.ones(c["pool"].shape[0], dtype=torch.bool)
    for i, n in enumerate(c["lengths"]):
        lo, hi, slot = int(c["cu"][i]), int(c["cu"][i + 1]), int(c["slots"][i])
        f = oracle.forward(c["x"][lo:hi], c["decay"][lo:hi], c["bias"] if bias else None, c["pool"][slot], decay_mode, input_mode)
        close(y[lo:hi], f["y"], f["off"], dtype, ("y", i))
        close(pool[slot], f["final"], f["final_off"], torch.float32, ("state", i))
        untouched[slot] = False
    assert torch.equal(pool[untouched], c["pool"][untouched])


@pytest.mark.parametrize("channels", [1, 7, 8, 64, 130, 200])
@pytest.mark.parametrize("lengths", [[1], [1, 1, 1], [3, 1, 2], [63], [64], [65], [1, 15, 16, 17, 65], [129, 1, 200], [128, 64]])
def test_lengths_and_channels(lengths, channels):
    c = case(lengths, channels, torch.bfloat16, "logits")
    y, pool = serve(c, "logits", "unit")
    check_serve(c, y, pool, "logits", "unit")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("decay_mode,input_mode", MODES)
def test_types_and_modes(dtype, decay_mode, input_mode):
    bias = decay_mode == "logits"
    for lengths, channels in (([70, 1, 131, 5], 72), ([1] * 9, 136), ([33], 19)):
        c = case(lengths, channels, dtype, decay_mode, seed=3)
        y, pool = serve(c, decay_mode, input_mode, bias=bias)
        check_serve(c, y, pool, decay_mode, input_mode, bias=bias)


@pytest.mark.parametrize("decay_mode,input_mode", MODES)
def test_long_sequence_with_slow_channels(decay_mode, input_mode):
    """6000 tokens and channels that forget over thousands of them: every join of tiles counts."""
    c = case([6000, 2100], 40, torch.float32, decay_mode, seed=5, slow=True)
    y, pool = serve(c, decay_mode, input_mode)
    check_serve(c, y, pool, decay_mode, input_mode)


def test_many_sequences_of_one_token():
    c = case([1] * 700, 264, torch.float16, "logits", seed=6)
    y, pool = serve(c, "logits", "complement", bias=True, max_seqlen=1)
    check_serve(c, y, pool, "logits", "complement", bias=True)


def test_many_short_sequences():
    g = torch.Generator().manual_seed(4)
    c = case(torch.randint(1, 9, (300,), generator=g).tolist(), 96, torch.bfloat16, "logits", seed=7)
    y, pool = serve(c, "logits", "unit")
    check_serve(c, y, pool, "logits", "unit")


def test_tokens_one_by_one_agree_with_one_call():
    """The state carries everything: feeding a sequence token by token gives what one call gives, within the bounds of
    both."""
    c = case([40, 40], 72, torch.float32, "logits", seed=8)
    _, pool = serve(c, "logits", "unit")
    step_pool = c["pool"].to(DEV)
    rows = []
    for t in range(40):
        one = dict(c, x=c["x"][t::40].contiguous(), decay=c["decay"][t::40].contiguous(), cu=torch.tensor([0, 1, 2], dtype=torch.int32))
        rows.append(serve(one, "logits", "unit", pool=step_pool)[0])
    y = torch.stack(rows, 1).reshape(80, 72)
    check_serve(c, y, step_pool.cpu(), "logits", "unit")
    assert torch.allclose(pool, step_pool.cpu(), rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset,width", [(0, 64), (3, 64), (8, 200), (1, 33)])
def test_rows_of_a_wider_projection(dtype, offset, width):
    """x and decay as column slices of one tensor: rows far apart, starts aligned to the element only."""
    from flashrwkv2_b200 import infer_tmix_gated_scan_fp32io16_forward_varlen as op

    c = case([70, 3, 60], width, dtype, "logits", seed=9)
    wide = torch.full((133, 2 * width + offset + 5), math.nan, dtype=dtype)
    wide[:, offset:offset + width], wide[:, offset + width:offset + 2 * width] = c["x"], c["decay"]
    wide = wide.to(DEV)
    pool = c["pool"].to(DEV)
    y = op(wide[:, offset:offset + width], wide[:, offset + width:offset + 2 * width], state_pool=pool, cu_seqlens=c["cu"].to(DEV),
           state_indices=c["slots"].to(DEV))
    assert y.is_contiguous()
    check_serve(c, y.cpu(), pool.cpu(), "logits", "unit")


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_row_for_all_tokens(dtype):
    """Rows at distance 0 (an expanded tensor), from a start that is aligned to the element only."""
    from flashrwkv2_b200 import infer_tmix_gated_scan_fp32io16_forward_varlen as op

    c = case([300, 290], 70, dtype, "logits", seed=16)
    row = torch.full((73,), math.nan, dtype=dtype)
    row[1:71] = c["x"][0]
    c["x"] = c["x"][:1].expand(590, 70).contiguous()
    x = row.to(DEV)[1:71].expand(590, 70)
    assert x.stride(0) == 0
    pool = c["pool"].to(DEV)
    y = op(x, c["decay"].to(DEV), state_pool=pool, cu_seqlens=c["cu"].to(DEV), state_indices=c["slots"].to(DEV))
    check_serve(c, y.cpu(), pool.cpu(), "logits", "unit")


def test_very_many_sequences():
    """Several sequences to a unit of work; short ones, which the step kernel serves, among them."""
    g = torch.Generator().manual_seed(5)
    c = case(torch.randint(1, 33, (1100,), generator=g).tolist(), 992, torch.bfloat16, "logits", seed=17)
    y, pool = serve(c, "logits", "unit")
    check_serve(c, y, pool, "logits", "unit")
    c, initial, dy, dfinal = train_case(torch.randint(1, 20, (1100,), generator=g).tolist(), 992, torch.bfloat16, "logits", 18)
    got = train(c["x"], c["decay"], initial, dy, dfinal, "logits", "unit", cu=c["cu"])
    check_train(c, got, initial, dy, dfinal, "logits", "unit")


def test_offsets_beyond_two_to_the_thirty_one_elements():
    """66000 rows of 32800 channels: the last rows lie past 2^31 elements.  Channels are independent, so the last eight of them
    against the oracle say whether every offset is right."""
    from flashrwkv2_b200 import infer_tmix_gated_scan_fp32io16_forward_varlen as op

    rows, channels = 66000, 32800
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    small = case([rows - 3000, 3000], 8, torch.bfloat16, "retention", seed=19, spare=0)
    x, decay = (torch.zeros(rows, channels, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    x[:, -8:], decay[:, -8:] = small["x"].to(DEV), small["decay"].to(DEV)
    pool = torch.zeros(2, channels, device=DEV)
    pool[:, -8:] = small["pool"].to(DEV)
    y = op(x, decay, state_pool=pool, cu_seqlens=small["cu"].to(DEV), state_indices=small["slots"].to(DEV), decay_mode="retention")
    check_serve(small, y[:, -8:].cpu(), pool[:, -8:].cpu(), "retention", "unit")
    assert float(y[:, :-8].abs().max()) == 0 and float(pool[:, :-8].abs().max()) == 0


def test_extreme_logits_and_retentions():
    big = torch.tensor([-math.inf, -200.0, -90.0, -30.0, -17.0, 17.0, 30.0, 100.0, math.inf, 0.0])
    c = case([50], 10, torch.float32, "logits", seed=10)
    c["decay"] = big.repeat(50, 1)
    y, pool = serve(c, "logits", "unit")
    check_serve(c, y, pool, "logits", "unit")
    c["decay"] = torch.tensor([0.0, 1.0, 1e-20, 1e-4, 0.5, 0.9999999, 1 - 2.0 ** -12, 0.3, 1e-38, 0.0]).repeat(50, 1)
    y, pool = serve(c, "retention", "complement")
    check_serve(c, y, pool, "retention", "complement")


@pytest.mark.parametrize("poison", [math.nan, math.inf])
def test_a_bad_sequence_leaves_its_neighbours_alone(poison):
    for lengths in ([30, 20, 45, 200, 90], [1] * 5):
        c = case(lengths, 40, torch.float32, "logits", seed=11)
        clean_y, clean_pool = serve(c, "logits", "unit")
        lo, hi = int(c["cu"][2]), int(c["cu"][3])
        c["x"][lo:hi, 7] = poison
        c["pool"][int(c["slots"][2]), 9] = poison
        y, pool = serve(c, "logits", "unit")
        hit = torch.zeros_like(y, dtype=torch.bool)
        hit[lo:hi, 7] = hit[lo:hi, 9] = True
        assert torch.equal(y[~hit], clean_y[~hit]) and not torch.isfinite(y[hit]).any()
        state_hit = torch.zeros_like(pool, dtype=torch.bool)
        state_hit[int(c["slots"][2]), [7, 9]] = True
        assert torch.equal(pool[~state_hit], clean_pool[~state_hit])


def test_run_to_run_bit_identical():
    c = case([3000, 17, 900], 72, torch.float32, "logits", seed=12)
    first = serve(c, "logits", "complement")
    for _ in range(3):
        again = serve(c, "logits", "complement")
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_bad_metadata_raises_with_a_static_ticket_and_fails_closed_with_a_capacity_ticket():
    from flashrwkv2_b200 import infer_tmix_gated_scan_fp32io16_forward_varlen as op
    from flashrwkv2_b200 import prepare_tmix_wkv7_recurrent_metadata as prepare

    c = case([40, 100], 24, torch.bfloat16, "logits", seed=13)
    twice = dict(c, slots=torch.tensor([1, 1], dtype=torch.int32))
    with pytest.raises(RuntimeError, match="unique"):
        serve(twice, "logits", "unit")
    count = lambda v: torch.tensor([v], dtype=torch.int32, device=DEV)
    for slots, bounds in (([1, 1], [0, 40, 140]), ([0, 9], [0, 40, 140]), ([0, 1], [0, 140, 140]), ([0, 1], [0, 40, 139])):
        cu, ix = torch.tensor(bounds, dtype=torch.int32, device=DEV), torch.tensor(slots, dtype=torch.int32, device=DEV)
        ticket = prepare(cu, ix, state_pool_size=4, token_capacity=140, sequence_capacity=2, max_seqlen_capacity=140,
                         num_active_tokens=count(140), num_active_sequences=count(2))
        pool = c["pool"].to(DEV)
        y = op(c["x"].to(DEV), c["decay"].to(DEV), state_pool=pool, cu_seqlens=cu, state_indices=ix, validated_metadata=ticket)
        assert torch.isnan(y).all() and torch.equal(pool.cpu(), c["pool"])


def test_capacity_ticket_in_a_graph_with_rewritten_metadata():
    """Warm-up with nothing active, capture, then replays with other lengths: rows behind the last sequence stay."""
    from flashrwkv2_b200 import infer_tmix_gated_scan_fp32io16_forward_varlen as op
    from flashrwkv2_b200 import prepare_tmix_wkv7_recurrent_metadata as prepare

    cap, n_cap, channels = 400, 4, 72
    c = case([cap], channels, torch.bfloat16, "logits", seed=14, spare=5)
    x, decay, pool = c["x"].to(DEV), c["decay"].to(DEV), c["pool"].to(DEV)
    cu = torch.zeros(n_cap + 1, dtype=torch.int32, device=DEV)
    slots = torch.zeros(n_cap, dtype=torch.int32, device=DEV)
    n_tok, n_seq = (torch.zeros(1, dtype=torch.int32, device=DEV) for _ in range(2))

    def call():
        ticket = prepare(cu, slots, state_pool_size=6, token_capacity=cap, sequence_capacity=n_cap, max_seqlen_capacity=cap,
                         num_active_tokens=n_tok, num_active_sequences=n_seq)
        return op(x, decay, state_pool=pool, cu_seqlens=cu, state_indices=slots, validated_metadata=ticket)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call()
    torch.cuda.synchronize()
    assert torch.equal(pool.cpu(), c["pool"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        y = call()
    for lengths in ([100, 1, 64], [400], [1], [5, 5, 5, 300]):
        n, total = len(lengths), sum(lengths)
        part = dict(c, x=c["x"][:total], decay=c["decay"][:total], lengths=lengths,
                    cu=torch.tensor([0] + lengths).cumsum(0).to(torch.int32), slots=torch.tensor([4, 1, 0, 3][:n], dtype=torch.int32))
        cu.fill_(-7)
        cu[:n + 1].copy_(part["cu"])
        slots.fill_(99)
        slots[:n].copy_(part["slots"])
        n_tok.fill_(total)
        n_seq.fill_(n)
        pool.copy_(c["pool"])
        y.fill_(123.0)
        graph.replay()
        torch.cuda.synchronize()
        check_serve(part, y[:total].cpu(), pool.cpu(), "logits", "unit")
        assert (y[total:] == 123.0).all()


def test_two_graphs_and_an_eager_call_interleaved():
    """Each captured call owns its scratch: replays of two graphs on two streams at once, with an eager call between."""
    from flashrwkv2_b200 import pretrain_tmix_gated_scan_fp32io16 as op

    sets = []
    for seed in (20, 21):
        c = case([2500], 72, torch.float32, "logits", seed=seed)
        x, d = c["x"].to(DEV)[None], c["decay"].to(DEV)[None]
        want = [t.clone() for t in op(x, d)]
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            op(x, d)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            got = op(x, d)
        sets.append((graph, stream, got, want, (x, d)))
    for _ in range(5):
        for graph, stream, got, _, _ in sets:
            for t in got:
                t.zero_()
        torch.cuda.synchronize()
        for graph, stream, *_ in sets:
            with torch.cuda.stream(stream):
                graph.replay()
        eager = op(*sets[0][4])
        torch.cuda.synchronize()
        for _, _, got, want, _ in sets:
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(eager[0], sets[0][3][0])


def test_one_ticket_serves_wkv7_and_the_gated_scan():
    from flashrwkv2_b200 import (infer_tmix_gated_scan_fp32io16_forward_varlen, infer_tmix_wkv7_prefill_fp32io16_forward_varlen,
                                 prepare_tmix_wkv7_recurrent_metadata)
    from flashrwkv2_b200.workloads import make_workload

    t = make_workload("c3", n_seq=3, seq_len=50, heads=2).tensors
    d = {k: v.to(DEV) for k, v in t.items()}
    total, n = d["r"].shape[0], d["state_indices"].numel()
    ticket = prepare_tmix_wkv7_recurrent_metadata(d["cu_seqlens"], d["state_indices"], state_pool_size=d["state_pool"].shape[0],
                                                  total_tokens=total)
    common = dict(cu_seqlens=d["cu_seqlens"], state_indices=d["state_indices"], validated_metadata=ticket)
    y = infer_tmix_wkv7_prefill_fp32io16_forward_varlen(*(d[k] for k in "rwkvab"), state_pool=d["state_pool"],
                                                        decay_mode="retention", **common)
    rows = y.reshape(total, -1)
    memory = torch.zeros(d["state_pool"].shape[0], rows.shape[1], device=DEV)
    decay = d["w"].reshape(total, -1)
    z = infer_tmix_gated_scan_fp32io16_forward_varlen(rows, decay, state_pool=memory, decay_mode="retention",
                                                      input_mode="complement", **common)
    lengths = (d["cu_seqlens"][1:] - d["cu_seqlens"][:-1]).tolist()
    c = dict(x=rows.cpu(), decay=decay.cpu(), pool=torch.zeros_like(memory).cpu(), slots=t["state_indices"], cu=t["cu_seqlens"],
             lengths=lengths)
    assert len(lengths) == n
    check_serve(c, z.cpu(), memory.cpu(), "retention", "complement")


def test_another_stream():
    c = case([500, 90], 64, torch.bfloat16, "logits", seed=15)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        y, pool = serve(c, "logits", "unit")
    check_serve(c, y, pool, "logits", "unit")


# ---- training form


def train(x, decay, initial, dy, dfinal, decay_mode, input_mode, cu=None):
    from flashrwkv2_b200 import pretrain_tmix_gated_scan_fp32io16 as op

    leaves = [t.to(DEV).requires_grad_() for t in (x, decay)]
    h0 = None if initial is None else initial.to(DEV).requires_grad_()
    y, final = op(*leaves, initial_state=h0, cu_seqlens=None if cu is None else cu.to(DEV), decay_mode=decay_mode,
                  input_mode=input_mode)
    outputs, grads = [], []
    for out, grad in ((y, dy), (final, dfinal)):
        if grad is not None:
            outputs.append(out)
            grads.append(grad.to(DEV))
    got = torch.autograd.grad(outputs, leaves + ([] if h0 is None else [h0]), grads)
    torch.cuda.synchronize()
    return [t.detach().cpu() for t in (y, final, *got)]


def check_train(c, got, initial, dy, dfinal, decay_mode, input_mode):
    dtype, channels = c["x"].dtype, c["x"].shape[-1]
    y, final, dx, dd = (t.reshape(-1, channels) for t in got[:4])
    zeros = torch.zeros(len(c["lengths"]), channels)
    dy = torch.zeros(c["x"].shape) if dy is None else dy
    for i in range(len(c["lengths"])):
        lo, hi = int(c["cu"][i]), int(c["cu"][i + 1])
        w = oracle.backward(c["x"][lo:hi], c["decay"][lo:hi], (zeros if initial is None else initial)[i], dy[lo:hi],
                            (zeros if dfinal is None else dfinal)[i], decay_mode, input_mode)
        close(y[lo:hi], w["y"], w["off"], dtype, ("y", i))
        close(final[i], w["final"], w["final_off"], torch.float32, ("final", i))
        close(dx[lo:hi], w["dx"], w["dx_off"], dtype, ("dx", i))
        close(dd[lo:hi], w["ddecay"], w["ddecay_off"], dtype, ("ddecay", i))
        if initial is not None:
            close(got[4][i], w["dinitial"], w["dinitial_off"], torch.float32, ("dinitial", i))


def train_case(lengths, channels, dtype, decay_mode, seed):
    c = case(lengths, channels, dtype, decay_mode, seed)
    g = torch.Generator().manual_seed(seed + 77)
    n = len(lengths)
    return (c, torch.randn(n, channels, generator=g), torch.randn(c["x"].shape, generator=g).to(dtype),
            torch.randn(n, channels, generator=g))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("decay_mode,input_mode", MODES)
def test_training_packed(dtype, decay_mode, input_mode):
    for lengths, channels in (([1, 63, 64, 65, 130], 72), ([3], 1), ([200, 7], 19)):
        c, initial, dy, dfinal = train_case(lengths, channels, dtype, decay_mode, 30)
        got = train(c["x"], c["decay"], initial, dy, dfinal, decay_mode, input_mode, cu=c["cu"])
        check_train(c, got, initial, dy, dfinal, decay_mode, input_mode)


@pytest.mark.parametrize("batch,tokens,channels", [(1, 1, 8), (3, 1, 5), (2, 64, 64), (3, 100, 40), (1, 700, 136)])
def test_training_dense(batch, tokens, channels):
    c, initial, dy, dfinal = train_case([tokens] * batch, channels, torch.float32, "logits", 31)
    shape = (batch, tokens, channels)
    got = train(c["x"].view(shape), c["decay"].view(shape), initial, dy.view(shape), dfinal, "logits", "complement")
    assert got[0].shape == got[2].shape == shape
    check_train(c, got, initial, dy, dfinal, "logits", "complement")
    packed = train(c["x"], c["decay"], initial, dy, dfinal, "logits", "complement", cu=c["cu"])
    for a, b in zip(got, packed):
        assert torch.equal(a.reshape(-1), b.reshape(-1))


@pytest.mark.parametrize("decay_mode", ["logits", "retention"])
def test_training_long_with_slow_channels(decay_mode):
    c = case([3000, 1100], 40, torch.float32, decay_mode, seed=5, slow=True)
    g = torch.Generator().manual_seed(3)
    initial, dfinal = torch.randn(2, 40, generator=g), torch.randn(2, 40, generator=g)
    dy = torch.randn(4100, 40, generator=g)
    got = train(c["x"], c["decay"], initial, dy, dfinal, decay_mode, "unit", cu=c["cu"])
    check_train(c, got, initial, dy, dfinal, decay_mode, "unit")


def test_training_without_initial_state_or_without_one_of_the_gradients():
    c, initial, dy, dfinal = train_case([90, 40], 24, torch.float32, "logits", 32)
    check_train(c, train(c["x"], c["decay"], None, dy, dfinal, "logits", "unit", cu=c["cu"]), None, dy, dfinal, "logits", "unit")
    check_train(c, train(c["x"], c["decay"], initial, dy, None, "logits", "unit", cu=c["cu"]), initial, dy, None, "logits", "unit")
    check_train(c, train(c["x"], c["decay"], initial, None, dfinal, "logits", "unit", cu=c["cu"]), initial, None, dfinal, "logits", "unit")


def test_training_rows_of_a_wider_projection_and_an_expanded_gradient():
    from flashrwkv2_b200 import pretrain_tmix_gated_scan_fp32io16 as op

    c, _, _, _ = train_case([70, 70], 33, torch.float32, "logits", 33)
    wide = torch.cat([c["x"], c["decay"]], 1).view(2, 70, 66).to(DEV).requires_grad_()
    y, _ = op(*wide.chunk(2, -1))
    y.sum().backward()
    got = wide.grad.cpu()
    zeros, ones = torch.zeros(2, 33), torch.ones(140, 33)
    y = y.detach().cpu().reshape(140, 33)
    for i in range(2):
        w = oracle.backward(c["x"][70 * i:70 * i + 70], c["decay"][70 * i:70 * i + 70], zeros[i], ones[:70], zeros[i], "logits", "unit")
        close(y[70 * i:70 * i + 70], w["y"], w["off"], torch.float32, "y")
        close(got[i, :, :33], w["dx"], w["dx_off"], torch.float32, "dx")
        close(got[i, :, 33:], w["ddecay"], w["ddecay_off"], torch.float32, "ddecay")


@pytest.mark.parametrize("decay_mode,input_mode", MODES)
def test_training_gradient_against_differences(decay_mode, input_mode):
    """Central differences of the fp32 forward pass along a random direction of every input.  f = sum(y w) in float64, so its
    error is that of y: at most 2^-20 of sum |y w| a side, over 2 step; the third derivative adds step^2 of the scale."""
    from flashrwkv2_b200 import pretrain_tmix_gated_scan_fp32io16 as op

    c, initial, dy, dfinal = train_case([70, 9], 12, torch.float32, decay_mode, 34)
    if decay_mode == "retention":
        c["decay"] = c["decay"] * 0.9
    got = train(c["x"], c["decay"], initial, dy, dfinal, decay_mode, input_mode, cu=c["cu"])
    g = torch.Generator().manual_seed(9)
    base = [c["x"], c["decay"], initial]
    step = 2.0 ** -7
    for k, grad in enumerate((got[2], got[3], got[4])):
        v = torch.randn(base[k].shape, generator=g) * (0.02 if k == 1 and decay_mode == "retention" else 1.0)
        told, size = [], 0.0
        for sign in (1, -1):
            moved = [t.double() if j != k else t.double() + sign * step * v.double() for j, t in enumerate(base)]
            y, final = op(moved[0].float().to(DEV), moved[1].float().to(DEV), initial_state=moved[2].float().to(DEV),
                          cu_seqlens=c["cu"].to(DEV), decay_mode=decay_mode, input_mode=input_mode)
            told.append(float((y.cpu().double() * dy).sum() + (final.cpu().double() * dfinal).sum()))
            size = max(size, float((y.cpu().double() * dy).abs().sum() + (final.cpu().double() * dfinal).abs().sum()))
        slope = (told[0] - told[1]) / (2 * step)
        want = float((grad.double() * v).sum())
        allowed = 2.0 ** -20 * size / step + (16 * step * step * size if k == 1 else 0.0)
        assert abs(slope - want) <= allowed, (k, slope, want, allowed)


def test_training_bad_bounds_make_everything_nan():
    c, initial, dy, dfinal = train_case([40, 30], 16, torch.bfloat16, "logits", 35)
    for bounds in ([0, 80, 70], [0, 40, 69], [1, 40, 70], [0, 0, 70]):
        got = train(c["x"], c["decay"], initial, dy, dfinal, "logits", "unit", cu=torch.tensor(bounds, dtype=torch.int32))
        assert all(torch.isnan(t).all() for t in got), bounds


def test_training_step_captured_and_replayed():
    from flashrwkv2_b200 import pretrain_tmix_gated_scan_fp32io16 as op

    c, initial, dy, dfinal = train_case([300, 90, 1], 72, torch.bfloat16, "logits", 36)
    want = train(c["x"], c["decay"], initial, dy, dfinal, "logits", "unit", cu=c["cu"])
    x, decay, h0 = (torch.zeros_like(t, device=DEV).requires_grad_() for t in (c["x"], c["decay"], initial))
    cu, gy, gf = torch.tensor([0, 391, 391, 391], dtype=torch.int32, device=DEV), dy.to(DEV), dfinal.to(DEV)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())

    def step():
        y, final = op(x, decay, initial_state=h0, cu_seqlens=cu)
        return [y.detach(), final.detach(), *torch.autograd.grad((y, final), (x, decay, h0), (gy, gf))]

    with torch.cuda.stream(stream):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = step()
    with torch.no_grad():
        x.copy_(c["x"])
        decay.copy_(c["decay"])
        h0.copy_(initial)
        cu.copy_(c["cu"])
    for _ in range(3):
        for t in out:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a.cpu(), b)


def test_training_changed_input_is_noticed():
    from flashrwkv2_b200 import pretrain_tmix_gated_scan_fp32io16 as op

    x = torch.randn(1, 10, 8, device=DEV)
    decay = torch.randn(1, 10, 8, device=DEV, requires_grad=True)
    y, _ = op(x, decay)
    x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_training_is_differentiable_once():
    from flashrwkv2_b200 import pretrain_tmix_gated_scan_fp32io16 as op

    x, decay = (torch.randn(1, 10, 8, device=DEV, requires_grad=True) for _ in range(2))
    y, _ = op(x, decay)
    plain, = torch.autograd.grad(y.sum(), x, retain_graph=True)
    recorded, = torch.autograd.grad(y.sum(), x, create_graph=True)
    assert torch.equal(plain, recorded)
    with pytest.raises(RuntimeError, match="differentiable once"):
        recorded.sum().backward()


def test_training_without_gradients_builds_no_graph():
    from flashrwkv2_b200 import pretrain_tmix_gated_scan_fp32io16 as op

    x, decay = (torch.randn(1, 10, 8, device=DEV, requires_grad=True) for _ in range(2))
    with torch.no_grad():
        y, final = op(x, decay)
    assert not y.requires_grad and not final.requires_grad
    y, final = op(x.detach(), decay.detach())
    assert not y.requires_grad and not final.requires_grad
    y, final = op(x.detach(), decay)  # one input alone
    assert torch.autograd.grad(y.sum() + final.sum(), decay)[0].shape == decay.shape
