"""GPU parity of the token log probabilities, the entropy, the top alternatives and their gradient.

Expectation: oracle.token_logprobs_oracle in float64, which also gives the bound of fp32 arithmetic for every value; a gradient
in 16 bits may differ by that and half a step of its type.  Ids have to be equal."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import token_logprobs_oracle as oracle
from oracle.gated_scan_oracle import half_step

pytestmark = pytest.mark.gpu

DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def case(rows, vocab, dtype, seed=0, scale=2.5):
    g = torch.Generator().manual_seed(seed + 7 * rows + vocab)
    return ((scale * torch.randn(rows, vocab, generator=g)).to(dtype), torch.randint(0, vocab, (rows,), generator=g),
            torch.randn(rows, generator=g), torch.randn(rows, generator=g))


def near(got, want, off, what):
    got, want = got.detach().cpu().double(), want.cpu()
    plain = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    odd = ~plain & ~torch.isnan(want)
    assert torch.equal(got[odd], want[odd]), what
    excess = (got - want).abs()[plain] - off.cpu()[plain]
    assert not plain.any() or float(excess.max()) <= 0, (what, float(excess.max()))


def score(logits, ids, temperature=1.0, top_k=0, **more):
    from flashrwkv2_b200 import rl_infctx_head_token_logprobs as op

    out = op(logits.to(DEV), ids.to(DEV), temperature=temperature, top_k=top_k, **more)
    torch.cuda.synchronize()
    return out


def check(logits, ids, out, temperature=1.0, top_k=0, **more):
    r = oracle.rows(logits, ids, temperature, **more)
    near(out.logprobs, r["logprobs"], r["logprobs_off"], "logprobs")
    near(out.entropy, r["entropy"], r["entropy_off"], "entropy")
    assert out.logprobs.dtype == out.entropy.dtype == torch.float32
    if not top_k:
        assert out.top_ids is None and out.top_logprobs is None
        return
    want = oracle.top(logits, top_k)
    live = r["live"][..., None]
    assert out.top_ids.dtype == torch.int64
    assert torch.equal(out.top_ids.cpu(), torch.where(live, want, -1))
    told = torch.where(live, r["logp"].gather(-1, want), torch.full_like(want, -math.inf, dtype=torch.float64))
    near(out.top_logprobs, told, r["top_off"].gather(-1, want), "top_logprobs")


def gradient(logits, ids, temperature, a, b, **more):
    from flashrwkv2_b200 import rl_infctx_head_token_logprobs as op

    x = logits.to(DEV).requires_grad_()
    out = op(x, ids.to(DEV), temperature=temperature, **more)
    grad, = torch.autograd.grad((out.logprobs, out.entropy), x, (a.to(DEV), b.to(DEV)))
    torch.cuda.synchronize()
    return grad


def check_gradient(logits, ids, grad, temperature, a, b, **more):
    want, off, _ = oracle.gradient(logits, ids, temperature, a, b, **more)
    assert grad.dtype == logits.dtype and grad.shape == logits.shape
    off = off + half_step(logits.dtype, want.nan_to_num(0)) + off * torch.finfo(logits.dtype).eps
    near(grad, want, off, "dlogits")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 2), (3, 7), (5, 31), (2, 257), (4, 1000), (7, 4099), (1, 65536), (3, 50277), (200, 515),
                                        (2, 131073)])
def test_sizes(rows, vocab, dtype):
    logits, ids, a, b = case(rows, vocab, dtype)
    top_k = min(vocab, 20)
    check(logits, ids, score(logits, ids, top_k=top_k), top_k=top_k)
    check(logits, ids, score(logits, ids))
    check_gradient(logits, ids, gradient(logits, ids, 1.0, a, b), 1.0, a, b)


@pytest.mark.parametrize("temperature", [1e-30, 1e30])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_the_ends_of_the_temperature_range(dtype, temperature):
    """At 1e-30 all of the probability is on the largest logits, at 1e30 it is even."""
    logits, ids, a, b = case(6, 2000, dtype, seed=2)
    check(logits, ids, score(logits, ids, temperature, 5), temperature, 5)
    check_gradient(logits, ids, gradient(logits, ids, temperature, a, b), temperature, a, b)


@pytest.mark.parametrize("temperature", [0.3, 1.0, 2.5, 100.0])
@pytest.mark.parametrize("top_k", [1, 5, 32])
def test_temperature_and_top_k(temperature, top_k):
    logits, ids, a, b = case(6, 2000, torch.bfloat16, seed=1)
    check(logits, ids, score(logits, ids, temperature, top_k), temperature, top_k)
    check_gradient(logits, ids, gradient(logits, ids, temperature, a, b), temperature, a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [300, 8192, 40001])
def test_ties_rank_by_id(dtype, vocab):
    """All equal; two values; the largest value many times in one place; -0 beside +0."""
    g = torch.Generator().manual_seed(vocab)
    logits = torch.zeros(5, vocab)
    logits[1] = torch.randint(0, 2, (vocab,), generator=g).float()
    logits[2, vocab // 2:] = 3.0
    logits[3] = -torch.zeros(vocab)
    logits[3, ::3] = 0.0
    logits[4] = torch.randint(-3, 4, (vocab,), generator=g).float()
    logits = logits.to(dtype)
    ids = torch.randint(0, vocab, (5,), generator=g)
    check(logits, ids, score(logits, ids, top_k=32), top_k=32)


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_rows(dtype):
    """-inf in most places, in all but one, in all; the type's lowest value likewise; the given token masked or not."""
    vocab, low = 3001, torch.finfo(dtype).min
    logits, ids, a, b = case(9, vocab, dtype, seed=2)
    g = torch.Generator().manual_seed(5)
    for row, fill in ((0, -math.inf), (1, low)):
        hide = torch.rand(vocab, generator=g) < 0.95
        logits[row, hide] = fill
    ids[1] = int((logits[1] > low).nonzero()[0])
    for row, fill in ((2, -math.inf), (3, low)):
        keep = logits[row, 77].clone()
        logits[row] = fill
        logits[row, 77] = keep
        ids[row] = 77
    logits[4] = -math.inf
    logits[5] = low
    logits[6, :] = -math.inf
    logits[6, 2999] = 1.0
    ids[6] = 5
    logits[7, int(ids[7])] = -math.inf
    check(logits, ids, score(logits, ids, top_k=32), top_k=32)
    check_gradient(logits, ids, gradient(logits, ids, 1.0, a, b), 1.0, a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [math.nan, -math.nan, math.inf])
def test_nan_and_infinity_stay_in_their_row(dtype, bad):
    logits, ids, a, b = case(4, 2100, dtype, seed=3)
    clean = score(logits, ids, top_k=4)
    logits[1, 700] = logits[1, 2099] = bad
    logits[2] = bad
    out = score(logits, ids, top_k=4)
    for row in (1, 2):
        assert torch.isnan(out.logprobs[row]) and torch.isnan(out.entropy[row]) and torch.isnan(out.top_logprobs[row]).all()
    assert out.top_ids[1, :2].tolist() == [700, 2099] and out.top_ids[2].tolist() == [0, 1, 2, 3]
    for row in (0, 3):
        for x, y in zip(clean, out):
            assert torch.equal(x[row], y[row])
    grad = gradient(logits, ids, 1.0, a, b)
    assert torch.isnan(grad[1:3]).all() and torch.isfinite(grad[[0, 3]]).all()


def test_left_out_and_unknown_ids():
    logits, ids, a, b = case(6, 1500, torch.bfloat16, seed=4)
    ids[1], ids[3], ids[4] = -100, -1, 1500
    logits[1] = math.nan  # not looked at
    out = score(logits, ids, top_k=3)
    assert out.logprobs[1] == 0 and out.entropy[1] == 0 and (out.top_ids[1] == -1).all() and (out.top_logprobs[1] == -math.inf).all()
    assert torch.isnan(out.logprobs[[3, 4]]).all() and torch.isfinite(out.entropy).all()
    grad = gradient(logits, ids, 1.0, a, b)
    assert (grad[1] == 0).all() and torch.isnan(grad[3:5]).all() and torch.isfinite(grad[[0, 2, 5]]).all()
    other = torch.where(ids == -100, 7, ids)
    out = score(logits, other, ignore_index=7, top_k=3)
    assert out.logprobs[1] == 0 and (out.top_ids[1] == -1).all()
    big = torch.full_like(ids, 2 ** 40)  # wider than 32 bits and still outside
    assert torch.isnan(score(logits[[0] * 6], big).logprobs).all()


@pytest.mark.parametrize("ids_dtype", [torch.int64, torch.int32])
def test_shifted_batch_without_a_copy(ids_dtype):
    """logits[:, :-1] against ids[:, 1:], as a language model is scored; odd rows start anywhere."""
    from flashrwkv2_b200 import rl_infctx_head_token_logprobs as op

    for vocab, dtype in ((513, torch.bfloat16), (1024, torch.float16), (77, torch.float32)):
        g = torch.Generator().manual_seed(vocab)
        logits = torch.randn(3, 6, vocab, generator=g).to(dtype)
        ids = torch.randint(0, vocab, (3, 6), generator=g).to(ids_dtype)
        x = logits.to(DEV).requires_grad_()
        out = op(x[:, :-1], ids.to(DEV)[:, 1:], top_k=2)
        check(logits[:, :-1], ids[:, 1:], out, top_k=2)
        a, b = torch.randn(3, 5, generator=g), torch.randn(3, 5, generator=g)
        grad, = torch.autograd.grad((out.logprobs, out.entropy), x, (a.to(DEV), b.to(DEV)))
        assert (grad[:, -1] == 0).all()
        check_gradient(logits[:, :-1], ids[:, 1:].long(), grad[:, :-1], 1.0, a, b)


def test_columns_of_a_wider_tensor():
    """A padded vocabulary cut to its true size: rows start at every alignment of the element."""
    g = torch.Generator().manual_seed(8)
    for dtype in DTYPES:
        wide = torch.full((6, 1211), math.nan, dtype=dtype)
        wide[:, 3:1106] = torch.randn(6, 1103, generator=g).to(dtype)
        ids = torch.randint(0, 1103, (6,), generator=g)
        wide_gpu = wide.to(DEV)
        check(wide[:, 3:1106], ids, score(wide_gpu[:, 3:1106], ids, top_k=9), top_k=9)
        a, b = torch.randn(6, generator=g), torch.randn(6, generator=g)
        x = wide_gpu[:, 3:1106]
        check_gradient(wide[:, 3:1106], ids, gradient(x, ids, 1.0, a, b), 1.0, a, b)


def test_a_common_offset_costs_no_precision():
    logits, ids, a, b = case(4, 3000, torch.float32, seed=6)
    logits = (logits * 256).round() / 256  # so that the sum below is exact
    moved = logits + 4096.0
    one, two = score(logits, ids, top_k=5), score(moved, ids, top_k=5)
    for x, y in zip(one, two):
        assert torch.equal(x, y)
    assert torch.equal(gradient(logits, ids, 1.0, a, b), gradient(moved, ids, 1.0, a, b))


def test_wide_range_of_logits():
    for dtype in DTYPES:
        logits, ids, a, b = case(4, 2500, dtype, seed=7, scale=300.0)
        check(logits, ids, score(logits, ids, top_k=4), top_k=4)
        check_gradient(logits, ids, gradient(logits, ids, 1.0, a, b), 1.0, a, b)


def test_no_rows_one_row_and_no_row_dimension():
    from flashrwkv2_b200 import rl_infctx_head_token_logprobs as op

    empty = torch.zeros(0, 9, device=DEV, requires_grad=True)
    out = op(empty, torch.zeros(0, dtype=torch.int64, device=DEV), top_k=2)
    assert out.logprobs.shape == (0,) and out.top_ids.shape == (0, 2)
    assert torch.autograd.grad(out.logprobs.sum(), empty)[0].shape == (0, 9)
    row = torch.randn(9, device=DEV)
    out = op(row, torch.tensor(4, device=DEV), top_k=2)
    assert out.logprobs.shape == () and out.top_ids.shape == (2,)
    check(row.cpu()[None], torch.tensor([4]), type(out)(*(t[None] for t in out)), top_k=2)


def test_one_of_the_gradients_alone():
    from flashrwkv2_b200 import rl_infctx_head_token_logprobs as op

    logits, ids, a, b = case(3, 700, torch.float32, seed=9)
    for first in (True, False):
        x = logits.to(DEV).requires_grad_()
        out = op(x, ids.to(DEV))
        grad, = torch.autograd.grad(out.logprobs if first else out.entropy, x, (a if first else b).to(DEV))
        zero = torch.zeros(3)
        check_gradient(logits, ids, grad, 1.0, a if first else zero, zero if first else b)
    x = logits.to(DEV).requires_grad_()
    op(x, ids.to(DEV), top_k=3).logprobs.sum().backward()  # an expanded gradient
    check_gradient(logits, ids, x.grad, 1.0, torch.ones(3), torch.zeros(3))


def test_gradient_against_differences():
    """Central differences in fp32: logprobs are off by `logprobs_off` a side, over 2 step; the third derivative of both outputs is
    below 16, in the direction's norm."""
    from flashrwkv2_b200 import rl_infctx_head_token_logprobs as op

    logits, ids, a, b = case(5, 60, torch.float32, seed=10, scale=1.0)
    grad = gradient(logits, ids, 0.8, a, b).cpu().double()
    g = torch.Generator().manual_seed(1)
    v, step = torch.randn(5, 60, generator=g), 2.0 ** -6
    told = []
    for sign in (1, -1):
        out = op((logits + sign * step * v).to(DEV), ids.to(DEV), temperature=0.8)
        told.append(float((out.logprobs.cpu().double() * a).sum() + (out.entropy.cpu().double() * b).sum()))
    r = oracle.rows(logits, ids, 0.8)
    noise = float((r["logprobs_off"] * a.abs() + r["entropy_off"] * b.abs()).sum()) + 2.0 ** -24 * 16 * 60 / 0.8
    curve = float(((a.abs() + b.abs()) * 16 * (v.abs().amax(1) / 0.8) ** 3).sum()) * step * step / 6
    assert abs((told[0] - told[1]) / (2 * step) - float((grad * v).sum())) <= noise / step + curve


def test_run_to_run_bit_identical_and_batch_independent():
    """A row's results do not depend on its neighbours, and two runs agree in every bit."""
    logits, ids, a, b = case(40, 9001, torch.bfloat16, seed=11)
    first, again = score(logits, ids, top_k=20), score(logits, ids, top_k=20)
    for x, y in zip(first, again):
        assert torch.equal(x, y)
    assert torch.equal(gradient(logits, ids, 1.0, a, b), gradient(logits, ids, 1.0, a, b))


def test_captured_and_replayed_on_another_stream():
    from flashrwkv2_b200 import rl_infctx_head_token_logprobs as op

    logits, ids, a, b = case(20, 3003, torch.bfloat16, seed=12)
    want = [t.clone() for t in score(logits, ids, 0.9, 7)] + [gradient(logits, ids, 0.9, a, b)]
    x, i = torch.zeros_like(logits, device=DEV).requires_grad_(), torch.zeros_like(ids, device=DEV)
    ga, gb = a.to(DEV), b.to(DEV)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())

    def step():
        out = op(x, i, temperature=0.9, top_k=7)
        return [out.logprobs.detach(), out.entropy.detach(), out.top_ids, out.top_logprobs,
                *torch.autograd.grad((out.logprobs, out.entropy), x, (ga, gb))]

    with torch.cuda.stream(stream):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = step()
    with torch.no_grad():
        x.copy_(logits)
        i.copy_(ids)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(got, want):
            assert torch.equal(p, q)


def test_rows_beyond_two_to_the_thirty_one_elements():
    """Offsets past 32 bits: a row whose start lies past 2^31 elements of its tensor."""
    vocab, rows = 65537, 32800
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    logits = torch.zeros(rows, vocab, dtype=torch.bfloat16, device=DEV)
    pick = torch.tensor([0, 17000, 32767, 32768, 32799])
    small, ids, a, b = case(5, vocab, torch.bfloat16, seed=13)
    logits[pick.to(DEV)] = small.to(DEV)
    full_ids = torch.full((rows,), -100, dtype=torch.int64)
    full_ids[pick] = ids
    from flashrwkv2_b200 import rl_infctx_head_token_logprobs as op

    x = logits.requires_grad_()
    out = op(x, full_ids.to(DEV), top_k=3)
    check(small, ids, type(out)(*(t[pick.to(DEV)] for t in out)), top_k=3)
    ga, gb = torch.zeros(rows), torch.zeros(rows)
    ga[pick], gb[pick] = a, b
    grad, = torch.autograd.grad((out.logprobs, out.entropy), x, (ga.to(DEV), gb.to(DEV)))
    check_gradient(small, ids, grad[pick.to(DEV)], 1.0, a, b)
    assert float(grad[1].abs().max()) == 0


def test_rollouts_through_scan_head_and_loss():
    """As they are used together: packed rollouts from carried states through the gated scan, a head, the log probabilities and a
    policy-gradient loss with an entropy bonus; outputs and gradients against float64 autograd.

    Tolerance: everything is fp32; the scan is off by at most 2^-18 of its values (its gate), the two products of 24 terms by 2^-18
    of theirs, and a logit passes at most to a difference of itself: 2^-14 relative to each tensor's largest value holds all."""
    from flashrwkv2_b200 import pretrain_tmix_gated_scan_fp32io16, rl_infctx_head_token_logprobs

    g = torch.Generator().manual_seed(14)
    lengths, width, vocab = [70, 1, 33], 24, 211
    total = sum(lengths)
    leaves = dict(x=torch.randn(total, width, generator=g), decay=torch.randn(total, width, generator=g),
                  h0=torch.randn(3, width, generator=g), head=torch.randn(vocab, width, generator=g) / 5)
    ids = torch.randint(0, vocab, (total,), generator=g)
    ids[::9] = -100
    adv = torch.randn(total, generator=g)
    cu = torch.tensor([0, 70, 71, 104], dtype=torch.int32)

    gpu = {k: v.to(DEV).requires_grad_() for k, v in leaves.items()}
    y, final = pretrain_tmix_gated_scan_fp32io16(gpu["x"], gpu["decay"], initial_state=gpu["h0"], cu_seqlens=cu.to(DEV))
    out = rl_infctx_head_token_logprobs(y @ gpu["head"].t(), ids.to(DEV), temperature=0.9)
    loss = -(out.logprobs * adv.to(DEV)).sum() - 0.01 * out.entropy.sum() + final.square().sum() / 2
    loss.backward()
    loss = loss.detach()

    cpu = {k: v.double().requires_grad_() for k, v in leaves.items()}
    rho = torch.exp(-math.exp(-0.5) * torch.sigmoid(cpu["decay"]))
    rows, finals = [], []
    for s in range(3):
        h = cpu["h0"][s]
        for t in range(int(cu[s]), int(cu[s + 1])):
            h = rho[t] * h + cpu["x"][t]
            rows.append(h)
        finals.append(h)
    logp = torch.log_softmax(torch.stack(rows) @ cpu["head"].t() / 0.9, -1)
    live = (ids != -100).double()
    picked = logp[torch.arange(total), ids.clamp_min(0)] * live
    entropy = -(logp.exp() * logp).sum(-1) * live
    want = -(picked * adv).sum() - 0.01 * entropy.sum() + torch.stack(finals).square().sum() / 2
    want.backward()
    want, picked, finals = want.detach(), picked.detach(), [f.detach() for f in finals]
    assert abs(float(loss) - float(want)) <= 2.0 ** -14 * float((picked * adv).abs().sum() + torch.stack(finals).square().sum())
    for k in leaves:
        top = float(cpu[k].grad.abs().max())
        assert float((gpu[k].grad.cpu().double() - cpu[k].grad).abs().max()) <= 2.0 ** -14 * top, k


def test_differentiable_once_and_no_graph_without_need():
    from flashrwkv2_b200 import rl_infctx_head_token_logprobs as op

    logits, ids, a, b = case(3, 40, torch.float32, seed=15)
    x, ids = logits.to(DEV).requires_grad_(), ids.to(DEV)
    out = op(x, ids, top_k=2)
    assert out.logprobs.requires_grad and out.entropy.requires_grad and not out.top_logprobs.requires_grad
    recorded, = torch.autograd.grad(out.logprobs.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        recorded.sum().backward()
    with torch.no_grad():
        assert not op(x, ids).logprobs.requires_grad
    assert not op(x.detach(), ids).logprobs.requires_grad
    out = op(x, ids)
    with torch.no_grad():
        x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.logprobs.sum().backward()
