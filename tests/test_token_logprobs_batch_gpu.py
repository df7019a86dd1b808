"""GPU: what a row's results owe to the rows that are scored with it: nothing to their values, last bits to their number."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import token_logprobs_oracle as oracle

pytestmark = pytest.mark.gpu

DEV = "cuda"


def score(logits, ids):
    from flashrwkv2_b200 import rl_infctx_head_token_logprobs as op

    x = logits.detach().requires_grad_()
    out = op(x, ids, temperature=0.9, top_k=20)
    grad, = torch.autograd.grad((out.logprobs, out.entropy), x, [torch.full((ids.numel(),), w, device=DEV) for w in (1.5, 0.25)])
    return dict(logprobs=out.logprobs.detach(), entropy=out.entropy.detach(), top_ids=out.top_ids, top_logprobs=out.top_logprobs,
                grad=grad)


def same(a, b):
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))


@pytest.mark.parametrize("dtype,vocab", [(torch.bfloat16, 65536), (torch.float16, 50304), (torch.float32, 33336),
                                         (torch.bfloat16, 17000), (torch.bfloat16, 2048), (torch.bfloat16, 33333)])
def test_rows_among_other_rows(dtype, vocab):
    """Among as many others with other values: the same bits.  Among more, where a row is taken by four, two or one CTA: the same
    alternatives, and floats within the bound of fp32 sums in any order."""
    g = torch.Generator().manual_seed(vocab)
    rows = (2.5 * torch.randn(8, vocab, generator=g)).to(dtype)
    rows[2, vocab // 3:] = -math.inf
    rows[3] = torch.finfo(dtype).min
    rows[4, 5] = math.nan
    ids = torch.randint(0, vocab // 3, (8,), generator=g)
    want = oracle.rows(rows, ids, 0.9)
    off = dict(logprobs=want["logprobs_off"], entropy=want["entropy_off"])
    rows, ids = rows.to(DEV), ids.to(DEV)
    first = None
    for count in (20, 150, 400, 1000):
        told = []
        for seed in (1, 2):
            more = torch.randn(count, vocab, device=DEV, generator=torch.Generator(DEV).manual_seed(seed)).to(dtype)
            more[::7] = math.nan if seed == 1 else -math.inf
            told.append(score(torch.cat([rows, more]), torch.cat([ids, torch.zeros(count, dtype=torch.int64, device=DEV)])))
        for key in told[0]:
            assert same(told[0][key][:8], told[1][key][:8]), (count, key)
        first = first or told[0]
        keep = [0, 1, 2, 3, 5, 6, 7]
        assert torch.equal(told[0]["top_ids"][:8], first["top_ids"][:8])
        for key in off:
            a, b = (t[key][:8].cpu().double()[keep] for t in (told[0], first))
            assert bool(((a - b).abs() <= 2 * off[key][keep]).all()), (count, key)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("temperature", [4.0, 1e3, 1e30])
def test_logits_further_apart_than_the_largest_number(dtype, temperature):
    """The difference of two finite logits may pass fp32's range where the temperature brings it back."""
    from flashrwkv2_b200 import rl_infctx_head_token_logprobs as op

    big = torch.finfo(dtype).max
    logits = torch.zeros(4, 700, dtype=dtype)
    logits[0, 3], logits[0, 5] = big, -big
    logits[1] = -big
    logits[1, 699] = big
    logits[2] = big
    logits[2, :20] = -big
    logits[3, 9] = -math.inf
    ids = torch.tensor([5, 0, 7, 9])
    out = op(logits.to(DEV), ids.to(DEV), temperature=temperature, top_k=32)
    want = oracle.rows(logits, ids, temperature)
    got = out.logprobs.cpu().double()
    assert got[3] == -math.inf and bool(torch.isfinite(got[:3]).all())
    assert bool(((got - want["logprobs"]).abs()[:3] <= want["logprobs_off"][:3]).all())
    assert bool(((out.entropy.cpu().double() - want["entropy"]).abs() <= want["entropy_off"]).all())
    top = oracle.top(logits, 32)
    assert torch.equal(out.top_ids.cpu(), top)
    told, off = (want[key].gather(-1, top) for key in ("logp", "top_off"))
    finite = torch.isfinite(told)
    assert bool(((out.top_logprobs.cpu().double() - told).abs()[finite] <= off[finite]).all())
