"""CPU checks of the gated scan's and the token log probabilities' entry points: refusals, and the oracles' own arithmetic.

The checks live in the compiled module and run before anything touches a device, so calls with CPU tensors reach all of
them; the last one refuses the device."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import gated_scan_oracle, token_logprobs_oracle


@pytest.fixture(autouse=True)
def native_module(monkeypatch):
    import flashrwkv2_b200 as pkg
    from flashrwkv2_b200 import _C_sm100

    monkeypatch.setattr(pkg, "_C", _C_sm100)


def scan_arguments(**changes):
    t = torch.zeros(5, 6, dtype=torch.bfloat16)
    args = dict(x=t, decay_logits=t.clone(), state_pool=torch.zeros(3, 6), cu_seqlens=torch.tensor([0, 2, 5], dtype=torch.int32),
                state_indices=torch.tensor([2, 0], dtype=torch.int32))
    args.update(changes)
    return args


@pytest.mark.parametrize("changes,error,text", [
    (dict(x=None), TypeError, "incompatible function arguments"),
    (dict(x=torch.zeros(5, 6, dtype=torch.float64)), TypeError, "bfloat16, float16 or float32"),
    (dict(decay_logits=torch.zeros(5, 6)), TypeError, "x's dtype"),
    (dict(decay_logits=torch.zeros(5, 7, dtype=torch.bfloat16)), ValueError, "x's shape"),
    (dict(x=torch.zeros(1, 5, 6, dtype=torch.bfloat16)), ValueError, "packed shape"),
    (dict(x=torch.zeros(0, 6, dtype=torch.bfloat16)), ValueError, "nonzero"),
    (dict(x=torch.zeros(6, 5, dtype=torch.bfloat16).t()), ValueError, "unit stride"),
    (dict(state_pool=torch.zeros(3, 7)), ValueError, "state_pool must have shape"),
    (dict(state_pool=torch.zeros(3, 6, dtype=torch.float16)), TypeError, "state_pool must have dtype float32"),
    (dict(state_pool=torch.zeros(3, 12)[:, ::2]), ValueError, "state_pool must be contiguous"),
    (dict(cu_seqlens=torch.tensor([0, 5], dtype=torch.int32)), ValueError, "cu_seqlens must have shape"),
    (dict(cu_seqlens=torch.tensor([0, 2, 5])), TypeError, "int32"),
    (dict(state_indices=torch.tensor([2, 0])), TypeError, "int32"),
    (dict(cu_seqlens=torch.zeros(7, dtype=torch.int32), state_indices=torch.zeros(6, dtype=torch.int32)), ValueError,
     "every sequence needs a token"),
    (dict(decay_bias=torch.zeros(5, dtype=torch.bfloat16)), ValueError, "shape"),
    (dict(decay_bias=torch.zeros(6)), TypeError, "x's dtype"),
    (dict(decay_bias=torch.zeros(6, dtype=torch.bfloat16), decay_mode="retention"), ValueError, "only applies"),
    (dict(decay_mode="exp"), ValueError, "decay_mode"),
    (dict(input_mode="norm"), ValueError, "input_mode"),
    (dict(), ValueError, "x must be CUDA"),
])
def test_gated_scan_refusals(changes, error, text):
    from flashrwkv2_b200 import infer_tmix_gated_scan_fp32io16_forward_varlen as op

    with pytest.raises(error, match=text):
        op(**scan_arguments(**changes))


@pytest.mark.parametrize("changes,error,text", [
    (dict(x=torch.zeros(5, 6)), ValueError, r"\[B,T,C\]"),
    (dict(x=torch.zeros(2, 0, 6)), ValueError, "nonzero"),
    (dict(decay_logits=torch.zeros(2, 5, 6, dtype=torch.float16)), TypeError, "x's dtype"),
    (dict(x=torch.zeros(5, 2, 6).transpose(0, 1)), ValueError, "regular distance"),
    (dict(initial_state=torch.zeros(2, 6, dtype=torch.bfloat16)), TypeError, "initial_state must have dtype float32"),
    (dict(initial_state=torch.zeros(3, 6)), ValueError, r"initial_state must have shape \[N,C\]"),
    (dict(cu_seqlens=torch.tensor([0, 5], dtype=torch.int32)), ValueError, "packed shape"),
    (dict(x=torch.zeros(5, 6), decay_logits=torch.zeros(5, 6), cu_seqlens=torch.tensor([0, 5])), TypeError, "int32"),
    (dict(x=torch.zeros(5, 6), decay_logits=torch.zeros(5, 6), cu_seqlens=torch.zeros(1, dtype=torch.int32)), ValueError,
     r"\[N\+1\]"),
    (dict(x=torch.zeros(2, 6), decay_logits=torch.zeros(2, 6), cu_seqlens=torch.zeros(4, dtype=torch.int32)), ValueError,
     "needs a token"),
    (dict(decay_mode="none"), ValueError, "decay_mode"),
    (dict(), ValueError, "x must be CUDA"),
])
def test_gated_scan_training_refusals(changes, error, text):
    from flashrwkv2_b200 import pretrain_tmix_gated_scan_fp32io16 as op

    args = dict(x=torch.zeros(2, 5, 6), decay_logits=torch.zeros(2, 5, 6))
    args.update(changes)
    with pytest.raises(error, match=text):
        op(**args)


@pytest.mark.parametrize("changes,error,text", [
    (dict(logits=torch.zeros(3, 8, dtype=torch.float64)), TypeError, "bfloat16, float16 or float32"),
    (dict(token_ids=torch.zeros(3)), TypeError, "int64 or int32"),
    (dict(token_ids=torch.zeros(2, dtype=torch.int64)), ValueError, "shape of logits"),
    (dict(logits=torch.zeros(3, 0)), ValueError, "V > 0"),
    (dict(logits=torch.zeros(8, 3).t()), ValueError, "unit stride"),
    (dict(logits=torch.zeros(5, 4, 3, 8).transpose(0, 2)[:, :, ::2], token_ids=torch.zeros(3, 4, 3, dtype=torch.int64)),
     ValueError, "two strides"),
    (dict(temperature=0.0), ValueError, "temperature"),
    (dict(temperature=-1.0), ValueError, "temperature"),
    (dict(temperature=math.nan), ValueError, "temperature"),
    (dict(temperature=math.inf), ValueError, "temperature"),
    (dict(temperature=1e-42), ValueError, "temperature"),
    (dict(top_k=-1), ValueError, "top_k"),
    (dict(top_k=33), ValueError, "top_k"),
    (dict(), ValueError, "logits must be CUDA"),
])
def test_token_logprobs_refusals(changes, error, text):
    from flashrwkv2_b200 import rl_infctx_head_token_logprobs as op

    args = dict(logits=torch.zeros(3, 8), token_ids=torch.zeros(3, dtype=torch.int64))
    args.update(changes)
    with pytest.raises(error, match=text):
        op(**args)


@pytest.mark.parametrize("temperature", [3e-39, 1e-38, 9e-31, 1.1e30, 3e38])
def test_temperatures_whose_reciprocal_overflows_or_is_subnormal_are_refused(temperature):
    """1 / 3e-39 is finite in fp32 but not times log2 e: rows would come out as NaN."""
    from flashrwkv2_b200 import _lib, rl_infctx_head_token_logprobs as op

    with pytest.raises(ValueError, match="temperature"):
        op(torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64), temperature=temperature)
    lib = _lib.load()
    assert lib.frwkv_sm100_token_logprobs(16, 1, 1, 8, 8, 16, 1, -100, 8, 0, temperature, 0, 16, 16, 16, 0, 0, 0) != 0
    assert "temperature" in _lib.last_error()
    assert lib.frwkv_sm100_token_logprobs_backward(16, 1, 1, 8, 8, 16, 1, -100, 8, 0, temperature, 16, 16, 16, 16, 16, 0) != 0
    assert "temperature" in _lib.last_error()


def test_operators_fail_loudly_without_backend(monkeypatch):
    import flashrwkv2_b200 as pkg

    monkeypatch.setattr(pkg, "_C", None)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        pkg.infer_tmix_gated_scan_fp32io16_forward_varlen(**scan_arguments())
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        pkg.pretrain_tmix_gated_scan_fp32io16(torch.zeros(1, 2, 3), torch.zeros(1, 2, 3))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        pkg.rl_infctx_head_token_logprobs(torch.zeros(1, 2), torch.zeros(1, dtype=torch.int64))


def test_c_entries_refuse_bad_arguments():
    from flashrwkv2_b200 import _lib

    lib = _lib.load()

    def scan(pool=16, n_seq=1, total=100, channels=64, io=0, decay=0, gate=0, bias=0):
        return lib.frwkv_sm100_gated_scan(16, 16, 16, pool, 16, 64, 16, 64, bias, 16, n_seq, total, channels, io, decay, gate, 0, 0)

    for bad, text in ((dict(pool=0), "non-null"), (dict(n_seq=0), "1..65535"), (dict(n_seq=65536, total=70000), "1..65535"),
                      (dict(total=0), "token"), (dict(channels=0), "channel"), (dict(total=0x7fffffff), "2^31"), (dict(io=3), "dtype"), (dict(decay=2), "mode"),
                      (dict(gate=-1), "mode"), (dict(bias=16, decay=1), "decay_bias")):
        assert scan(**bad) != 0 and text in _lib.last_error(), bad
    assert lib.frwkv_sm100_gated_scan_train_forward(0, 0, 16, 64, 16, 64, 0, 16, 16, 16, 3, 100, 64, 0, 0, 0, 0, 0) != 0
    assert "multiple of the sequence count" in _lib.last_error()
    assert lib.frwkv_sm100_gated_scan_train_backward(0, 0, 16, 64, 16, 64, 0, 0, 16, 0, 16, 16, 0, 1, 100, 64, 0, 0, 0, 0, 0) != 0
    assert "non-null" in _lib.last_error()

    def rows(outer=1, inner=1, vocab=8, io=0, temperature=1.0, k=0, ids=16):
        return lib.frwkv_sm100_token_logprobs(16, outer, inner, 8, 8, ids, 1, -100, vocab, io, temperature, k, 16, 16, 16, 0, 0, 0)

    for bad, text in ((dict(ids=0), "non-null"), (dict(outer=0), "row count"), (dict(outer=1 << 20, inner=1 << 20), "row count"),
                      (dict(vocab=0), "vocab"), (dict(io=9), "dtype"), (dict(temperature=0.0), "temperature"),
                      (dict(k=33), "top_k"), (dict(k=4), "top_k")):
        assert rows(**bad) != 0 and text in _lib.last_error(), bad


@pytest.mark.parametrize("decay_mode", ["logits", "retention"])
@pytest.mark.parametrize("input_mode", ["unit", "complement"])
def test_scan_oracle_gradient_is_the_autograd_gradient(decay_mode, input_mode):
    g = torch.Generator().manual_seed(1)
    x, d, dy = (torch.randn(9, 4, generator=g, dtype=torch.float64) for _ in range(3))
    if decay_mode == "retention":
        d = torch.rand(9, 4, generator=g, dtype=torch.float64)
    h0, dfinal = torch.randn(4, generator=g, dtype=torch.float64), torch.randn(4, generator=g, dtype=torch.float64)
    leaves = [t.clone().requires_grad_() for t in (x, d, h0)]
    h, rows = leaves[2], []
    for t in range(9):
        rho = torch.exp(-math.exp(-0.5) * torch.sigmoid(leaves[1][t])) if decay_mode == "logits" else leaves[1][t]
        h = rho * h + (leaves[0][t] if input_mode == "unit" else (1 - rho) * leaves[0][t])
        rows.append(h)
    ((torch.stack(rows) * dy).sum() + (h * dfinal).sum()).backward()
    want = gated_scan_oracle.backward(x, d, h0, dy, dfinal, decay_mode, input_mode)
    for leaf, key in zip(leaves, ("dx", "ddecay", "dinitial")):
        assert torch.allclose(leaf.grad, want[key], rtol=1e-12, atol=1e-13), key


def test_logprob_oracle_gradient_is_the_autograd_gradient():
    g = torch.Generator().manual_seed(2)
    x = (3 * torch.randn(5, 11, generator=g, dtype=torch.float64)).requires_grad_()
    ids = torch.randint(0, 11, (5,), generator=g)
    a, b = torch.randn(5, generator=g, dtype=torch.float64), torch.randn(5, generator=g, dtype=torch.float64)
    logp = torch.log_softmax(x / 0.7, -1)
    entropy = -(logp.exp() * logp).sum(-1)
    ((logp[torch.arange(5), ids] * a).sum() + (entropy * b).sum()).backward()
    want, _, r = token_logprobs_oracle.gradient(x.detach(), ids, 0.7, a, b)
    assert torch.allclose(x.grad, want, rtol=1e-12, atol=1e-13)
    assert torch.allclose(r["entropy"], entropy) and torch.allclose(r["logprobs"], logp[torch.arange(5), ids])
