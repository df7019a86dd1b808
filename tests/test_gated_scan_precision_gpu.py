"""GPU precision of the gated scan where errors add up: channels whose decay is slow and the same at every token.

Worst-case bounds over thousands of tokens are too wide to see a bias (an error that always has the same sign), so these
compare root mean square errors against float64 with those of a plain fp32 walk, token by token, of the same inputs."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
RATE = math.exp(-0.5)
MODES = [(d, i) for d in ("logits", "retention") for i in ("unit", "complement")]
DELTAS = (1e-3, 1.2e-4, 1.2e-5, 1e-6)  # 1 - rho


def steady_case(batch, tokens, channels, decay_mode, seed=0):
    """x, decay, dy [B, T, C] fp32 and the states; a quarter of the channels at each of DELTAS, spread by 30 %."""
    g = torch.Generator().manual_seed(seed)
    delta = torch.tensor(DELTAS, dtype=torch.float64).repeat_interleave(channels // 4)
    delta = delta * (1 + 0.3 * torch.rand(channels, generator=g, dtype=torch.float64))
    if decay_mode == "logits":
        s = -torch.log1p(-delta) / RATE
        decay = torch.log(s / (1 - s))
    else:
        decay = 1 - delta
    x, dy = (torch.randn(batch, tokens, channels, generator=g).to(DEV) for _ in range(2))
    initial, dfinal = (torch.randn(batch, channels, generator=g).to(DEV) for _ in range(2))
    return x, decay.float().to(DEV).expand(batch, tokens, channels).contiguous(), initial, dy, dfinal


def gate(decay, decay_mode):
    """rho - 1 and d rho / d decay in float64, of one token's decays."""
    d = decay.double()
    if decay_mode == "retention":
        return d - 1, torch.ones_like(d)
    s = torch.sigmoid(d)
    fall = torch.expm1(-RATE * s)
    return fall, -RATE * s * torch.sigmoid(-d) * (1 + fall)


def walk(x, decay, initial, dy, dfinal, decay_mode, input_mode, dtype):
    """Token by token in `dtype`, from gates that were rounded to it once: y, final, dx, ddecay, dinitial."""
    fall, slope = (t.to(dtype) for t in gate(decay[0, 0], decay_mode))
    x, dy, h, g = (t.to(dtype) for t in (x, dy, initial, dfinal))
    weight = -fall if input_mode == "complement" else torch.ones_like(fall)
    y, before = torch.empty_like(x), torch.empty_like(x)
    for t in range(x.shape[1]):
        before[:, t] = h - x[:, t] if input_mode == "complement" else h
        h = h + (fall * h + weight * x[:, t])
        y[:, t] = h
    dx, dd = torch.empty_like(x), torch.empty_like(x)
    for t in range(x.shape[1] - 1, -1, -1):
        g = dy[:, t] + g
        dx[:, t] = weight * g
        dd[:, t] = g * before[:, t] * slope
        g = g + fall * g
    return dict(y=y, final=h, dx=dx, ddecay=dd, dinitial=g)


def rms_by_delta(t):
    return t.double().reshape(-1, len(DELTAS), t.shape[-1] // len(DELTAS)).square().mean((0, 2)).sqrt()


def check(got, exact, plain, gates):
    """At most twice the plain walk's error, and `gates` beside it: what the gate's own approximations may cost, relative to the
    values (a retention is given, its gate costs nothing)."""
    for key in got:
        size, off, allowed = (rms_by_delta(t) for t in (exact[key], got[key].double() - exact[key], plain[key].double() - exact[key]))
        limit = 2 * allowed + gates * size
        assert bool((off <= limit).all()), (key, (off / size).tolist(), (allowed / size).tolist())


# One sequence on a cluster of CTAs; so many that each is walked by one CTA; one that ends inside a tile.
@pytest.mark.parametrize("batch,tokens,channels", [(1, 6000, 64), (20, 2048, 512), (2, 1111, 20)])
@pytest.mark.parametrize("decay_mode,input_mode", MODES)
def test_steady_slow_channels(decay_mode, input_mode, batch, tokens, channels):
    """The gate from a logit of -6 to -14: an exponent of up to 20 rounded to 2^-20 of one, two approximate functions of 2^-22 and
    a polynomial of 2^-23, so 1 - rho is off by 2^-19 of itself at most, and with it, in sums over many tokens, a state; a
    gradient of the decay meets three such factors."""
    from flashrwkv2_b200 import infer_tmix_gated_scan_fp32io16_forward_varlen, pretrain_tmix_gated_scan_fp32io16

    x, decay, initial, dy, dfinal = steady_case(batch, tokens, channels, decay_mode)
    exact = walk(x, decay, initial, dy, dfinal, decay_mode, input_mode, torch.float64)
    plain = walk(x, decay, initial, dy, dfinal, decay_mode, input_mode, torch.float32)
    leaves = [t.requires_grad_() for t in (x, decay, initial)]
    y, final = pretrain_tmix_gated_scan_fp32io16(x, decay, initial_state=initial, decay_mode=decay_mode, input_mode=input_mode)
    dx, dd, dh = torch.autograd.grad((y, final), leaves, (dy, dfinal))
    logits = decay_mode == "logits"
    check(dict(y=y.detach(), final=final.detach(), dx=dx, dinitial=dh), exact, plain, 2.0 ** -19 if logits else 0.0)
    check(dict(ddecay=dd), exact, plain, 3 * 2.0 ** -19 if logits else 0.0)

    pool = initial.detach().clone()
    cu = torch.arange(0, batch * tokens + 1, tokens, dtype=torch.int32, device=DEV)
    served = infer_tmix_gated_scan_fp32io16_forward_varlen(
        x.detach().view(-1, channels), decay.detach().view(-1, channels), state_pool=pool, cu_seqlens=cu,
        state_indices=torch.arange(batch, dtype=torch.int32, device=DEV), decay_mode=decay_mode, input_mode=input_mode)
    check(dict(y=served.view(batch, tokens, channels), final=pool), exact, plain, 2.0 ** -19 if logits else 0.0)


@pytest.mark.parametrize("input_mode", ["unit", "complement"])
def test_gradient_of_saturated_gates(input_mode):
    """Logits of -40 to 30 and beyond, one token each: the decay's gradient against float64, relative to itself.

    exp(-logit) is off by 2^-22 and by its exponent's rounding, 2^-19 for |logit| <= 44, times log 2; two sigmoids, the rest of
    five factors: 2^-23 and 2^-24 each.  2^-18 holds all, and fp32's smallest normal number what is below it."""
    from flashrwkv2_b200 import pretrain_tmix_gated_scan_fp32io16

    for dtype in (torch.float32, torch.bfloat16):
        logits = torch.cat([torch.arange(-40, 40.5, 0.5), torch.tensor([-math.inf, -200.0, -100.0, -88.0, 60.0, 88.0, 120.0, math.inf])])
        n = logits.numel()
        g = torch.Generator().manual_seed(1)
        x, dy = (torch.randn(1, 1, n, generator=g).to(dtype).to(DEV) for _ in range(2))
        h0, dfinal = (torch.randn(1, n, generator=g).to(DEV) for _ in range(2))
        decay = logits.to(dtype).view(1, 1, n).to(DEV).requires_grad_()
        y, final = pretrain_tmix_gated_scan_fp32io16(x, decay, initial_state=h0, input_mode=input_mode)
        got, = torch.autograd.grad((y, final), decay, (dy, dfinal))
        s, rest = torch.sigmoid(decay.detach().double()), torch.sigmoid(-decay.detach().double())
        slope = -RATE * s * rest * torch.exp(-RATE * s)
        # the sum and the difference in it are fp32: their roundings do not hit the slope alone
        dg, dh = dy.double() + dfinal.double(), h0.double() - (x.double() if input_mode == "complement" else 0.0)
        want = dg * dh * slope
        reach = (dy.double().abs() + dfinal.double().abs()) * (h0.double().abs() + x.double().abs()) * slope.abs()
        allowed = 2.0 ** -18 * want.abs() + 2.0 ** -23 * reach + torch.finfo(dtype).eps / 2 * want.abs() * (1 + 2.0 ** -17)
        allowed = allowed + 2.0 ** -126 * (1 + (dg * dh).abs())
        allowed = torch.where(decay.detach().double().abs() <= 44, allowed, allowed + 2.0 ** -15 * want.abs())
        assert bool(((got.double() - want).abs() <= allowed).all()), ((got.double() - want).abs() / want.abs()).max()
