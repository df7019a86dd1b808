"""Float64 token log probabilities, entropy, top alternatives and their gradient, with bounds on fp32 arithmetic.  Test
infrastructure.

Bounds: e = 2^-24 is half a step of fp32.  A scaled difference z = (x - m) / T is off by at most 4e |z|, its exponential by that
and 2^-21 of itself, or by 2^-126 in all: fp32 has no normal number below that, so a probability may become one or zero there (its
relative error is then unbounded, which no relative term covers).  Sums over the vocabulary are chains of at most V / 128 + 64 additions, however they are split."""

from __future__ import annotations

import math

import torch

E = 2.0 ** -24


def rows(logits, ids, temperature, ignore_index=-100):
    x = logits.double()
    vocab = x.shape[-1]
    m = x.amax(-1, keepdim=True)
    z = (x - m) / temperature
    empty = (m == -math.inf)[..., 0]
    z = torch.where(empty[..., None], torch.full_like(z, -math.inf), z)
    log_s = torch.where(empty, torch.zeros_like(m[..., 0]), torch.log(torch.exp(z).sum(-1)))
    logp = z - log_s[..., None]
    p = torch.exp(logp)
    finite_z = torch.where(p > 0, z, torch.zeros_like(z))
    entropy = torch.where(empty, torch.zeros_like(log_s), log_s - (p * finite_z).sum(-1))
    reach = (p * finite_z.abs()).sum(-1)
    sum_off = (vocab / 128 + 64) * E + 2.0 ** -21 + 4 * E * reach
    live = ids != ignore_index
    known = (ids >= 0) & (ids < vocab)
    picked = logp.gather(-1, ids.clamp(0, vocab - 1).long()[..., None])[..., 0]
    picked = torch.where(known, picked, torch.full_like(picked, math.nan))
    zero = torch.zeros_like(picked)
    return dict(z=z, p=p, logp=logp, live=live, known=known, empty=empty, sum_off=sum_off, reach=reach,
                logprobs=torch.where(live, picked, zero),
                logprobs_off=sum_off + 8 * E * (picked.abs() + log_s.abs()),
                entropy=torch.where(live, entropy, zero), entropy_off=2 * sum_off * (1 + reach) + 4 * E * log_s.abs(),
                top_off=sum_off[..., None] + 8 * E * (logp.abs() + log_s.abs()[..., None]))


def top(logits, k):
    """Ids of the k largest logits, lowest id first among equals, NaN above all: stable sort."""
    x = logits.double()
    x = torch.where(torch.isnan(x), torch.full_like(x, math.inf), x * 1.0)
    key = torch.where(torch.isnan(logits.double()), torch.ones_like(x), torch.zeros_like(x))
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    order = order.gather(-1, torch.sort(key.gather(-1, order), dim=-1, descending=True, stable=True).indices)
    return order[..., :k]


def gradient(logits, ids, temperature, dlogprobs, dentropy, ignore_index=-100):
    """dlogits and its bound before rounding to the logits' type."""
    r = rows(logits, ids, temperature, ignore_index)
    a, b = dlogprobs.double()[..., None], dentropy.double()[..., None]
    logp = torch.where(r["p"] > 0, r["logp"], torch.zeros_like(r["p"]))
    weight = a + b * (logp + r["entropy"][..., None])
    grad = torch.where(r["p"] > 0, -r["p"] * weight, torch.zeros_like(r["p"]))
    p_off = r["p"] * (8 * E * r["z"].abs().nan_to_num(0, posinf=0, neginf=0) + r["sum_off"][..., None] + 2.0 ** -21) + 2.0 ** -126
    off = p_off * (a.abs() + b.abs() * (logp.abs() + r["entropy"][..., None]))
    off = off + r["p"] * b.abs() * (r["top_off"].nan_to_num(0, posinf=0) + r["entropy_off"][..., None]) + 8 * E * grad.abs()
    at = ids.clamp(0, logits.shape[-1] - 1).long()[..., None]
    picked = torch.zeros_like(grad).scatter(-1, at, 1.0)
    grad = grad + a * picked
    off = off + 8 * E * (a.abs() * picked)
    grad = torch.where((r["live"] & ~r["known"])[..., None], torch.full_like(grad, math.nan), grad)
    skip = (~r["live"] | (r["empty"] & r["known"]))[..., None]
    return torch.where(skip, torch.zeros_like(grad), grad) / temperature, off / temperature, r
