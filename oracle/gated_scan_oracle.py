"""Float64 gated scan, token by token, with running bounds on what fp32 arithmetic may be off by.  Test infrastructure.

Bounds: e = 2^-24 is half a step of fp32.  One state update costs at most eight roundings of values no larger than hbar
(the scan of |u|), whether the tokens are walked or joined as affine maps; an error made at one token decays like the state
itself.  The gate from a logit is off by at most 2^-18 of 1 - rho (two approximate functions of 2^-22 and an exponent of up to
|logit| <= 32 rounded to 2^-24 of itself); a given retention is exact.  The gate's derivative is a product of such factors, off
by at most 2^-17 of itself.

These are bounds for the worst case: over thousands of tokens they grow too wide to show an error that always has the same sign,
which is compared with a plain fp32 walk instead.
"""

from __future__ import annotations

import math

import torch

E = 2.0 ** -24
RATE = math.exp(-0.5)


def half_step(dtype: torch.dtype, value: torch.Tensor) -> torch.Tensor:
    """Largest error of rounding `value` to dtype: half an eps of it, and of the smallest normal number below that."""
    info = torch.finfo(dtype)
    return 0.5 * info.eps * torch.maximum(value.abs() * (1 + 1e-6), torch.full_like(value, info.smallest_normal))


def gate(decay, bias, decay_mode):
    """rho, 1 - rho, its absolute error, and d(1 - rho)/d decay with its absolute error."""
    d = decay.double() if bias is None else decay.double() + bias.double()
    if decay_mode == "retention":
        return d, 1 - d, E * (1 - d).abs(), torch.full_like(d, -1.0), torch.zeros_like(d)
    s = torch.sigmoid(d)
    rho, delta = torch.exp(-RATE * s), -torch.expm1(-RATE * s)
    slope = RATE * s * torch.sigmoid(-d) * rho
    return rho, delta, 2.0 ** -18 * delta, slope, 2.0 ** -17 * slope + 2.0 ** -126


def forward(x, decay, bias, initial, decay_mode, input_mode):
    """One sequence: x, decay [T, C], initial [C] -> dict of float64 rows and bounds."""
    rho, delta, ddelta, slope, dslope = gate(decay, bias, decay_mode)
    x = x.double()
    u = delta * x if input_mode == "complement" else x
    u_off = ddelta * x.abs() if input_mode == "complement" else torch.zeros_like(x)
    h, bar, off = initial.double(), initial.double().abs(), torch.zeros_like(initial, dtype=torch.float64)
    rows, offs, befores, before_offs = [], [], [], []
    for t in range(x.shape[0]):
        befores.append(h)
        before_offs.append(off)
        off = rho[t].abs() * off + ddelta[t] * bar + u_off[t]
        h = rho[t] * h + u[t]
        bar = rho[t].abs() * bar + u[t].abs()
        off = off + 8 * E * bar
        rows.append(h)
        offs.append(off)
    return dict(y=torch.stack(rows), off=torch.stack(offs), before=torch.stack(befores), before_off=torch.stack(before_offs),
                final=h, final_off=off, rho=rho, delta=delta, ddelta=ddelta, slope=slope, dslope=dslope)


def backward(x, decay, initial, dy, dfinal, decay_mode, input_mode):
    f = forward(x, decay, None, initial, decay_mode, input_mode)
    x, dy = x.double(), dy.double()
    complement = input_mode == "complement"
    carry, bar, off = dfinal.double(), dfinal.double().abs(), torch.zeros_like(dfinal, dtype=torch.float64)
    out = {k: torch.empty_like(x) for k in ("dx", "dx_off", "ddecay", "ddecay_off")}
    for t in range(x.shape[0] - 1, -1, -1):
        g, g_bar = dy[t] + carry, dy[t].abs() + bar
        g_off = off + 8 * E * g_bar
        delta, source = f["delta"][t], (x[t] if complement else torch.zeros_like(x[t])) - f["before"][t]
        reach = (x[t].abs() if complement else 0) + f["before"][t].abs()
        out["dx"][t] = delta * g if complement else g
        out["dx_off"][t] = (delta.abs() * g_off + f["ddelta"][t] * g_bar if complement else g_off)
        d, d_off = g * source, g_off * reach + g_bar * f["before_off"][t] + 4 * E * g_bar * reach
        out["ddecay"][t] = d * f["slope"][t]
        out["ddecay_off"][t] = d_off * f["slope"][t].abs() + g_bar * reach * f["dslope"][t] + 2 * E * out["ddecay"][t].abs()
        carry, bar = f["rho"][t] * g, f["rho"][t].abs() * g_bar
        off = f["rho"][t].abs() * g_off + f["ddelta"][t] * g_bar + 4 * E * g_bar
    return dict(f, **out, dinitial=carry, dinitial_off=off)
