"""Shared by the tests of gated_linear: inputs, the definition in 64 bits, and bounds on how far off a
result may be, element by element.

u is half a step of the result's type (2^-8 bf16, 2^-24 float32), e = 2^-24 one float32 rounding. A sum
of n products is off by at most (n + 2) e times the sum of their magnitudes, whatever its order. The
activations' slopes are at most 1.13 and change by at most 0.8 a unit; the activations and their slopes
are evaluated to 16 e of the larger of 1 and |a|.
"""
import math

import torch

DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16
E = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def inputs(seed, M, D, F, dtype):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    def normal(*s):
        return torch.randn(*s, generator=g, device=DEV)
    x, wg, wu = normal(M, D).to(dtype), (normal(F, D) / math.sqrt(D)).to(dtype), (normal(F, D) / math.sqrt(D)).to(dtype)
    return x, wg, wu, normal(M, F).to(dtype)


def activation(a, kind):
    """act(a), act'(a) in 64 bits."""
    if kind == "silu":
        s = torch.sigmoid(a)
        return a * s, s * (1 + a * (1 - s))
    phi = torch.special.erfc(-a / math.sqrt(2)) / 2
    return a * phi, phi + a * torch.exp(-a * a / 2) / math.sqrt(2 * math.pi)


def results(x, wg, wu, dh, kind):
    """{name: (value, bound)} of h, dx, dgate and dup, in 64 bits."""
    u = half_step(x.dtype)
    x, wg, wu, dh = (v.detach().double() for v in (x, wg, wu, dh))
    M, D = x.shape
    F = wg.shape[0]
    a, b = x @ wg.t(), x @ wu.t()
    ea, eb = ((D + 2) * E * (x.abs() @ w.abs().t()) for w in (wg, wu))
    act, slope = activation(a, kind)
    near = 16 * E * a.abs().clamp(min=1)
    e_act, e_slope = 1.13 * ea + near, 0.8 * ea + near
    h = act * b
    out = {"h": (h, (e_act * (b.abs() + eb) + act.abs() * eb + 2 * E * h.abs()) * (1 + u) + u * h.abs())}
    da, db = dh * b * slope, dh * act
    e_da = dh.abs() * (e_slope * (b.abs() + eb) + slope.abs() * eb) + (3 * E + u) * da.abs()
    e_db = dh.abs() * e_act + (3 * E + u) * db.abs()
    dx = da @ wg + db @ wu
    size = (2 * F + 2) * E
    out["dx"] = (dx, (e_da * (1 + size)) @ wg.abs() + (e_db * (1 + size)) @ wu.abs()
                 + size * (da.abs() @ wg.abs() + db.abs() @ wu.abs()) + u * dx.abs())
    size = (M + 2) * E
    for name, d, e in (("dgate", da, e_da), ("dup", db, e_db)):
        w = d.t() @ x
        out[name] = (w, (e.t() * (1 + size)) @ x.abs() + size * (d.abs().t() @ x.abs()) + u * w.abs())
    return out


def within(got, want, what):
    value, bound = want
    assert got.shape == value.shape, (what, got.shape, value.shape)
    off = (got.detach().double() - value).abs() - 1.001 * bound - 1e-37
    assert bool(torch.isfinite(got).all()), what
    assert not bool((off > 0).any()), (what, float(off.max()), float(value.abs().max()))


def call(seq, x, wg, wu, dh, kind):
    x, wg, wu = (v.detach().requires_grad_() for v in (x, wg, wu))
    h = seq.gated_linear(x, wg, wu, activation=kind)
    return dict(zip(("h", "dx", "dgate", "dup"), (h.detach(), *torch.autograd.grad(h, (x, wg, wu), dh))))


def check(got, x, wg, wu, dh, kind):
    want = results(x, wg, wu, dh, kind)
    for name in want:
        within(got[name], want[name], name)
