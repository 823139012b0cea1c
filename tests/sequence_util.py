"""Shared by the GPU tests of the sequence operators: inputs, 64-bit copies, and the bounds
that results of each type are held to."""
import math

import torch

import sequence_oracle as oracle

DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def normal(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def wide(t):
    return None if t is None else t.detach().double().requires_grad_(t.requires_grad)


def error(got, want):
    """The 2-norm of the error over that of the wanted values."""
    got, want = got.detach().double(), want.detach().double()
    assert got.shape == want.shape, (got.shape, want.shape)
    return float((got - want).norm()) / max(float(want.norm()), 1e-300)


def close(got, want, what, bound):
    assert bool(torch.isfinite(got).all()), what
    e = error(got, want)
    assert e <= bound, (what, e, bound)


def scan_inputs(g, B, T, H, P, G, N, dtype, carried=False, full=True):
    own = {"x": normal(g, B, T, H, P, dtype=dtype), "dt": normal(g, B, T, H, dtype=dtype),
           "A": -torch.exp(torch.linspace(0.0, math.log(16.0), H, device=DEV)),
           "B": normal(g, B, T, G, N, dtype=dtype), "C": normal(g, B, T, G, N, dtype=dtype),
           "D": normal(g, H) if full else None, "dt_bias": normal(g, H) - 4 if full else None,
           "h": normal(g, B, H, P, N) if carried else None}
    return {k: None if v is None else v.requires_grad_() for k, v in own.items()}


def run_scan(seq, own, lengths=None):
    return seq.state_scan(own["x"], own["dt"], own["A"], own["B"], own["C"], own["D"], dt_bias=own["dt_bias"],
                          initial_state=own["h"], lengths=lengths, return_state=True)


def ref_scan(ref, lengths=None):
    return oracle.scan(ref["x"], ref["dt"], ref["A"], ref["B"], ref["C"], ref["D"], ref["dt_bias"], ref["h"], lengths)


def small_conv(dtype=F32):
    """x, weight, bias, window."""
    g = gen(31)
    return (normal(g, 2, 6, 8, dtype=dtype), normal(g, 8, 4), normal(g, 8), normal(g, 2, 3, 8, dtype=dtype))


def small_scan(dtype=F32):
    """(state_scan's arguments, a state)."""
    g = gen(32)
    return dict(x=normal(g, 2, 6, 2, 8, dtype=dtype), dt=normal(g, 2, 6, 2, dtype=dtype),
                A=-torch.ones(2, device=DEV), B=normal(g, 2, 6, 1, 4, dtype=dtype), C=normal(g, 2, 6, 1, 4, dtype=dtype),
                D=normal(g, 2), dt_bias=normal(g, 2)), normal(g, 2, 2, 8, 4)
