"""The sequence operators at sizes at which every loop of their kernels goes round more than
once: workgroups that walk a group's heads, tiles of features and chunks, segments of wide
states, rows of a norm and runs of a convolution beyond the grid's, sums of partial rows in
two passes. Gradients against differences along themselves.

Bounds, on the 2-norm of an output's error over that of the output: a bf16 result's rounding
is at most 2^-9 of each element; what is rounded is a float32 sum of products whose factors
carry errors of at most 2^-18 (two bf16 parts) or a few 2^-24: 1e-5, and 4e-5 for the
gradients of dt, A and dt_bias, whose terms cancel."""
import math

import pytest
import torch

import sequence_oracle as oracle
from sequence_util import BF16, DEV, F32, close, gen, normal, ref_scan, run_scan, scan_inputs, wide

pytestmark = pytest.mark.gpu


def bound(t, of=1e-5):
    return of + (2.0 ** -9 if t.dtype == BF16 else 0.0)


def compare(out, want, own, ref, g, cancelling=()):
    """Outputs, and the gradients of a random combination of them."""
    for i, (a, b) in enumerate(zip(out, want)):
        close(a, b, f"output {i}", bound(a))
    dout = [normal(g, *a.shape, dtype=a.dtype) for a in out]
    names = [k for k, v in own.items() if v is not None]
    grads = torch.autograd.grad(out, [own[k] for k in names], dout)
    exact = torch.autograd.grad(want, [ref[k] for k in names], [d.double() for d in dout])
    for name, a, b in zip(names, grads, exact):
        close(a, b, f"d{name}", bound(a, 4e-5 if name in cancelling else 1e-5))
    return dict(zip(names, grads))


SCAN = [  # batch, length, heads, dim, groups, state, type, carried, ragged
    (1100, 40, 3, 32, 1, 16, BF16, False, False),   # one chunk, no states: a workgroup walks three heads
    (1100, 40, 3, 32, 1, 16, F32, True, True),      # the same with states
    (1030, 66, 2, 33, 1, 17, BF16, True, True),     # heads and chunks, single elements
    (530, 5, 4, 64, 2, 64, BF16, True, False),      # sums of more than 512 partial rows
    (1030, 3, 2, 64, 1, 128, BF16, True, True),
    (1030, 3, 2, 64, 1, 100, F32, False, True),
    (260, 5, 3, 96, 1, 24, F32, True, True),        # heads and tiles of features
    (260, 70, 3, 96, 1, 40, BF16, True, True),
    (100, 5, 4, 16, 1, 8, BF16, True, True),        # three workgroups share four heads
    (1, 600, 2, 64, 1, 128, BF16, True, True),      # segments of 64 x 128 states
    (2, 520, 1, 64, 1, 128, F32, True, True),
    (1, 777, 2, 32, 1, 128, BF16, False, False),
    (3, 1100, 2, 64, 2, 64, BF16, True, True),      # segments whose chunks are not all alike
]


@pytest.mark.parametrize("case", SCAN, ids=lambda c: "x".join(map(str, c[:6])) + ("b" if c[6] == BF16 else "f"))
def test_scan(case):
    from astra_cuda import sequence as seq
    B, T, H, P, G, N, dtype, carried, ragged = case
    print("scan", case, flush=True)
    g = gen(61)
    own = scan_inputs(g, B, T, H, P, G, N, dtype, carried)
    ref = {k: wide(v) for k, v in own.items()}
    lengths = torch.randint(0, T + 1, (B,), generator=g, device=DEV, dtype=torch.int32) if ragged else None
    if ragged:
        lengths[0] = T - 1
    out, want = run_scan(seq, own, lengths), ref_scan(ref, lengths)
    grads = compare(out, want, own, ref, g, ("dt", "A", "dt_bias"))
    if ragged:
        over = ~(torch.arange(T, device=DEV)[None] < lengths[:, None])
        assert not bool(out[0][over].any())
        for name in ("x", "dt", "B", "C"):
            assert not bool(grads[name][over].any()), name


CONV = [  # batch, length, width, taps, type, carried, ragged
    (9000, 9, 64, 4, BF16, True, True),
    (2100, 6, 1024, 4, BF16, False, False),
    (2100, 6, 1024, 3, F32, True, False),
    (9000, 3, 33, 2, F32, False, True),
    (2, 9001, 48, 4, BF16, True, False),
]


@pytest.mark.parametrize("case", CONV, ids=lambda c: "x".join(map(str, c[:4])) + ("b" if c[4] == BF16 else "f"))
def test_conv(case):
    from astra_cuda import sequence as seq
    B, T, D, K, dtype, carried, ragged = case
    print("conv", case, flush=True)
    g = gen(62)
    own = {"x": normal(g, B, T, D, dtype=dtype).requires_grad_(), "weight": normal(g, D, K).requires_grad_(),
           "bias": normal(g, D).requires_grad_(),
           "window": normal(g, B, K - 1, D, dtype=dtype).requires_grad_() if carried else None}
    ref = {k: wide(v) for k, v in own.items()}
    lengths = torch.randint(0, T + 1, (B,), generator=g, device=DEV, dtype=torch.int32) if ragged else None
    out = seq.short_conv(own["x"], own["weight"], own["bias"], initial_state=own["window"], lengths=lengths,
                         return_state=True)
    want = oracle.conv(ref["x"], ref["weight"], ref["bias"], ref["window"], lengths)
    grads = compare(out, want, own, ref, g)
    if ragged:
        over = ~(torch.arange(T, device=DEV)[None] < lengths[:, None])
        assert not bool(out[0][over].any()) and not bool(grads["x"][over].any())


JOIN = [  # rows, width, type, residual type, gate, scale
    (40000, 64, BF16, BF16, "full", "full"),    # 16 threads a row
    (20000, 256, BF16, BF16, "full", "full"),   # 32
    (10000, 512, BF16, F32, "row", "one"),      # 64, one to four vectors each
    (9000, 1000, BF16, BF16, "full", "full"),
    (9000, 1536, BF16, BF16, "full", "full"),
    (9000, 768, F32, F32, "full", "one"),
    (9000, 37, F32, F32, "full", "full"),
    (3000, 4096, BF16, F32, "row", "full"),     # 256, two and four vectors each
    (2500, 6144, BF16, BF16, "full", "full"),
    (2500, 3000, F32, F32, "full", None),
    (2500, 1025, BF16, F32, "full", "full"),
    (700, 12000, BF16, BF16, "full", "full"),   # 1,024
    (1200, 16384, F32, F32, "full", "full"),
    (600, 9001, F32, F32, "row", "one"),
]


@pytest.mark.parametrize("case", JOIN, ids=lambda c: f"{c[0]}x{c[1]}{'b' if c[2] == BF16 else 'f'}{c[4]}")
def test_join(case):
    from astra_cuda import sequence as seq
    R, D, dtype, rtype, gate, scale = case
    print("join", case, flush=True)
    g = gen(63)
    own = {"residual": normal(g, R, D, dtype=rtype), "block": normal(g, R, D, dtype=dtype), "post": normal(g, D),
           "next": normal(g, D), "gate": normal(g, R, D if gate == "full" else 1, dtype=dtype),
           "scale": None if scale is None else normal(g, D if scale == "full" else 1)}
    own = {k: None if v is None else v.requires_grad_() for k, v in own.items()}
    ref = {k: wide(v) for k, v in own.items()}
    out = seq.join_norm(own["residual"], own["block"], own["post"], own["next"], gate=own["gate"], scale=own["scale"])
    want = oracle.join(ref["residual"], ref["block"], ref["post"], ref["next"], ref["gate"], ref["scale"])
    compare(out, want, own, ref, g)


@pytest.mark.parametrize("case", [(20000, 256, BF16), (9000, 1024, F32), (3000, 5000, BF16)], ids=str)
def test_rms_norm(case):
    from astra_cuda import sequence as seq
    R, D, dtype = case
    g = gen(64)
    own = {"x": normal(g, R, D, dtype=dtype).requires_grad_(), "weight": normal(g, D).requires_grad_()}
    ref = {k: wide(v) for k, v in own.items()}
    compare((seq.rms_norm(own["x"], own["weight"]),), (oracle.join(ref["x"], None, None, ref["weight"])[1],), own, ref, g)


# ------------------------------------------------------------------ against differences

def along_the_gradient(value, own):
    """The derivative of `value` along each input's own gradient, by a difference of two
    values. The step moves an input of n elements by 2^-8 sqrt(n) in all, so the difference's
    third-order term is some 2^-16 of the values' curvature, and the float32 outputs (2^-24
    of sums of some thousands over two steps) less than 1e-2."""
    grads = torch.autograd.grad(value(own), list(own.values()))
    for (name, v), grad in zip(own.items(), grads):
        size = float(grad.double().norm())
        d = (grad.double() / size * math.sqrt(v.numel())).to(v.dtype)
        step = 2.0 ** -8
        with torch.no_grad():
            up, down = value({**own, name: v + step * d}), value({**own, name: v - step * d})
        numeric, formula = float((up - down) / (2 * step)), float((grad.double() * d.double()).sum())
        assert abs(numeric - formula) <= 1e-3 * formula + 1e-2, (name, numeric, formula)


def test_gradients_against_differences():
    from astra_cuda import sequence as seq
    g = gen(65)
    own = scan_inputs(g, 2, 90, 2, 16, 1, 8, F32, True)
    wy, wh = normal(g, 2, 90, 2, 16).double(), normal(g, 2, 2, 16, 8).double()

    def scan(p):
        y, h = run_scan(seq, p)
        return (y.double() * wy).sum() + (h.double() * wh).sum()

    along_the_gradient(scan, own)
    own = {"x": normal(g, 2, 50, 24), "weight": normal(g, 24, 4), "bias": normal(g, 24), "window": normal(g, 2, 3, 24)}
    own = {k: v.requires_grad_() for k, v in own.items()}
    wc, wl = normal(g, 2, 50, 24).double(), normal(g, 2, 3, 24).double()

    def conv(p):
        y, last = seq.short_conv(p["x"], p["weight"], p["bias"], initial_state=p["window"], return_state=True)
        return (y.double() * wc).sum() + (last.double() * wl).sum()

    along_the_gradient(conv, own)
    for gate in (40, 1):
        own = {"residual": normal(g, 30, 40), "block": normal(g, 30, 40), "post": normal(g, 40), "next": normal(g, 40),
               "gate": normal(g, 30, gate), "scale": normal(g, 40 if gate == 40 else 1)}
        own = {k: v.requires_grad_() for k, v in own.items()}
        wj, wn = normal(g, 30, 40).double(), normal(g, 30, 40).double()

        def join(p):
            joined, normed = seq.join_norm(p["residual"], p["block"], p["post"], p["next"], gate=p["gate"], scale=p["scale"])
            return (joined.double() * wj).sum() + (normed.double() * wn).sum()

        along_the_gradient(join, own)
