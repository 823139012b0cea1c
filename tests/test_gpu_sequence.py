"""The sequence operators against their definitions in float64 (tests/sequence_oracle.py),
forward, backward and a position at a time, at the sizes where they can go wrong: lengths
of 0 and 1, around a chunk's 64 positions and a segment's end, odd widths and states,
strided and unaligned rows, ragged and empty rows with NaN and infinities after their
ends, shared heads, carried states, other streams, graphs, and refusals.

Tolerances are on the 2-norm of an output's error over that of the output. A float32
result is a sum of products whose factors carry errors of at most 2^-18 (two bf16 parts,
the scan of bf16 inputs) or a few 2^-24 (float32 inputs): 1e-5 covers both with the sums'
own rounding. A bf16 result adds its rounding, at most 2^-9 of each element: 2^-8."""
import ctypes
import math

import pytest
import torch

import sequence_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


def close(got, want, what, scale=1.0):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bound = (2.0 ** -8 if got.dtype == BF16 else 1e-5) * scale
    got, want = got.detach().double(), want.detach().double()
    assert bool(torch.isfinite(got).all()), what
    err, norm = float((got - want).norm()), float(want.norm())
    assert err <= bound * norm + 1e-12, (what, err / max(norm, 1e-300))


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def normal(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def wide(t):
    return None if t is None else t.detach().double().requires_grad_(t.requires_grad)


def compare_grads(own_out, own_in, ref_out, ref_in, g, what, used=None, scale=1.0):
    """Gradients of the same random combination of the outputs, on both sides."""
    names = [n for n, t in own_in.items() if t is not None]
    outs = [i for i in range(len(own_out)) if own_out[i] is not None and (used is None or i in used)]
    seeds = [normal(g, *own_out[i].shape, dtype=own_out[i].dtype) for i in outs]
    got = torch.autograd.grad([own_out[i] for i in outs], [own_in[n] for n in names], seeds, allow_unused=True)
    want = torch.autograd.grad([ref_out[i] for i in outs], [ref_in[n] for n in names], [s.double() for s in seeds],
                               allow_unused=True)
    for n, a, b in zip(names, got, want):
        b = torch.zeros_like(ref_in[n]) if b is None else b
        assert a is not None and a.dtype == own_in[n].dtype, (what, n)
        close(a, b, f"{what} d{n}", scale)


# ------------------------------------------------------------------------- short_conv

CONV = [  # batch, length, width, taps, type, carried, ragged, silu, bias
    (3, 1, 8, 4, F32, False, False, True, True),
    (2, 2, 16, 4, BF16, True, False, True, True),
    (4, 65, 24, 4, BF16, True, True, True, True),
    (5, 40, 640, 4, BF16, False, False, True, True),
    (2, 133, 33, 3, F32, True, True, False, False),
    (7, 9, 7, 2, BF16, False, True, True, False),
    (1, 3001, 20, 4, F32, True, False, True, True),
    (300, 40, 72, 3, F32, False, True, True, True),
]


@pytest.mark.parametrize("case", CONV, ids=lambda c: "x".join(str(v) for v in c[:4]))
def test_conv(case):
    from astra_cuda import sequence as seq
    B, T, D, K, dtype, carried, ragged, silu, with_bias = case
    print("conv", case, flush=True)
    g = gen(1)
    own = {"x": normal(g, B, T, D, dtype=dtype).requires_grad_(), "weight": normal(g, D, K).requires_grad_(),
           "bias": normal(g, D).requires_grad_() if with_bias else None,
           "window": normal(g, B, K - 1, D, dtype=dtype).requires_grad_() if carried else None}
    lengths = torch.randint(0, T + 1, (B,), generator=g, device=DEV, dtype=torch.int32) if ragged else None
    if ragged:
        lengths[0] = 0
        lengths[-1] = T
    ref = {k: wide(v) for k, v in own.items()}
    act = "silu" if silu else None
    y, last = seq.short_conv(own["x"], own["weight"], own["bias"], activation=act, initial_state=own["window"],
                             lengths=lengths, return_state=True)
    ry, rlast = oracle.conv(ref["x"], ref["weight"], ref["bias"], ref["window"], lengths, silu)
    close(y, ry, "y")
    assert torch.equal(last.double(), rlast)
    compare_grads((y, last), own, (ry, rlast), ref, g, "both")
    y = seq.short_conv(own["x"], own["weight"], own["bias"], activation=act, initial_state=own["window"],
                       lengths=lengths)
    ry, _ = oracle.conv(ref["x"], ref["weight"], ref["bias"], ref["window"], lengths, silu)
    compare_grads((y,), own, (ry,), ref, g, "y alone")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [1, 24, 33])
def test_conv_steps_are_the_sequence(dtype, D):
    """T steps, the window moved on in place, give the whole call's outputs and window."""
    from astra_cuda import sequence as seq
    g = gen(2)
    B, T, K = 5, 9, 4
    x, w, b = normal(g, B, T, D, dtype=dtype), normal(g, D, K), normal(g, D)
    window = normal(g, B, K - 1, D, dtype=dtype)
    y, last = seq.short_conv(x, w, b, initial_state=window, return_state=True)
    state = window.clone()
    for t in range(T):
        assert torch.equal(seq.short_conv_step(x[:, t], state, w, b), y[:, t]), t
    assert torch.equal(state, last)


def test_conv_strided_rows_and_garbage_after_the_end():
    """x as a part of a wider tensor at an odd offset; NaN and infinities after the rows'
    ends and in their output gradients reach nothing."""
    from astra_cuda import sequence as seq
    g = gen(3)
    B, T, D, K = 4, 70, 32, 4
    lengths = torch.tensor([0, 1, 64, 70], device=DEV, dtype=torch.int64)
    for dtype in (F32, BF16):
        for offset in (0, 3):
            whole = normal(g, B, T, 2 * D + 8, dtype=dtype)
            x = whole[..., offset:offset + D]
            for b in range(B):
                x[b, int(lengths[b]):] = float("nan") if b % 2 else float("inf")
            w, bias = normal(g, D, K).requires_grad_(), normal(g, D).requires_grad_()
            x = x.requires_grad_()
            y, last = seq.short_conv(x, w, bias, lengths=lengths, return_state=True)
            clean = torch.nan_to_num(x.detach().double(), 0, 0, 0).requires_grad_()
            rw, rb = wide(w), wide(bias)
            ry, rlast = oracle.conv(clean, rw, rb, None, lengths)
            close(y, ry, "y")
            close(last, rlast, "last")
            dy = normal(g, B, T, D, dtype=dtype)
            rgrads = torch.autograd.grad(ry, [clean, rw, rb], dy.double())
            for b in range(B):
                dy[b, int(lengths[b]):] = float("nan")
            for n, a, b in zip("xwb", torch.autograd.grad(y, [x, w, bias], dy), rgrads):
                close(a, b, n)


def test_conv_without_positions():
    from astra_cuda import sequence as seq
    window = normal(gen(4), 3, 3, 8).requires_grad_()
    x, w = torch.zeros(3, 0, 8, device=DEV, requires_grad=True), torch.ones(8, 4, device=DEV, requires_grad=True)
    y, last = seq.short_conv(x, w, initial_state=window, return_state=True)
    assert y.shape == (3, 0, 8) and torch.equal(last, window)
    dw, dwin = torch.autograd.grad(last.sum(), [w, window])
    assert not dw.any() and torch.equal(dwin, torch.ones_like(dwin))
    none = torch.zeros(0, 5, 8, device=DEV, requires_grad=True)
    y, last = seq.short_conv(none, w, return_state=True)
    assert y.shape == (0, 5, 8) and last.shape == (0, 3, 8)
    assert not torch.autograd.grad(y.sum(), [w])[0].any()


# ------------------------------------------------------------------------- state_scan

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


SCAN = [  # batch, length, heads, dim, groups, state, type, carried, ragged, D and dt_bias
    (2, 1, 1, 64, 1, 64, F32, False, False, True),
    (2, 1, 2, 16, 1, 16, BF16, True, False, True),
    (3, 40, 8, 64, 1, 64, BF16, False, False, True),
    (3, 63, 4, 32, 2, 16, F32, True, True, True),
    (2, 64, 2, 48, 1, 24, BF16, True, False, False),
    (2, 65, 2, 33, 2, 17, F32, True, True, True),
    (2, 65, 3, 33, 1, 17, BF16, False, True, True),
    (2, 100, 4, 64, 1, 128, BF16, True, True, True),
    (1, 130, 2, 40, 1, 100, F32, False, False, False),
    (2, 200, 4, 128, 2, 32, F32, True, False, True),
    (2, 200, 2, 128, 2, 64, BF16, True, True, True),
    (1, 700, 2, 32, 1, 32, BF16, True, True, True),
    (1, 1, 1, 1, 1, 1, F32, True, False, True),
    (300, 5, 2, 16, 2, 8, BF16, True, True, True),
    (2, 300, 6, 96, 3, 64, F32, False, True, True),
]


@pytest.mark.parametrize("case", SCAN, ids=lambda c: "x".join(str(v) for v in c[:6]) + ("b" if c[6] == BF16 else "f"))
def test_scan(case):
    from astra_cuda import sequence as seq
    B, T, H, P, G, N, dtype, carried, ragged, full = case
    print("scan", case, flush=True)
    g = gen(5)
    own = scan_inputs(g, B, T, H, P, G, N, dtype, carried, full)
    ref = {k: wide(v) for k, v in own.items()}
    lengths = None
    if ragged:
        lengths = torch.randint(0, T + 1, (B,), generator=g, device=DEV, dtype=torch.int32)
        lengths[0] = T - 1 if B == 1 else 0
    out, want = run_scan(seq, own, lengths), ref_scan(ref, lengths)
    close(out[0], want[0], "y")
    close(out[1], want[1], "state")
    # the gradients of A, dt_bias and dt are sums with cancellation: a few times the bound
    compare_grads(out, own, want, ref, g, "both", scale=4.0)
    compare_grads(run_scan(seq, own, lengths), own, ref_scan(ref, lengths), ref, g, "y alone", used=(0,), scale=4.0)
    with torch.no_grad():
        again = run_scan(seq, own, lengths)
    assert torch.equal(again[0], out[0]) and torch.equal(again[1], out[1])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(3, 8, 64, 2, 64), (2, 2, 33, 1, 17), (2, 1, 32, 1, 128), (5, 4, 16, 4, 24),
                                   (2, 2, 8, 1, 100), (2, 1, 3, 1, 65)])
def test_scan_steps_are_the_sequence(dtype, shape):
    from astra_cuda import sequence as seq
    B, H, P, G, N = shape
    T = 6
    g = gen(6)
    own = scan_inputs(g, B, T, H, P, G, N, dtype, True)
    with torch.no_grad():
        want = ref_scan({k: wide(v) for k, v in own.items()})
        h = own["h"].clone()
        ys = [seq.state_scan_step(own["x"][:, t], own["dt"][:, t], own["A"], own["B"][:, t], own["C"][:, t], h,
                                  D=own["D"], dt_bias=own["dt_bias"]) for t in range(T)]
    close(torch.stack(ys, 1), want[0], "y")
    close(h, want[1], "state")


def test_scan_of_a_long_row_in_segments_and_pieces():
    """A row of many chunks is split into segments; played in pieces with the state carried
    between them it gives the same, and gradients flow through the pieces."""
    from astra_cuda import sequence as seq
    g = gen(7)
    for dtype in (F32, BF16):
        own = scan_inputs(g, 1, 2500, 2, 32, 1, 16, dtype, True)
        ref = {k: wide(v) for k, v in own.items()}
        out, want = run_scan(seq, own), ref_scan(ref)
        close(out[0], want[0], "y")
        close(out[1], want[1], "state")
        compare_grads(out, own, want, ref, g, "whole", scale=4.0)
        h, ys = own["h"], []
        for t0, t1 in ((0, 1), (1, 1300), (1300, 1300), (1300, 2500)):
            part = {k: v[:, t0:t1] if k in ("x", "dt", "B", "C") else v for k, v in own.items()}
            y, h = run_scan(seq, {**part, "h": h})
            ys.append(y)
        pieces = (torch.cat(ys, 1), h)
        close(pieces[0], want[0], "y of pieces")
        close(pieces[1], want[1], "state of pieces")
        compare_grads(pieces, own, ref_scan(ref), ref, g, "pieces", scale=4.0)


def test_scan_gradient_against_differences():
    """The directional derivative of a fixed function of the outputs, in float32."""
    from astra_cuda import sequence as seq
    g = gen(8)
    own = scan_inputs(g, 2, 90, 2, 16, 1, 8, F32, True)
    wy, wh = normal(g, 2, 90, 2, 16).double(), normal(g, 2, 2, 16, 8).double()

    def value(p):
        y, h = run_scan(seq, p)
        return (y.double() * wy).sum() + (h.double() * wh).sum()

    grads = torch.autograd.grad(value(own), list(own.values()))
    for name, grad in zip(own, grads):
        d = normal(g, *own[name].shape)
        step = 2.0 ** -8
        with torch.no_grad():
            up = value({**own, name: own[name] + step * d})
            down = value({**own, name: own[name] - step * d})
        numeric, formula = float((up - down) / (2 * step)), float((grad.double() * d.double()).sum())
        size = float(grad.double().norm() * d.double().norm())
        # the difference's third-order term and float32 outputs (2^-24 of their sum over 2 steps)
        assert abs(numeric - formula) <= 1e-3 * size + 1e-2, (name, numeric, formula)


def test_scan_strided_rows_and_garbage_after_the_end():
    """x, B and C as parts of one tensor at offsets that allow wide accesses or not, dt
    transposed; NaN and infinities after the rows' ends reach nothing."""
    from astra_cuda import sequence as seq
    g = gen(9)
    B, T, H, P, G, N = 4, 130, 2, 32, 1, 16
    lengths = torch.tensor([0, 1, 64, 129], device=DEV, dtype=torch.int32)
    live = torch.arange(T, device=DEV)[None] < lengths[:, None]
    for dtype in (F32, BF16):
        for offset in (0, 1):
            own = scan_inputs(g, B, T, H, P, G, N, dtype, True)
            whole = normal(g, B, T, H * P + 2 * G * N + 4, dtype=dtype)
            x, b, c = whole[..., offset:offset + H * P + 2 * G * N].split([H * P, G * N, G * N], -1)
            dt = normal(g, B, H, T, dtype=dtype).transpose(1, 2)
            parts = {"x": x.unflatten(-1, (H, P)), "B": b.unflatten(-1, (G, N)), "C": c.unflatten(-1, (G, N)), "dt": dt}
            ref = {k: wide(v) for k, v in {**own, **parts}.items()}
            for k in parts:
                ref[k] = ref[k].detach().requires_grad_()
            whole[~live] = float("nan")
            dt[1, 1:] = float("inf")
            dt[2, 64:] = float("nan")
            own.update({k: v.requires_grad_() for k, v in parts.items()})
            out, want = run_scan(seq, own, lengths), ref_scan(ref, lengths)
            close(out[0], want[0], "y")
            close(out[1], want[1], "state")
            dy, dh = normal(g, B, T, H, P, dtype=dtype), normal(g, B, H, P, N)
            rgrads = torch.autograd.grad(want, list(ref.values()), [dy.double(), dh.double()])
            dy[~live] = float("nan")
            for n, a, r in zip(own, torch.autograd.grad(out, list(own.values()), [dy, dh]), rgrads):
                close(a, r, f"d{n}", 4.0)
            # a row of length 0 keeps its state
            assert torch.equal(out[1][0], own["h"][0])


def test_scan_extreme_steps():
    """Steps that underflow to zero, and decays that underflow to zero within a chunk."""
    from astra_cuda import sequence as seq
    g = gen(10)
    for dtype in (F32, BF16):
        own = scan_inputs(g, 2, 150, 2, 32, 1, 16, dtype, True)
        with torch.no_grad():
            own["dt"][0, 10:20] = -200.0
            own["dt"][1, 30] = 60.0
            own["dt"][1, 100:140] = 20.0
        ref = {k: wide(v) for k, v in own.items()}
        out, want = run_scan(seq, own), ref_scan(ref)
        close(out[0], want[0], "y")
        close(out[1], want[1], "state")
        compare_grads(out, own, want, ref, g, "extreme", scale=4.0)


def test_scan_without_positions():
    from astra_cuda import sequence as seq
    own = scan_inputs(gen(11), 2, 0, 2, 8, 1, 4, F32, True)
    y, h = run_scan(seq, own)
    assert y.shape == (2, 0, 2, 8) and torch.equal(h, own["h"])
    dA, dh = torch.autograd.grad(h.sum(), [own["A"], own["h"]])
    assert not dA.any() and torch.equal(dh, torch.ones_like(dh))
    own["h"] = None
    assert not run_scan(seq, own)[1].any()
    own = scan_inputs(gen(11), 0, 5, 2, 8, 1, 4, F32)
    y, h = run_scan(seq, own)
    assert y.shape == (0, 5, 2, 8) and h.shape == (0, 2, 8, 4)
    assert not torch.autograd.grad(y.sum(), [own["A"]])[0].any()


def test_scan_states_past_32_bits():
    """States whose offsets pass 2^31 elements: the last env's step is the oracle's."""
    from astra_cuda import sequence as seq
    B, H, P, N = 33_000, 8, 64, 128
    g = gen(12)
    own = scan_inputs(g, 1, 1, H, P, 1, N, BF16, True)
    x, dt, Bm, Cm = (own[k].detach()[:, 0].expand(B, *own[k].shape[2:]) for k in ("x", "dt", "B", "C"))
    h = torch.zeros(B, H, P, N, device=DEV)
    h[-1] = own["h"].detach()[0]
    with torch.no_grad():
        y = seq.state_scan_step(x, dt, own["A"], Bm, Cm, h, D=own["D"], dt_bias=own["dt_bias"])
        want = ref_scan({k: wide(v) for k, v in own.items()})
    close(y[-1:], want[0][:, 0], "y")
    close(h[-1:], want[1], "state")


# -------------------------------------------------------------------------- join_norm

JOIN = [  # rows, width, type, residual type, gate, scale, next
    (1, 1, F32, F32, "full", "full", True),
    (3, 7, BF16, F32, "row", "one", True),
    (5, 64, BF16, BF16, "full", "full", True),
    (130, 256, BF16, BF16, "full", "full", True),
    (9, 500, F32, F32, "row", None, True),
    (6, 1000, BF16, BF16, "none", "full", True),
    (4, 1537, BF16, F32, "full", "one", True),
    (5, 2048, F32, F32, "full", "full", True),
    (3, 4096, BF16, F32, "row", "full", True),
    (3, 5001, F32, F32, "full", "full", True),
    (2, 8192, F32, F32, "none", None, True),
    (2, 16384, BF16, BF16, "full", "full", True),
    (2, 16383, BF16, F32, "row", "full", True),
    (6000, 48, F32, F32, "full", "one", True),
    (17, 384, BF16, F32, "full", "full", False),
]


@pytest.mark.parametrize("case", JOIN, ids=lambda c: f"{c[0]}x{c[1]}{'b' if c[2] == BF16 else 'f'}{c[4]}")
def test_join(case):
    from astra_cuda import sequence as seq
    R, D, dtype, rtype, gate, scale, nxt = case
    print("join", case, flush=True)
    g = gen(13)
    own = {"residual": normal(g, R, D, dtype=rtype), "block": normal(g, R, D, dtype=dtype),
           "post": normal(g, D), "next": normal(g, D) if nxt else None,
           "gate": None if gate == "none" else normal(g, R, D if gate == "full" else 1, dtype=dtype),
           "scale": None if scale is None else normal(g, D if scale == "full" else 1)}
    own = {k: None if v is None else v.requires_grad_() for k, v in own.items()}
    ref = {k: wide(v) for k, v in own.items()}
    out = seq.join_norm(own["residual"], own["block"], own["post"], own["next"], gate=own["gate"], scale=own["scale"])
    want = oracle.join(**{"residual": ref["residual"], "block": ref["block"], "post": ref["post"], "nxt": ref["next"],
                          "gate": ref["gate"], "scale": ref["scale"]})
    close(out[0], want[0], "joined")
    if nxt:
        close(out[1], want[1], "normed")
    else:
        assert out[1] is None
    compare_grads(out, own, want, ref, g, "both", scale=2.0)
    if nxt:
        for used in ((0,), (1,)):
            again = seq.join_norm(own["residual"], own["block"], own["post"], own["next"], gate=own["gate"],
                                  scale=own["scale"])
            rgain = oracle.join(ref["residual"], ref["block"], ref["post"], ref["next"], ref["gate"], ref["scale"])
            compare_grads(again, own, rgain, ref, g, f"output {used}", used=used, scale=2.0)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [5, 256, 3000])
def test_rms_norm(dtype, D):
    from astra_cuda import sequence as seq
    g = gen(14)
    own = {"x": normal(g, 3, 4, D, dtype=dtype).requires_grad_(), "weight": normal(g, D).requires_grad_()}
    ref = {k: wide(v) for k, v in own.items()}
    out, want = seq.rms_norm(own["x"], own["weight"]), oracle.join(ref["x"], None, None, ref["weight"])[1]
    close(out, want, "normed")
    compare_grads((out,), own, (want,), ref, g, "rms", scale=2.0)


def test_join_strided_zero_rows_and_shapes():
    """Rows of a wider tensor at offsets that allow wide accesses or not, rows of zeros,
    leading dimensions, no rows at all."""
    from astra_cuda import sequence as seq
    g = gen(15)
    for offset in (0, 3):
        whole = normal(g, 4, 6, 3 * 64 + 8, dtype=BF16)
        r, u, gate = (whole[..., offset + 64 * i:offset + 64 * (i + 1)] for i in range(3))
        u[0] = 0
        r[0, 1] = 0
        own = {"residual": r.requires_grad_(), "block": u.requires_grad_(), "gate": gate.requires_grad_(),
               "post": normal(g, 64).requires_grad_(), "next": normal(g, 64).requires_grad_()}
        ref = {k: wide(v) for k, v in own.items()}
        out = seq.join_norm(own["residual"], own["block"], own["post"], own["next"], gate=own["gate"])
        want = oracle.join(ref["residual"], ref["block"], ref["post"], ref["next"], ref["gate"])
        assert out[0].shape == (4, 6, 64)
        close(out[0], want[0], "joined")
        close(out[1], want[1], "normed")
        compare_grads(out, own, want, ref, g, "strided", scale=2.0)
    w = torch.ones(8, device=DEV, requires_grad=True)
    none = torch.zeros(0, 8, device=DEV)
    joined, normed = seq.join_norm(none, none, w, w)
    assert joined.shape == normed.shape == (0, 8)
    assert not torch.autograd.grad(normed.sum() + joined.sum(), [w])[0].any()


# ------------------------------------------------------------------- how they are called

def test_other_stream_and_graph_replays():
    """The calls run on the current stream, and a captured step replays with new inputs."""
    from astra_cuda import sequence as seq
    g = gen(16)
    B, H, P, N, K = 64, 4, 32, 32, 4
    D = H * P + 2 * N
    w, bias = normal(g, D, K), normal(g, D)
    A, skip, dtb = -torch.ones(H, device=DEV), normal(g, H), normal(g, H) - 4
    xs, dts = normal(g, 6, B, D, dtype=BF16), normal(g, 6, B, H, dtype=BF16)

    def move(x, dt, window, h):
        mixed = seq.short_conv_step(x, window, w, bias)
        xp, b, c = mixed.split([H * P, N, N], -1)
        return seq.state_scan_step(xp.unflatten(-1, (H, P)), dt, A, b[:, None], c[:, None], h, D=skip, dt_bias=dtb)

    def fresh():
        return torch.zeros(B, K - 1, D, device=DEV, dtype=BF16), torch.zeros(B, H, P, N, device=DEV)

    window, h = fresh()
    want = [move(xs[t], dts[t], window, h).clone() for t in range(6)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    window2, h2 = fresh()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = [move(xs[t], dts[t], window2, h2) for t in range(6)]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(h, h2)
    window3, h3 = fresh()
    x, dt = xs[0].clone(), dts[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = move(x, dt, window3, h3)
    window3.zero_()
    h3.zero_()
    for t in range(6):
        x.copy_(xs[t])
        dt.copy_(dts[t])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[t]), t
    assert torch.equal(h3, h) and torch.equal(window3, window)


def test_results_do_not_change_from_call_to_call():
    """No sum depends on the order in which workgroups finish."""
    from astra_cuda import sequence as seq
    g = gen(17)
    own = scan_inputs(g, 40, 100, 4, 64, 2, 64, BF16, True)

    def once():
        y, h = run_scan(seq, own)
        return torch.autograd.grad([y, h], list(own.values()), [torch.ones_like(y), torch.ones_like(h)])

    first = once()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, once()))


def test_refusals():
    from astra_cuda import sequence as seq
    x = torch.zeros(2, 5, 4, 8, device=DEV)
    dt, A = torch.zeros(2, 5, 4, device=DEV), -torch.ones(4, device=DEV)
    B = torch.zeros(2, 5, 2, 16, device=DEV)
    bad = [
        lambda: seq.state_scan(x.cpu(), dt, A, B, B),
        lambda: seq.state_scan(x.half(), dt.half(), A, B.half(), B.half()),
        lambda: seq.state_scan(x, dt.bfloat16(), A, B, B),
        lambda: seq.state_scan(x, dt[:, :4], A, B, B),
        lambda: seq.state_scan(x, dt, A[:3], B, B),
        lambda: seq.state_scan(x, dt, A, torch.zeros(2, 5, 3, 16, device=DEV), torch.zeros(2, 5, 3, 16, device=DEV)),
        lambda: seq.state_scan(x, dt, A, B, B[..., :8]),
        lambda: seq.state_scan(x, dt, A, torch.zeros(2, 5, 2, 129, device=DEV), torch.zeros(2, 5, 2, 129, device=DEV)),
        lambda: seq.state_scan(x, dt, A, B, B, initial_state=torch.zeros(2, 4, 8, 15, device=DEV)),
        lambda: seq.state_scan(x, dt, A, B, B, lengths=torch.zeros(3, device=DEV, dtype=torch.int32)),
        lambda: seq.state_scan(x, dt, A, B, B, lengths=torch.zeros(2, device=DEV)),
        lambda: seq.state_scan(x[0], dt, A, B, B),
        lambda: seq.state_scan_step(x[:, 0], dt[:, 0], A, B[:, 0], B[:, 0], torch.zeros(2, 4, 8, 16)),
        lambda: seq.state_scan_step(x[:, 0], dt[:, 0], A, B[:, 0], B[:, 0],
                                    torch.zeros(2, 4, 16, 8, device=DEV).transpose(2, 3)),
        lambda: seq.state_scan_step(x[:, 0].requires_grad_(), dt[:, 0], A, B[:, 0], B[:, 0],
                                    torch.zeros(2, 4, 8, 16, device=DEV)),
        lambda: seq.short_conv(x[..., 0], torch.zeros(4, 5, device=DEV)),
        lambda: seq.short_conv(x[..., 0], torch.zeros(4, 1, device=DEV)),
        lambda: seq.short_conv(x[..., 0], torch.zeros(3, 4, device=DEV)),
        lambda: seq.short_conv(x[..., 0], torch.zeros(4, 4, device=DEV), activation="relu"),
        lambda: seq.short_conv(x[..., 0], torch.zeros(4, 4, device=DEV), initial_state=torch.zeros(2, 4, 4, device=DEV)),
        lambda: seq.short_conv_step(x[:, 0, :, 0], torch.zeros(2, 3, 4, device=DEV, dtype=BF16),
                                    torch.zeros(4, 4, device=DEV)),
        lambda: seq.join_norm(x, x[:1], torch.ones(8, device=DEV), None),
        lambda: seq.join_norm(x.bfloat16(), x, torch.ones(8, device=DEV), None),
        lambda: seq.join_norm(x, x, torch.ones(7, device=DEV), None),
        lambda: seq.join_norm(x, x, torch.ones(8, device=DEV), None, gate=x[..., :2]),
        lambda: seq.join_norm(x, x, torch.ones(8, device=DEV), None, scale=torch.ones(2, device=DEV)),
        lambda: seq.rms_norm(torch.zeros(1, 16385, device=DEV), torch.zeros(16385, device=DEV)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError, match="Astra Fatal Error"):
            call()
            pytest.fail(f"call {i} was not refused")


def test_refusals_of_the_c_entry_points():
    from astra_cuda import _native
    lib = _native.lib()
    n = ctypes.c_size_t(0)
    f = _native.StateScan(batch=1, length=5, heads=3, dim=8, groups=2, state=16, type=0)
    assert lib.astra_state_scan_forward(ctypes.addressof(f), None) == 1 and "heads" in _native.last_error()
    f.groups, f.state = 1, 200
    assert lib.astra_state_scan_workspace_size(ctypes.addressof(f), ctypes.byref(n)) == 1
    f.state = 16
    assert lib.astra_state_scan_forward(ctypes.addressof(f), None) == 1 and "NULL" in _native.last_error()
    f.type = 7
    assert lib.astra_state_scan_forward(ctypes.addressof(f), None) == 1
    assert lib.astra_state_scan_forward(None, None) == 1
    c = _native.ShortConv(batch=1, length=5, width=8, taps=5)
    assert lib.astra_short_conv_forward(ctypes.addressof(c), None) == 1 and "taps" in _native.last_error()
    j = _native.JoinNorm(rows=2, width=20000)
    assert lib.astra_join_norm_forward(ctypes.addressof(j), None) == 1 and "width" in _native.last_error()
    j.width = 8
    assert lib.astra_join_norm_forward(ctypes.addressof(j), None) == 1
    # a workspace that is too small is refused before anything is launched
    w = torch.zeros(8, 4, device=DEV)
    x = torch.zeros(1, 5, 8, device=DEV)
    c = _native.ShortConv(x=x.data_ptr(), weight=w.data_ptr(), batch=1, length=5, x_stride_b=40, x_stride_t=8, width=8,
                          taps=4)
    g = _native.ShortConvGrad(c, dy=x.data_ptr(), dweight=w.data_ptr(), workspace=x.data_ptr(), workspace_bytes=16)
    assert lib.astra_short_conv_backward(ctypes.addressof(g), None) == 1 and "workspace_bytes" in _native.last_error()
