"""Infinities and NaN at positions that count: they reach what the definitions say they
reach. Outputs of earlier positions stay what they are without them, outputs and gradients
after a row's end stay zero, and a head that forgets at once (A = -inf) is an ordinary head."""
import math

import pytest
import torch

import sequence_oracle as oracle
from sequence_util import BF16, DEV, F32, close, gen, normal, ref_scan, run_scan, scan_inputs, wide

pytestmark = pytest.mark.gpu
TYPES = [F32, BF16]
SHAPES = [(1, 64, 1, 128), (2, 64, 1, 64), (3, 32, 1, 16), (2, 33, 2, 17)]  # heads, dim, groups, state


def same(a, b):
    return torch.equal(a.nan_to_num(nan=12345.0), b.nan_to_num(nan=12345.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_no_output_depends_on_later_positions(shape, dtype):
    from astra_cuda import sequence as seq
    H, P, G, N = shape
    print("causal", shape, dtype, flush=True)
    g = gen(41)
    for T, carried in ((40, False), (150, True)):
        own = {k: None if v is None else v.detach() for k, v in scan_inputs(g, 1, T, H, P, G, N, dtype, carried).items()}
        y = run_scan(seq, own)[0]
        assert bool(torch.isfinite(y).all())
        for at in (0, 1, 17, 31, 38):
            for name in ("x", "dt", "B", "C"):
                for bad in (math.inf, -math.inf, math.nan):
                    if name == "dt" and bad == -math.inf:
                        continue  # a step of zero
                    spoilt = own[name].clone()
                    spoilt[0, at].view(-1)[0] = bad
                    got = run_scan(seq, {**own, name: spoilt})[0]
                    assert torch.equal(got[:, :at], y[:, :at]), (name, bad, at, T)
                    if name == "x":  # only the first feature of the first head took it in
                        assert not bool(torch.isfinite(got[:, at:, 0, 0]).any()), (bad, at, T)
                        rest = torch.ones(H, P, dtype=torch.bool, device=DEV)
                        rest[0, 0] = False
                        assert torch.equal(got[:, :, rest], y[:, :, rest]), (bad, at, T)
                    if name == "C":  # only this position reads with it
                        assert torch.equal(got[:, at + 1:], y[:, at + 1:]), (bad, at, T)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_rows_end_in_zeros_whatever_they_held(shape, dtype):
    """A state, an input or a gradient that is not finite while a row lasts: outputs and
    gradients of the positions after it are zero, and other rows do not notice."""
    from astra_cuda import sequence as seq
    H, P, G, N = shape
    print("zeros", shape, dtype, flush=True)
    g = gen(42)
    T = 140
    lengths = torch.tensor([10, 70, 0, 140], device=DEV, dtype=torch.int32)
    live = torch.arange(T, device=DEV)[None] < lengths[:, None]
    own = scan_inputs(g, 4, T, H, P, G, N, dtype, True)
    dy, dh = normal(g, 4, T, H, P, dtype=dtype), normal(g, 4, H, P, N)

    def both(p, dy, dh):
        out = run_scan(seq, p, lengths)
        return out, torch.autograd.grad(out, [p[k] for k in ("x", "dt", "B", "C", "h")], [dy, dh])

    (y, h), grads = both(own, dy, dh)
    for name in ("x", "dt", "B", "C", "h", "dy", "dh"):
        for bad in (math.inf, math.nan):
            spoilt = {"dy": dy, "dh": dh, **own}[name].detach().clone()
            spoilt[:3].view(3, -1)[:, 0] = bad  # position 0, or the state's first value
            p = dict(own)
            if name in p:
                p[name] = spoilt.requires_grad_()
            (y2, h2), grads2 = both(p, spoilt if name == "dy" else dy, spoilt if name == "dh" else dh)
            assert not bool(y2[~live].any()), (name, bad)
            for n, v in zip(("dx", "ddt", "dB", "dC"), grads2):
                assert not bool(v[~live].any()), (name, bad, n)
            assert torch.equal(y2[3], y[3]) and torch.equal(h2[3], h[3]), (name, bad)
            assert all(torch.equal(a[3], b[3]) for a, b in zip(grads2, grads)), (name, bad)
            if name not in ("h", "dh"):  # a row without positions keeps its state
                assert torch.equal(h2[2], own["h"][2]) and torch.equal(grads2[4][2], dh[2]), (name, bad)
            elif name == "h":
                assert same(h2[2], p["h"][2])


@pytest.mark.parametrize("dtype", TYPES)
def test_a_head_without_memory(dtype):
    """A = -inf: every position forgets what was before it. The same as a decay that
    underflows, and as the definition."""
    from astra_cuda import sequence as seq
    g = gen(43)
    for T in (1, 40, 200):
        own = {k: v.detach() for k, v in scan_inputs(g, 2, T, 2, 32, 1, 16, dtype, True).items()}
        own["A"] = torch.tensor([-math.inf, -1.0], device=DEV)
        got = run_scan(seq, own)
        want = ref_scan({k: wide(v) for k, v in own.items()})
        for i, what in enumerate(("y", "state")):
            close(got[i], want[i], (what, T), 2.0 ** -8 if got[i].dtype == BF16 else 1e-5)
        own["A"] = torch.tensor([-1e30, -1.0], device=DEV)
        again = run_scan(seq, own)
        assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


def test_conv_rows_end_in_zeros_whatever_they_held():
    from astra_cuda import sequence as seq
    g = gen(44)
    B, T, D, K = 3, 70, 16, 4
    lengths = torch.tensor([5, 66, 0], device=DEV, dtype=torch.int32)
    live = torch.arange(T, device=DEV)[None] < lengths[:, None]
    for dtype in TYPES:
        x = normal(g, B, T, D, dtype=dtype)
        w, window = normal(g, D, K), normal(g, B, K - 1, D, dtype=dtype)
        x[0, 4, 0] = math.inf
        x[1, 65, 1] = math.nan
        window[2] = math.inf
        x.requires_grad_()
        y, last = seq.short_conv(x, w, initial_state=window, lengths=lengths, return_state=True)
        assert not bool(y[~live].any())
        assert torch.equal(last[2], window[2])
        want = oracle.conv(x.detach().double(), w.double(), None, window.double(), lengths)[0]
        assert torch.equal(torch.isfinite(y), torch.isfinite(want))
        dx, = torch.autograd.grad(y, [x], torch.ones_like(y))
        assert not bool(dx[~live].any())
