"""The float32 gradients of bf16 scans: dA and ddt_bias are sums of what the states and their
gradients give, each of which is float32, and as exact as float32 sums of them.

Each test leaves one of the terms that make d(dt A), with a state (or a state's gradient)
whose values have a mean of 16 times their spread and a factor of zero mean, so that what is
left of the sum is 1/16 of its terms. In float32 the terms' and the sums' roundings are a few
2^-24 of the terms, of random sign: 16 2^-24 = 1e-6 of the result each, 1e-5 with the sums of
the partial sums. Two bf16 parts of a state leave 16 2^-18 / sqrt(6) = 2.5e-5."""
import pytest
import torch

from sequence_util import BF16, close, gen, normal, ref_scan, run_scan, scan_inputs, wide

pytestmark = pytest.mark.gpu
BOUND = 1e-5
SHAPES = [(4, 64, 1, 128), (4, 64, 1, 64), (4, 32, 1, 64), (4, 64, 1, 32), (4, 32, 1, 32), (2, 33, 1, 100)]


def zero_mean(g, *shape):
    v = normal(g, *shape)
    return v - v.mean(-1, keepdim=True)


def gradients(own, dy, dh):
    from astra_cuda import sequence as seq
    ref = {k: wide(v) for k, v in own.items()}
    names = ["A", "dt_bias"]
    got = torch.autograd.grad(run_scan(seq, own), [own[k] for k in names], [dy, dh])
    want = torch.autograd.grad(ref_scan(ref), [ref[k] for k in names], [dy.double(), dh.double()])
    return zip(names, got, want)


def inputs(g, T, H, P, G, N):
    own = scan_inputs(g, 3, T, H, P, G, N, BF16, True)
    with torch.no_grad():
        own["A"].mul_(1e-2)  # states last over the chunk
    return own


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_states_against_their_gradients(shape):
    """<dh, h> alone: no outputs count, and B is zero."""
    g = gen(71)
    H, P, G, N = shape
    print("dot", shape, flush=True)
    for T in (30, 64):
        own = inputs(g, T, *shape)
        with torch.no_grad():
            own["B"].zero_()
            own["h"].add_(16)
        dh = zero_mean(g, 3, H, P * N).view(3, H, P, N)
        for name, a, b in gradients(own, torch.zeros_like(own["x"]), dh):
            close(a, b, f"d{name} of {T}", BOUND)


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_states_against_the_outputs_gradients(shape):
    """C . (h dY) alone: x is zero, and the last state does not count."""
    g = gen(72)
    H, P, G, N = shape
    print("outputs", shape, flush=True)
    for T in (30, 64):
        own = inputs(g, T, *shape)
        with torch.no_grad():
            own["x"].zero_()
            own["h"].add_(16)
            own["C"].copy_(zero_mean(g, 3, T, G, N))
        dy = normal(g, 3, T, H, P, dtype=BF16)
        for name, a, b in gradients(own, dy, torch.zeros_like(own["h"])):
            close(a, b, f"d{name} of {T}", BOUND)


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_inputs_against_the_states_gradients(shape):
    """B . (dh x) alone: the state before is zero, and no outputs count."""
    g = gen(73)
    H, P, G, N = shape
    print("inputs", shape, flush=True)
    for T in (30, 64):
        own = inputs(g, T, *shape)
        with torch.no_grad():
            own["h"].zero_()
            own["B"].copy_(zero_mean(g, 3, T, G, N))
        dh = normal(g, 3, H, P, N) + 16
        for name, a, b in gradients(own, torch.zeros_like(own["x"]), dh):
            close(a, b, f"d{name} of {T}", BOUND)
