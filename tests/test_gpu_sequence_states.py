"""States of bf16 scans enter the products as float32 values do: where the terms of h C
(or dh B) cancel, what is left is still right to bf16's own rounding.

Bounds, on the 2-norm of an output's error over that of the output. A state enters a product
as the sum of two bf16 values, 2^-18 of each of its values at most. With a state of mean m
and a C of zero mean over the N values, y's terms are m times as large as what is left of
them after the sum, so a state's part of the error is at most m 2^-18 sqrt(N) of y's norm
even if every rounding had the same sign: for m = 16, N = 128 that is 7e-4, and a bf16
result's rounding is at most 2^-9 = 1.95e-3: 2.65e-3 together. One bf16 value for a state
leaves 2.9e-2 there."""
import pytest
import torch

from sequence_util import BF16, DEV, F32, close, error, gen, normal, ref_scan, run_scan, scan_inputs, wide

pytestmark = pytest.mark.gpu
BOUND = 2.65e-3

SHAPES = [  # heads, dim, groups, state: every tile of the kernels, and parts of tiles
    (4, 64, 1, 128), (2, 32, 1, 128), (2, 64, 2, 64), (2, 32, 1, 64), (2, 64, 1, 32), (4, 32, 2, 32),
    (2, 33, 1, 100), (2, 128, 1, 48),
]


def cancelling(g, *shape):
    """bf16 rows whose values sum to almost nothing."""
    v = normal(g, *shape)
    return (v - v.mean(-1, keepdim=True)).to(BF16)


def inputs(g, B, T, H, P, G, N, mean):
    own = scan_inputs(g, B, T, H, P, G, N, BF16, True, False)
    with torch.no_grad():
        own["A"].mul_(1e-3)  # states last
        own["dt"].sub_(4)
        own["C"].copy_(cancelling(g, B, T, G, N))
        own["B"].copy_(cancelling(g, B, T, G, N))
        own["h"].add_(mean)
    return own


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_read_out_of_a_state_with_a_mean(shape):
    from astra_cuda import sequence as seq
    H, P, G, N = shape
    print("states", shape, flush=True)
    g = gen(21)
    for T in (40, 200):
        own = inputs(g, 2, T, H, P, G, N, 16.0)
        with torch.no_grad():
            got, want = run_scan(seq, own), ref_scan({k: wide(v) for k, v in own.items()})
        close(got[0], want[0], f"y of {T}", BOUND)
        close(got[1], want[1], f"state of {T}", 1e-5)


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_input_gradient_from_a_state_s_gradient_with_a_mean(shape):
    """dx where it comes from the last state's gradient, of mean 16, and B cancels it. The
    outputs' own gradient is zero, so dx is nothing else; D is absent."""
    from astra_cuda import sequence as seq
    H, P, G, N = shape
    print("states", shape, flush=True)
    g = gen(22)
    for T in (40, 200):
        own = inputs(g, 2, T, H, P, G, N, 0.0)
        ref = {k: wide(v) for k, v in own.items()}
        dh = normal(g, 2, H, P, N) + 16
        out, want = run_scan(seq, own), ref_scan(ref)
        got = torch.autograd.grad(out, [own["x"]], [torch.zeros_like(out[0]), dh])[0]
        exact = torch.autograd.grad(want, [ref["x"]], [torch.zeros_like(want[0]), dh.double()])[0]
        close(got, exact, f"dx of {T}", BOUND)


def test_whole_sequences_and_steps_agree():
    """The same positions through state_scan and through state_scan_step, which keeps its
    state in float32: each within the bound of the definition, over three chunks."""
    from astra_cuda import sequence as seq
    g = gen(23)
    T = 150
    own = inputs(g, 3, T, 2, 64, 1, 128, 16.0)
    with torch.no_grad():
        y, last = run_scan(seq, own)
        h = own["h"].clone()
        ys = [seq.state_scan_step(own["x"][:, t], own["dt"][:, t], own["A"], own["B"][:, t], own["C"][:, t], h)
              for t in range(T)]
    assert error(y, torch.stack(ys, 1)) <= 2 * BOUND
    assert error(last, h) <= 1e-5


def test_float_states_are_as_exact():
    from astra_cuda import sequence as seq
    g = gen(24)
    own = inputs(g, 2, 200, 2, 64, 1, 128, 16.0)
    own = {k: None if v is None else v.detach().to(F32) for k, v in own.items()}
    assert own["x"].device == torch.device(DEV)
    with torch.no_grad():
        got, want = run_scan(seq, own), ref_scan({k: wide(v) for k, v in own.items()})
    # 16 times the terms, each with a few 2^-24
    close(got[0], want[0], "y", 1e-5)
