"""The direct terms of float32 scans, D x in y and D dy in dx, are rounded once, and not as
often as the sum of the other positions' terms is.

Bounds, on the 2-norm of the error over that of the output: one multiply-add, 2^-24 of each
element at most, 6.0e-8; the other positions' part is at most a fifth of the output here
(asserted), and a float32 sum of at most 64 products over 2 x 64 or fewer: 2e-7 of itself,
4e-8 of the output. Together 1e-7."""
import pytest
import torch

from sequence_util import F32, close, gen, normal, ref_scan, run_scan, scan_inputs, wide

pytestmark = pytest.mark.gpu
BOUND = 1e-7


@pytest.mark.parametrize("shape", [(4, 64, 1, 128), (4, 64, 2, 64), (2, 32, 1, 64), (4, 64, 1, 32), (4, 32, 1, 16),
                                   (3, 33, 1, 17), (2, 96, 1, 40)], ids=lambda s: "x".join(map(str, s)))
def test_direct_terms(shape):
    H, P, G, N = shape
    from astra_cuda import sequence as seq
    print("direct", shape, flush=True)
    g = gen(81)
    for T, carried in ((40, False), (64, True), (150, True)):
        own = scan_inputs(g, 3, T, H, P, G, N, F32, carried)
        with torch.no_grad():
            own["D"].copy_(10 + 10 * normal(g, H).abs())
            own["B"].mul_(N ** -0.5)
            own["C"].mul_(N ** -0.5)
            if carried:
                own["h"].mul_(0.5)
        ref = {k: wide(v) for k, v in own.items()}
        out, want = run_scan(seq, own), ref_scan(ref)
        direct = ref["D"][:, None] * ref["x"]
        assert float((want[0] - direct).norm()) <= 0.2 * float(want[0].norm())
        close(out[0], want[0], f"y of {T}", BOUND)
        dy = normal(g, *out[0].shape)
        got, = torch.autograd.grad(out[0], [own["x"]], dy)
        exact, = torch.autograd.grad(want[0], [ref["x"]], dy.double())
        assert float((exact - ref["D"][:, None] * dy.double()).norm()) <= 0.2 * float(exact.norm())
        close(got, exact, f"dx of {T}", BOUND)
