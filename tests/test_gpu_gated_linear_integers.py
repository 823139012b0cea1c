"""gated_linear of whole numbers, bit by bit (gated_integers.py says why that is possible), at sizes where rows
are cut into many slices, and in every form of its tiles with rows and hidden widths off their edges."""
import pytest
import torch

import gated_integers
from gated_util import BF16, DEV, F32, call, check
from gated_util import inputs as normal_inputs

pytestmark = pytest.mark.gpu

# Tiles of 128 x 192 results: h of all (but float32 rows of 1,020), with the projections kept and not; da and db with
# the projections computed again, which bf16 rows of 1,017 to 1,023 do anyway; dx of the first in bf16 (weights turned).
WIDE = [(8195, 2056, 4100), (8195, 1024, 4104), (8195, 1020, 4104), (3001, 1021, 3001)]
SIZES = [(1, 1, 1), (1, 256, 1024), (2, 7, 3), (16, 32, 17), (33, 128, 40), (64, 96, 130), (65, 64, 128), (129, 33, 65),
         (200, 520, 1000), (257, 1000, 136), (300, 4096, 520), (2049, 256, 512), (4100, 100, 4096), (20_000, 40, 72),
         (70_001, 24, 16), (8200, 1031, 72), (8193, 1024, 600), (16_400, 1048, 1032), (6145, 1100, 2100)] + WIDE


def run(seq, x, gate, up, dh, kind, **choice):
    leaves = [v.detach().requires_grad_() for v in (x, gate, up)]
    h = seq.gated_linear(*leaves, activation=kind, **choice)
    return dict(zip(("h", "dx", "dgate", "dup"), (h.detach(), *torch.autograd.grad(h, leaves, dh))))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_every_bit(size, dtype):
    from astra_cuda import sequence as seq
    print("gated integers", size, dtype, flush=True)
    x, gate, up, dh = gated_integers.inputs(sum(size), *size, dtype, DEV)
    want = gated_integers.results(x, gate, up, dh)
    for kind in ("silu", "gelu"):
        for choice in ({}, {"recompute": True}, {"exact_gradients": True}):
            got = run(seq, x, gate, up, dh, kind, **choice)
            for k in want:
                assert torch.equal(got[k], want[k]), (k, kind, choice, int((got[k] != want[k]).sum()))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("size", [(20_000, 40, 72), (8200, 1031, 72), (8193, 1024, 600), (8195, 1020, 4104)],
                         ids=lambda s: "x".join(map(str, s)))
def test_one_row_s_gradient(size, dtype):
    """Of all rows one alone has a gradient: the first, the last, and those about the ends of a step."""
    from astra_cuda import sequence as seq
    M = size[0]
    x, gate, up, full = gated_integers.inputs(7, *size, dtype, DEV)
    for m in (0, 31, 32, 63, 64, 575, 576, M // 2, M - 65, M - 2, M - 1):
        dh = torch.zeros_like(full)
        dh[m] = full[m]
        got = run(seq, x, gate, up, dh, "silu")
        want = gated_integers.results(x[m:m + 1], gate, up, dh[m:m + 1])
        assert torch.equal(got["dx"][m:m + 1], want["dx"]) and not bool(got["dx"][:m].any() or got["dx"][m + 1:].any()), m
        assert torch.equal(got["dgate"], want["dgate"]) and torch.equal(got["dup"], want["dup"]), m


@pytest.mark.parametrize("kind", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("size", WIDE, ids=lambda s: "x".join(map(str, s)))
def test_wide_tiles(size, dtype, kind):
    from astra_cuda import sequence as seq
    print("gated wide", size, dtype, kind, flush=True)
    x, wg, wu, dh = normal_inputs(sum(size), *size, dtype)
    got = call(seq, x, wg, wu, dh, kind)
    check(got, x, wg, wu, dh, kind)
    check(run(seq, x, wg, wu, dh, kind, recompute=True), x, wg, wu, dh, kind)
    with torch.no_grad():
        assert torch.equal(seq.gated_linear(x, wg, wu, activation=kind), got["h"])
