"""What the tests of whole numbers see, on the CPU: mistakes planted in what they compare with."""
import pytest
import torch

import gated_integers

F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("M,D,F", [(70_001, 24, 16), (20_000, 40, 72), (8200, 1031, 72), (8193, 256, 600)])
def test_rows_that_are_lost_show(M, D, F, dtype):
    """A slice of the rows, a step of one, and the part of a step at the end: without any of them both weights'
    gradients are others."""
    x, gate, up, dh = gated_integers.inputs(M, M, D, F, dtype, "cpu")
    da, db, _ = gated_integers.slopes(x, gate, up, dh)
    want = gated_integers.results(x, gate, up, dh)
    wx = x.double()
    for rows in (32, 64, 288, 576):
        starts = list(range(0, M, rows))
        for first in starts[:: max(1, len(starts) // 12)] + starts[-1:]:
            part = slice(first, min(first + rows, M))
            for name, d in (("dgate", da), ("dup", db)):
                lost = (d.t() @ wx - d[part].t() @ wx[part]).to(dtype)
                assert not torch.equal(lost, want[name]), (name, rows, first)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_columns_that_are_lost_or_exchanged_show(dtype):
    x, gate, up, dh = gated_integers.inputs(1, 300, 520, 200, dtype, "cpu")
    want = gated_integers.results(x, gate, up, dh)
    for j in (1, 7, 63, 64, 511, 519):
        bad = x.clone()
        bad[:, j] = 0
        assert not torch.equal(gated_integers.results(bad, gate, up, dh)["h"], want["h"]), j
    for j in (3, 65, 510):
        bad = x.clone()
        bad[:, [j, j + 8]] = x[:, [j + 8, j]]
        assert not torch.equal(gated_integers.results(bad, gate, up, dh)["h"], want["h"]), j
    for j in (0, 17, 199):
        bad = dh.clone()
        bad[:, j] = 0
        assert not torch.equal(gated_integers.results(x, gate, up, bad)["dx"], want["dx"]), j
