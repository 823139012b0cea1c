"""log_probs of rows whose entries are alike, or nearly all of them: sums are whole numbers, and a piece, a
vector or an entry that is left out or counted twice shows."""
import math

import pytest
import torch

from probs_util import BF16, DEV, E, F32

pytestmark = pytest.mark.gpu

# One or few rows in pieces of 4,096 or 8,192 entries (3,663 pieces, of which a thread of the join has 4; 1,025; 17), rows by
# workgroups, rows by lanes.
SHAPES = [(1, 30_000_001), (1, 8_400_000), (3, 8_388_609), (7, 131_072), (64, 131_073), (200, 50_003), (600, 50_003), (2000, 2049),
          (9000, 1000), (9000, 513), (300, 257), (5, 9)]


def bound(n):
    """Of log Z: the sum is exact up to 2^24 and one of a power of two times whole numbers beyond, in at most 16
    additions a rounding each; the logarithm to 2 of its own, and the differences from it to 2 more."""
    return (16 + 4 * (math.log(n) + 1)) * E


@pytest.mark.parametrize("top", [0, 3])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("R,n", SHAPES)
def test_entries_that_are_alike(R, n, dtype, top):
    from astra_cuda import sequence as seq
    print("alike", R, n, dtype, top, flush=True)
    logits = torch.full((R, n), 1.5, device=DEV, dtype=dtype)
    choice = torch.arange(R, device=DEV) * 7919 % n
    out = seq.log_probs(logits, choice, top=top)
    for v in out[:2]:
        assert float((v.double().abs() - math.log(n)).abs().max()) <= bound(n)
    assert math.log(n) - math.log(n - min(8, n - 1)) > 2 * bound(n) or n > 10 ** 6
    assert math.log(n) - math.log(n - min(4096, n - 1)) > 10 * bound(n)  # (what is lost of less than a piece)
    if top:
        assert torch.equal(out[3], torch.arange(top, device=DEV).expand(R, top))
        assert float((out[2].double() + math.log(n)).abs().max()) <= bound(n)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("R,n", SHAPES)
def test_one_entry_above_all(R, n, dtype):
    """exp(-200) is 0 beside 1: the log probability of the one is 0, of any other -200; wherever it lies, the
    last entry of all and the ends of pieces among the places."""
    from astra_cuda import sequence as seq
    places = sorted({p for p in (0, 1, n // 2, n - 9, n - 1, 4095, 4096, 8191, 8192, 16_384 * 40 + 3, n - 8192, n - 4097) if 0 <= p < n})
    logits = torch.zeros(R, n, device=DEV, dtype=dtype)
    rows = torch.arange(R, device=DEV)
    for i, p in enumerate(places):
        at = (torch.full((R,), p, device=DEV) + rows * (i % 2)) % n
        logits[rows, at] = 200.0
        lp, h, tl, ti = seq.log_probs(logits, at, top=2)
        assert not bool(lp.any()) and not bool(h.any()), p
        assert torch.equal(ti[:, 0], at) and not bool(tl[:, 0].any()), p
        assert torch.equal(ti[:, 1], (at == 0).long()) and bool((tl[:, 1] == -200).all()), p
        lp, h = seq.log_probs(logits, (at + 1) % n)
        assert bool((lp == -200).all()) and not bool(h.any()), p
        logits[rows, at] = 0.0
