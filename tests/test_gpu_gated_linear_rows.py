"""gated_linear at more rows than one launch has threads for."""
import pytest
import torch

from gated_util import DEV, F32, inputs, results, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [2 ** 24 + 37, 2 ** 28 + 37])
def test_gradients_from_kept_projections(M):
    """Rows of which the first and the last 50 alone are not zero: the kept projections' gradients take 16
    threads a row, and 2^28 rows are 2^32 threads. (137 GB of rows, 69 of gradients of their projections.)"""
    from astra_cuda import sequence as seq
    torch.cuda.empty_cache()
    D, F = 128, 1
    if torch.cuda.mem_get_info()[0] < M * 4 * (D + 64 + 4 * F) + (8 << 30):
        pytest.skip("not enough memory")
    print("gated", M, D, F, flush=True)
    few, wg, wu, dh_few = inputs(31, 51, D, F, F32)
    x, dh = torch.zeros(M, D, device=DEV), torch.zeros(M, F, device=DEV)
    for whole, part in ((x, few), (dh, dh_few)):
        whole[:1], whole[-50:] = part[:1], part[1:]
    wg.requires_grad_()
    wu.requires_grad_()
    h = seq.gated_linear(x, wg, wu)
    dgate, dup = torch.autograd.grad(h, (wg, wu), dh)
    want = results(few, wg, wu, dh_few, "silu")  # (rows of zeros add nothing, and no rounding)
    within(torch.cat([h[:1], h[-50:]]), want["h"], "h")
    assert not bool(h[1:-50].any())
    within(dgate, want["dgate"], "dgate")
    within(dup, want["dup"], "dup")
