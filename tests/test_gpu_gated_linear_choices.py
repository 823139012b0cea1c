"""What a caller of gated_linear can choose: what is kept for the backward pass."""
import pytest
import torch

from gated_util import BF16, DEV, F32, check, inputs

pytestmark = pytest.mark.gpu


def call(seq, x, wg, wu, dh, kind, **choice):
    leaves = [v.detach().requires_grad_() for v in (x, wg, wu)]
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    h = seq.gated_linear(*leaves, activation=kind, **choice)
    kept = torch.cuda.memory_allocated() - before - h.numel() * h.element_size()
    return dict(zip(("h", "dx", "dgate", "dup"), (h.detach(), *torch.autograd.grad(h, leaves, dh)))), kept


@pytest.mark.parametrize("kind", ["silu", "gelu"])
@pytest.mark.parametrize("M,D,F,dtype", [(1, 1024, 65, BF16), (40, 1030, 200, BF16), (300, 1024, 257, BF16),
                                         (2049, 1100, 1024, BF16), (8200, 1032, 264, BF16), (1, 128, 40, F32),
                                         (50, 129, 130, F32), (700, 256, 683, F32), (300, 4096, 520, F32)])
def test_recomputed_projections(M, D, F, dtype, kind):
    """They are not kept (but for what the allocator adds to a tensor of this size)."""
    from astra_cuda import sequence as seq
    x, wg, wu, dh = inputs(M + D, M, D, F, dtype)
    got, kept = call(seq, x, wg, wu, dh, kind, recompute=True)
    usual, kept_usual = call(seq, x, wg, wu, dh, kind)
    assert kept <= 512 and kept_usual >= 8 * M * F
    assert torch.equal(got["h"], usual["h"])
    check(got, x, wg, wu, dh, kind)
    again, _ = call(seq, x, wg, wu, dh, kind, recompute=True)
    assert all(torch.equal(got[k], again[k]) for k in got)


def test_narrow_blocks_keep_nothing_anyway():
    from astra_cuda import sequence as seq
    for recompute in (False, True):
        x, wg, wu, dh = inputs(3, 500, 64, 96, BF16)
        got, kept = call(seq, x, wg, wu, dh, "silu", recompute=recompute)
        assert kept <= 512
        check(got, x, wg, wu, dh, "silu")


def test_recomputed_projections_in_a_graph():
    from astra_cuda import sequence as seq
    sets = [inputs(40 + i, 300, 1024, 264, BF16) for i in range(3)]
    want = [call(seq, *s, "silu", recompute=True)[0] for s in sets]
    x, wg, wu, dh = (v.clone() for v in sets[0])
    leaves = [v.requires_grad_() for v in (x, wg, wu)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h = seq.gated_linear(*leaves, recompute=True)
        got = [h, *torch.autograd.grad(h, leaves, dh)]
    for i in (0, 1, 2, 0):
        with torch.no_grad():
            for a, b in zip((x, wg, wu, dh), sets[i]):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a.detach(), b) for a, b in zip(got, want[i].values())), i
        again = call(seq, *sets[(i + 1) % 3], "silu", recompute=True)[0]
        assert all(torch.equal(again[k], want[(i + 1) % 3][k]) for k in again)
