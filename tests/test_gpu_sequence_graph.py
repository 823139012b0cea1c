"""Whole-sequence calls in a captured graph: forward and backward, with kernels that need more
LDS than a launch gets unasked, segments and chunks. Every replay gives what an eager call
gives, with the program's own eager work between the replays."""
import pytest
import torch

from sequence_util import BF16, DEV, F32, gen, normal, run_scan, scan_inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", [
    (1, 2100, 2, 64, 1, 128, BF16), (2, 70, 4, 64, 1, 64, BF16), (2, 150, 2, 32, 1, 16, F32), (1, 200, 2, 64, 1, 128, F32),
], ids=lambda c: "x".join(map(str, c[:6])))
def test_scan_forward_and_backward_replay(case):
    from astra_cuda import sequence as seq
    *shape, dtype = case
    print("graph", case, flush=True)
    g = gen(51)
    own = scan_inputs(g, *shape, dtype, True)
    B, T, H, P, _, N = shape
    dy, dh = normal(g, B, T, H, P, dtype=dtype), normal(g, B, H, P, N)

    def once():
        out = run_scan(seq, own)
        return (*out, *torch.autograd.grad(out, list(own.values()), [dy, dh]))

    inputs = [{k: v.detach().clone() for k, v in scan_inputs(gen(52 + i), *shape, dtype, True).items()} for i in range(3)]

    def load(i):
        with torch.no_grad():
            for k, v in own.items():
                v.copy_(inputs[i][k])

    want = []
    for i in range(3):
        load(i)
        want.append([v.detach().clone() for v in once()])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = once()
    for i in (0, 1, 2, 1, 0):
        load(i)
        graph.replay()
        torch.cuda.synchronize()
        for k, (a, b) in enumerate(zip(got, want[i])):
            assert torch.equal(a.detach(), b), (i, k)
        load((i + 1) % 3)  # eager work of the same program
        again = once()
        assert all(torch.equal(a.detach(), b) for a, b in zip(again, want[(i + 1) % 3]))


def test_conv_and_join_forward_and_backward_replay():
    from astra_cuda import sequence as seq
    g = gen(53)
    x = normal(g, 3, 100, 64, dtype=BF16).requires_grad_()
    w, b = normal(g, 64, 4).requires_grad_(), normal(g, 64).requires_grad_()
    r, post, nxt = normal(g, 3, 100, 64).requires_grad_(), normal(g, 64).requires_grad_(), normal(g, 64).requires_grad_()
    scale = normal(g, 1).requires_grad_()
    dj, dn = normal(g, 3, 100, 64), normal(g, 3, 100, 64, dtype=BF16)
    leaves = [x, w, b, r, post, nxt, scale]

    def once():
        u = seq.short_conv(x, w, b)
        out = seq.join_norm(r, u, post, nxt, scale=scale)
        return (*out, *torch.autograd.grad(out, leaves, [dj, dn]))

    want = [v.detach().clone() for v in once()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = once()
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a.detach(), b) for a, b in zip(got, want))
        assert all(torch.equal(a.detach(), b) for a, b in zip(once(), want))
    assert r.device == torch.device(DEV)
