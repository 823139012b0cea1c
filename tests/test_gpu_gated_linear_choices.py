"""What a caller of gated_linear can choose: what is kept for the backward pass, and how exact bfloat16
gradients are."""
import ctypes
import math

import pytest
import torch

from gated_util import BF16, DEV, E, F32, activation, check, half_step, inputs, results, within

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


def exact_gradients(x, wg, wu, dh, kind):
    """{name: (value, bound)} of the gradients in 64 bits, where da and db enter their products to 2^-17 and not
    to 2^-8: of v in [1, 2) the first number loses at most 2^-8, half a step of which is at most 2^-17."""
    u, rest = half_step(x.dtype), 2.0 ** -17
    x, wg, wu, dh = (v.detach().double() for v in (x, wg, wu, dh))
    (M, D), F = x.shape, wg.shape[0]
    a, b = x @ wg.t(), x @ wu.t()
    ea, eb = ((D + 2) * E * (x.abs() @ w.abs().t()) for w in (wg, wu))
    act, slope = activation(a, kind)
    near = 16 * E * a.abs().clamp(min=1)
    e_act, e_slope = 1.13 * ea + near, 0.8 * ea + near
    da, db = dh * b * slope, dh * act
    e_da = dh.abs() * (e_slope * (b.abs() + eb) + slope.abs() * eb) + (3 * E + rest) * da.abs()
    e_db = dh.abs() * e_act + (3 * E + rest) * db.abs()
    dx, n = da @ wg + db @ wu, (4 * F + 2) * E
    out = {"dx": (dx, (e_da * (1 + n)) @ wg.abs() + (e_db * (1 + n)) @ wu.abs()
                  + n * (da.abs() @ wg.abs() + db.abs() @ wu.abs()) + u * dx.abs())}
    n = (2 * M + 2) * E
    for name, d, e in (("dgate", da, e_da), ("dup", db, e_db)):
        w = d.t() @ x
        out[name] = (w, (e.t() * (1 + n)) @ x.abs() + n * (d.abs().t() @ x.abs()) + u * w.abs())
    return out


@pytest.mark.parametrize("kind", ["silu", "gelu"])
@pytest.mark.parametrize("M,D,F", [(1, 1, 1), (1, 256, 1024), (40, 128, 40), (130, 33, 65), (200, 520, 1000), (257, 1000, 136),
                                   (300, 4096, 520), (2049, 256, 512), (8200, 1031, 72), (8193, 1024, 600), (20_000, 40, 72),
                                   (16_400, 136, 1032), (8195, 1024, 4104)])
def test_exact_gradients(M, D, F, kind):
    """Rounded once: off by hardly more than 64 bits rounded to bfloat16, and the same h."""
    from astra_cuda import sequence as seq
    print("exact", M, D, F, kind, flush=True)
    x, wg, wu, dh = inputs(M + F, M, D, F, BF16)
    got, _ = call(seq, x, wg, wu, dh, kind, exact_gradients=True)
    usual, _ = call(seq, x, wg, wu, dh, kind)
    assert torch.equal(got["h"], usual["h"])
    want = exact_gradients(x, wg, wu, dh, kind)
    for name in want:
        within(got[name], want[name], name)
        if got[name].numel() > 1000:
            # In the mean, of independent roundings: that of the result, and da's and db's 2^-17 (and float32
            # sums of up to 2 M terms, which are some 2^-20 here) instead of 2^-8 from each.
            off, least = ((v.double() - want[name][0]).norm() / want[name][0].norm()
                          for v in (got[name], want[name][0].to(BF16)))
            assert float(off) <= 1.02 * float(least), (name, float(off), float(least))
    for choice in ({"recompute": True}, {}):
        again, _ = call(seq, x, wg, wu, dh, kind, exact_gradients=True, **choice)
        if not choice:
            assert all(torch.equal(got[k], again[k]) for k in got)
        for name in want:
            within(again[name], want[name], name)


@pytest.mark.parametrize("which", [(0,), (1,), (2,), (0, 2), (1, 2)])
@pytest.mark.parametrize("M,D,F", [(100, 48, 56), (8200, 1024, 72)])
def test_exact_gradients_that_are_asked_for(M, D, F, which):
    from astra_cuda import sequence as seq
    x, wg, wu, dh = inputs(6, M, D, F, BF16)
    want, _ = call(seq, x, wg, wu, dh, "silu", exact_gradients=True)
    leaves = [v.detach().clone().requires_grad_(i in which) for i, v in enumerate((x, wg, wu))]
    got = torch.autograd.grad(seq.gated_linear(*leaves, exact_gradients=True), [leaves[i] for i in which], dh)
    for i, d in zip(which, got):
        assert torch.equal(d, want[("dx", "dgate", "dup")[i]])


def test_exact_float_gradients_are_the_usual_ones():
    from astra_cuda import sequence as seq
    x, wg, wu, dh = inputs(8, 300, 72, 100, F32)
    got, want = (call(seq, x, wg, wu, dh, "silu", exact_gradients=e)[0] for e in (True, False))
    assert all(torch.equal(got[k], want[k]) for k in want)


def test_exact_gradients_that_are_not_finite():
    """da beyond the largest bfloat16 is an infinity, not what is left of one."""
    from astra_cuda import sequence as seq
    top = torch.finfo(BF16).max
    x = torch.tensor([[1.0, 0.0], [1.0, 0.0], [1.0, 2.0]], device=DEV, dtype=BF16)
    wg, wu = torch.tensor([[64.0, 0.0]], device=DEV, dtype=BF16), torch.tensor([[1.0, 0.0]], device=DEV, dtype=BF16)
    dh = torch.tensor([[1.0], [top], [math.nan]], device=DEV, dtype=BF16)
    got, _ = call(seq, x, wg, wu, dh, "silu", exact_gradients=True)  # act(64) = 64 and its slope 1: da = dh, db = 64 dh
    assert got["dx"][0].tolist() == [128.0, 0.0] and float(got["dx"][1, 0]) == math.inf
    assert bool(torch.isnan(got["dx"][2]).all()) and bool(torch.isnan(got["dup"]).any())


def test_exact_gradients_by_the_c_entry():
    """Its workspace is larger, and no byte beyond it is written."""
    from astra_cuda import _native
    lib = _native.lib()
    exact = 256  # ASTRA_SEQ_EXACT_GRADIENTS
    for M, D, F in ((300, 64, 128), (8200, 1024, 72)):
        x, wg, wu, dh = inputs(14, M, D, F, BF16)
        h = torch.empty_like(dh)
        f = _native.GatedLinear(x=x.data_ptr(), gate=wg.data_ptr(), up=wu.data_ptr(), h=h.data_ptr(), rows=M, x_stride=D,
                                gate_stride=D, up_stride=D, width=D, hidden=F, type=1, activation=1)
        n, need = [], "astra_gated_linear_grad_workspace_size"
        for f.activation in (1, 1 | exact):
            n.append(ctypes.c_size_t(0))
            assert getattr(lib, need)(ctypes.addressof(f), ctypes.byref(n[-1])) == 0
        assert n[1].value == n[0].value + M * 2 * 128 * 2
        stream = torch.cuda.current_stream().cuda_stream
        spare = ctypes.c_size_t(0)
        assert lib.astra_gated_linear_workspace_size(ctypes.addressof(f), ctypes.byref(spare)) == 0
        partial = torch.empty(max(spare.value, 1), dtype=torch.uint8, device=DEV)
        f.workspace, f.workspace_bytes = partial.data_ptr(), spare.value
        assert lib.astra_gated_linear_forward(ctypes.addressof(f), stream) == 0
        grads = [torch.empty_like(v) for v in (x, wg, wu)]
        b = _native.GatedLinearGrad(f=f, dh=dh.data_ptr(), dx=grads[0].data_ptr(), dgate=grads[1].data_ptr(), dup=grads[2].data_ptr())
        ws = torch.full((n[1].value + 4096,), 77, dtype=torch.uint8, device=DEV)
        b.workspace, b.workspace_bytes = ws.data_ptr(), n[1].value - 1
        assert lib.astra_gated_linear_backward(ctypes.addressof(b), stream) == 1
        b.workspace_bytes = n[1].value
        assert lib.astra_gated_linear_backward(ctypes.addressof(b), stream) == 0
        torch.cuda.synchronize()
        assert bool((ws[n[1].value:] == 77).all())
        want = exact_gradients(x, wg, wu, dh, "silu")
        within(h, results(x, wg, wu, dh, "silu")["h"], "h")
        for name, d in zip(("dx", "dgate", "dup"), grads):
            within(d, want[name], name)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("choice", [{"recompute": True}, {"exact_gradients": True}, {"recompute": True, "exact_gradients": True}], ids=str)
def test_choices_with_no_rows_and_other_shapes(choice, dtype):
    from astra_cuda import sequence as seq
    x, wg, wu, dh = inputs(7, 0, 1032, 40, dtype)
    got, _ = call(seq, x, wg, wu, dh, "silu", **choice)
    assert got["dx"].shape == (0, 1032) and not got["dgate"].any() and not got["dup"].any()
    x, wg, wu, dh = inputs(9, 96, 136, 72, dtype)
    want, _ = call(seq, x, wg, wu, dh, "gelu", **choice)
    # rows beside others, and with leading dimensions
    wide = torch.full((96, 150), math.nan, device=DEV, dtype=dtype)
    wide[:, 9:145] = x
    got, _ = call(seq, wide[:, 9:145], wg, wu, dh, "gelu", **choice)
    assert all(torch.equal(got[k], want[k]) for k in want)
    got, _ = call(seq, x.view(4, 24, 136), wg, wu, dh.view(4, 24, 72), "gelu", **choice)
    assert all(torch.equal(got[k].flatten(0, -2), want[k]) for k in want)


def test_exact_gradients_in_two_graphs_and_beside_them():
    """Two graphs of one pass each, replayed in turn on streams of their own while eager passes run."""
    from astra_cuda import sequence as seq
    sets = [inputs(50 + i, 8200, 1024, 200, BF16) for i in range(3)]
    want = [call(seq, *s, "silu", exact_gradients=True)[0] for s in sets]
    graphs = []
    for i in range(2):
        x, wg, wu, dh = (v.clone() for v in sets[i])
        leaves = [v.requires_grad_() for v in (x, wg, wu)]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            h = seq.gated_linear(*leaves, exact_gradients=True)
            got = [h, *torch.autograd.grad(h, leaves, dh)]
        graphs.append((graph, (x, wg, wu, dh), got, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for turn in range(3):
        for i, (graph, into, got, stream) in enumerate(graphs):
            with torch.cuda.stream(stream), torch.no_grad():
                for a, b in zip(into, sets[(turn + i) % 3]):
                    a.copy_(b)
                graph.replay()
        eager = call(seq, *sets[turn], "silu", exact_gradients=True)[0]
        torch.cuda.synchronize()
        assert all(torch.equal(eager[k], want[turn][k]) for k in eager)
        for i, (graph, into, got, stream) in enumerate(graphs):
            assert all(torch.equal(a.detach(), b) for a, b in zip(got, want[(turn + i) % 3].values())), (turn, i)
