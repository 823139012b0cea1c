"""gated_linear and its gradients against the definition in 64 bits, with bounds per element: sizes at
and around the tiles' edges, operands that do not lie as the tiles want them, values that are not
finite, and the modes a call can be made in."""
import math

import pytest
import torch

from gated_util import BF16, DEV, F32, call, check, half_step, inputs, results, within

pytestmark = pytest.mark.gpu

SIZES = [
    (1, 1, 1), (1, 256, 1024), (2, 7, 3), (15, 8, 16), (16, 32, 17), (17, 64, 64), (33, 128, 40), (64, 96, 130),
    (65, 64, 128), (127, 72, 129), (128, 128, 64), (129, 33, 65), (200, 520, 1000), (256, 64, 256), (257, 1000, 136),
    (1000, 136, 1111), (2049, 256, 512), (4100, 100, 4096), (20_000, 40, 72), (70_001, 24, 16), (513, 1031, 2050),
    (8200, 1031, 72), (8193, 1024, 600), (16_400, 136, 1032),
]


@pytest.mark.parametrize("kind", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_values_and_gradients(size, dtype, kind):
    from astra_cuda import sequence as seq
    print("gated", size, dtype, kind, flush=True)
    x, wg, wu, dh = inputs(sum(size), *size, dtype)
    got = call(seq, x, wg, wu, dh, kind)
    check(got, x, wg, wu, dh, kind)
    with torch.no_grad():
        assert torch.equal(seq.gated_linear(x, wg, wu, activation=kind), got["h"])
    again = call(seq, x, wg, wu, dh, kind)
    assert all(torch.equal(got[k], again[k]) for k in got)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_large_widths(dtype):
    """Many steps of the contraction, and more tiles than a band has."""
    from astra_cuda import sequence as seq
    for size in ((2304, 2048, 2560), (300, 4096, 4104)):
        x, wg, wu, dh = inputs(3, *size, dtype)
        check(call(seq, x, wg, wu, dh, "silu"), x, wg, wu, dh, "silu")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("M", [3, 64, 150])
@pytest.mark.parametrize("D", [40, 37, 200])
def test_operands_inside_larger_memory(dtype, M, D):
    """What lies beside an operand's rows, behind them or before them is never used: it is NaN."""
    from astra_cuda import sequence as seq
    for shift, pad in ((0, 24), (0, 1), (8, 8), (3, 10)):
        x, wg, wu, dh = inputs(M + D, M, D, 72, dtype)
        def inside(v):
            big = torch.full((v.shape[0] + 2, shift + v.shape[1] + pad), math.nan, device=DEV, dtype=dtype)
            big[1:-1, shift:shift + v.shape[1]] = v
            return big[1:-1, shift:shift + v.shape[1]]
        got = call(seq, inside(x), inside(wg), inside(wu), inside(dh), "silu")
        check(got, x, wg, wu, dh, "silu")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_views(dtype):
    """Halves of one weight, a transposed input, leading dimensions, a broadcast input, one weight twice."""
    from astra_cuda import sequence as seq
    x, wg, wu, dh = inputs(5, 96, 64, 48, dtype)
    want = call(seq, x, wg, wu, dh, "gelu")
    both = torch.cat([wg, wu]).requires_grad_()
    h = seq.gated_linear(x.view(4, 24, 64), both[:48], both[48:], activation="gelu")
    assert h.shape == (4, 24, 48) and torch.equal(h.detach().view(96, 48), want["h"])
    d, = torch.autograd.grad(h, both, dh.view(4, 24, 48))
    assert torch.equal(d, torch.cat([want["dgate"], want["dup"]]))
    xt = x.t().contiguous().requires_grad_()
    h = seq.gated_linear(xt.t(), wg, wu, activation="gelu")
    assert torch.equal(h.detach(), want["h"])
    d, = torch.autograd.grad(h, xt, dh)
    assert torch.equal(d.t(), want["dx"])
    one = x[:1].detach().clone().requires_grad_()
    h = seq.gated_linear(one.expand(96, 64), wg, wu, activation="gelu")
    d, = torch.autograd.grad(h, one, dh)
    rows = call(seq, one.detach().expand(96, 64).contiguous(), wg, wu, dh, "gelu")
    assert torch.equal(h.detach(), rows["h"])
    # the rows' sum: 96 of them, rounded once more by torch
    total, size = rows["dx"].double().sum(0, keepdim=True), rows["dx"].double().abs().sum(0, keepdim=True)
    assert bool(((d.double() - total).abs() <= 98 * half_step(dtype) * size).all())
    w = wg.detach().clone().requires_grad_()
    h = seq.gated_linear(x, w, w)
    d, = torch.autograd.grad(h, w, dh)
    twice = call(seq, x, wg, wg, dh, "silu")
    assert torch.equal(d, twice["dgate"] + twice["dup"])
    v = x[0]
    assert torch.equal(seq.gated_linear(v, wg, wu), seq.gated_linear(v[None], wg, wu)[0])


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("which", [(0,), (1,), (2,), (0, 2), (1, 2)])
def test_gradients_that_are_asked_for(dtype, which):
    from astra_cuda import sequence as seq
    x, wg, wu, dh = inputs(6, 100, 48, 56, dtype)
    want = call(seq, x, wg, wu, dh, "silu")
    leaves = [v.detach().clone() for v in (x, wg, wu)]
    for i in which:
        leaves[i].requires_grad_()
    got = torch.autograd.grad(seq.gated_linear(*leaves), [leaves[i] for i in which], dh)
    for i, d in zip(which, got):
        assert torch.equal(d, want[("dx", "dgate", "dup")[i]])


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_rows_that_overlap(dtype):
    """Rows that begin inside the row before them: an infinity in the last one is in no other, nor in
    what would lie behind it. (The slope at infinity is 1 + inf * 0, so dgate is NaN; dup is not.)"""
    from astra_cuda import sequence as seq
    M, D, F = 100, 64, 24
    memory = torch.rand((M - 1) * 8 + D, device=DEV).to(dtype) + 1
    memory[-1] = math.inf
    x = memory.as_strided((M, D), (8, 1))
    w, dh = torch.ones(F, D, device=DEV, dtype=dtype), torch.ones(M, F, device=DEV, dtype=dtype)
    got, want = call(seq, x, w, w, dh, "silu"), call(seq, x.contiguous(), w, w, dh, "silu")
    assert bool(torch.isposinf(want["dup"]).all())
    assert all(torch.equal(got[k].nan_to_num(-1.0, -2.0), want[k].nan_to_num(-1.0, -2.0)) for k in want)


def test_projections_that_are_not_wanted():
    """The C entry writes as many floats as it says, none where that is none."""
    import ctypes
    from astra_cuda import _native
    lib = _native.lib()
    for M in (40, 300):
        x, wg, wu, dh = inputs(14, M, 64, 128, BF16)
        h, spare = torch.empty_like(dh), torch.full((2, M, 128), 7.0, device=DEV)
        f = _native.GatedLinear(x=x.data_ptr(), gate=wg.data_ptr(), up=wu.data_ptr(), h=h.data_ptr(),
                                projections=spare.data_ptr(), rows=M, x_stride=64, gate_stride=64, up_stride=64,
                                width=64, hidden=128, type=1, activation=1)
        n = ctypes.c_size_t(1)
        assert lib.astra_gated_linear_projections(ctypes.addressof(f), ctypes.byref(n)) == 0 and n.value == 0
        assert lib.astra_gated_linear_workspace_size(ctypes.addressof(f), ctypes.byref(n)) == 0 and n.value == 0
        assert lib.astra_gated_linear_forward(ctypes.addressof(f), torch.cuda.current_stream().cuda_stream) == 0
        grads = [torch.empty_like(v) for v in (x, wg, wu)]
        b = _native.GatedLinearGrad(f=f, dh=dh.data_ptr(), dx=grads[0].data_ptr(), dgate=grads[1].data_ptr(), dup=grads[2].data_ptr())
        assert lib.astra_gated_linear_grad_workspace_size(ctypes.addressof(f), ctypes.byref(n)) == 0
        ws = torch.empty(n.value, dtype=torch.uint8, device=DEV)
        b.workspace, b.workspace_bytes = ws.data_ptr(), n.value
        assert lib.astra_gated_linear_backward(ctypes.addressof(b), torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        assert bool((spare == 7).all())
        check(dict(zip(("h", "dx", "dgate", "dup"), (h, *grads))), x, wg, wu, dh, "silu")


def test_copies_of_more_than_64_gib():
    """Rows that do not start on 16 bytes, more than one launch has threads for. (One row serves all.)"""
    from astra_cuda import sequence as seq
    M, D, F = 2 ** 25 + 5, 1024, 8
    x, wg, wu, dh = inputs(17, 1, D + 1, F, BF16)
    x, wg, wu = x[:, 1:], wg[:, 1:], wu[:, 1:]
    h = seq.gated_linear(x.expand(M, D), wg, wu)
    assert bool((h == h[0]).all())
    within(h[:1], results(x, wg, wu, dh, "silu")["h"], "h")


def test_more_than_2_to_the_31_results():
    """Of whose gradient the last rows alone are not zero."""
    from astra_cuda import sequence as seq
    M, D, F = 2_200_001, 8, 1000
    _, wg, wu, _ = inputs(15, 1, D, F, BF16)
    x = torch.randn(M, D, device=DEV).to(BF16)
    dh = torch.zeros(M, F, device=DEV, dtype=BF16)
    dh[-70:] = torch.randn(70, F, device=DEV).to(BF16)
    got = call(seq, x, wg, wu, dh, "silu")
    want = results(x[-70:], wg, wu, dh[-70:], "silu")
    assert not bool(got["dx"][:-70].any())
    for k in ("h", "dx", "dgate", "dup"):
        within(got[k][-70:] if k in ("h", "dx") else got[k], want[k], k)


def test_no_rows():
    from astra_cuda import sequence as seq
    for dtype in (F32, BF16):
        x, wg, wu, dh = inputs(7, 0, 24, 40, dtype)
        got = call(seq, x, wg, wu, dh, "silu")
        assert got["h"].shape == (0, 40) and got["dx"].shape == (0, 24)
        assert not got["dgate"].any() and not got["dup"].any()
        assert seq.gated_linear(x.view(3, 0, 24), wg, wu).shape == (3, 0, 40)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("M", [40, 300])
def test_values_that_are_not_finite_stay_in_their_rows(dtype, M):
    from astra_cuda import sequence as seq
    x, wg, wu, dh = inputs(8, M, 72, 100, dtype)
    good = call(seq, x, wg, wu, dh, "silu")
    bad = x.clone()
    bad[M - 1, 71], bad[M // 2, 0] = math.inf, math.nan
    got = call(seq, bad, wg, wu, dh, "silu")
    rows = torch.ones(M, dtype=torch.bool, device=DEV)
    rows[[M - 1, M // 2]] = False
    for k in ("h", "dx"):
        assert torch.equal(got[k][rows], good[k][rows]), k
    assert bool(torch.isnan(got["h"][M // 2]).all()) and not bool(torch.isfinite(got["h"][M - 1]).any())
    w = wg.clone()
    w[99, 71] = math.nan
    got = call(seq, x, w, wu, dh, "silu")
    assert torch.equal(got["h"][:, :99], good["h"][:, :99]) and bool(torch.isnan(got["h"][:, 99]).all())
    assert torch.equal(got["dgate"][:99], good["dgate"][:99]) and torch.equal(got["dup"][:99], good["dup"][:99])


@pytest.mark.parametrize("kind", ["silu", "gelu"])
def test_far_values_of_the_activations(kind):
    """a from -200 to 200 through a weight of 1, against 64 bits; and the largest floats."""
    from astra_cuda import sequence as seq
    a = torch.cat([torch.linspace(-200, 200, 4001, device=DEV), torch.linspace(-15, 15, 3001, device=DEV)])
    x = torch.stack([a, torch.ones_like(a)], 1)
    w, one = torch.tensor([[1.0, 0.0]], device=DEV), torch.tensor([[0.0, 1.0]], device=DEV)
    dh = torch.ones(len(a), 1, device=DEV)
    check(call(seq, x, w, one, dh, kind), x, w, one, dh, kind)
    big = torch.tensor([[1e30, 1.0], [3e38, 1.0], [-1e30, 1.0], [-3e38, 1.0]], device=DEV)
    got = call(seq, big, w, one, dh[:4], kind)
    assert torch.equal(got["h"][:2], big[:2, :1]) and not bool(got["h"][2:].any())
    assert torch.equal(got["dx"][:, 0], torch.tensor([1.0, 1.0, 0.0, 0.0], device=DEV))


@pytest.mark.parametrize("kind", ["silu", "gelu"])
def test_gradients_against_differences(kind):
    """Along random directions, L = sum(h dh) in 64 bits over the kernel's float32 h. With steps of s
    the difference is off by s^2 / 6 times a third derivative of order L's own terms, and by 2^-24
    sqrt(terms) over s: both below 1e-3 of the terms' norm at s = 1e-2."""
    from astra_cuda import sequence as seq
    x, wg, wu, dh = inputs(9, 130, 64, 96, F32)
    got = call(seq, x, wg, wu, dh, kind)
    g = torch.Generator(device=DEV)
    g.manual_seed(10)
    leaves = [x, wg, wu]
    for i, name in enumerate(("dx", "dgate", "dup")):
        v = torch.randn(leaves[i].shape, generator=g, device=DEV)
        v = v / v.norm() * leaves[i].norm()
        step = 1e-2
        ends = []
        for s in (step, -step):
            moved = list(leaves)
            moved[i] = leaves[i] + s * v
            ends.append(seq.gated_linear(*moved, activation=kind).double() * dh.double())
        slope = float((ends[0] - ends[1]).sum()) / (2 * step)
        scale = float(got[name].double().norm() * v.double().norm())
        assert abs(slope - float((got[name].double() * v.double()).sum())) <= 1e-3 * scale, name


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("size", [(20, 64, 96), (300, 72, 100), (3000, 33, 130)], ids=lambda s: "x".join(map(str, s)))
def test_forward_and_backward_replay(size, dtype):
    from astra_cuda import sequence as seq
    print("graph", size, dtype, flush=True)
    sets = [inputs(20 + i, *size, dtype) for i in range(3)]
    want = [call(seq, *s, "silu") for s in sets]
    x, wg, wu, dh = (v.clone() for v in sets[0])
    leaves = [v.requires_grad_() for v in (x, wg, wu)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h = seq.gated_linear(*leaves)
        got = [h, *torch.autograd.grad(h, leaves, dh)]
    for i in (0, 1, 2, 1, 0):
        with torch.no_grad():
            for a, b in zip((x, wg, wu, dh), sets[i]):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a.detach(), b) for a, b in zip(got, want[i].values())), i
        again = call(seq, *sets[(i + 1) % 3], "silu")
        assert all(torch.equal(again[k], want[(i + 1) % 3][k]) for k in again)


def test_another_stream():
    from astra_cuda import sequence as seq
    x, wg, wu, dh = inputs(11, 700, 264, 520, BF16)
    want = call(seq, x, wg, wu, dh, "silu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = torch.zeros_like(x)
        for _ in range(20):
            late = late + x
        got = call(seq, late / 20, wg, wu, dh, "silu")
    side.synchronize()
    ref = call(seq, (late / 20), wg, wu, dh, "silu")
    assert all(torch.equal(got[k], ref[k]) for k in got) and want["h"].shape == got["h"].shape


def test_refusals():
    from astra_cuda import sequence as seq
    import torch.autograd.forward_ad as fwd
    x, wg, wu, dh = inputs(12, 6, 16, 8, F32)
    for bad in (lambda: seq.gated_linear(x.double(), wg, wu), lambda: seq.gated_linear(x.half(), wg.half(), wu.half()),
                lambda: seq.gated_linear(x, wg.to(BF16), wu), lambda: seq.gated_linear(x, wg, wu.to(BF16)),
                lambda: seq.gated_linear(x, wg[:, :8], wu), lambda: seq.gated_linear(x, wg, wu[:4]),
                lambda: seq.gated_linear(x, wg[0], wu[0]), lambda: seq.gated_linear(x, wg.cpu(), wu),
                lambda: seq.gated_linear(x[:, :0], wg[:, :0], wu[:, :0]), lambda: seq.gated_linear(x, wg[:0], wu[:0]),
                lambda: seq.gated_linear(x[0, 0], wg, wu), lambda: seq.gated_linear(x, wg, wu, activation="relu"),
                lambda: torch.jit.trace(seq.gated_linear, (x, wg, wu), check_trace=False)):
        with pytest.raises(RuntimeError, match="Astra Fatal Error"):
            bad()
    for i in range(3):
        with fwd.dual_level():
            duals = [x, wg, wu]
            duals[i] = fwd.make_dual(duals[i].clone(), torch.ones_like(duals[i]))
            with pytest.raises(RuntimeError, match="Astra Fatal Error.*forward-mode"):
                seq.gated_linear(*duals)
    x.requires_grad_()
    h = seq.gated_linear(x, wg, wu)
    with pytest.raises(RuntimeError, match="Astra Fatal Error.*once"):
        torch.autograd.grad(h, x, dh, create_graph=True)
