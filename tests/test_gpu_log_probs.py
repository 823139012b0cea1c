"""log_probs and its gradient against the definition in 64 bits: parts from one entry to many, masks that
leave nothing, choices that do not count or do not exist, values at the ends of their types, ties, rows
that lie anywhere, and the modes a call can be made in."""
import math

import pytest
import torch

from probs_util import BF16, DEV, F32, check, part, within

pytestmark = pytest.mark.gpu


def make(seed, R, sizes, dtype, scale=2.0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    W = sum(sizes)
    logits = (scale * torch.randn(R, W, generator=g, device=DEV)).to(dtype)
    choice = torch.stack([torch.randint(0, n, (R,), generator=g, device=DEV) for n in sizes], 1)
    mask = torch.rand(R, W, generator=g, device=DEV) < 0.6
    return logits, choice, mask


SIZES = [[1], [2], [7], [8], [9], [31], [64], [65], [127, 127, 6, 6], [10, 10, 3, 3], [300], [511], [512], [513],
         [1023], [1024], [1025], [2048], [2049, 5], [5, 4097, 1, 600], [1, 1, 1], [16] * 16, [8191], [8192], [50_003]]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "-".join(map(str, s[:4])))
def test_values_gradients_and_top(sizes, dtype):
    from astra_cuda import sequence as seq
    print("log_probs", sizes[:4], dtype, flush=True)
    for R in (1, 3, 130):
        logits, choice, mask = make(R, R, sizes, dtype)
        top = min(min(sizes), 7)
        for m in (None, mask, mask[:1]):
            for t in (0, top):
                check(seq, logits, choice, sizes, m, t, R)
        check(seq, logits, choice.to(torch.int32), sizes, mask, top, R)
        check(seq, logits, None, sizes, mask, top, R)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("R,sizes", [(600, [1500]), (2000, [3001, 9]), (20_000, [127, 127, 6, 6]), (70_001, [5]), (513, [20_000]),
                                      (8192, [1000, 513]), (8195, [2048, 600]), (9000, [1025]), (8193, [1500, 2049])],
                         ids=str)
def test_many_rows(R, sizes, dtype):
    from astra_cuda import sequence as seq
    logits, choice, mask = make(R, R, sizes, dtype)
    choice[torch.rand(R, device=DEV) < 0.2] = -1
    for m in (None, mask):
        out, d = check(seq, logits, choice, sizes, m, min(min(sizes), 5), 1)
    again, d2 = check(seq, logits, choice, sizes, mask, min(min(sizes), 5), 1)
    assert torch.equal(d.nan_to_num(3.0), d2.nan_to_num(3.0)) and all(torch.equal(a, b) for a, b in zip(out, again))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("top", [1, 4, 5, 33, 64])
@pytest.mark.parametrize("n", [256, 257, 511, 700, 1024, 1025, 2000])
def test_top_of_many_rows(n, top, dtype):
    """Rows with many ties, few or no allowed entries, and choices that do not count among them."""
    from astra_cuda import sequence as seq
    R = 8200
    logits, choice, mask = make(n + top, R, [n], dtype)
    logits[::3] = logits[::3].round()
    logits[5], mask[6], mask[7, 3:], choice[8] = 0.0, False, False, -1
    check(seq, logits, choice, [n], mask, top, 9)
    logits, choice, mask = make(n + top, R, [n, 300], dtype)
    check(seq, logits, choice, [n, 300], None, top, 10)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("top", [1, 2, 20, 63, 64])
@pytest.mark.parametrize("n", [64, 100, 513, 1024, 1025, 30_000, 131_072])
def test_top_with_ties_and_orders(n, top, dtype):
    """Random with many ties, rising, falling, all alike, and fewer allowed than asked for."""
    from astra_cuda import sequence as seq
    g = torch.Generator(device=DEV)
    g.manual_seed(n + top)
    rise = torch.linspace(-10, 10, n, device=DEV)
    rows = [torch.randn(n, generator=g, device=DEV), torch.randint(-3, 4, (n,), generator=g, device=DEV).float(), rise,
            -rise, torch.zeros(n, device=DEV), torch.where(torch.arange(n, device=DEV) % 2 == 0, 0.0, -0.0)]
    few = torch.full((n,), -math.inf, device=DEV)
    few[torch.randperm(n, generator=g, device=DEV)[:5]] = torch.tensor([1.0, 1.0, 3.0, -2.0, 0.5], device=DEV)
    logits = torch.stack(rows + [few]).to(dtype)
    choice = torch.zeros(len(logits), 1, dtype=torch.int64, device=DEV)
    check(seq, logits, choice, [n], None, top, 2)
    check(seq, logits, choice, [n], torch.rand(logits.shape, generator=g, device=DEV) < 0.5, top, 2)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("n", [6, 127, 700, 3000])
def test_rows_with_nothing_allowed_and_choices_that_do_not_count(n, dtype):
    from astra_cuda import sequence as seq
    logits, choice, mask = make(n, 40, [n, 5], dtype)
    mask[3], mask[7, :n], mask[9, n:] = False, False, False
    logits[11], logits[12, :n] = -math.inf, -math.inf
    choice[20], choice[21, 0], choice[22, 1] = -1, -1, -1
    logits[20], logits[21, :n] = math.nan, math.nan     # not read
    logits[22, n:] = math.inf
    choice[25, 0], choice[26, 1], choice[27, 0] = n, -2, -(2 ** 33)
    choice[28, 1] = 2 ** 32 + 1
    for top in (0, 3):
        out, d = check(seq, logits, choice, [n, 5], mask, top, 3)
        out = [v.detach() for v in out]
        assert not bool(d[3].any()) and not bool(d[20].any()) and not bool(d[11].any())
        assert float(out[1][3, 0]) == 0 and float(out[0][20, 0]) == 0 and float(out[0][3, 1]) == -math.inf
        assert bool(torch.isnan(out[0][25, 0])) and bool(torch.isnan(out[0][28, 1])) and bool(torch.isnan(out[0][27, 0]))
        if top:
            assert bool((out[3][3] == -1).all()) and bool((out[3][20] == -1).all())


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("n", [6, 127, 700, 3000])
def test_values_at_the_ends_of_their_type(n, dtype):
    """Masks by the lowest value, all entries at it, and the largest beside the lowest."""
    from astra_cuda import sequence as seq
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    logits, choice, mask = make(n, 12, [n], dtype)
    logits[0, 1:], logits[1], logits[2], logits[3, :3] = low, low, high, high
    logits[3, 3:] = low
    logits[4, : n // 2], logits[5, -1] = low, high
    logits[6] = 1e30
    choice[:] = 0
    check(seq, logits, choice, [n], None, min(n, 4), 4)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("n", [6, 127, 700, 3000])
def test_values_that_are_not_finite(n, dtype):
    """They make their own row and part NaN where they are allowed, and nothing where they are not."""
    from astra_cuda import sequence as seq
    logits, choice, mask = make(n, 30, [n, n], dtype)
    mask[:] = True
    good, gd = check(seq, logits, choice, [n, n], mask, 3, 5)
    logits[4, 2], logits[5, n + 1], logits[6, n - 1] = math.nan, math.inf, math.inf
    logits[7], logits[8, :n] = math.nan, math.inf
    mask[10, 1], mask[11, n + 2], mask[12, 0] = False, False, False
    good2, gd2 = check(seq, logits.nan_to_num(0.0, 0.0), choice, [n, n], mask, 3, 5)
    logits[10, 1], logits[11, n + 2], logits[12, 0] = math.nan, math.inf, -math.inf
    x = logits.detach().requires_grad_()
    out = seq.log_probs(x, choice, sizes=[n, n], mask=mask, top=3)
    g = torch.Generator(device=DEV)
    g.manual_seed(5)
    dl, dh = (torch.randn(30, 2, generator=g, device=DEV) for _ in range(2))
    d, = torch.autograd.grad(out[:2], x, [dl, dh])
    bad = torch.zeros(30, 2, dtype=torch.bool, device=DEV)
    bad[4, 0], bad[5, 1], bad[6, 0], bad[7], bad[8, 0] = True, True, True, True, True
    for v, w in zip(out[:2], good2[:2]):
        assert torch.equal(torch.isnan(v), bad) and torch.equal(v[~bad], w[~bad])
    assert torch.equal(out[3][~bad], good2[3][~bad])
    wide = bad.repeat_interleave(n, 1)
    assert torch.equal(torch.isnan(d), wide) and torch.equal(d[~wide], gd2[~wide])
    clean = torch.ones(30, dtype=torch.bool, device=DEV)
    clean[[4, 5, 6, 7, 8, 10, 11, 12]] = False
    assert torch.equal(d[clean], gd[clean]) and torch.equal(out[0][clean], good[0][clean])


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("sizes", [[13], [127, 6], [600], [1301], [5000, 3]], ids=str)
def test_rows_inside_larger_memory(sizes, dtype):
    """Any alignment of a row; what lies between rows is NaN, and not used."""
    from astra_cuda import sequence as seq
    R, W = 21, sum(sizes)
    logits, choice, mask = make(8, R, sizes, dtype)
    for shift, pad in ((0, 3), (1, 0), (5, 8), (8, 0)):
        big = torch.full((R + 2, shift + W + pad), math.nan, device=DEV, dtype=dtype)
        big[1:-1, shift:shift + W] = logits
        allowed = torch.ones(R + 2, shift + W + pad, dtype=torch.bool, device=DEV)
        allowed[1:-1, shift:shift + W] = mask
        check(seq, big[1:-1, shift:shift + W], choice, sizes, allowed[1:-1, shift:shift + W], 2, 6)


def test_shapes_and_views():
    from astra_cuda import sequence as seq
    logits, choice, mask = make(9, 24, [10, 6], F32)
    want = seq.log_probs(logits, choice, sizes=[10, 6], mask=mask, top=2)
    got = seq.log_probs(logits.view(2, 3, 4, 16), choice.view(2, 3, 4, 2), sizes=(10, 6), mask=mask.view(2, 3, 4, 16), top=2)
    assert [v.shape for v in got] == [(2, 3, 4, 2), (2, 3, 4, 2), (2, 3, 4, 2, 2), (2, 3, 4, 2, 2)]
    assert all(torch.equal(a.reshape(b.shape), b) for a, b in zip(got, want))
    t = logits.t().contiguous().requires_grad_()
    lp, h = seq.log_probs(t.t(), choice, sizes=[10, 6], mask=mask)
    assert torch.equal(lp, want[0]) and torch.equal(h, want[1])
    d, = torch.autograd.grad(lp.sum() + h.sum(), t)
    x = logits.clone().requires_grad_()
    lp, h = seq.log_probs(x, choice, sizes=[10, 6], mask=mask)
    d2, = torch.autograd.grad(lp.sum() + h.sum(), x)
    assert torch.equal(d.t(), d2)
    # every other choice of a wider tensor, a mask of one row, a broadcast row of logits
    wide = torch.stack([choice, choice + 100], -1)[..., 0]
    assert torch.equal(seq.log_probs(logits, wide, sizes=[10, 6], mask=mask)[0], want[0])
    one = seq.log_probs(logits, choice, sizes=[10, 6], mask=mask[0])
    assert torch.equal(one[0], seq.log_probs(logits, choice, sizes=[10, 6], mask=mask[:1].expand(24, 16).contiguous())[0])
    row = logits[:1].clone().requires_grad_()
    lp, h = seq.log_probs(row.expand(24, 16), choice, sizes=[10, 6])
    d, = torch.autograd.grad(lp.sum(), row)
    assert d.shape == (1, 16) and bool(torch.isfinite(d).all())
    lp, h = seq.log_probs(logits[0], choice[0, 0])
    assert lp.shape == () and h.shape == ()
    lp, h = seq.log_probs(logits[:0], choice[:0], sizes=[10, 6])
    assert lp.shape == (0, 2)
    none, h, tl, ti = seq.log_probs(logits, top=1)
    assert none is None and h.shape == (24,) and tl.shape == (24, 1) and torch.equal(ti[:, 0], logits.argmax(1))


def test_one_output_s_gradient_alone():
    from astra_cuda import sequence as seq
    for n in (9, 2000):
        logits, choice, _ = make(10, 50, [n], BF16)
        x = logits.requires_grad_()
        zero = torch.zeros(50, device=DEV)
        g = torch.randn(50, device=DEV)
        for i in range(2):
            out = seq.log_probs(x, choice[:, 0], top=2)
            d, = torch.autograd.grad(out[i], x, g, retain_graph=True)
            both = [zero, zero]
            both[i] = g
            e, = torch.autograd.grad(out[:2], x, both)
            assert torch.equal(d, e)
        assert out[2].requires_grad is False and out[3].requires_grad is False


def test_gradients_against_differences():
    """Of sum(dl log_prob + dh entropy) along random directions of unit root mean square, in float32:
    steps of 1e-2 leave a third derivative's 1e-4 and roundings of 2^-24 x 10 / 1e-2 a row."""
    from astra_cuda import sequence as seq
    for sizes in ([127, 127, 6, 6], [2500]):
        logits, choice, mask = make(11, 64, sizes, F32)
        mask.scatter_(1, choice[:, :1], True)
        given = sizes if len(sizes) > 1 else None
        c = choice if given else choice[:, 0]
        dl, dh = torch.randn(c.shape, device=DEV).double(), torch.randn(c.shape, device=DEV).double()
        # (choices that are left out have no gradient, and a log probability of -inf)
        def total(x):
            lp, h = seq.log_probs(x, c, sizes=given, mask=mask)
            return (torch.where(torch.isinf(lp), 0.0, lp.double()) * dl + h.double() * dh).sum()
        x = logits.clone().requires_grad_()
        d, = torch.autograd.grad(total(x), x)
        for _ in range(3):
            v = torch.randn_like(logits)
            slope = (total(logits + 1e-2 * v) - total(logits - 1e-2 * v)) / 2e-2
            scale = float(dl.abs().sum() + dh.abs().sum())
            assert abs(float(slope) - float((d.double() * v).sum())) <= 1e-3 * scale


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("sizes", [[10, 10, 3, 3], [1000], [9001]], ids=str)
def test_forward_and_backward_replay(sizes, dtype):
    from astra_cuda import sequence as seq
    print("graph", sizes, dtype, flush=True)
    sets = [make(30 + i, 50, sizes, dtype) for i in range(3)]
    dl, dh = torch.randn(50, len(sizes), device=DEV), torch.randn(50, len(sizes), device=DEV)
    logits, choice, mask = (v.clone() for v in sets[0])
    def once(x, c, m):
        out = seq.log_probs(x, c, sizes=sizes, mask=m, top=2)
        return (*out, *torch.autograd.grad(out[:2], x, [dl, dh]))
    want = [[v.detach() for v in once(s[0].clone().requires_grad_(), s[1], s[2])] for s in sets]
    logits.requires_grad_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = once(logits, choice, mask)
    for i in (0, 1, 2, 1, 0):
        with torch.no_grad():
            for a, b in zip((logits, choice, mask), sets[i]):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a.detach(), b) for a, b in zip(got, want[i])), i
        s = sets[(i + 1) % 3]
        again = once(s[0].clone().requires_grad_(), s[1], s[2])
        assert all(torch.equal(a.detach(), b) for a, b in zip(again, want[(i + 1) % 3]))


def test_many_entries():
    """More than 2^31 bytes of logits, and a single row of many entries."""
    from astra_cuda import sequence as seq
    R, n = 9000, 130_001
    g = torch.Generator(device=DEV)
    g.manual_seed(12)
    logits = torch.randn(R, n, generator=g, device=DEV, dtype=BF16)
    choice = torch.randint(0, n, (R,), generator=g, device=DEV)
    x = logits.requires_grad_()
    out = seq.log_probs(x, choice, top=2)
    dl, dh = torch.randn(R, device=DEV), torch.randn(R, device=DEV)
    d, = torch.autograd.grad(out[:2], x, [dl, dh])
    at = torch.tensor([0, 1, 8258, 8259, 8260, R - 2, R - 1], device=DEV)
    want = part(logits.detach()[at], None, choice[at], 2, dl[at], dh[at], BF16)
    within(out[0][at], want["log_prob"], "log_prob")
    within(out[1][at], want["entropy"], "entropy")
    within(d[at], want["dlogits"], "dlogits")
    assert torch.equal(out[3][at], want["top_index"])
    del x, logits, d
    big = torch.randn(1, 30_000_001, generator=g, device=DEV)
    check(seq, big, torch.tensor([[29_999_999]], device=DEV), [30_000_001], None, 3, 7)


def test_many_rows_of_larger_parts():
    """More workgroups than one launch may have: a row of logits, or of pieces of one, for each. (One row
    of memory serves all.)"""
    from astra_cuda import sequence as seq
    logits, choice, _ = make(14, 1, [1025], BF16)
    R = 2 ** 24 + 5
    want = part(logits, None, choice[:, 0], 0, None, None, BF16)
    got = seq.log_probs(logits.expand(R, 1025), choice[:, 0].expand(R))
    for v, k in zip(got, ("log_prob", "entropy")):
        assert bool((v == v[0]).all())
        within(v[:1], want[k], k)
    logits, choice, _ = make(15, 1, [9000], BF16)
    R = 2 ** 22 + 5
    want = part(logits, None, choice[:, 0], 1, None, None, BF16)
    got = seq.log_probs(logits.expand(R, 9000), choice[:, 0].expand(R), top=1)
    for v, k in zip(got, ("log_prob", "entropy", "top_log_prob")):
        assert bool((v == v[0]).all())
        within(v[:1], want[k], k)
    assert bool((got[3] == want["top_index"]).all())


def test_gradient_of_many_rows_of_larger_parts():
    from astra_cuda import sequence as seq
    logits, choice, _ = make(16, 1, [1025], BF16)
    R = 2 ** 24 + 5
    x = logits.expand(R, 1025).detach().requires_grad_()
    lp, h = seq.log_probs(x, choice[:, 0].expand(R))
    d, = torch.autograd.grad([lp, h], x, [torch.ones_like(lp), torch.ones_like(h)])
    one = part(logits, None, choice[:, 0], 0, torch.ones(1, device=DEV), torch.ones(1, device=DEV), BF16)
    within(d[:1], one["dlogits"], "dlogits")
    assert all(bool((d[i:i + 2 ** 20] == d[0]).all()) for i in range(0, R, 2 ** 20))


def test_refusals():
    from astra_cuda import sequence as seq
    import torch.autograd.forward_ad as fwd
    logits, choice, mask = make(13, 6, [10, 6], F32)
    for bad in (lambda: seq.log_probs(logits.double(), choice, sizes=[10, 6]), lambda: seq.log_probs(logits.cpu(), choice, sizes=[10, 6]),
                lambda: seq.log_probs(logits, choice, sizes=[10, 5]), lambda: seq.log_probs(logits, choice, sizes=[16, 0]),
                lambda: seq.log_probs(logits, choice, sizes=[10, 7]), lambda: seq.log_probs(logits, choice, sizes=[]),
                lambda: seq.log_probs(logits, choice, sizes=[1] * 17), lambda: seq.log_probs(logits, choice, sizes=[26, -10]),
                lambda: seq.log_probs(logits, choice), lambda: seq.log_probs(logits, choice[:, 0], sizes=[10, 6]),
                lambda: seq.log_probs(logits, choice.float(), sizes=[10, 6]), lambda: seq.log_probs(logits, choice.cpu(), sizes=[10, 6]),
                lambda: seq.log_probs(logits, choice, sizes=[10, 6], mask=mask.float()),
                lambda: seq.log_probs(logits, choice, sizes=[10, 6], mask=mask[:, :10]),
                lambda: seq.log_probs(logits, choice, sizes=[10, 6], mask=mask[:5]),
                lambda: seq.log_probs(logits, choice, sizes=[10, 6], mask=mask[None]),
                lambda: seq.log_probs(logits, choice, sizes=[10, 6], mask=mask.cpu()),
                lambda: seq.log_probs(logits, choice, sizes=[10, 6], top=7), lambda: seq.log_probs(logits, choice, sizes=[10, 6], top=-1),
                lambda: seq.log_probs(logits.repeat(1, 10), choice[:, 0], top=65), lambda: seq.log_probs(logits[:, :0]),
                lambda: seq.log_probs(logits[0, 0]),
                lambda: torch.jit.trace(lambda x: seq.log_probs(x, choice[:, 0]), (logits,), check_trace=False)):
        with pytest.raises(RuntimeError, match="Astra Fatal Error"):
            bad()
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match="Astra Fatal Error.*forward-mode"):
            seq.log_probs(fwd.make_dual(logits.clone(), torch.ones_like(logits)), choice[:, 0])
    x = logits.requires_grad_()
    with pytest.raises(RuntimeError, match="Astra Fatal Error.*once"):
        torch.autograd.grad(seq.log_probs(x, choice[:, 0])[1].sum(), x, create_graph=True)
