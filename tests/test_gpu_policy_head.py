"""The feed-forward block and the head of a policy as they are used together: norm, gated_linear,
projection, join_norm, head, log_probs, and the gradients of a policy's loss back to every weight."""
import math

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SIZES = [30, 30, 6, 6]


def weights(seed, D=96, hidden=200):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    def normal(*s):
        return torch.randn(*s, generator=g, device=DEV)
    w = {"r": normal(40, 12, D), "first": 1 + 0.1 * normal(D), "gate": normal(hidden, D) / math.sqrt(D),
         "up": normal(hidden, D) / math.sqrt(D), "out": normal(D, hidden) / math.sqrt(hidden), "post": 1 + 0.1 * normal(D),
         "next": 1 + 0.1 * normal(D), "scale": 0.5 + 0.1 * normal(D), "head": normal(sum(SIZES), D) / math.sqrt(D)}
    choice = torch.stack([torch.randint(0, n, (40, 12), generator=g, device=DEV) for n in SIZES], -1)
    allowed = torch.rand(40, 12, sum(SIZES), generator=g, device=DEV) < 0.7
    at = torch.tensor([0, 30, 60, 66], device=DEV)
    allowed.scatter_(-1, choice + at, True)  # what was chosen was allowed
    lengths = torch.randint(1, 13, (40,), generator=g, device=DEV)
    choice[torch.arange(12, device=DEV)[None] >= lengths[:, None]] = -1  # games that are over
    return w, choice, allowed, normal(40, 12)


def own(w, choice, allowed, advantage):
    from astra_cuda import sequence as seq
    n = seq.rms_norm(w["r"], w["first"])
    u = F.linear(seq.gated_linear(n, w["gate"], w["up"]), w["out"])
    r, n = seq.join_norm(w["r"], u, w["post"], w["next"], scale=w["scale"])
    log_prob, entropy = seq.log_probs(F.linear(n, w["head"]), choice, sizes=SIZES, mask=allowed)
    return -(advantage * log_prob.sum(-1) + 0.01 * entropy.sum(-1)).sum() / 100 + r.square().sum() / 1000


def plain(w, choice, allowed, advantage):
    """The same in 64 bits, from torch's operations."""
    def rms(v):
        return v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-6)
    n = rms(w["r"]) * w["first"]
    u = (F.silu(n @ w["gate"].t()) * (n @ w["up"].t())) @ w["out"].t()
    r = w["r"] + w["scale"] * rms(u) * w["post"]
    logits = (rms(r) * w["next"]) @ w["head"].t()
    total = r.square().sum() / 1000
    for i, (x, m) in enumerate(zip(logits.split(SIZES, -1), allowed.split(SIZES, -1))):
        l = torch.log_softmax(x.masked_fill(~m, -math.inf), -1)
        l = torch.where(m, l, 0.0)
        c = choice[..., i]
        on = c != -1
        chosen = torch.gather(l, -1, c.clamp(min=0)[..., None])[..., 0]
        h = -(torch.where(m, l.exp(), 0.0) * l).sum(-1)
        total = total - torch.where(on, advantage * chosen + 0.01 * h, 0.0).sum() / 100
    return total


def test_loss_and_gradients():
    """Float32 throughout. Sums of up to 200 products are off by at most 200 x 2^-24 = 1.2e-5 of the sum
    of their magnitudes, there are five products one behind the other, and norms and softmax pass
    relative errors on: 1e-3 of a gradient's norm is far above what they add up to."""
    w, choice, allowed, advantage = weights(1)
    leaves = {k: v.clone().requires_grad_() for k, v in w.items()}
    wide = {k: v.double().requires_grad_() for k, v in w.items()}
    got, want = own(leaves, choice, allowed, advantage), plain(wide, choice, allowed, advantage.double())
    assert abs(float(got.detach()) - float(want.detach())) <= 1e-4 * abs(float(want.detach()))
    for (k, a), b in zip(zip(leaves, torch.autograd.grad(got, list(leaves.values()))),
                         torch.autograd.grad(want, list(wide.values()))):
        assert bool(torch.isfinite(a).all()), k
        assert float((a.double() - b).norm()) <= 1e-3 * float(b.norm()), k


def test_a_captured_update():
    """The loss and its gradients as one graph, replayed on other inputs between eager ones."""
    sets = [weights(s) for s in (2, 3, 4)]
    def grads(w, *rest):
        leaves = {k: v.requires_grad_() for k, v in w.items()}
        loss = own(leaves, *rest)
        return [loss.detach(), *torch.autograd.grad(loss, list(leaves.values()))]
    want = [grads({k: v.clone() for k, v in s[0].items()}, *s[1:]) for s in sets]
    held = {k: v.clone() for k, v in sets[0][0].items()}
    rest = [v.clone() for v in sets[0][1:]]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = grads(held, *rest)
    for i in (0, 1, 2, 1, 0):
        with torch.no_grad():
            for k in held:
                held[k].copy_(sets[i][0][k])
            for a, b in zip(rest, sets[i][1:]):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        # (the loss ends in torch's own sums and products, which may run otherwise when captured)
        for a, b in zip(got, want[i]):
            assert float((a - b).norm()) <= 1e-5 * float(b.norm())
        again = grads({k: v.clone() for k, v in sets[(i + 1) % 3][0].items()}, *sets[(i + 1) % 3][1:])
        assert all(float((a - b).norm()) <= 1e-5 * float(b.norm()) for a, b in zip(again, want[(i + 1) % 3]))


def test_a_move_and_whole_games_agree():
    """A few rows and many go through different kernels: the same to the products' roundings."""
    from astra_cuda import sequence as seq
    w, choice, allowed, _ = weights(5)
    n = seq.rms_norm(w["r"], w["first"])
    whole = seq.gated_linear(n, w["gate"], w["up"])
    by_move = torch.stack([seq.gated_linear(n[:, t], w["gate"], w["up"]) for t in range(12)], 1)
    size = n.double().abs() @ w["gate"].double().abs().t() + n.double().abs() @ w["up"].double().abs().t()
    top = (1 + (n @ w["gate"].t()).abs() + (n @ w["up"].t()).abs()).double()
    assert bool(((whole - by_move).double().abs() <= 2 * 98 * 2.0 ** -24 * 1.13 * size * top).all())
    logits = F.linear(whole @ w["out"].t(), w["head"])
    lp, h = seq.log_probs(logits, choice, sizes=SIZES, mask=allowed)
    parts = [seq.log_probs(logits[:, t], choice[:, t], sizes=SIZES, mask=allowed[:, t]) for t in range(12)]
    assert torch.equal(lp, torch.stack([p[0] for p in parts], 1)) and torch.equal(h, torch.stack([p[1] for p in parts], 1))


def test_two_streams_and_two_graphs_at_once():
    """Calls that use a workspace (copies, slices, pieces) side by side, eager and replayed, share none."""
    from astra_cuda import sequence as seq
    g = torch.Generator(device=DEV)
    g.manual_seed(6)
    def make():
        x = torch.randn(300, 1003, generator=g, device=DEV).bfloat16().requires_grad_()
        w = [(torch.randn(210, 1003, generator=g, device=DEV) / 30).bfloat16().requires_grad_() for _ in range(2)]
        logits = torch.randn(5, 90_001, generator=g, device=DEV).requires_grad_()
        choice = torch.randint(0, 90_001, (5,), generator=g, device=DEV)
        return x, w, logits, choice, torch.randn(300, 210, generator=g, device=DEV).bfloat16(), torch.randn(5, generator=g, device=DEV)
    def run(x, w, logits, choice, dh, dl):
        h = seq.gated_linear(x, *w, activation="gelu")
        lp, e, tl, ti = seq.log_probs(logits, choice, top=9)
        return [h.detach(), lp.detach(), e.detach(), tl, ti, *torch.autograd.grad(h, (x, *w), dh), *torch.autograd.grad([lp, e], logits, [dl, dl])]
    sets = [make(), make()]
    want = [run(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        got = []
        for s, stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                got.append(run(*s))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))
    graphs, outs = [], []
    for s in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(run(*s))
    for _ in range(5):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(outs, want) for a, b in zip(x, y))
