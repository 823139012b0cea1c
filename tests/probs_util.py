"""Shared by the tests of log_probs: the definition in 64 bits, and bounds on how far off a result may be.

e = 2^-24 is one float32 rounding, u half a step of the logits' type. A part of n entries is summed by
at least 64 lanes where n is over 512, and by chains of at most 16 below, then over lanes and
wavefronts: Z is off by at most z = (n / 64 + 64 + 2 mean |x - m|) e of itself, each of its terms
by 2 |x - m| + 4 roundings. Everything else is a few roundings of the numbers it adds.
"""
import math

import torch

DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16
E = 2.0 ** -24


def part(x, mask, choice, top, dl, dh, dtype):
    """One part, [R, n] logits: {name: (value, bound)}; `choice` may be None, dl and dh [R]."""
    u = torch.finfo(dtype).eps / 2
    x = x.detach().double()
    R, n = x.shape
    live = x != -math.inf
    if mask is not None:
        live = live & mask
    counts = torch.ones(R, dtype=torch.bool, device=x.device) if choice is None else choice != -1
    live = live & counts[:, None]
    some = live.any(1)
    m = torch.where(live, x, -math.inf).amax(1)
    m = torch.where(some, m, 0.0)[:, None]
    d = torch.where(live, x - m, 0.0)
    t = torch.where(live, torch.exp(d), 0.0)
    Z = torch.where(some, t.sum(1), 1.0)[:, None]
    p, logz = t / Z, torch.log(Z)
    spread = (p * d.abs()).sum(1, keepdim=True)
    H = logz + spread
    l = torch.where(live, d - logz, -math.inf)
    zrel = (n / 64 + 64 + 2 * spread) * E
    el = zrel + 4 * E * (d.abs() + logz + 1)
    eH = zrel + spread * (3 * zrel + 4 * E) + 4 * E * (H + 1) + (p * d.abs() * (2 * d.abs() + 4)).sum(1, keepdim=True) * E
    out = {"entropy": (torch.where(some, H[:, 0], 0.0), eH[:, 0])}
    g = torch.zeros_like(x)
    size = torch.zeros_like(x)
    fl = torch.where(live, l, 0.0)
    ep = p * (el + 4 * E * (fl.abs() + 1))
    if dh is not None:
        g = g - dh.double()[:, None] * p * (fl + H)
        size = size + dh.double().abs()[:, None] * (ep * (fl + H).abs() + p * (el + eH + 4 * E * (fl.abs() + H)))
    if choice is not None:
        inside = (choice >= 0) & (choice < n)
        at = choice.clamp(0, n - 1).long()[:, None]
        lc = torch.gather(l, 1, at)[:, 0]
        value = torch.where(counts, torch.where(inside, lc, math.nan), 0.0)
        out["log_prob"] = (value, torch.gather(el, 1, at)[:, 0])
        if dl is not None:
            hot = torch.zeros_like(p).scatter_(1, at, 1.0)
            s = torch.where(torch.isinf(lc), 0.0, dl.double())
            s = torch.where(inside, s, math.nan)[:, None]
            g = g + torch.where(live, s * (hot - p), 0.0)
            size = size + dl.double().abs()[:, None] * (ep + 2 * E)
    g = torch.where(live, g, 0.0)
    out["dlogits"] = (g, (size + 8 * E * g.abs()) * (1 + u) + u * g.abs())
    if top:
        order = torch.sort(torch.where(live & ~torch.isnan(x), x, -math.inf), dim=1, descending=True, stable=True)
        index = torch.where(order.values[:, :top] > -math.inf, order.indices[:, :top], -1)
        at = index.clamp(min=0)
        out["top_index"] = index
        out["top_log_prob"] = (torch.where(index >= 0, torch.gather(l, 1, at), -math.inf), torch.gather(el, 1, at))
    return out


def within(got, want, what):
    value, bound = want
    got = got.detach().double()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(value)), what
    # -3.4e38 - 3.4e38 is below every float32, and is -inf when rounded to one
    value = torch.where(value.abs() > 2.0 ** 128, value.sign() * math.inf, value)
    odd = torch.isinf(value)
    assert torch.equal(got[odd], value[odd]) and not bool(torch.isinf(got[~odd]).any()), what
    fine = torch.isfinite(value)
    off = (got[fine] - value[fine]).abs() - 1.001 * bound[fine] - 1e-37
    assert not bool((off > 0).any()), (what, float(off.max()))


def check(seq, logits, choice, sizes, mask=None, top=0, seed=0, whole=None):
    """A call with gradients against the definition, part by part. `whole`: sizes as the call has them."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    R, P = logits.shape[0], len(sizes)
    x = logits.detach().requires_grad_()
    given = list(sizes) if P > 1 or whole else None
    def of_call(v):
        return v if given is not None or v is None else v[:, 0]
    with torch.no_grad():
        plain = seq.log_probs(logits, of_call(choice), sizes=given, mask=mask, top=top)
    out = seq.log_probs(x, of_call(choice), sizes=given, mask=mask, top=top)
    for a, b in zip(plain, out):
        assert (a is None and b is None) or torch.equal(a.nan_to_num(7.0), b.detach().nan_to_num(7.0))
    dl, dh = (torch.randn(R, P, generator=g, device=DEV) for _ in range(2))
    leaves = [out[1]] if choice is None else [out[0], out[1]]
    d, = torch.autograd.grad(leaves, x, [of_call(dh)] if choice is None else [of_call(dl), of_call(dh)])
    assert d.shape == x.shape and d.dtype == x.dtype
    begin = 0
    for i, n in enumerate(sizes):
        m = None if mask is None else mask.expand(R, -1)[:, begin:begin + n]
        c = None if choice is None else choice[:, i]
        want = part(logits[:, begin:begin + n], m, c, top, dl[:, i], dh[:, i], logits.dtype)
        pick = (lambda v: v[:, i]) if given is not None else (lambda v: v)
        if choice is not None:
            within(pick(out[0]), want["log_prob"], ("log_prob", i))
        within(pick(out[1]), want["entropy"], ("entropy", i))
        within(d[:, begin:begin + n], want["dlogits"], ("dlogits", i))
        if top:
            assert torch.equal(pick(out[3]), want["top_index"]), ("top_index", i)
            within(pick(out[2]), want["top_log_prob"], ("top_log_prob", i))
        begin += n
    return out, d
