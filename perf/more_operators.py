"""What is measured of a policy's feed-forward block and of its head, through the public calls of
``astra_cuda.sequence``.

``gated_linear`` is the gated feed-forward block before its way back: both projections of a
block's normed input, the activation of one and its product with the other. ``log_probs`` is
what a head's logits are asked for: the log probability of each part of the move that was made,
the entropy of what could have been made, and the likeliest alternatives. Each is measured as a
rollout calls it, a few rows at a time, and as an update does, over whole games with gradients.

Where ``own`` is false, the operators are computed from elementary torch operations in 32 bits.
"""
import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if os.path.join(ROOT, "astra-cuda_amd") not in sys.path:
    sys.path.insert(0, os.path.join(ROOT, "astra-cuda_amd"))

own = False

TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # One env, one move: a policy that plays by hand. Nothing but latency.
        dict(name="gated_step_1", kind="gated", dtype="bf16", rows=1, width=256, hidden=1024, activation="silu"),
        # A move of 64 envs by a wide policy: the weights are read for few rows.
        dict(name="gated_step_wide", kind="gated", dtype="bf16", rows=64, width=4096, hidden=8192, activation="silu"),
        # Training on whole games: 2,048 envs with 40 moves.
        dict(name="gated_game_train", kind="gated_train", dtype="bf16", rows=81_920, width=256, hidden=1024,
             activation="silu"),
        # The same in 32 bits: 300 games of 100 moves, a hidden width of 8/3 that is no multiple of anything.
        dict(name="gated_game_train_f32", kind="gated_train", dtype="f32", rows=30_000, width=256, hidden=683,
             activation="gelu"),
        # Training a wide policy on records.
        dict(name="gated_wide_train", kind="gated_train", dtype="bf16", rows=16_384, width=4096, hidden=8192,
             activation="silu"),
        # A record read before play goes on, at odd sizes, forward alone.
        dict(name="gated_prompt_odd", kind="gated", dtype="bf16", rows=4097, width=1000, hidden=2731,
             activation="gelu"),
        # The example policy's head for a move of 64 envs: two prices of 10 and two sizes of 3.
        dict(name="log_move_64", kind="log_probs", dtype="f32", rows=64, sizes="10,10,3,3", mask="none", ragged=False,
             top=0),
        # Training on whole games with the game's 127 prices and sizes of 0 to 5, illegal moves masked, and games
        # that end at different moves.
        dict(name="log_game_train", kind="log_probs_train", dtype="bf16", rows=81_920, sizes="127,127,6,6",
             mask="given", ragged=True, top=0),
        # Training on records written in tokens.
        dict(name="log_tokens_train", kind="log_probs_train", dtype="bf16", rows=8192, sizes="50000", mask="none",
             ragged=False, top=0),
        # The same in 32 bits, with an odd number of tokens, some of them ruled out by logits of -inf.
        dict(name="log_tokens_train_f32", kind="log_probs_train", dtype="f32", rows=2000, sizes="32003", mask="inf",
             ragged=True, top=0),
        # One token for each of 64 envs, with the alternatives that a log keeps.
        dict(name="log_tokens_top", kind="log_probs", dtype="bf16", rows=64, sizes="131072", mask="none", ragged=False,
             top=20),
        # One token of one env: few rows, so the length has to be split.
        dict(name="log_token_one", kind="log_probs", dtype="f32", rows=1, sizes="65537", mask="none", ragged=False,
             top=5),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _sizes(case):
    return [int(n) for n in case["sizes"].split(",")]


def draw(rng):
    """One more case of the ranges that the listed ones stand for."""
    kind = rng.choice(["gated", "gated_train", "gated_train", "log_probs", "log_probs_train", "log_probs_train"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if kind.startswith("gated"):
        width, hidden = _log_int(rng, 32, 4096), _log_int(rng, 64, 12_288)
        if rng.random() < 0.7:
            width, hidden = (width + 7) // 8 * 8, (hidden + 7) // 8 * 8
        # (the plain form's products cost the same for both types)
        most = min(100_000, 200_000_000_000 // (width * hidden), 400_000_000 // max(width, hidden))
        return dict(kind=kind, dtype=dtype, rows=_log_int(rng, 1, max(1, most)), width=width, hidden=hidden,
                    activation=rng.choice(["silu", "silu", "gelu"]))
    if rng.random() < 0.5:
        price, size = _log_int(rng, 2, 400), _log_int(rng, 2, 30)
        sizes = rng.choice([[price, price, size, size], [price, price, size, size], [price, size], [price]])
    else:
        sizes = [_log_int(rng, 400, 150_000)]
    top = rng.choice([0, 1, 5, 20]) if kind == "log_probs" else 0
    most = (10_000_000 if top else 200_000_000) // sum(sizes)
    return dict(kind=kind, dtype=dtype, rows=_log_int(rng, 1, min(200_000, most)), sizes=",".join(map(str, sizes)),
                mask=rng.choice(["none", "given", "inf"]), ragged=rng.random() < 0.4, top=min(top, min(sizes)))


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    kind, dtype, rows = case["kind"], TYPES[case["dtype"]], case["rows"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    s = {"case": case, "kind": kind}
    if kind.startswith("gated"):
        width, hidden = case["width"], case["hidden"]
        s["x"] = normal(rows, width).to(dtype)
        s["gate"], s["up"] = ((normal(hidden, width) / math.sqrt(width)).to(dtype) for _ in range(2))
        s["leaves"], s["grads"] = ["x", "gate", "up"], [normal(rows, hidden).to(dtype)]
    else:
        sizes = _sizes(case)
        logits = 2 * normal(rows, sum(sizes))
        allowed = torch.rand(logits.shape, generator=g, device="cuda") < 0.7 if case["mask"] != "none" else None
        if case["mask"] == "inf":
            logits.masked_fill_(~allowed, -math.inf)
        s["logits"] = logits.to(dtype)
        s["mask"] = allowed if case["mask"] == "given" else None
        s["sizes"] = sizes if len(sizes) > 1 else None
        # choices drawn from the policy itself; none where nothing is allowed, or where a game is over
        seen = s["logits"].float()
        if s["mask"] is not None:
            seen = seen.masked_fill(~allowed, -math.inf)
        race = seen - torch.log(-torch.log(torch.rand(seen.shape, generator=g, device="cuda").clamp(1e-20, 1 - 1e-7)))
        picked = [p.max(-1) for p in race.split(sizes, dim=-1)]
        choice = torch.stack([torch.where(v > -math.inf, i, -1) for v, i in picked], -1)
        if case["ragged"]:
            choice[torch.rand(rows, generator=g, device="cuda") < 0.25] = -1
        s["choice"] = choice if len(sizes) > 1 else choice[:, 0]
        # of a mean over the moves: an advantage each, and a bonus for entropy
        s["leaves"] = ["logits"]
        s["grads"] = [normal(*s["choice"].shape) / rows, torch.full(s["choice"].shape, -0.01 / rows, device="cuda")]
    if kind.endswith("train"):
        for k in s["leaves"]:
            s[k].requires_grad_()
    return s


# ---------------------------------------------------------------- plain forms

def _plain_gated(x, gate, up, activation):
    xf = x.float()
    a, b = torch.matmul(xf, gate.float().t()), torch.matmul(xf, up.float().t())
    if activation == "silu":
        act = a * torch.sigmoid(a)
    else:
        act = a * 0.5 * (1 + torch.erf(a * math.sqrt(0.5)))
    return (act * b).to(x.dtype)


def _plain_part(logits, choice, mask, top):
    x = logits.float()
    live = x > -math.inf
    if mask is not None:
        live = live & mask
    counts = choice != -1
    some = live.any(-1, keepdim=True)
    x = torch.where(live & some, x, 0.0)
    most = torch.where(live, x.detach(), -math.inf).amax(-1, keepdim=True)
    most = torch.where(some, most, 0.0)
    e = torch.where(live, torch.exp(torch.where(live, x - most, 0.0)), 0.0)
    total = torch.where(some, e.sum(-1, keepdim=True), 1.0)
    lp = torch.where(live, x - most - torch.log(total), 0.0)
    at = choice.clamp(min=0)[:, None]
    chosen = torch.where(torch.gather(live, 1, at)[:, 0], torch.gather(lp, 1, at)[:, 0], -math.inf)
    out = [torch.where(counts, chosen, 0.0), torch.where(counts, -(e / total * lp).sum(-1), 0.0)]
    if top:
        lp = torch.where(live & counts[:, None], lp, -math.inf)
        best, index = torch.sort(torch.where(live & counts[:, None], x, -math.inf), dim=-1, descending=True, stable=True)
        index = torch.where(best[:, :top] > -math.inf, index[:, :top], -1)
        out += [torch.where(index >= 0, torch.gather(lp, 1, index.clamp(min=0)), -math.inf), index]
    return out


def _plain_log_probs(s):
    sizes, choice, mask = _sizes(s["case"]), s["choice"], s["mask"]
    if len(sizes) == 1:
        return tuple(_plain_part(s["logits"], choice, mask, s["case"]["top"]))
    masks = [None] * len(sizes) if mask is None else mask.split(sizes, dim=-1)
    parts = [_plain_part(x, choice[:, i], m, s["case"]["top"])
             for i, (x, m) in enumerate(zip(s["logits"].split(sizes, dim=-1), masks))]
    return tuple(torch.stack(v, 1) for v in zip(*parts))


def run(s):
    case, train = s["case"], s["kind"].endswith("train")
    if own:
        from astra_cuda import sequence
    with torch.set_grad_enabled(train):
        if s["kind"].startswith("gated"):
            if own:
                out = (sequence.gated_linear(s["x"], s["gate"], s["up"], activation=case["activation"]),)
            else:
                out = (_plain_gated(s["x"], s["gate"], s["up"], case["activation"]),)
        elif own:
            out = sequence.log_probs(s["logits"], s["choice"], sizes=s["sizes"], mask=s["mask"], top=case["top"])
        else:
            out = _plain_log_probs(s)
    if not train:
        return out
    grads = torch.autograd.grad(out[:len(s["grads"])], [s[k] for k in s["leaves"]], s["grads"])
    return tuple(v.detach() for v in out), grads


def work(case):
    rows, e, train = case["rows"], 2 if case["dtype"] == "bf16" else 4, case["kind"].endswith("train")
    if case["kind"].startswith("gated"):
        D, F = case["width"], case["hidden"]
        # forwards two products; their gradients two each
        forward = e * (rows * D + 2 * D * F + rows * F)
        return {"bytes": forward * (2 if train else 1), "flops": (12 if train else 4) * rows * D * F}
    sizes = _sizes(case)
    n, parts = rows * sum(sizes), rows * len(sizes)
    forward = n * (e + (1 if case["mask"] == "given" else 0)) + parts * (16 + 12 * case["top"])
    if not train:
        return {"bytes": forward, "flops": 8 * n}
    return {"bytes": forward + n * e + 8 * parts, "flops": 16 * n}


# ------------------------------------------------- the definitions, in 64 bits

def _exact_gated(s, case):
    x, wg, wu, dh = (v.detach().double() for v in (s["x"], s["gate"], s["up"], s["grads"][0]))
    a, b = x @ wg.T, x @ wu.T
    if case["activation"] == "silu":
        sg = 1 / (1 + torch.exp(-a))
        act, slope = a * sg, sg * (1 + a * (1 - sg))
    else:
        phi = torch.special.erfc(-a / math.sqrt(2)) / 2
        act, slope = a * phi, phi + a * torch.exp(-a * a / 2) / math.sqrt(2 * math.pi)
    h = act * b
    if case["kind"] == "gated":
        return (h,)
    da, db = dh * b * slope, dh * act
    return (h,), (da @ wg + db @ wu, da.T @ x, db.T @ x)


def _exact_part(logits, mask, choice, top, grads):
    x = logits.detach().double()
    if mask is not None:
        x = x.masked_fill(~mask, -math.inf)
    x = torch.where((choice == -1)[:, None], -math.inf, x)
    lse = torch.logsumexp(x, 1)
    lp = x - torch.where(torch.isinf(lse), 0.0, lse)[:, None]
    p = lp.exp()
    h = -torch.where(p > 0, p * lp, 0.0).sum(1)
    hot = torch.zeros_like(p).scatter_(1, choice.clamp(min=0)[:, None], (choice != -1).double()[:, None])
    chosen = torch.where(choice == -1, 0.0, torch.gather(lp, 1, choice.clamp(min=0)[:, None])[:, 0])
    out = [chosen, h]
    if top:
        out += [torch.topk(lp, top, 1)[0], None]
    if grads is None:
        return out, None
    dlp, dh = (v.double()[:, None] for v in grads)
    d = dlp * (hot - p) - dh * torch.where(p > 0, p * (lp + h[:, None]), 0.0)
    return out, torch.where((choice == -1)[:, None], 0.0, d)


def _exact_log_probs(s, case):
    sizes, train = _sizes(case), case["kind"].endswith("train")
    if len(sizes) == 1:
        out, d = _exact_part(s["logits"], s["mask"], s["choice"], case["top"], s["grads"] if train else None)
        return (tuple(out), (d,)) if train else tuple(out)
    parts, at = [], 0
    for i, n in enumerate(sizes):
        mask = None if s["mask"] is None else s["mask"][:, at:at + n]
        parts.append(_exact_part(s["logits"][:, at:at + n], mask, s["choice"][:, i], case["top"],
                                 [g[:, i] for g in s["grads"]] if train else None))
        at += n
    out = tuple(None if v[0] is None else torch.stack(v, 1) for v in zip(*(p[0] for p in parts)))
    return (out, (torch.cat([p[1] for p in parts], 1),)) if train else out


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return (_exact_gated if case["kind"].startswith("gated") else _exact_log_probs)(s, case)
