"""The sequence operators from their definitions, position by position, in float64 with
torch's autograd: the oracle of tests/test_gpu_sequence.py."""
import torch


def _live(lengths, B, T, device):
    if lengths is None:
        return torch.ones(B, T, dtype=torch.bool, device=device)
    return torch.arange(T, device=device)[None] < lengths.clamp(0, T)[:, None]


def conv(x, weight, bias=None, window=None, lengths=None, silu=True):
    """(y, the last K-1 inputs); every argument float64."""
    B, T, D = x.shape
    K = weight.shape[1]
    live = _live(lengths, B, T, x.device)
    seen = [x.new_zeros(B, D) if window is None else window[:, k] for k in range(K - 1)]
    ys = []
    for t in range(T):
        on = live[:, t, None]
        now = torch.where(on, x[:, t], 0.0)
        taps = seen + [now]
        p = sum(weight[:, k] * taps[k] for k in range(K))
        if bias is not None:
            p = p + bias
        ys.append(torch.where(on, p * torch.sigmoid(p) if silu else p, 0.0))
        seen = [torch.where(on, taps[k + 1], taps[k]) for k in range(K - 1)]
    y = torch.stack(ys, 1) if T else x.new_zeros(B, 0, D)
    return y, torch.stack(seen, 1)


def scan(x, dt, A, B, C, D=None, dt_bias=None, h=None, lengths=None):
    """(y, the state after the last position); every argument float64."""
    n, T, H, P = x.shape
    G, N = B.shape[2:]
    live = _live(lengths, n, T, x.device)
    h = x.new_zeros(n, H, P, N) if h is None else h
    ys = []
    for t in range(T):
        on = live[:, t]
        xt = torch.where(on[:, None, None], x[:, t], 0.0)
        Bt, Ct = (torch.where(on[:, None, None], v[:, t], 0.0).repeat_interleave(H // G, 1)[:, :, None] for v in (B, C))
        raw = dt[:, t] if dt_bias is None else dt[:, t] + dt_bias
        step = torch.where(on[:, None], torch.nn.functional.softplus(raw, threshold=50.0), 0.0)
        h = torch.exp(step * A)[..., None, None] * h + (step[..., None] * xt)[..., None] * Bt
        y = (h * Ct).sum(-1)
        if D is not None:
            y = y + D[:, None] * xt
        ys.append(y)
    return torch.stack(ys, 1) if T else x.new_zeros(n, 0, H, P), h


def join(residual, block, post, nxt, gate=None, scale=None, eps=1e-6):
    """(joined, normed); every argument float64."""
    def rms(v):
        return v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)
    r = residual
    if block is not None:
        u = rms(block) * post
        if scale is not None:
            u = u * scale
        if gate is not None:
            u = u * torch.sigmoid(gate)
        r = r + u
    return r, None if nxt is None else rms(r) * nxt
