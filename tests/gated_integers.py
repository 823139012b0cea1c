"""gated_linear of whole numbers, where every sum is exact whatever its order: results differ in no bit from
64 bits rounded once, and a row, a step or a slice that is lost or counted twice shows.

The activations of 50 and more are the number itself with a slope of 1, in float32: exp(-50) is below 2^-70.
x is -2 to 2 with ones in its first column; a row of gate has 64 there and up to 3 ones of either sign, a row
of up 8 at most; dh is -1, 0 or 1. So a is 58 to 70, b, da, h and db are at most 16, 16, 1,120 and 70 (a, b,
da and db are bfloat16 numbers), and no sum's terms add up to 2^24.
"""
import torch


def inputs(seed, M, D, F, dtype, device):
    g = torch.Generator()
    g.manual_seed(seed)
    x = torch.randint(-2, 3, (M, D), generator=g).float()
    x[:, 0] = 1
    def ones(n):
        w = torch.zeros(F, D)
        for _ in range(n):
            at = torch.randint(0, D, (F, 1), generator=g)
            w.scatter_(1, at, torch.randint(0, 2, (F, 1), generator=g).float() * 2 - 1)
        return w
    gate, up = ones(3), ones(8)
    gate[:, 0] = 64
    dh = torch.randint(-1, 2, (M, F), generator=g).float()
    return tuple(v.to(device=device, dtype=dtype) for v in (x, gate, up, dh))


def slopes(x, gate, up, dh):
    """da and db in 64 bits; h."""
    x, gate, up, dh = (v.detach().double() for v in (x, gate, up, dh))
    a, b = x @ gate.t(), x @ up.t()
    assert float(a.min()) >= 50 and float(a.max()) <= 70 and float(b.abs().max()) <= 16
    return dh * b, dh * a, a * b


def results(x, gate, up, dh):
    da, db, h = slopes(x, gate, up, dh)
    wx, wg, wu = x.double(), gate.double(), up.double()
    # (each sum's terms, by their magnitudes)
    size = max(float((da.abs() @ wg.abs() + db.abs() @ wu.abs()).max()), float((db.abs().t() @ wx.abs()).max()),
               float((da.abs().t() @ wx.abs()).max()))
    assert size < 2 ** 24, size
    out = {"h": h, "dx": da @ wg + db @ wu, "dgate": da.t() @ wx, "dup": db.t() @ wx}
    return {k: v.to(x.dtype) for k, v in out.items()}
