"""The sigmoid of the gates and of the convolution's activation, element by element over
the arguments at which it is small: float32 results are right to a few of their own
roundings there too.

Bounds: the exponential and the reciprocal are each good to 2^-23, the exponent's product is
carried in two parts, one addition and the product with what is gated are 2^-24 each; the
norm of a constant block is exact but for its inverse root (2^-23) and three roundings:
2^-23 + 2^-23 + 2^-23 + 5 2^-24 = 6.6e-7 of each element at most."""
import pytest
import torch

from sequence_util import DEV, F32

pytestmark = pytest.mark.gpu
BOUND = 7e-7


def test_small_gates():
    from astra_cuda import sequence as seq
    gate = torch.linspace(-85.0, 20.0, 64 * 100, device=DEV).view(100, 64)
    block = torch.full((100, 64), 3.0, device=DEV)
    zero, one = torch.zeros(100, 64, device=DEV), torch.ones(64, device=DEV)
    joined, _ = seq.join_norm(zero, block, one, None, gate=gate)
    rms = 3.0 / (9.0 + 1e-6) ** 0.5
    want = torch.sigmoid(gate.double()) * rms
    worst = float(((joined.double() - want) / want).abs().max())
    assert worst <= BOUND, worst
    row, _ = seq.join_norm(zero, block, one, None, gate=gate[:, :1].contiguous())
    worst = float(((row.double() - want[:, :1]) / want[:, :1]).abs().max())
    assert worst <= BOUND, worst


def test_small_bf16_gates_of_a_float_residual():
    """The joined stream is float32 although block and gate are bf16."""
    from astra_cuda import sequence as seq
    gate = torch.linspace(-85.0, 20.0, 64 * 100, device=DEV).view(100, 64).bfloat16()
    block = torch.full((100, 64), 3.0, device=DEV, dtype=torch.bfloat16)
    zero, one = torch.zeros(100, 64, device=DEV), torch.ones(64, device=DEV)
    want = torch.sigmoid(gate.double()) * (3.0 / (9.0 + 1e-6) ** 0.5)
    joined, _ = seq.join_norm(zero, block, one, None, gate=gate)
    assert joined.dtype == F32
    worst = float(((joined.double() - want) / want).abs().max())
    assert worst <= BOUND, worst


def test_small_activations():
    """silu(p) = p sigmoid(p) for the same range: p is exact (one tap of 1)."""
    from astra_cuda import sequence as seq
    x = torch.linspace(-85.0, 20.0, 8 * 500, device=DEV).view(1, 500, 8)
    w = torch.tensor([0.0, 1.0], device=DEV).expand(8, 2).contiguous()
    xl = x.clone().requires_grad_()
    y = seq.short_conv(xl, w)
    p = x.double()
    want = p * torch.sigmoid(p)
    worst = float(((y.detach().double() - want)[p != 0] / want[p != 0]).abs().max())
    assert worst <= BOUND, worst


def test_slopes_of_small_steps():
    """The derivative of softplus by its argument: ddt of one position with A = 0 is
    x . (dh B) sigmoid(dt)."""
    from astra_cuda import sequence as seq
    n = 1000
    dt = torch.linspace(-80.0, 20.0, n, device=DEV).view(n, 1, 1).requires_grad_()
    one = torch.ones(n, 1, 1, 1, device=DEV)
    y = seq.state_scan(one, dt, torch.zeros(1, device=DEV), one, one)
    got, = torch.autograd.grad(y, [dt], torch.ones_like(y))
    want = torch.sigmoid(dt.detach().double())
    # also the quotient (sum with dt) / dt and two roundings: 2^-23 + 2 2^-24 more
    worst = float(((got.double() - want) / want).abs().max())
    assert worst <= BOUND + 2.0 ** -22, worst
    assert got.dtype == F32


def test_closed_and_open_gates():
    """Gates beyond the range of the exponential, infinities among them: 0 and 1; NaN stays."""
    from astra_cuda import sequence as seq
    values = [-float("inf"), -1e30, -3e4, -205.0, -104.0, -95.0, 95.0, 104.0, 205.0, 3e4, 1e30, float("inf"), float("nan")]
    for dtype in (F32, torch.bfloat16):
        gate = torch.tensor(values, device=DEV).to(dtype)[:, None].expand(-1, 8).contiguous()
        block, one = torch.ones(len(values), 8, device=DEV, dtype=dtype), torch.ones(8, device=DEV)
        for g in (gate, gate[:, :1].contiguous()):
            joined, _ = seq.join_norm(torch.zeros_like(block), block, one, None, gate=g)
            assert float(joined[:6].abs().max()) <= 2.0 ** -126
            assert bool(((joined[6:12] - 1).abs() <= 1e-6).all())  # rms(1) is 1 / sqrt(1 + eps)
            assert bool(torch.isnan(joined[12]).all())
