"""Derivatives and traces that the sequence operators cannot give are refused instead of lost."""
import pytest
import torch

from sequence_util import gen, normal, small_conv, small_scan

pytestmark = pytest.mark.gpu


def calls(seq):
    """Every operator as (function of its tensors, its tensors)."""
    x, w, b, window = small_conv()
    p, h = small_scan()
    g = gen(33)
    r, u, gate, post, nxt, scale = (normal(g, 3, 8), normal(g, 3, 8), normal(g, 3, 8), normal(g, 8), normal(g, 8),
                                    normal(g, 8))
    ps = {k: (v if k in ("A", "D", "dt_bias") else v[:, 0]) for k, v in p.items()}
    return {
        "short_conv": (lambda x, w, b, s: seq.short_conv(x, w, b, initial_state=s), (x, w, b, window)),
        "short_conv_step": (lambda x, s, w, b: seq.short_conv_step(x, s, w, b), (x[:, 0], window, w, b)),
        "state_scan": (lambda x, dt, A, B, C, D, bias, h: seq.state_scan(x, dt, A, B, C, D, dt_bias=bias, initial_state=h),
                       (*p.values(), h)),
        "state_scan_step": (lambda x, dt, A, B, C, D, bias, h: seq.state_scan_step(x, dt, A, B, C, h, D, dt_bias=bias),
                            (*ps.values(), h)),
        "join_norm": (lambda r, u, p, n, g, s: seq.join_norm(r, u, p, n, gate=g, scale=s), (r, u, post, nxt, gate, scale)),
        "rms_norm": (lambda x, w: seq.rms_norm(x, w), (r, nxt)),
    }


NAMES = ["short_conv", "short_conv_step", "state_scan", "state_scan_step", "join_norm", "rms_norm"]


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_derivatives_are_refused(name):
    import torch.autograd.forward_ad as fwd
    from astra_cuda import sequence as seq
    fn, args = calls(seq)[name]
    for i in range(len(args)):
        for no_grad in (False, True):
            with fwd.dual_level(), torch.set_grad_enabled(not no_grad):
                duals = list(args)
                duals[i] = fwd.make_dual(args[i].clone(), torch.ones_like(args[i]))
                with pytest.raises(RuntimeError, match="Astra Fatal Error.*forward-mode"):
                    fn(*duals)
    with fwd.dual_level():
        fn(*args)  # no tangent, nothing to lose
    if not name.endswith("step"):
        with fwd.dual_level():
            duals = list(args)
            duals[0] = fwd.make_dual(args[0].clone().requires_grad_(), torch.ones_like(args[0]))
            with pytest.raises(RuntimeError, match="Astra Fatal Error.*forward-mode"):
                fn(*duals)


@pytest.mark.parametrize("name", NAMES)
def test_traces_are_refused(name):
    """A trace would hold the allocation of the result and not what fills it."""
    from astra_cuda import sequence as seq
    fn, args = calls(seq)[name]
    with pytest.raises(RuntimeError, match="Astra Fatal Error.*trace"):
        torch.jit.trace(fn, args, check_trace=False)
    fn(*args)
