"""A step in place raises the version of the state that it moves on, as torch's own operations
in place do: what saved the state for a backward pass notices."""
import pytest
import torch

from sequence_util import BF16, F32, small_conv, small_scan

pytestmark = pytest.mark.gpu


def scan_step(seq, p, h, t=0):
    return seq.state_scan_step(p["x"][:, t], p["dt"][:, t], p["A"], p["B"][:, t], p["C"][:, t], h, p["D"],
                               dt_bias=p["dt_bias"])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_step_on_a_saved_window_is_noticed(dtype):
    from astra_cuda import sequence as seq
    x, w, b, window = small_conv(dtype)
    w.requires_grad_()
    y = seq.short_conv(x, w, b, initial_state=window)
    before = window._version
    with torch.no_grad():
        seq.short_conv_step(x[:, 0], window, w, b)
    assert window._version == before + 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.float().sum().backward()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_step_on_a_saved_state_is_noticed(dtype):
    from astra_cuda import sequence as seq
    p, h = small_scan(dtype)
    p["A"].requires_grad_()
    y = seq.state_scan(**{k: v for k, v in p.items() if k not in ("D", "dt_bias")}, D=p["D"], dt_bias=p["dt_bias"],
                       initial_state=h)
    before = h._version
    with torch.no_grad():
        scan_step(seq, p, h)
    assert h._version == before + 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.float().sum().backward()


def test_a_step_on_a_view_of_a_saved_state_is_noticed():
    """A state that a torch operation saved, moved on through a detached view of it."""
    from astra_cuda import sequence as seq
    p, h = small_scan()
    h.requires_grad_()
    loss = h.square().sum()
    with torch.no_grad():
        scan_step(seq, p, h.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_steps_in_inference_mode_and_on_inference_tensors():
    """Those have no version; a rollout uses them."""
    from astra_cuda import sequence as seq
    x, w, b, window = small_conv()
    p, h = small_scan()
    with torch.inference_mode():
        window2, h2 = window.clone(), h.clone()
        y, z = seq.short_conv_step(x[:, 0], window2, w, b), scan_step(seq, p, h2)
    with torch.no_grad():
        assert torch.equal(seq.short_conv_step(x[:, 0], window, w, b), y) and torch.equal(window, window2)
        assert torch.equal(scan_step(seq, p, h), z) and torch.equal(h, h2)
        assert torch.equal(seq.short_conv_step(x[:, 1], window, w, b), seq.short_conv_step(x[:, 1], window2, w, b))
        assert torch.equal(scan_step(seq, p, h, 1), scan_step(seq, p, h2, 1))
