"""Sizes that no launch or workspace has room for are refused by the sequence operators' C entries, on the
CPU, before any device call."""
import ctypes

import pytest

from test_gated_linear_abi import _gated
from test_sequence_abi import _lib


def _probs(**kw):
    from astra_cuda import _native
    f = dict(logits=4096, choice=8192, log_prob=4096, entropy=4096, stats=4096, rows=3, stride=15, parts=2, choice_bytes=8,
             sizes=(10, 5))
    f.update(kw)
    f["sizes"] = (ctypes.c_int32 * 16)(*f["sizes"])
    return _native.LogProbs(**f)


@pytest.mark.parametrize("rows", [2 ** 38 + 1, 2 ** 43, 2 ** 62, 2 ** 63 - 1])
@pytest.mark.parametrize("name,make", [("gated_linear", _gated), ("log_probs", _probs)])
def test_more_rows_than_sizes_of_64_bits(name, make, rows):
    lib = _lib()
    from astra_cuda import _native
    f = make(rows=rows)
    n = ctypes.c_size_t(0)
    assert getattr(lib, f"astra_{name}_workspace_size")(ctypes.addressof(f), ctypes.byref(n)) == 1
    assert getattr(lib, f"astra_{name}_forward")(ctypes.addressof(f), None) == 1
    if name == "gated_linear":
        assert lib.astra_gated_linear_grad_workspace_size(ctypes.addressof(f), ctypes.byref(n)) == 1
        assert lib.astra_gated_linear_projections(ctypes.addressof(f), ctypes.byref(n)) == 1
        g = _native.GatedLinearGrad(f=f, dh=4096, dx=4096, workspace=4096, workspace_bytes=1 << 62)
        assert lib.astra_gated_linear_backward(ctypes.addressof(g), None) == 1
    else:
        g = _native.LogProbsGrad(f=f, dlogits=4096)
        assert lib.astra_log_probs_backward(ctypes.addressof(g), None) == 1
    f = make(rows=2 ** 38)
    assert getattr(lib, f"astra_{name}_workspace_size")(ctypes.addressof(f), ctypes.byref(n)) == 0


@pytest.mark.parametrize("type", [0, 1])
@pytest.mark.parametrize("width,batch", [(1, 2 ** 32), (129, 2 ** 25), (1, 2 ** 39)])
def test_convolutions_of_more_than_2_to_the_32_threads(type, width, batch):
    from astra_cuda import _native
    lib = _lib()
    f = _native.ShortConv(x=4098, weight=4096, y=4098, last=4098, batch=batch, length=1, width=width, taps=3, type=type,
                          x_stride_b=width, x_stride_t=width)
    assert lib.astra_short_conv_forward(ctypes.addressof(f), None) == 1
    assert "blocks" in _native.last_error()
    o = _native.ShortConvOne(x=4098, weight=4096, window=4098, y=4098, batch=batch, width=width, taps=3, type=type,
                             x_stride_b=width)
    assert lib.astra_short_conv_step(ctypes.addressof(o), None) == 1
    assert "blocks" in _native.last_error()


@pytest.mark.parametrize("type", [0, 1])
@pytest.mark.parametrize("batch", [2 ** 24, 2 ** 31])
def test_scans_of_more_than_2_to_the_32_threads(type, batch):
    """(16 heads of one feature and state each.)"""
    from astra_cuda import _native
    lib = _lib()
    p = dict(x=4096, dt=4096, b=4096, c=4096, A=4096)
    size = dict(batch=batch, heads=16, dim=1, groups=16, state=1, type=type)
    f = _native.StateScan(**p, y=4096, length=1, **size)
    assert lib.astra_state_scan_forward(ctypes.addressof(f), None) == 1
    assert "blocks" in _native.last_error()
    g = _native.StateScanGrad(f=f, dy=4096, dx=4096, ddt=4096, db=4096, dc=4096, workspace=4096, workspace_bytes=1 << 62)
    assert lib.astra_state_scan_backward(ctypes.addressof(g), None) == 1
    assert "blocks" in _native.last_error()
    o = _native.StateScanOne(**p, h=4096, y=4096, **size)
    assert lib.astra_state_scan_step(ctypes.addressof(o), None) == 1
    assert "blocks" in _native.last_error()


@pytest.mark.parametrize("activation", [256, 259, 1 | 128, 1 | 256 | 512, 2 | 1 << 30, -1])
def test_gated_linear_flags(activation):
    """Exact gradients go with an activation, and nothing else does."""
    from astra_cuda import _native
    lib, n = _lib(), ctypes.c_size_t(0)
    f = _gated(activation=activation)
    assert lib.astra_gated_linear_grad_workspace_size(ctypes.addressof(f), ctypes.byref(n)) == 1
    assert "activation" in _native.last_error()
    for kind in (1, 2):
        assert lib.astra_gated_linear_grad_workspace_size(ctypes.addressof(_gated(activation=kind | 256)), ctypes.byref(n)) == 0
    exact, flt = n.value, ctypes.c_size_t(0)
    assert lib.astra_gated_linear_grad_workspace_size(ctypes.addressof(_gated(activation=1)), ctypes.byref(n)) == 0
    assert exact == n.value + 500 * 2 * 128 * 2
    sizes = []
    for a in (1, 1 | 256):  # float gradients are no different
        assert lib.astra_gated_linear_grad_workspace_size(ctypes.addressof(_gated(activation=a, type=0)), ctypes.byref(flt)) == 0
        sizes.append(flt.value)
    assert sizes[0] == sizes[1]
