"""gated_linear's C ABI on the CPU: the structures' layout, refusals before any device call, workspace
sizes, and the compiled binding's refusal of host tensors."""
import ctypes
import os
import subprocess

import pytest
import torch

from test_sequence_abi import ROOT, _lib


def test_structures_have_the_header_s_layout(tmp_path):
    from astra_cuda import _native
    pairs = {"astra_gated_linear": _native.GatedLinear, "astra_gated_linear_grad": _native.GatedLinearGrad}
    body = "".join(f'printf("%zu\\n", sizeof({c}));' + "".join(
        f'printf("%zu\\n", offsetof({c}, {n}));' for n, _ in py._fields_) for c, py in pairs.items())
    src = tmp_path / "layout.c"
    src.write_text(f'#include <stdio.h>\n#include "sequence/astra_sequence.h"\nint main(void) {{ {body} return 0; }}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = [v for c, py in pairs.items() for v in [ctypes.sizeof(py)] + [getattr(py, n).offset for n, _ in py._fields_]]
    assert got == want


def _gated(**kw):
    from astra_cuda import _native
    f = dict(x=4096, gate=8192, up=16384, h=32768, rows=500, x_stride=64, gate_stride=64, up_stride=64, width=64,
             hidden=128, type=1, activation=1)
    f.update(kw)
    return _native.GatedLinear(**f)


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(width=0), dict(hidden=0), dict(type=2), dict(type=-1),
                                 dict(activation=0), dict(activation=3), dict(x_stride=-64), dict(gate_stride=-1),
                                 dict(width=1 << 21), dict(hidden=1 << 21), dict(x=None), dict(gate=None),
                                 dict(up=None), dict(h=None), dict(x_stride=65)])
def test_refuses(bad):
    """(Rows that do not start on 16 bytes need a workspace.)"""
    from astra_cuda import _native
    lib = _lib()
    f = _gated(**bad)
    assert lib.astra_gated_linear_forward(ctypes.addressof(f), None) == 1
    b = _native.GatedLinearGrad(f=f, dh=4096, dx=4096)
    assert lib.astra_gated_linear_backward(ctypes.addressof(b), None) == 1
    assert lib.astra_gated_linear_forward(None, None) == 1 and lib.astra_gated_linear_backward(None, None) == 1


def test_workspaces():
    lib = _lib()

    def size(name, f):
        n = ctypes.c_size_t(0)
        assert getattr(lib, name)(ctypes.addressof(f), ctypes.byref(n)) == 0
        return n.value

    need = "astra_gated_linear_workspace_size"
    assert size(need, _gated()) == 0
    assert size(need, _gated(x_stride=72)) == 0
    assert size(need, _gated(x_stride=65)) == 500 * 64 * 2
    assert size(need, _gated(x=4098)) == 500 * 64 * 2
    assert size(need, _gated(width=63)) == (500 + 2 * 128) * 64 * 2
    assert size(need, _gated(width=63, type=0)) == (500 + 2 * 128) * 64 * 4
    assert size(need, _gated(width=63, rows=64)) == 0  # few rows are read as they lie
    grad = "astra_gated_linear_grad_workspace_size"
    assert size(grad, _gated(rows=0)) == 0
    assert size(grad, _gated()) >= 500 * 2 * 128 * 2
    b = _gated(hidden=129)
    assert size(grad, b) >= 500 * 2 * 136 * 2
    from astra_cuda import _native
    g = _native.GatedLinearGrad(f=b, dh=4096, dx=4096, workspace=4096, workspace_bytes=16)
    assert lib.astra_gated_linear_backward(ctypes.addressof(g), None) == 1
    g = _native.GatedLinearGrad(f=b, dh=4096, dx=4096, workspace=4100, workspace_bytes=1 << 40)
    assert lib.astra_gated_linear_backward(ctypes.addressof(g), None) == 1


def test_limits_and_host_tensors():
    from astra_cuda import sequence
    from test_sequence_abi import _text
    assert f"ASTRA_SEQ_MAX_LINEAR_WIDTH {sequence.MAX_LINEAR_WIDTH}" in _text()
    x, w = torch.zeros(3, 8), torch.ones(4, 8)
    with pytest.raises(RuntimeError, match="Astra Fatal Error"):
        sequence.gated_linear(x, w, w)
