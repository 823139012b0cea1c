"""The sequence operators' C ABI on the CPU: the library exports what
include/sequence/astra_sequence.h declares, the ctypes structures have the header's layout,
bad arguments are refused before any device call, workspace sizes are consistent, and the
compiled binding refuses tensors that are not on a HIP device."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "sequence", "astra_sequence.h")


def _lib():
    from astra_cuda import _native
    from astra_cuda.build import LIB_PATH, build
    if not os.path.exists(LIB_PATH):
        build()
    return _native.lib()


def _text():
    return re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)


def test_library_exports_and_prototypes_cover_the_header():
    from astra_cuda._native import SEQUENCE_PROTOTYPES
    declared = sorted(set(re.findall(r"\b(astra_\w+)\s*\(", _text())))
    assert sorted(SEQUENCE_PROTOTYPES) == declared
    lib = _lib()
    assert not [n for n in declared if not hasattr(lib, n)]


def test_structures_have_the_header_s_layout(tmp_path):
    """Every field's offset, and the sizes, as a C compiler lays the header out."""
    from astra_cuda import _native
    pairs = {"astra_short_conv": _native.ShortConv, "astra_short_conv_grad": _native.ShortConvGrad,
             "astra_short_conv_one": _native.ShortConvOne, "astra_state_scan": _native.StateScan,
             "astra_state_scan_grad": _native.StateScanGrad, "astra_state_scan_one": _native.StateScanOne,
             "astra_join_norm": _native.JoinNorm, "astra_join_norm_grad": _native.JoinNormGrad}
    body = "".join(f'printf("%zu\\n", sizeof({c}));' + "".join(
        f'printf("%zu\\n", offsetof({c}, {n}));' for n, _ in py._fields_) for c, py in pairs.items())
    src = tmp_path / "layout.c"
    src.write_text(f'#include <stdio.h>\n#include "sequence/astra_sequence.h"\nint main(void) {{ {body} return 0; }}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = [v for c, py in pairs.items() for v in [ctypes.sizeof(py)] + [getattr(py, n).offset for n, _ in py._fields_]]
    assert got == want


def test_constants():
    from astra_cuda import sequence
    text = open(HEADER).read()
    for name in ("MAX_TAPS", "MAX_STATE", "MAX_NORM_WIDTH"):
        assert getattr(sequence, name) == int(re.search(rf"ASTRA_SEQ_{name} (\d+)", text).group(1))


def _scan(**kw):
    from astra_cuda import _native
    f = dict(batch=2, length=300, heads=4, dim=64, groups=2, state=64, type=0)
    f.update(kw)
    return _native.StateScan(**f)


@pytest.mark.parametrize("bad", [dict(heads=3), dict(groups=0), dict(state=0), dict(state=129), dict(dim=0),
                                 dict(batch=-1), dict(length=-1), dict(type=2), dict(heads=0)])
def test_scan_refuses(bad):
    lib, n = _lib(), ctypes.c_size_t(0)
    f = _scan(**bad)
    assert lib.astra_state_scan_workspace_size(ctypes.addressof(f), ctypes.byref(n)) == 1
    assert lib.astra_state_scan_forward(ctypes.addressof(f), None) == 1


def test_scan_workspaces():
    """Chunk states from the second chunk on; segments only where few rows leave room."""
    lib = _lib()

    def size(fn, f):
        n = ctypes.c_size_t(0)
        assert fn(ctypes.addressof(f), ctypes.byref(n)) == 0
        return n.value

    assert size(lib.astra_state_scan_chunk_states, _scan(length=64)) == 0
    assert size(lib.astra_state_scan_chunk_states, _scan(length=65)) == 2 * 4 * 2 * 64 * 64
    assert size(lib.astra_state_scan_chunk_states, _scan(length=0)) == 0
    assert size(lib.astra_state_scan_workspace_size, _scan(length=128)) == 0
    assert size(lib.astra_state_scan_workspace_size, _scan(length=100_000)) > 0
    assert size(lib.astra_state_scan_workspace_size, _scan(length=100_000, batch=4096)) == 0
    for f in (_scan(), _scan(length=1), _scan(batch=5000, length=40)):
        assert size(lib.astra_state_scan_grad_workspace_size, f) > 0


@pytest.mark.parametrize("bad", [dict(taps=1), dict(taps=5), dict(width=0), dict(type=5), dict(activation=2),
                                 dict(batch=-1)])
def test_conv_refuses(bad):
    from astra_cuda import _native
    f = dict(batch=1, length=5, width=8, taps=4)
    f.update(bad)
    c = _native.ShortConv(**f)
    assert _lib().astra_short_conv_forward(ctypes.addressof(c), None) == 1
    f.pop("length")
    o = _native.ShortConvOne(**f)
    assert _lib().astra_short_conv_step(ctypes.addressof(o), None) == 1


@pytest.mark.parametrize("bad", [dict(width=0), dict(width=16385), dict(type=1, residual_type=2), dict(rows=-1),
                                 dict(type=0, residual_type=1), dict(block=None, next=None),
                                 dict(gate=64, gate_width=3), dict(scale=64, scale_width=2), dict(post=None)])
def test_join_refuses(bad):
    from astra_cuda import _native
    f = dict(residual=64, block=64, post=64, next=64, joined=64, normed=64, rows=2, width=8, residual_stride=8,
             block_stride=8)
    f.update(bad)
    j = _native.JoinNorm(**f)
    assert _lib().astra_join_norm_forward(ctypes.addressof(j), None) == 1


def test_null_structures_and_pointers_are_refused():
    from astra_cuda import _native
    lib = _lib()
    for name in ("astra_short_conv_forward", "astra_short_conv_backward", "astra_short_conv_step",
                 "astra_state_scan_forward", "astra_state_scan_backward", "astra_state_scan_step",
                 "astra_join_norm_forward", "astra_join_norm_backward"):
        assert getattr(lib, name)(None, None) == 1, name
        assert "NULL" in _native.last_error()
    f = _scan()
    assert lib.astra_state_scan_forward(ctypes.addressof(f), None) == 1 and "NULL" in _native.last_error()


def test_the_compiled_binding_refuses_host_tensors():
    from astra_cuda import sequence
    x, w = torch.zeros(1, 4, 8), torch.ones(8, 4)
    for call in (lambda: sequence.short_conv(x, w), lambda: sequence.rms_norm(x, w[:, 0]),
                 lambda: sequence.join_norm(x, x, w[:, 0], None),
                 lambda: sequence.state_scan(x[..., None], x, w[:, 0], x[..., None], x[..., None])):
        with pytest.raises(RuntimeError, match="Astra Fatal Error"):
            call()
