"""log_probs' C ABI on the CPU: the structures' layout, refusals before any device call, and the compiled
binding's refusal of host tensors."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

from test_sequence_abi import ROOT, _lib, _text


def test_structures_have_the_header_s_layout(tmp_path):
    from astra_cuda import _native
    pairs = {"astra_log_probs": _native.LogProbs, "astra_log_probs_grad": _native.LogProbsGrad}
    body = "".join(f'printf("%zu\\n", sizeof({c}));' + "".join(
        f'printf("%zu\\n", offsetof({c}, {n}));' for n, _ in py._fields_) for c, py in pairs.items())
    src = tmp_path / "layout.c"
    src.write_text(f'#include <stdio.h>\n#include "sequence/astra_sequence.h"\nint main(void) {{ {body} return 0; }}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = [v for c, py in pairs.items() for v in [ctypes.sizeof(py)] + [getattr(py, n).offset for n, _ in py._fields_]]
    assert got == want


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(parts=0), dict(parts=17), dict(type=2), dict(top=-1), dict(top=65),
                                 dict(top=6), dict(choice_bytes=2), dict(stride=-1), dict(mask_stride=-5),
                                 dict(sizes=(10, 0)), dict(sizes=(10, -1)), dict(sizes=(1 << 30, 1)), dict(logits=None),
                                 dict(entropy=None), dict(log_prob=None), dict(choice=None), dict(top=2),
                                 dict(sizes=(2 ** 31 - 1, 2 ** 31 - 1))])
def test_refuses(bad):
    from astra_cuda import _native
    lib = _lib()
    f = dict(logits=4096, choice=8192, log_prob=4096, entropy=4096, rows=3, stride=15, parts=2, choice_bytes=8, sizes=(10, 5))
    f.update(bad)
    f["sizes"] = (ctypes.c_int32 * 16)(*f["sizes"])
    s = _native.LogProbs(**f)
    assert lib.astra_log_probs_forward(ctypes.addressof(s), None) == 1
    g = _native.LogProbsGrad(f=s)
    assert lib.astra_log_probs_backward(ctypes.addressof(g), None) == 1
    assert lib.astra_log_probs_forward(None, None) == 1 and lib.astra_log_probs_backward(None, None) == 1


def test_limits_and_host_tensors():
    from astra_cuda import sequence
    for name in ("MAX_PARTS", "MAX_TOP", "MAX_ENTRIES"):
        assert getattr(sequence, name) == int(re.search(rf"ASTRA_SEQ_{name} (\d+)", _text()).group(1))
    with pytest.raises(RuntimeError, match="Astra Fatal Error"):
        sequence.log_probs(torch.zeros(3, 8))
