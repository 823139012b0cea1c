"""Lengths of rows as a caller may hold them."""
import pytest
import torch

from sequence_util import DEV, small_conv, small_scan

pytestmark = pytest.mark.gpu


def test_long_lengths_are_clamped_and_not_cut_off():
    """Lengths of 64 bits beyond what 32 hold."""
    from astra_cuda import sequence as seq
    x, w, b, _ = small_conv()
    p, _ = small_scan()
    far = torch.tensor([2 ** 32, -2 ** 32 + 3], device=DEV)
    near = torch.tensor([6, 0], device=DEV)
    for lengths in (far, torch.tensor([2 ** 31, -2 ** 63], device=DEV), torch.tensor([2 ** 63 - 1, -1], device=DEV)):
        assert torch.equal(seq.short_conv(x, w, b, lengths=lengths), seq.short_conv(x, w, b, lengths=near))
        assert torch.equal(seq.state_scan(**p, lengths=lengths), seq.state_scan(**p, lengths=near))
