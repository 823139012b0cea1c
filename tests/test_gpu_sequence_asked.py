"""Gradients that a backward pass does not ask for are not computed, though their tensors require them: nothing
is allocated for them, and those that are asked for are the same as in a whole pass."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _tensors(seed, shapes, dtype):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return [(0.3 * torch.randn(*s, generator=g, device=DEV)).to(d or dtype).requires_grad_() for s, d in shapes]


def _gated(seq, leaves):
    return (seq.gated_linear(*leaves),)


def _conv(seq, leaves):
    x, weight, bias, window = leaves
    return seq.short_conv(x, weight, bias, initial_state=window, return_state=True)


def _bare_conv(seq, leaves):
    x, weight, window = leaves
    return seq.short_conv(x, weight, initial_state=window, return_state=True)


def _scan(seq, leaves):
    x, dt, A, B, C, bias, h = leaves
    return seq.state_scan(x, dt, A, B, C, dt_bias=bias, initial_state=h, return_state=True)


def _join(seq, leaves):
    residual, block, post, nxt, gate, scale = leaves
    return seq.join_norm(residual, block, post, nxt, gate=gate, scale=scale)


def _last_join(seq, leaves):
    residual, block, post, scale = leaves
    return seq.join_norm(residual, block, post, None, scale=scale)[:1]


F32 = torch.float32
W = 512
CALLS = {
    "gated_linear": (_gated, [((3000, 256), None), ((W, 256), None), ((W, 256), None)], range(3)),
    "short_conv": (_conv, [((8, 400, W), None), ((W, 4), F32), ((W,), F32), ((8, 3, W), None)], (0, 1, 2, 3)),
    "short_conv without a bias": (_bare_conv, [((8, 400, W), None), ((W, 4), F32), ((8, 3, W), None)], (0, 1, 2)),
    # (the gradients of x, dt, B and C come together)
    "state_scan": (_scan, [((4, 200, 4, 32), None), ((4, 200, 4), None), ((4,), F32), ((4, 200, 2, 32), None),
                           ((4, 200, 2, 32), None), ((4,), F32), ((4, 4, 32, 32), F32)], (2, 5, 6)),
    "join_norm": (_join, [((2000, W), None), ((2000, W), None), ((W,), F32), ((W,), F32), ((2000, W), None), ((W,), F32)], range(6)),
    "join_norm without a next": (_last_join, [((2000, W), None), ((2000, W), None), ((W,), F32), ((W,), F32)], range(4)),
}


@pytest.mark.parametrize("dtype", [F32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("name", CALLS)
def test_gradients_that_are_not_asked_for(name, dtype):
    from astra_cuda import sequence as seq
    call, shapes, single = CALLS[name]
    leaves = _tensors(1, shapes, dtype)
    out = call(seq, leaves)
    grads = [torch.randn(v.shape, device=DEV).to(v.dtype) for v in out]

    def backward(which):
        before = torch.cuda.memory_stats()["allocated_bytes.all.allocated"]
        got = torch.autograd.grad(out, [leaves[i] for i in which], grads, retain_graph=True)
        return got, torch.cuda.memory_stats()["allocated_bytes.all.allocated"] - before

    every, all_bytes = backward(range(len(leaves)))
    for i in single:
        (got,), bytes_ = backward([i])
        assert torch.equal(got, every[i]), i
        spared = sum(leaves[j].numel() * leaves[j].element_size() for j in single if j != i)
        assert bytes_ <= all_bytes - spared, (i, bytes_, all_bytes, spared)
    # through backward(), into the leaves that collect
    some = list(single)[:2]
    torch.autograd.backward(out, grads, inputs=[leaves[i] for i in some])
    for i, v in enumerate(leaves):
        assert v.grad is None if i not in some else torch.equal(v.grad, every[i]), i
