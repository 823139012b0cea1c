"""``astra_cuda.sequence`` -- the sequence layer of a recurrent policy, as HIP kernels.

A game of hidden information asks a policy to remember the moves it has seen. These
operators are one layer of such a policy, over whole games in training and a move at a
time in rollouts with a state of fixed size per env (include/sequence/astra_sequence.h):

``short_conv``       every channel filtered by its own few taps, causally, then SiLU
``state_scan``       a selective state space scan: per head a decaying state, with input,
                     read-out and step size given per position
``join_norm``        what stands between two blocks: the norm after one, its gate and
                     residual scale, the residual sum, the norm before the next
``gated_linear``     the gated feed-forward block before its way back: both projections, the
                     activation and the product
``log_probs``        log probability of a move, entropy and likeliest alternatives from logits
``short_conv_step``, ``state_scan_step``   one position, the state moved on in place

All but the steps are differentiable in every floating point tensor they take, backwards and
once: tensors with a forward-mode tangent are refused, and so is being part of a torch.jit
trace. A step raises its state's version: a backward pass that had saved the state refuses to
run, as after torch's own operations in place.

Tensors are float32 or bfloat16 on one HIP device. Sums, states and norms are float32
throughout, and each result is rounded to its type once; what is computed in between enters
the matrix products of a bfloat16 scan as the sum of two bfloat16 values (2^-18), or of three
where it ends in a float32 result. Calls run on the caller's current stream and do not
synchronise. Tensors may be strided as long as their last dimension is contiguous (others
are copied); rows of 16-byte aligned, multiple-of-8 (bf16) or 4 (float32) elements are
accessed widest.

``lengths`` (int32 or int64 ``[B]``) says how many positions of each row count: what comes after
is not read (it may hold anything), its outputs and gradients are zero, and states are
those after position ``lengths[b]``; a row of length 0 keeps its initial state.

Values that are not finite reach the outputs that the definitions say and no others. The
gradients of up to 64 positions before and after them may be NaN as well.

Errors follow ``astra_cuda.order_matching``: ``RuntimeError("Astra Fatal Error: ...")``.
The checks, the calls and their autograd nodes are compiled (``astra_cuda._C.sequence``,
csrc/sequence_bindings.cpp): a call of one position takes less time on the GPU than a
Python body would on the host.
"""
from __future__ import annotations

import torch  # noqa: F401  (before the compiled binding)

MAX_TAPS = 4        # ASTRA_SEQ_MAX_TAPS
MAX_STATE = 128     # ASTRA_SEQ_MAX_STATE
MAX_NORM_WIDTH = 16384  # ASTRA_SEQ_MAX_NORM_WIDTH
MAX_LINEAR_WIDTH = 1048576  # ASTRA_SEQ_MAX_LINEAR_WIDTH
MAX_PARTS = 16      # ASTRA_SEQ_MAX_PARTS
MAX_TOP = 64        # ASTRA_SEQ_MAX_TOP
MAX_ENTRIES = 1 << 30  # ASTRA_SEQ_MAX_ENTRIES

_ops = None


def _compiled():
    """astra_cuda._C.sequence, loaded by the first call: importing the package needs only
    what it is used for."""
    global _ops
    if _ops is None:
        from . import _native
        _native.lib()
        from ._C import sequence
        _ops = sequence
    return _ops


def short_conv(x, weight, bias=None, *, activation="silu", initial_state=None, lengths=None, return_state=False):
    """Causal convolution of each channel with its own taps, then ``activation``.

    ``y[b,t,d] = act(bias[d] + sum_k weight[d,k] x[b,t-K+1+k,d])`` for ``x`` ``[B,T,D]``,
    ``weight`` ``[D,K]`` (2 to 4 taps), ``bias`` ``[D]``; ``activation``: ``"silu"`` or None.
    ``initial_state`` ``[B,K-1,D]`` of x's type holds the inputs before x (default zeros).
    Returns y, or ``(y, state)`` with ``return_state``: the last K-1 inputs, for what follows.
    """
    return (_ops or _compiled()).short_conv(x, weight, bias, activation, initial_state, lengths, return_state)


def short_conv_step(x, state, weight, bias=None, *, activation="silu"):
    """One position of ``short_conv``: ``x`` ``[B,D]``, returns y ``[B,D]``; ``state``
    ``[B,K-1,D]`` (contiguous, x's type) is moved on by x in place. No gradient."""
    return (_ops or _compiled()).short_conv_step(x, state, weight, bias, activation)


def state_scan(x, dt, A, B, C, D=None, *, dt_bias=None, initial_state=None, lengths=None, return_state=False):
    """Selective state space scan over whole sequences.

    Per head, with ``step = softplus(dt + dt_bias)``: ``h_t = exp(step_t A) h_{t-1} +
    step_t x_t (x) B_t`` and ``y_t = h_t C_t + D x_t``. ``x`` ``[batch, length, heads, dim]``,
    ``dt`` ``[batch, length, heads]``, ``B`` and ``C`` ``[batch, length, groups, state]`` of x's
    type (each group serves heads / groups neighbouring heads; state up to 128); ``A``
    (negative for decay), ``D`` and ``dt_bias`` ``[heads]``. ``initial_state``
    ``[batch, heads, dim, state]``, default zeros. Returns y, or ``(y, state)`` with
    ``return_state``: the float32 state after the last position.
    """
    return (_ops or _compiled()).state_scan(x, dt, A, B, C, D, dt_bias, initial_state, lengths, return_state)


def state_scan_step(x, dt, A, B, C, state, D=None, *, dt_bias=None):
    """One position of ``state_scan``: ``x`` ``[batch, heads, dim]``, ``dt`` ``[batch, heads]``,
    ``B`` and ``C`` ``[batch, groups, state]``; returns y. ``state`` (float32, contiguous,
    ``[batch, heads, dim, state]``) is moved on in place. No gradient."""
    return (_ops or _compiled()).state_scan_step(x, dt, A, B, C, state, D, dt_bias)


def join_norm(residual, block, post_weight, next_weight, *, gate=None, scale=None, eps=1e-6):
    """From one block to the next: returns ``(joined, normed)``.

    ``joined = residual + scale * sigmoid(gate) * rms(block) * post_weight`` and
    ``normed = rms(joined) * next_weight`` with ``rms(v) = v / sqrt(mean(v^2) + eps)`` over the
    last dimension (normed is taken from joined before its rounding). ``residual`` and
    ``block`` ``[..., D]``; the residual is of block's type or float32, and ``joined`` with
    it. ``gate`` ``[..., D]`` or ``[..., 1]`` (None: no gate) and ``scale`` ``[D]`` or ``[1]``
    (None: 1); the weights ``[D]``. ``next_weight=None``: normed is None, for the last block.
    """
    return (_ops or _compiled()).join_norm(residual, block, post_weight, next_weight, gate, scale, eps)


def rms_norm(x, weight, *, eps=1e-6):
    """``x / sqrt(mean(x^2) + eps) * weight`` over the last dimension: the norm before the
    first block, where there is nothing to join yet."""
    return (_ops or _compiled()).rms_norm(x, weight, eps)


def gated_linear(x, gate_weight, up_weight, *, activation="silu", recompute=False, exact_gradients=False):
    """The gated feed-forward block before its way back: ``act(x gate_weight^T) * (x up_weight^T)``.

    ``x`` ``[..., D]``, the weights ``[F, D]`` of x's type, as those of two ``nn.Linear``; returns
    ``[..., F]``. ``activation``: ``"silu"``, or ``"gelu"`` (v times the normal distribution function
    at v, by erf). Bfloat16 products are summed in float32 and the result is rounded once; the
    gradients of the two projections are rounded to x's type before their own products, which makes
    bfloat16 gradients 1.4 times as far off as their own rounding does. With ``exact_gradients`` these
    products take them as two bfloat16 numbers each, and the gradients are rounded once, for twice
    the products (float32 gradients are no different). A forward
    pass that is differentiated keeps its inputs, and from a width of 1,024 (float32: 128) on the
    two projections in float32, 8 bytes an element of the result, because the backward pass is faster
    with them; with ``recompute`` it keeps its inputs alone and the backward pass computes the
    projections again, which is as exact.
    """
    return (_ops or _compiled()).gated_linear(x, gate_weight, up_weight, activation, recompute, exact_gradients)


def log_probs(logits, choice=None, *, sizes=None, mask=None, top=0):
    """What a head's ``logits`` ``[..., W]`` say: returns ``(log_prob, entropy)``, and with ``top`` k
    ``(log_prob, entropy, top_log_prob, top_index)``.

    ``sizes`` cuts a row into the parts of a move, each a distribution of its own (default: one
    part of W entries); outputs are ``[..., parts]``, without ``sizes`` ``[...]``. ``choice`` of that
    shape (int32 or int64) is the entry of each part whose log probability is wanted (None: no
    log_prob). ``mask`` (bool, broadcast along the leading dimensions) says which entries are
    allowed; logits of -inf are not, either. ``top_log_prob`` and ``top_index`` ``[..., k]`` are the
    likeliest allowed entries, ties to the lower index, -inf and -1 where there are fewer.

    A choice of -1 says that a part does not count (a game that is over): its logits may be
    anything, its log_prob, entropy and gradient are 0. The log probability of an entry that is left out is
    -inf and has no gradient, that of a choice outside of its part is NaN. Where nothing is allowed
    the entropy is 0. An allowed NaN or infinity makes its part's log probabilities, entropy and
    gradient NaN. log_prob and entropy are float32 and differentiable in logits; the top ones are not.
    """
    return (_ops or _compiled()).log_probs(logits, choice, sizes, mask, top)
