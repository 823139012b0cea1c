"""``astra_cuda.sequence`` -- the sequence layer of a recurrent policy, as HIP kernels.

A game of hidden information asks a policy to remember the moves it has seen. These
operators are one layer of such a policy, over whole games in training and a move at a
time in rollouts with a state of fixed size per env (include/astra_sequence.h):

``short_conv``       every channel filtered by its own few taps, causally, then SiLU
``state_scan``       a selective state space scan: per head a decaying state, with input,
                     read-out and step size given per position
``join_norm``        what stands between two blocks: the norm after one, its gate and
                     residual scale, the residual sum, the norm before the next
``short_conv_step``, ``state_scan_step``   one position, the state moved on in place

The first three are differentiable in every tensor they take (once). Tensors are float32
or bfloat16 on one HIP device; sums, states and norms are float32 throughout, and each
result is rounded to its type once. Calls run on the caller's current stream and do not
synchronise. Tensors may be strided as long as their last dimension is contiguous (others
are copied); rows of 16-byte aligned, multiple-of-8 (bf16) or 4 (float32) elements are
accessed widest.

``lengths`` (int32 ``[B]``) says how many positions of each row count: what comes after
is not read (it may hold anything), its outputs and gradients are zero, and states are
those after position ``lengths[b]``; a row of length 0 keeps its initial state.

Errors follow ``astra_cuda.order_matching``: ``RuntimeError("Astra Fatal Error: ...")``.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _native
from .order_matching import _check, _fatal, _raw_stream

MAX_TAPS = 4        # ASTRA_SEQ_MAX_TAPS
MAX_STATE = 128     # ASTRA_SEQ_MAX_STATE
MAX_NORM_WIDTH = 16384  # ASTRA_SEQ_MAX_NORM_WIDTH

_PLAIN = (torch.Tensor, torch.nn.Parameter)
_TYPES = {torch.float32: 0, torch.bfloat16: 1}  # ASTRA_SEQ_F32, ASTRA_SEQ_BF16
_ACTIVATIONS = {None: 0, "silu": 1}             # ASTRA_SEQ_LINEAR, ASTRA_SEQ_SILU


def _need(cond: bool, what: str) -> None:
    if not cond:
        _fatal(f"sequence.py {what}")


def _data(name: str, t, like=None, shape=None):
    """A float32 or bfloat16 tensor on a HIP device, of ``like``'s type and device."""
    if type(t) in _PLAIN and t.is_cuda and (
            t.dtype in _TYPES if like is None else t.dtype is like.dtype and t.device == like.device) and (
            shape is None or t.shape == shape):
        return t
    _need(isinstance(t, torch.Tensor), f"{name} must be a tensor")
    _need(t.is_cuda, f"{name} must be on a HIP device, got {t.device}")
    _need(t.dtype in _TYPES, f"{name} must be float32 or bfloat16, got {t.dtype}")
    if like is not None:
        _need(t.device == like.device, f"{name} must be on {like.device}, got {t.device}")
        _need(t.dtype == like.dtype, f"{name} must be {like.dtype}, got {t.dtype}")
    if shape is not None:
        _need(tuple(t.shape) == tuple(shape), f"{name} must have shape {list(shape)}, got {list(t.shape)}")
    return t


def _param(name: str, t, like, shape):
    """A parameter or state as a contiguous float32 tensor (None stays None)."""
    if t is None:
        return None
    if type(t) in _PLAIN and t.dtype is torch.float32 and t.shape == shape and t.device == like.device \
            and t.is_contiguous():
        return t
    _need(isinstance(t, torch.Tensor), f"{name} must be a tensor")
    _need(t.device == like.device, f"{name} must be on {like.device}, got {t.device}")
    _need(t.dtype.is_floating_point, f"{name} must be a floating point tensor, got {t.dtype}")
    _need(tuple(t.shape) == tuple(shape), f"{name} must have shape {list(shape)}, got {list(t.shape)}")
    return t.float().contiguous()


def _lengths(t, like, batch: int):
    if t is None:
        return None
    _need(isinstance(t, torch.Tensor) and t.device == like.device, f"lengths must be a tensor on {like.device}")
    _need(t.dtype in (torch.int32, torch.int64), f"lengths must be int32 or int64, got {t.dtype}")
    _need(tuple(t.shape) == (batch,), f"lengths must have shape [{batch}], got {list(t.shape)}")
    return t.to(torch.int32).contiguous()


def _rows(t):
    """t with a contiguous last dimension (a dimension of size 1 has no stride to speak of)."""
    return t if t.shape[-1] == 1 or t.stride(-1) == 1 else t.contiguous()


def _p(t):
    return None if t is None else t.data_ptr()


def _with_grad(*tensors) -> bool:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _call(fn, struct, device) -> None:
    if torch.cuda.current_device() == device.index:
        rc = fn(ctypes.addressof(struct), _raw_stream(device.index))
    else:
        with torch.cuda.device(device):
            rc = fn(ctypes.addressof(struct), _raw_stream(device.index))
    if rc:
        _check(rc)


def _size(fn, struct) -> int:
    n = ctypes.c_size_t(0)
    _check(fn(ctypes.addressof(struct), ctypes.byref(n)))
    return n.value


def _workspace(nbytes: int, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _no_grad(name: str, *tensors) -> None:
    if _with_grad(*tensors):
        _fatal(f"sequence.py {name} moves its state on in place and has no gradient; "
               "call it under torch.no_grad(), or use the whole-sequence operator")


# ------------------------------------------------------------------------ short_conv

def _conv_forward(x, weight, bias, window, lengths, activation, want_last):
    B, T, D = x.shape
    K = weight.shape[1]
    y = torch.empty((B, T, D), dtype=x.dtype, device=x.device)
    last = torch.empty((B, K - 1, D), dtype=x.dtype, device=x.device) if want_last else None
    f = _native.ShortConv(_p(x), _p(weight), _p(bias), _p(window), _p(lengths), _p(y), _p(last), B, T,
                          x.stride(0), x.stride(1), D, K, _TYPES[x.dtype], activation)
    _call(_native.lib().astra_short_conv_forward, f, x.device)
    return y, last


class _ShortConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, window, lengths, activation, want_last):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, weight, bias, window, lengths)
        ctx.activation = activation
        return _conv_forward(x, weight, bias, window, lengths, activation, want_last)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        x, weight, bias, window, lengths = ctx.saved_tensors
        B, T, D = x.shape
        K = weight.shape[1]
        need = ctx.needs_input_grad
        if dy is None and dlast is None:
            return (None,) * 7
        dy = x.new_zeros((B, T, D)) if dy is None else dy.contiguous()
        dlast = None if dlast is None else dlast.contiguous()
        f = _native.ShortConv(_p(x), _p(weight), _p(bias), _p(window), _p(lengths), None, None, B, T,
                              x.stride(0), x.stride(1), D, K, _TYPES[x.dtype], ctx.activation)
        lib = _native.lib()
        dx = torch.empty((B, T, D), dtype=x.dtype, device=x.device) if need[0] else None
        dw = torch.empty_like(weight) if need[1] else None
        db = torch.empty_like(bias) if bias is not None and need[2] else None
        dwin = torch.empty_like(window) if window is not None and need[3] else None
        sums = dw is not None or db is not None
        nbytes = _size(lib.astra_short_conv_workspace_size, f) if sums else 0
        ws = _workspace(nbytes, x.device)
        g = _native.ShortConvGrad(f, _p(dy), _p(dlast), _p(dx), _p(dwin), _p(dw), _p(db), _p(ws), nbytes)
        _call(lib.astra_short_conv_backward, g, x.device)
        return dx, dw, db, dwin, None, None, None


def _conv_checks(x, weight, bias, activation, width):
    _need(isinstance(weight, torch.Tensor) and weight.dim() == 2, "weight must be a tensor [width, taps]")
    K = weight.shape[1]
    _need(2 <= K <= MAX_TAPS, f"weight must have 2 to {MAX_TAPS} taps, got {K}")
    _need(activation in _ACTIVATIONS, f"activation must be 'silu' or None, got {activation!r}")
    return K, _param("weight", weight, x, (width, K)), _param("bias", bias, x, (width,))


def short_conv(x, weight, bias=None, *, activation="silu", initial_state=None, lengths=None, return_state=False):
    """Causal convolution of each channel with its own taps, then ``activation``.

    ``y[b,t,d] = act(bias[d] + sum_k weight[d,k] x[b,t-K+1+k,d])`` for ``x`` ``[B,T,D]``,
    ``weight`` ``[D,K]`` (2 to 4 taps), ``bias`` ``[D]``; ``activation``: ``"silu"`` or None.
    ``initial_state`` ``[B,K-1,D]`` of x's type holds the inputs before x (default zeros).
    Returns y, or ``(y, state)`` with ``return_state``: the last K-1 inputs, for what follows.
    """
    _data("x", x)
    _need(x.dim() == 3, f"x must have shape [batch, length, width], got {list(x.shape)}")
    B, T, D = x.shape
    _need(D >= 1, "x must have at least one channel")
    K, w, b = _conv_checks(x, weight, bias, activation, D)
    if initial_state is not None:
        initial_state = _data("initial_state", initial_state, x, (B, K - 1, D)).contiguous()
    run = _ShortConv.apply if _with_grad(x, w, b, initial_state) else _conv_forward
    y, last = run(_rows(x), w, b, initial_state, _lengths(lengths, x, B), _ACTIVATIONS[activation], bool(return_state))
    return (y, last) if return_state else y


def short_conv_step(x, state, weight, bias=None, *, activation="silu"):
    """One position of ``short_conv``: ``x`` ``[B,D]``, returns y ``[B,D]``; ``state``
    ``[B,K-1,D]`` (contiguous, x's type) is moved on by x in place."""
    _data("x", x)
    _need(x.dim() == 2, f"x must have shape [batch, width], got {list(x.shape)}")
    _no_grad("short_conv_step", x, state, weight, bias)
    B, D = x.shape
    _need(D >= 1, "x must have at least one channel")
    K, w, b = _conv_checks(x, weight, bias, activation, D)
    _data("state", state, x, (B, K - 1, D))
    _need(state.is_contiguous(), "state must be contiguous")
    x = _rows(x)
    y = torch.empty((B, D), dtype=x.dtype, device=x.device)
    o = _native.ShortConvOne(x.data_ptr(), w.data_ptr(), _p(b), state.data_ptr(), y.data_ptr(), B, x.stride(0), D, K,
                             _TYPES[x.dtype], _ACTIVATIONS[activation])
    _call(_native.lib().astra_short_conv_step, o, x.device)
    return y


# ------------------------------------------------------------------------ state_scan

def _scan_struct(x, dt, A, B, C, D, dt_bias, initial, lengths, y, final, states, ws):
    return _native.StateScan(
        _p(x), _p(dt), _p(B), _p(C), _p(A), _p(D), _p(dt_bias), _p(initial), _p(lengths), _p(y), _p(final),
        _p(states), x.shape[0], x.shape[1], x.stride(0), x.stride(1), x.stride(2), dt.stride(0), dt.stride(1),
        dt.stride(2), B.stride(0), B.stride(1), B.stride(2), C.stride(0), C.stride(1), C.stride(2), x.shape[2],
        x.shape[3], B.shape[2], B.shape[3], _TYPES[x.dtype], _p(ws), ws.numel() if ws is not None else 0)


def _scan_forward(x, dt, A, B, C, D, dt_bias, initial, lengths, want_state, grad=False):
    lib = _native.lib()
    batch, _, H, P = x.shape
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    final = torch.empty((batch, H, P, B.shape[3]), dtype=torch.float32, device=x.device) if want_state else None
    f = _scan_struct(x, dt, A, B, C, D, dt_bias, initial, lengths, y, final, None, None)
    ws = _workspace(_size(lib.astra_state_scan_workspace_size, f), x.device)
    states = None
    if grad:
        n = _size(lib.astra_state_scan_chunk_states, f)
        states = torch.empty(n, dtype=torch.float32, device=x.device) if n else None
    f.chunk_states, f.workspace = _p(states), _p(ws)
    f.workspace_bytes = ws.numel() if ws is not None else 0
    _call(lib.astra_state_scan_forward, f, x.device)
    return (y, final, states) if grad else (y, final)


class _StateScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, A, B, C, D, dt_bias, initial, lengths, want_state):
        y, final, states = _scan_forward(x, dt, A, B, C, D, dt_bias, initial, lengths, want_state, True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, dt, A, B, C, D, dt_bias, initial, lengths, states)
        return y, final

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dfinal):
        x, dt, A, B, C, D, dt_bias, initial, lengths, states = ctx.saved_tensors
        if dy is None and dfinal is None:
            return (None,) * 10
        need = ctx.needs_input_grad
        lib = _native.lib()
        dy = torch.zeros(x.shape, dtype=x.dtype, device=x.device) if dy is None else dy.contiguous()
        dfinal = None if dfinal is None else dfinal.contiguous()
        f = _scan_struct(x, dt, A, B, C, D, dt_bias, initial, lengths, None, None, states, None)

        def like(t, dtype=None):
            return torch.empty(t.shape, dtype=dtype or t.dtype, device=t.device)

        dx, ddt, dB, dC = like(x), like(dt), like(B), like(C)
        dA = like(A) if need[2] else None
        dD = like(D) if D is not None and need[5] else None
        dbias = like(dt_bias) if dt_bias is not None and need[6] else None
        dinit = like(initial) if initial is not None and need[7] else None
        nbytes = _size(lib.astra_state_scan_grad_workspace_size, f)
        ws = _workspace(nbytes, x.device)
        g = _native.StateScanGrad(f, _p(dy), _p(dfinal), _p(dx), _p(ddt), _p(dB), _p(dC), _p(dA), _p(dD), _p(dbias),
                                  _p(dinit), _p(ws), nbytes)
        _call(lib.astra_state_scan_backward, g, x.device)
        return dx, ddt, dA, dB, dC, dD, dbias, dinit, None, None


def _scan_checks(x, dt, A, B, C, D, dt_bias, lead: int):
    """Shapes with ``lead`` leading dimensions (batch, or batch and length)."""
    names = "[batch, heads, dim]" if lead == 1 else "[batch, length, heads, dim]"
    _data("x", x)
    _need(x.dim() == lead + 2, f"x must have shape {names}, got {list(x.shape)}")
    rows, (H, P) = tuple(x.shape[:lead]), x.shape[lead:]
    _need(H >= 1 and P >= 1, f"x must have at least one head and feature, got {list(x.shape)}")
    _data("dt", dt, x, rows + (H,))
    _data("B", B, x)
    _need(B.dim() == lead + 2 and tuple(B.shape[:lead]) == rows,
          f"B must have shape {list(rows)} + [groups, state], got {list(B.shape)}")
    G, N = B.shape[lead:]
    _need(G >= 1 and H % G == 0, f"the number of heads ({H}) must be a multiple of B's groups ({G})")
    _need(1 <= N <= MAX_STATE, f"the state must have 1 to {MAX_STATE} values, got {N}")
    _data("C", C, x, B.shape)
    A = _param("A", A, x, (H,))
    _need(A is not None, "A must be a tensor")
    return A, _param("D", D, x, (H,)), _param("dt_bias", dt_bias, x, (H,))


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
    A, D, dt_bias = _scan_checks(x, dt, A, B, C, D, dt_bias, 2)
    batch, _, H, P = x.shape
    initial_state = _param("initial_state", initial_state, x, (batch, H, P, B.shape[3]))
    run = _StateScan.apply if _with_grad(x, dt, A, B, C, D, dt_bias, initial_state) else _scan_forward
    y, state = run(_rows(x), dt, A, _rows(B), _rows(C), D, dt_bias, initial_state, _lengths(lengths, x, batch),
                   bool(return_state))
    return (y, state) if return_state else y


def state_scan_step(x, dt, A, B, C, state, D=None, *, dt_bias=None):
    """One position of ``state_scan``: ``x`` ``[batch, heads, dim]``, ``dt`` ``[batch, heads]``,
    ``B`` and ``C`` ``[batch, groups, state]``; returns y. ``state`` (float32, contiguous,
    ``[batch, heads, dim, state]``) is moved on in place."""
    _no_grad("state_scan_step", x, dt, A, B, C, state, D, dt_bias)
    A, D, dt_bias = _scan_checks(x, dt, A, B, C, D, dt_bias, 1)
    batch, H, P = x.shape
    G, N = B.shape[1:]
    _need(isinstance(state, torch.Tensor) and state.dtype == torch.float32 and state.device == x.device,
          f"state must be a float32 tensor on {x.device}")
    _need(tuple(state.shape) == (batch, H, P, N) and state.is_contiguous(),
          f"state must be contiguous with shape {[batch, H, P, N]}, got {list(state.shape)}")
    x, B, C = _rows(x), _rows(B), _rows(C)
    y = torch.empty((batch, H, P), dtype=x.dtype, device=x.device)
    o = _native.StateScanOne(x.data_ptr(), dt.data_ptr(), B.data_ptr(), C.data_ptr(), A.data_ptr(), _p(D),
                             _p(dt_bias), state.data_ptr(), y.data_ptr(), batch, x.stride(0), x.stride(1),
                             dt.stride(0), dt.stride(1), B.stride(0), B.stride(1), C.stride(0), C.stride(1), H, P, G,
                             N, _TYPES[x.dtype])
    _call(_native.lib().astra_state_scan_step, o, x.device)
    return y


# ------------------------------------------------------------------------- join_norm

def _join_struct(residual, block, post, nxt, gate, scale, joined, normed, rstd, eps):
    like = residual if block is None else block
    return _native.JoinNorm(
        _p(residual), _p(block), _p(gate), _p(post), _p(nxt), _p(scale), _p(joined), _p(normed), _p(rstd),
        residual.shape[0], residual.stride(0), like.stride(0), 0 if gate is None else gate.stride(0),
        residual.shape[1], 0 if gate is None else gate.shape[1], 0 if scale is None else scale.shape[0],
        _TYPES[like.dtype], _TYPES[residual.dtype], eps)


def _join_forward(residual, block, post, nxt, gate, scale, eps, rstd=None):
    # every tensor is 2-D here, [rows, width]
    like = residual if block is None else block
    joined = torch.empty(residual.shape, dtype=residual.dtype, device=like.device) if block is not None else None
    normed = torch.empty(residual.shape, dtype=like.dtype, device=like.device) if nxt is not None else None
    if residual.shape[0]:
        f = _join_struct(residual, block, post, nxt, gate, scale, joined, normed, rstd, eps)
        _call(_native.lib().astra_join_norm_forward, f, like.device)
    return joined, normed


class _JoinNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, residual, block, post, nxt, gate, scale, eps):
        rstd = torch.empty((residual.shape[0], 2), dtype=torch.float32, device=residual.device)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(residual, block, post, nxt, gate, scale, rstd)
        ctx.eps = eps
        return _join_forward(residual, block, post, nxt, gate, scale, eps, rstd)

    @staticmethod
    @once_differentiable
    def backward(ctx, djoined, dnormed):
        residual, block, post, nxt, gate, scale, rstd = ctx.saved_tensors
        if djoined is None and dnormed is None:
            return (None,) * 7
        need = ctx.needs_input_grad
        djoined, dnormed = (None if t is None else t.contiguous() for t in (djoined, dnormed))
        f = _join_struct(residual, block, post, nxt, gate, scale, None, None, rstd, ctx.eps)

        def like(i, t):
            return torch.empty(t.shape, dtype=t.dtype, device=t.device) if t is not None and need[i] else None

        dres, dblock, dpost, dgate, dscale = like(0, residual), like(1, block), like(2, post), like(4, gate), like(5, scale)
        dnext = like(3, nxt)
        if residual.shape[0] == 0:
            return tuple(None if t is None else t.zero_() for t in (dres, dblock, dpost, dnext, dgate, dscale, None))
        nbytes = 0
        if dpost is not None or dnext is not None or dscale is not None:
            nbytes = _size(_native.lib().astra_join_norm_workspace_size, f)
        ws = _workspace(nbytes, residual.device)
        g = _native.JoinNormGrad(f, _p(djoined), _p(dnormed), _p(dres), _p(dblock), _p(dgate), _p(dpost), _p(dnext),
                                 _p(dscale), _p(ws), nbytes)
        _call(_native.lib().astra_join_norm_backward, g, residual.device)
        return dres, dblock, dpost, dnext, dgate, dscale, None


def _flat(t):
    """[..., D] as [rows, D] (a view where the strides allow it) with contiguous rows."""
    return _rows(t) if t.dim() == 2 else _rows(t.reshape(-1, t.shape[-1]))


def _join(residual, block, post, nxt, gate, scale, eps):
    run = _JoinNorm.apply if _with_grad(residual, block, post, nxt, gate, scale) else _join_forward
    return run(_flat(residual), None if block is None else _flat(block), post, nxt,
               None if gate is None else _flat(gate), scale, float(eps))


def join_norm(residual, block, post_weight, next_weight, *, gate=None, scale=None, eps=1e-6):
    """From one block to the next: returns ``(joined, normed)``.

    ``joined = residual + scale * sigmoid(gate) * rms(block) * post_weight`` and
    ``normed = rms(joined) * next_weight`` with ``rms(v) = v / sqrt(mean(v^2) + eps)`` over the
    last dimension (normed is taken from joined before its rounding). ``residual`` and
    ``block`` ``[..., D]``; the residual is of block's type or float32, and ``joined`` with
    it. ``gate`` ``[..., D]`` or ``[..., 1]`` (None: no gate) and ``scale`` ``[D]`` or ``[1]``
    (None: 1); the weights ``[D]``. ``next_weight=None``: normed is None, for the last block.
    """
    _data("block", block)
    _data("residual", residual)
    _need(residual.dtype in (block.dtype, torch.float32),
          f"residual must be {block.dtype} or float32, got {residual.dtype}")
    _need(residual.device == block.device, f"residual must be on {block.device}, got {residual.device}")
    _need(block.dim() >= 1 and block.shape == residual.shape,
          f"residual and block must have one shape, got {list(residual.shape)} and {list(block.shape)}")
    D = block.shape[-1]
    _need(1 <= D <= MAX_NORM_WIDTH, f"the width must be 1 to {MAX_NORM_WIDTH}, got {D}")
    if gate is not None:
        _data("gate", gate, block)
        _need(gate.shape in (block.shape, block.shape[:-1] + (1,)),
              f"gate must have shape {list(block.shape)} or {list(block.shape[:-1]) + [1]}, got {list(gate.shape)}")
    if scale is not None:
        _need(isinstance(scale, torch.Tensor) and tuple(scale.shape) in ((D,), (1,)),
              f"scale must be a tensor of shape [{D}] or [1]")
        scale = _param("scale", scale, block, scale.shape)
    post = _param("post_weight", post_weight, block, (D,))
    _need(post is not None, "post_weight must be a tensor")
    joined, normed = _join(residual, block, post, _param("next_weight", next_weight, block, (D,)), gate, scale, eps)
    return joined.view(block.shape), None if normed is None else normed.view(block.shape)


def rms_norm(x, weight, *, eps=1e-6):
    """``x / sqrt(mean(x^2) + eps) * weight`` over the last dimension: the norm before the
    first block, where there is nothing to join yet."""
    _data("x", x)
    _need(x.dim() >= 1, "x must have at least one dimension")
    D = x.shape[-1]
    _need(1 <= D <= MAX_NORM_WIDTH, f"the width must be 1 to {MAX_NORM_WIDTH}, got {D}")
    weight = _param("weight", weight, x, (D,))
    _need(weight is not None, "weight must be a tensor")
    return _join(x, None, None, weight, None, None, eps)[1].view(x.shape)
