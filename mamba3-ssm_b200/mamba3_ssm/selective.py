"""Selective state space scan with a decay of its own for each channel and state, and the short
depthwise causal convolution in front of it, for sequences (training, prompts) and single tokens.

    x = causal_conv(x, weight, bias, activation="silu")               # (batch, length, channels)
    y = ssm_scan_selective(x, delta, A, B, C, D, z=z, delta_bias=b)   # delta, B, C: projections of x
    x = causal_conv_step_(conv_state, x, weight, bias, activation="silu")                   # one token
    y = ssm_step_selective_(ssm_state, x, delta, A, B, C, D, z=z, delta_bias=b)

Next to ``ssm_scan_siso`` / ``ssm_scan_mimo``, whose decay is one number a head and whose input has two
taps: here every channel e and state n decays by exp(dt[e] A[e, n]). Tensors are (batch, length,
channels) with contiguous channels, read in place at any strides of batch and length (columns
of a projection's output), in fp32, bf16 or fp16; states and sums are fp32.

``lengths`` (batch) holds the positions that count of each sequence of a padded batch, on the device.
Positions from there on are not read; outputs and gradients are 0 there, and returned states are those in
front of them (an empty sequence returns its initial state). Values are cut to 0 .. length.
Gradients flow once and backwards to every floating operand (no second derivatives, no forward mode).
No counterpart in the reference's package.
"""

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib as L
from .ops import _inner, _require_cuda

__all__ = ["causal_conv", "causal_conv_step_", "ssm_scan_selective", "ssm_step_selective_"]

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


def _check(name, main, **others):
    """Dtype of the main operand; one CUDA device for all that are given; no forward-mode tangents."""
    what, t = main
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: {what} must be a tensor")
    _require_cuda(name, t)
    if t.dtype not in _FLOATS:
        raise TypeError(f"{name}: {what} must be float32, bfloat16 or float16, got {t.dtype}")
    at = t.get_device()
    for k, v in others.items():
        if v is not None:
            if not isinstance(v, torch.Tensor):
                raise TypeError(f"{name}: {k} must be a tensor")
            if v.get_device() != at:
                raise RuntimeError(f"{name}: {k} is on {v.device}, {what} on {t.device}")
    if getattr(forward_ad, "_current_level", 0) >= 0:
        for k, v in (main, *others.items()):
            if v is not None and forward_ad.unpack_dual(v).tangent is not None:
                raise NotImplementedError(f"{name}: no forward-mode derivative, but {k} carries a tangent")


def _shape(name, what, t, *shape):
    if t is not None and tuple(t.shape) != shape:
        raise ValueError(f"{name}: {what} of shape {tuple(t.shape)}, expected {shape}")


def _silu(name, activation):
    if activation not in (None, "silu"):
        raise ValueError(f"{name}: activation is None or 'silu', got {activation!r}")
    return int(activation == "silu")


def _lengths(name, lengths, batch):
    if lengths is None:
        return None
    if lengths.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{name}: lengths must be int64 or int32, got {lengths.dtype}")
    _shape(name, "lengths", lengths, batch)
    return lengths.long().contiguous()


def _no_grad_only(name, *ts):
    if torch.is_grad_enabled() and any([t is not None and t.requires_grad for t in ts]):
        raise RuntimeError(f"{name}: works in place, without gradients; call it under torch.no_grad()")


def _written(t):
    if not t.is_inference():
        torch.autograd.graph.increment_version(t)


def _needs_grad(*ts):
    return torch.is_grad_enabled() and any([t is not None and t.requires_grad for t in ts])


def _new(t, *shape, dtype=None):
    return torch.empty(shape, dtype=dtype or t.dtype, device=t.device)


# ------------------------------------------------------------------------------------------
# convolution
# ------------------------------------------------------------------------------------------
def _conv_forward(x, weight, bias, initial, lengths, silu, want):
    b, n, e = x.shape
    y = _new(x, b, n, e)
    last = _new(x, b, weight.shape[1] - 1, e) if want else None
    a = L.pack(x, weight, bias, initial, lengths, y, last)
    p = a.ptrs
    with L.on_device(x.device):
        rc = L.load().m3_causal_conv(p[0], p[1], p[2], p[3], p[4], silu, p[5], p[6], L.stream_ptr(x.device))
    L.check(rc, "m3_causal_conv")
    return y, last


class _CausalConvFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, initial, lengths, silu, want):
        ctx.save_for_backward(x, weight, bias, initial, lengths)
        ctx.silu = silu
        ctx.set_materialize_grads(False)
        return _conv_forward(x, weight, bias, initial, lengths, silu, want)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        x, weight, bias, initial, lengths = ctx.saved_tensors
        if dy is None and dlast is None:
            return (None,) * 7
        b, n, e = x.shape
        dy = torch.zeros_like(x) if dy is None else _inner(dy)
        dlast = None if dlast is None else _inner(dlast)
        dx = _new(x, b, n, e)
        dw = _new(weight, *weight.shape)
        db = None if bias is None else _new(bias, e)
        di = _new(x, *initial.shape) if initial is not None and ctx.needs_input_grad[3] else None
        lib = L.load()
        nbytes = lib.m3_causal_conv_bwd_workspace_size(b, n, e, weight.shape[1])
        ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        p = (a := L.pack(x, weight, bias, initial, lengths, dy, dlast, dx, dw, db, di)).ptrs
        with L.on_device(x.device):
            rc = lib.m3_causal_conv_bwd(*p[:5], ctx.silu, *p[5:], ws.data_ptr(), nbytes, L.stream_ptr(x.device))
        L.check(rc, "m3_causal_conv_bwd")
        del a
        return dx, dw, db, di, None, None, None


def _conv_weights(name, x, weight, bias, e):
    if weight.dim() != 2 or weight.shape[0] != e:
        raise ValueError(f"{name}: weight of shape {tuple(weight.shape)}, expected ({e}, taps)")
    if not 2 <= weight.shape[1] <= 4:
        raise ValueError(f"{name}: 2, 3 or 4 taps, got {weight.shape[1]}")
    _shape(name, "bias", bias, e)
    if weight.dtype is not x.dtype and weight.dtype is not torch.float32:
        weight = weight.float()
    if bias is not None and bias.dtype is not weight.dtype:
        bias = bias.to(weight.dtype)
    return _inner(weight), bias if bias is None else bias.contiguous()


def causal_conv(x, weight, bias=None, *, activation=None, initial_state=None, lengths=None, return_state=False):
    """y[b, t, e] = act(bias[e] + sum_k weight[e, k] x[b, t - K + 1 + k, e]) for x (batch, length,
    channels), weight (channels, K) with K = 2, 3 or 4, bias (channels); ``activation`` None or
    "silu". y has x's shape and dtype. Weight and bias may be fp32 or of x's dtype.

    ``initial_state`` (batch, K - 1, channels) of x's dtype: the rows in front of the first
    (zeros without it). With ``return_state`` returns (y, state), the last K - 1 rows in that layout: the
    initial state of a following piece, or the state of ``causal_conv_step_``. ``lengths``: see above."""
    name = "causal_conv"
    _check(name, ("x", x), weight=weight, bias=bias, initial_state=initial_state, lengths=lengths)
    if x.dim() != 3:
        raise ValueError(f"{name}: x is (batch, length, channels), got {tuple(x.shape)}")
    b, _, e = x.shape
    silu = _silu(name, activation)
    weight, bias = _conv_weights(name, x, weight, bias, e)
    if initial_state is not None:
        _shape(name, "initial_state", initial_state, b, weight.shape[1] - 1, e)
        if initial_state.dtype is not x.dtype:
            raise TypeError(f"{name}: initial_state must be of x's dtype {x.dtype}, got {initial_state.dtype}")
        initial_state = _inner(initial_state)
    args = (_inner(x), weight, bias, initial_state, _lengths(name, lengths, b), silu, bool(return_state))
    y, last = (_CausalConvFn.apply if _needs_grad(x, weight, bias, initial_state) else _conv_forward)(*args)
    return (y, last) if return_state else y


def causal_conv_step_(state, x, weight, bias=None, *, activation=None):
    """``causal_conv`` for one more row x (batch, channels): returns y (batch, channels) and moves
    ``state`` (batch, K - 1, channels, x's dtype) on by one row, in place. Without gradients."""
    name = "causal_conv_step_"
    _check(name, ("x", x), state=state, weight=weight, bias=bias)
    if x.dim() != 2:
        raise ValueError(f"{name}: x is (batch, channels), got {tuple(x.shape)}")
    _no_grad_only(name, x, state, weight, bias)
    b, e = x.shape
    silu = _silu(name, activation)
    weight, bias = _conv_weights(name, x, weight, bias, e)
    _shape(name, "state", state, b, weight.shape[1] - 1, e)
    if state.dtype is not x.dtype:
        raise TypeError(f"{name}: state must be of x's dtype {x.dtype}, got {state.dtype}")
    x = _inner(x)
    y = _new(x, b, e)
    p = (a := L.pack(state, x, weight, bias, y)).ptrs
    with L.on_device(x.device):
        rc = L.load().m3_causal_conv_step(*p[:4], silu, p[4], L.stream_ptr(x.device))
    L.check(rc, "m3_causal_conv_step")
    del a
    _written(state)
    return y


# ------------------------------------------------------------------------------------------
# scan
# ------------------------------------------------------------------------------------------
def _scan_forward(u, delta, A, B, C, D, z, bias, initial, lengths, softplus, want, keep=False):
    b, n, e = u.shape
    m = A.shape[1]
    lib = L.load()
    y = _new(u, b, n, e)
    last = _new(u, b, e, m, dtype=torch.float32) if want else None
    with L.on_device(u.device):
        nws = lib.m3_selective_scan_workspace_size(b, n, e, m, B.shape[2])
        nst = lib.m3_selective_scan_states_size(b, n, e, m) if keep else 0
        ws = torch.empty(nws, dtype=torch.uint8, device=u.device) if nws else None
        states = torch.empty(nst, dtype=torch.uint8, device=u.device) if keep else None
        p = (a := L.pack(u, delta, A, B, C, D, z, bias, initial, lengths, y, last)).ptrs
        rc = lib.m3_selective_scan(*p[:10], softplus, *p[10:], states.data_ptr() if nst else None, nst,
                                   ws.data_ptr() if nws else None, nws, L.stream_ptr(u.device))
    L.check(rc, "m3_selective_scan")
    del a
    return (y, last, states) if keep else (y, last)


class _SelectiveScanFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, delta, A, B, C, D, z, bias, initial, lengths, softplus, want):
        # the state in front of every eighth step is kept for the backward
        y, last, states = _scan_forward(u, delta, A, B, C, D, z, bias, initial, lengths, softplus, want, keep=True)
        ctx.save_for_backward(u, delta, A, B, C, D, z, bias, initial, lengths, states)
        ctx.softplus = softplus
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        u, delta, A, B, C, D, z, bias, initial, lengths, states = ctx.saved_tensors
        if dy is None and dlast is None:
            return (None,) * 12
        b, n, e = u.shape
        lib = L.load()
        dy = torch.zeros_like(u) if dy is None else _inner(dy)
        dlast = None if dlast is None else dlast.contiguous()
        du, ddelta = _new(u, b, n, e), _new(delta, b, n, e)
        dA, dB, dC = _new(A, *A.shape), _new(B, *B.shape), _new(C, *C.shape)
        dD = None if D is None else _new(D, e)
        dz = None if z is None else _new(z, b, n, e)
        dbias = None if bias is None else _new(bias, e)
        di = _new(A, *initial.shape) if initial is not None and ctx.needs_input_grad[8] else None
        with L.on_device(u.device):
            nws = lib.m3_selective_scan_bwd_workspace_size(b, n, e, A.shape[1], B.shape[2])
            ws = torch.empty(nws, dtype=torch.uint8, device=u.device)
            p = (a := L.pack(u, delta, A, B, C, D, z, bias, initial, lengths, dy, dlast, du, ddelta, dA, dB, dC, dD, dz,
                             dbias, di)).ptrs
            rc = lib.m3_selective_scan_bwd(*p[:10], ctx.softplus, *p[10:], states.data_ptr() or None, states.numel(),
                                           ws.data_ptr() or None, nws, L.stream_ptr(u.device))
        L.check(rc, "m3_selective_scan_bwd")
        del a
        return du, ddelta, dA, dB, dC, dD, dz, dbias, di, None, None, None


def _scan_operands(name, u, delta, A, B, C, D, z, bias, lead):
    """The operands in the layouts and dtypes of the kernels, B and C as (..., groups, states)."""
    e = u.shape[-1]
    if A.dim() != 2 or A.shape[0] != e or A.shape[1] == 0:
        raise ValueError(f"{name}: A of shape {tuple(A.shape)}, expected ({e}, states)")
    m = A.shape[1]
    if m > 128:
        raise ValueError(f"{name}: at most 128 states a channel, got {m}")
    _shape(name, "delta", delta, *u.shape)
    _shape(name, "z", z, *u.shape)
    _shape(name, "D", D, e)
    _shape(name, "delta_bias", bias, e)
    if B.dim() == len(lead) + 1:
        B = B.unsqueeze(-2)
    if C.dim() == len(lead) + 1:
        C = C.unsqueeze(-2)
    if B.dim() != len(lead) + 2 or B.shape[:-2] != lead or B.shape[-1] != m or C.shape != B.shape:
        raise ValueError(f"{name}: B and C are {(*lead, m)} or {(*lead, 'groups', m)}, got {tuple(B.shape)} and "
                         f"{tuple(C.shape)}")
    if B.shape[-2] == 0 or e % B.shape[-2]:
        raise ValueError(f"{name}: {e} channels do not divide into {B.shape[-2]} groups")
    if z is not None and z.dtype is not u.dtype:
        raise TypeError(f"{name}: z must be of u's dtype {u.dtype}, got {z.dtype}")
    if delta.dtype is not u.dtype and delta.dtype is not torch.float32:
        delta = delta.float()
    if B.dtype is not C.dtype or (B.dtype is not u.dtype and B.dtype is not torch.float32):
        B, C = B.float(), C.float()
    return (_inner(u), _inner(delta), A.float().contiguous(), _inner(B), _inner(C),
            None if D is None else D.float().contiguous(), None if z is None else _inner(z),
            None if bias is None else bias.float().contiguous())


def ssm_scan_selective(u, delta, A, B_proj, C_proj, D=None, *, z=None, delta_bias=None, delta_softplus=True,
                       initial_state=None, lengths=None, return_state=False):
    """With dt = softplus(delta + delta_bias) (without the softplus where ``delta_softplus`` is False):

        h[t, e, n] = exp(dt[t, e] A[e, n]) h[t - 1, e, n] + dt[t, e] u[t, e] B[t, n]
        y[t, e] = (sum_n C[t, n] h[t, e, n] + D[e] u[t, e]) * silu(z[t, e])

    u, delta, z (batch, length, channels); A (channels, states), at most 128 states; B_proj, C_proj
    (batch, length, states), or (batch, length, groups, states) for as many equal groups of
    channels; D, delta_bias (channels). Without z there is no gate, without D no skip. delta, B and C
    may be of u's dtype or fp32. Returns y in u's shape and dtype.

    ``initial_state`` (batch, channels, states): the state in front of the first position (zeros
    without it). With ``return_state`` returns (y, state) with the state behind the last one in fp32: the
    initial state of a following piece, or the state of ``ssm_step_selective_``. ``lengths``: see above.
    For the backward the call keeps the state in front of every eighth position."""
    name = "ssm_scan_selective"
    _check(name, ("u", u), delta=delta, A=A, B_proj=B_proj, C_proj=C_proj, D=D, z=z, delta_bias=delta_bias,
           initial_state=initial_state, lengths=lengths)
    if u.dim() != 3:
        raise ValueError(f"{name}: u is (batch, length, channels), got {tuple(u.shape)}")
    b, _, e = u.shape
    ops = _scan_operands(name, u, delta, A, B_proj, C_proj, D, z, delta_bias, u.shape[:2])
    if initial_state is not None:
        _shape(name, "initial_state", initial_state, b, e, A.shape[1])
        initial_state = initial_state.float().contiguous()
    args = (*ops, initial_state, _lengths(name, lengths, b), int(bool(delta_softplus)), bool(return_state))
    y, last = (_SelectiveScanFn.apply if _needs_grad(*ops, initial_state) else _scan_forward)(*args)
    return (y, last) if return_state else y


def ssm_step_selective_(state, u, delta, A, B_proj, C_proj, D=None, *, z=None, delta_bias=None, delta_softplus=True):
    """``ssm_scan_selective`` for one more position: u, delta, z (batch, channels), B_proj, C_proj
    (batch, states) or (batch, groups, states). Returns y (batch, channels) and updates ``state``
    (batch, channels, states) fp32 in place. Without gradients."""
    name = "ssm_step_selective_"
    _check(name, ("u", u), state=state, delta=delta, A=A, B_proj=B_proj, C_proj=C_proj, D=D, z=z, delta_bias=delta_bias)
    if u.dim() != 2:
        raise ValueError(f"{name}: u is (batch, channels), got {tuple(u.shape)}")
    _no_grad_only(name, state, u, delta, A, B_proj, C_proj, D, z, delta_bias)
    b, e = u.shape
    ops = _scan_operands(name, u, delta, A, B_proj, C_proj, D, z, delta_bias, u.shape[:1])
    _shape(name, "state", state, b, e, A.shape[1])
    if state.dtype is not torch.float32:
        raise TypeError(f"{name}: state must be float32, got {state.dtype}")
    y = _new(u, b, e)
    p = (a := L.pack(state, *ops, y)).ptrs
    with L.on_device(u.device):
        rc = L.load().m3_selective_step(*p[:9], int(bool(delta_softplus)), p[9], L.stream_ptr(u.device))
    L.check(rc, "m3_selective_step")
    del a
    _written(state)
    return y
