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
Parameters, step sizes, B and C of other real dtypes than the call allows are converted to fp32; complex ones are refused.
A sequence call takes at most 65535 sequences. A is finite (0 times an infinite one would be NaN at a step size of 0, as in padding).

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


_CODE = L._DTYPE_CODE
_F32 = torch.float32


def _check(name, what, t, names, others):
    """Dtype of the main operand; one CUDA device for all that are given; no forward-mode tangents."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: {what} must be a tensor")
    if not t.is_cuda:
        _require_cuda(name, t)
    if t.dtype not in _FLOATS:
        raise TypeError(f"{name}: {what} must be float32, bfloat16 or float16, got {t.dtype}")
    at = t.get_device()
    try:
        same = all([v is None or v.get_device() == at for v in others])
    except AttributeError:
        same = False
    if not same:
        for k, v in zip(names, others):
            if v is not None and not isinstance(v, torch.Tensor):
                raise TypeError(f"{name}: {k} must be a tensor")
            if v is not None and v.get_device() != at:
                raise RuntimeError(f"{name}: {k} is on {v.device}, {what} on {t.device}")
    if getattr(forward_ad, "_current_level", 0) >= 0:
        for k, v in ((what, t), *zip(names, others)):
            if v is not None and forward_ad.unpack_dual(v).tangent is not None:
                raise NotImplementedError(f"{name}: no forward-mode derivative, but {k} carries a tangent")


def _shape(name, what, t, shape):
    if t is not None and t.shape != shape:
        raise ValueError(f"{name}: {what} of shape {tuple(t.shape)}, expected {tuple(shape)}")


def _silu(name, activation):
    if activation is None:
        return 0
    if activation != "silu":
        raise ValueError(f"{name}: activation is None or 'silu', got {activation!r}")
    return 1


def _lengths(name, lengths, batch):
    if lengths is None:
        return None
    if lengths.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{name}: lengths must be int64 or int32, got {lengths.dtype}")
    _shape(name, "lengths", lengths, (batch,))
    return _dense(lengths if lengths.dtype is torch.int64 else lengths.long())


def _dense(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _f32(name, what, t):
    """Another real dtype as fp32; a complex one would lose its imaginary part."""
    if t.dtype.is_complex:
        raise TypeError(f"{name}: {what} must be real, got {t.dtype} (complex operands are not supported)")
    return t.float()


def _param(name, what, t):
    """A parameter of the channels as the kernels read it: fp32, contiguous."""
    if t is None:
        return None
    return _dense(t if t.dtype is _F32 else _f32(name, what, t))


def _needs_grad(ts):
    if not torch.is_grad_enabled():
        return False
    for t in ts:
        if t is not None and t.requires_grad:
            return True
    return False


def _no_grad_only(name, ts):
    if _needs_grad(ts):
        raise RuntimeError(f"{name}: works in place, without gradients; call it under torch.no_grad()")


def _like(t):
    """An uninitialised tensor of t's shape, dtype and order of dimensions in memory, with contiguous channels: of rows one
    element apart empty_like may turn the order round."""
    y = torch.empty_like(t)
    return y if y.stride(-1) == 1 or y.shape[-1] <= 1 else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _written(t):
    if not t.is_inference():
        torch.autograd.graph.increment_version(t)


# Records of the operands (see _lib.Records), for which the shapes are known by then: a call has up to two
# dozen operands, and finding out each one's shape again would cost more than the launches.
def _r1(t, a):
    return L.NO_RECORD if t is None else L.rec1(t, _CODE[t.dtype], a)


def _r2(t, a, b):
    return L.NO_RECORD if t is None else L.rec2(t, _CODE[t.dtype], a, b)


def _r3(t, a, b, c):
    return L.NO_RECORD if t is None else L.rec3(t, _CODE[t.dtype], a, b, c)


def _at(base, vals, i):
    """Address of record i, None where its operand is absent."""
    return base + 112 * i if vals[15 * i] else None


# ------------------------------------------------------------------------------------------
# convolution
# ------------------------------------------------------------------------------------------
def _conv_vals(x, weight, bias, initial, lengths, b, n, e, k):
    return [*_r3(x, b, n, e), *_r2(weight, e, k), *_r1(bias, e), *_r3(initial, b, k - 1, e), *_r1(lengths, b)]


def _conv_forward(x, weight, bias, initial, lengths, silu, want):
    b, n, e = x.shape
    k = weight.shape[1]
    dev = x.device
    y = _like(x)
    last = torch.empty((b, k - 1, e), dtype=x.dtype, device=dev) if want else None
    vals = _conv_vals(x, weight, bias, initial, lengths, b, n, e, k)
    vals += _r3(y, b, n, e)
    vals += _r3(last, b, k - 1, e)
    a = L.Records(vals)
    at = a.base
    with L.on_device(dev):
        rc = L.load().m3_causal_conv(at, at + 112, at + 224 if bias is not None else None,
                                     at + 336 if initial is not None else None, at + 448 if lengths is not None else None,
                                     silu, at + 560, at + 672 if want else None, L.stream_ptr(dev))
    if rc:
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
        k = weight.shape[1]
        dev = x.device
        dy = torch.zeros((b, n, e), dtype=x.dtype, device=dev) if dy is None else _inner(dy)
        dlast = None if dlast is None else _inner(dlast)
        dx = _like(x)
        dw = torch.empty((e, k), dtype=weight.dtype, device=dev)
        db = None if bias is None else torch.empty_like(bias)
        di = None
        if initial is not None and ctx.needs_input_grad[3]:
            di = torch.empty((b, k - 1, e), dtype=x.dtype, device=dev)
        vals = _conv_vals(x, weight, bias, initial, lengths, b, n, e, k)
        vals += (*_r3(dy, b, n, e), *_r3(dlast, b, k - 1, e), *_r3(dx, b, n, e), *_r2(dw, e, k), *_r1(db, e),
                 *_r3(di, b, k - 1, e))
        a = L.Records(vals)
        p = [_at(a.base, vals, i) for i in range(11)]
        lib = L.load()
        with L.on_device(dev):
            nbytes = lib.m3_causal_conv_bwd_workspace_size(b, n, e, k)
            ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev)
            rc = lib.m3_causal_conv_bwd(*p[:5], ctx.silu, *p[5:], ws.data_ptr(), nbytes, L.stream_ptr(dev))
        if rc:
            L.check(rc, "m3_causal_conv_bwd")
        return dx, dw, db, di, None, None, None


def _conv_weights(name, x, weight, bias, e):
    if weight.dim() != 2 or weight.shape[0] != e:
        raise ValueError(f"{name}: weight of shape {tuple(weight.shape)}, expected ({e}, taps)")
    if not 2 <= weight.shape[1] <= 4:
        raise ValueError(f"{name}: 2, 3 or 4 taps, got {weight.shape[1]}")
    _shape(name, "bias", bias, (e,))
    # the kernels read both in x's dtype or both in fp32, which holds all bits of either
    if (weight.dtype is not x.dtype and weight.dtype is not _F32) or (bias is not None and bias.dtype is not weight.dtype):
        weight = _f32(name, "weight", weight)
        bias = None if bias is None else _f32(name, "bias", bias)
    return _inner(weight), _dense(bias)


def causal_conv(x, weight, bias=None, *, activation=None, initial_state=None, lengths=None, return_state=False):
    """y[b, t, e] = act(bias[e] + sum_k weight[e, k] x[b, t - K + 1 + k, e]) for x (batch, length,
    channels), weight (channels, K) with K = 2, 3 or 4, bias (channels); ``activation`` None or
    "silu". y has x's shape and dtype. Weight and bias may be fp32 or of x's dtype, each by itself (two
    dtypes are brought to fp32 first).

    ``initial_state`` (batch, K - 1, channels) of x's dtype: the rows in front of the first
    (zeros without it). With ``return_state`` returns (y, state), the last K - 1 rows in that layout: the
    initial state of a following piece, or the state of ``causal_conv_step_``. ``lengths``: see above."""
    name = "causal_conv"
    _check(name, "x", x, ("weight", "bias", "initial_state", "lengths"), (weight, bias, initial_state, lengths))
    if x.dim() != 3:
        raise ValueError(f"{name}: x is (batch, length, channels), got {tuple(x.shape)}")
    b, _, e = x.shape
    silu = _silu(name, activation)
    weight, bias = _conv_weights(name, x, weight, bias, e)
    if initial_state is not None:
        _shape(name, "initial_state", initial_state, (b, weight.shape[1] - 1, e))
        if initial_state.dtype is not x.dtype:
            raise TypeError(f"{name}: initial_state must be of x's dtype {x.dtype}, got {initial_state.dtype}")
        initial_state = _inner(initial_state)
    args = (_inner(x), weight, bias, initial_state, _lengths(name, lengths, b), silu, bool(return_state))
    y, last = (_CausalConvFn.apply if _needs_grad(args[:4]) else _conv_forward)(*args)
    return (y, last) if return_state else y


def causal_conv_step_(state, x, weight, bias=None, *, activation=None):
    """``causal_conv`` for one more row x (batch, channels): returns y (batch, channels) and moves
    ``state`` (batch, K - 1, channels, x's dtype) on by one row, in place. Without gradients."""
    name = "causal_conv_step_"
    _check(name, "x", x, ("state", "weight", "bias"), (state, weight, bias))
    if x.dim() != 2:
        raise ValueError(f"{name}: x is (batch, channels), got {tuple(x.shape)}")
    _no_grad_only(name, (x, state, weight, bias))
    b, e = x.shape
    silu = _silu(name, activation)
    weight, bias = _conv_weights(name, x, weight, bias, e)
    k = weight.shape[1]
    _shape(name, "state", state, (b, k - 1, e))
    if state.dtype is not x.dtype:
        raise TypeError(f"{name}: state must be of x's dtype {x.dtype}, got {state.dtype}")
    x = _inner(x)
    dev = x.device
    y = torch.empty_like(x)
    if not y.is_contiguous():  # rows of x one element apart
        y = torch.empty((b, e), dtype=x.dtype, device=dev)
    code = _CODE[x.dtype]
    vals = [*L.rec3(state, code, b, k - 1, e), *L.rec2(x, code, b, e), *L.rec2(weight, _CODE[weight.dtype], e, k),
            *_r1(bias, e), y.data_ptr() or 1, code, 2, b, e, 0, 0, 0, 0, e, 1, 0, 0, 0, 0]
    a = L.Records(vals)
    at = a.base
    with L.on_device(dev):
        rc = L.load().m3_causal_conv_step(at, at + 112, at + 224, None if bias is None else at + 336, silu, at + 448,
                                          L.stream_ptr(dev))
    if rc:
        L.check(rc, "m3_causal_conv_step")
    _written(state)
    return y


# ------------------------------------------------------------------------------------------
# scan
# ------------------------------------------------------------------------------------------
def _scan_vals(u, delta, A, B, C, D, z, bias, initial, lengths, b, n, e, m):
    vals = [*_r3(u, b, n, e), *_r3(delta, b, n, e), *_r2(A, e, m)]
    code = _CODE[B.dtype]
    if B.dim() == 3:  # one group
        vals += (*L.rec4_of3(B, code, b, n, m), *L.rec4_of3(C, code, b, n, m))
    else:
        g = B.shape[2]
        vals += (*L.rec4(B, code, b, n, g, m), *L.rec4(C, code, b, n, g, m))
    vals += (*_r1(D, e), *_r3(z, b, n, e), *_r1(bias, e), *_r3(initial, b, e, m), *_r1(lengths, b))
    return vals


def _groups(B):
    return 1 if B.dim() == 3 else B.shape[2]


def _scan_forward(u, delta, A, B, C, D, z, bias, initial, lengths, softplus, want, keep=False):
    b, n, e = u.shape
    m = A.shape[1]
    dev = u.device
    lib = L.load()
    y = _like(u)
    last = torch.empty((b, e, m), dtype=_F32, device=dev) if want else None
    vals = _scan_vals(u, delta, A, B, C, D, z, bias, initial, lengths, b, n, e, m)
    vals += _r3(y, b, n, e)
    vals += _r3(last, b, e, m)
    a = L.Records(vals)
    p = [_at(a.base, vals, i) for i in range(12)]
    with L.on_device(dev):
        nws = lib.m3_selective_scan_workspace_size(b, n, e, m, _groups(B))
        nst = lib.m3_selective_scan_states_size(b, n, e, m) if keep else 0
        ws = torch.empty((nws,), dtype=torch.uint8, device=dev) if nws else None
        states = torch.empty((nst,), dtype=torch.uint8, device=dev) if keep else None
        rc = lib.m3_selective_scan(*p[:10], softplus, *p[10:], states.data_ptr() if nst else None, nst,
                                   ws.data_ptr() if nws else None, nws, L.stream_ptr(dev))
    if rc:
        L.check(rc, "m3_selective_scan")
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
        m = A.shape[1]
        g = _groups(B)
        dev, empty = u.device, torch.empty
        dy = torch.zeros((b, n, e), dtype=u.dtype, device=dev) if dy is None else _inner(dy)
        dlast = _dense(dlast)
        # (empty_like costs half of empty; it keeps the order of the dimensions in memory, which B's and C's gradients may not)
        like = torch.empty_like
        du, ddelta, dA = _like(u), _like(delta), like(A)
        dB = like(B) if B.is_contiguous() else empty(B.shape, dtype=B.dtype, device=dev)
        dC = like(C) if C.is_contiguous() else empty(B.shape, dtype=B.dtype, device=dev)
        dD = None if D is None else like(D)
        dz = None if z is None else _like(z)
        dbias = None if bias is None else like(bias)
        di = empty((b, e, m), dtype=_F32, device=dev) if initial is not None and ctx.needs_input_grad[8] else None
        vals = _scan_vals(u, delta, A, B, C, D, z, bias, initial, lengths, b, n, e, m)
        code = _CODE[B.dtype]
        vals += (*_r3(dy, b, n, e), *_r3(dlast, b, e, m), *_r3(du, b, n, e), *_r3(ddelta, b, n, e), *_r2(dA, e, m))
        if B.dim() == 3:
            vals += (*L.rec4_of3(dB, code, b, n, m), *L.rec4_of3(dC, code, b, n, m))
        else:
            vals += (*L.rec4(dB, code, b, n, g, m), *L.rec4(dC, code, b, n, g, m))
        vals += (*_r1(dD, e), *_r3(dz, b, n, e), *_r1(dbias, e), *_r3(di, b, e, m))
        a = L.Records(vals)
        p = [_at(a.base, vals, i) for i in range(21)]
        lib = L.load()
        with L.on_device(dev):
            nws = lib.m3_selective_scan_bwd_workspace_size(b, n, e, m, g)
            ws = empty((nws,), dtype=torch.uint8, device=dev)
            rc = lib.m3_selective_scan_bwd(*p[:10], ctx.softplus, *p[10:], states.data_ptr() or None, states.numel(),
                                           ws.data_ptr() or None, nws, L.stream_ptr(dev))
        if rc:
            L.check(rc, "m3_selective_scan_bwd")
        return du, ddelta, dA, dB, dC, dD, dz, dbias, di, None, None, None


def _scan_operands(name, u, delta, A, B, C, D, z, bias, lead):
    """The operands in the layouts and dtypes of the kernels."""
    shape, an, bs = u.shape, A.shape, B.shape
    e = shape[-1]
    if len(an) != 2 or an[0] != e or an[1] == 0:
        raise ValueError(f"{name}: A of shape {tuple(an)}, expected ({e}, states)")
    m = an[1]
    if m > 128:
        raise ValueError(f"{name}: at most 128 states a channel, got {m}")
    if delta.shape != shape:
        _shape(name, "delta", delta, shape)
    if z is not None and z.shape != shape:
        _shape(name, "z", z, shape)
    _shape(name, "D", D, (e,))
    _shape(name, "delta_bias", bias, (e,))
    if bs != (*lead, m) and (len(bs) != len(lead) + 2 or bs[:-2] != lead or bs[-1] != m) or C.shape != bs:
        raise ValueError(f"{name}: B and C are {(*lead, m)} or {(*lead, 'groups', m)}, got {tuple(bs)} and "
                         f"{tuple(C.shape)}")
    if len(bs) > len(lead) + 1 and (bs[-2] == 0 or e % bs[-2]):
        raise ValueError(f"{name}: {e} channels do not divide into {bs[-2]} groups")
    if z is not None and z.dtype is not u.dtype:
        raise TypeError(f"{name}: z must be of u's dtype {u.dtype}, got {z.dtype}")
    dtype, dd, bd = u.dtype, delta.dtype, B.dtype
    if dd is not dtype and dd is not _F32:
        delta = _f32(name, "delta", delta)
    if bd is not C.dtype or (bd is not dtype and bd is not _F32):
        B, C = _f32(name, "B_proj", B), _f32(name, "C_proj", C)
    return (_inner(u), _inner(delta), _param(name, "A", A), _inner(B), _inner(C), _param(name, "D", D),
            None if z is None else _inner(z), _param(name, "delta_bias", bias))


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
    _check(name, "u", u, ("delta", "A", "B_proj", "C_proj", "D", "z", "delta_bias", "initial_state", "lengths"),
           (delta, A, B_proj, C_proj, D, z, delta_bias, initial_state, lengths))
    if u.dim() != 3:
        raise ValueError(f"{name}: u is (batch, length, channels), got {tuple(u.shape)}")
    ops = _scan_operands(name, u, delta, A, B_proj, C_proj, D, z, delta_bias, u.shape[:2])
    b, _, e = u.shape
    if initial_state is not None:
        _shape(name, "initial_state", initial_state, (b, e, A.shape[1]))
        initial_state = _param(name, "initial_state", initial_state)
    args = (*ops, initial_state, _lengths(name, lengths, b), 1 if delta_softplus else 0, bool(return_state))
    y, last = (_SelectiveScanFn.apply if _needs_grad(args[:9]) else _scan_forward)(*args)
    return (y, last) if return_state else y


def ssm_step_selective_(state, u, delta, A, B_proj, C_proj, D=None, *, z=None, delta_bias=None, delta_softplus=True):
    """``ssm_scan_selective`` for one more position: u, delta, z (batch, channels), B_proj, C_proj
    (batch, states) or (batch, groups, states). Returns y (batch, channels) and updates ``state``
    (batch, channels, states) fp32 in place. Without gradients."""
    name = "ssm_step_selective_"
    given = (state, u, delta, A, B_proj, C_proj, D, z, delta_bias)
    _check(name, "u", u, ("state", "u", "delta", "A", "B_proj", "C_proj", "D", "z", "delta_bias"), given)
    if u.dim() != 2:
        raise ValueError(f"{name}: u is (batch, channels), got {tuple(u.shape)}")
    _no_grad_only(name, given)
    u, delta, A, B, C, D, z, bias = _scan_operands(name, u, delta, A, B_proj, C_proj, D, z, delta_bias, u.shape[:1])
    b, e = u.shape
    m = A.shape[1]
    _shape(name, "state", state, (b, e, m))
    if state.dtype is not _F32:
        raise TypeError(f"{name}: state must be float32, got {state.dtype}")
    dev = u.device
    y = _like(u)
    code = _CODE[B.dtype]
    vals = [*_r3(state, b, e, m), *_r2(u, b, e), *_r2(delta, b, e), *_r2(A, e, m)]
    if B.dim() == 2:  # one group
        vals += (*L.rec3_of2(B, code, b, m), *L.rec3_of2(C, code, b, m))
    else:
        g = B.shape[1]
        vals += (*L.rec3(B, code, b, g, m), *L.rec3(C, code, b, g, m))
    vals += (*_r1(D, e), *_r2(z, b, e), *_r1(bias, e), *_r2(y, b, e))
    a = L.Records(vals)
    p = [_at(a.base, vals, i) for i in range(10)]
    with L.on_device(dev):
        rc = L.load().m3_selective_step(*p[:9], 1 if delta_softplus else 0, p[9], L.stream_ptr(dev))
    if rc:
        L.check(rc, "m3_selective_step")
    _written(state)
    return y
