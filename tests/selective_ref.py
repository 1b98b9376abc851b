"""The selective scan and the causal convolution in float64, with their gradients written out, and the
same sums over the magnitudes of their terms, which the tests' error bounds are made of."""

import torch


def silu(v):
    return v * torch.sigmoid(v)


def silu_slope(v):
    p = torch.sigmoid(v)
    return p * (1 + v * (1 - p))


def silu_slope_terms(v):
    """The magnitudes of the slope's two terms s + s v (1 - s). They cancel at v = -1.2785, where the slope is 0 but a sigmoid
    that is off by a relative d (a few 2^-23) moves it by s |v| s d or so: the bound there is one on the terms."""
    p = torch.sigmoid(v)
    return p + p * v.abs() * (1 - p)


def valid(lengths, batch, length, device):
    n = torch.full((batch,), length, device=device) if lengths is None else lengths.clamp(0, length)
    return torch.arange(length, device=device) < n[:, None]


def scan(u, delta, A, B, C, D=None, z=None, bias=None, softplus=True, h0=None, lengths=None, dy=None, dstate=None,
         magnitudes=False):
    """Outputs y and state, and with dy the gradients, as a dict. With ``magnitudes`` every product counts
    with its absolute value, so that the results bound the sums of the terms' magnitudes."""
    mag = (lambda t: t.abs()) if magnitudes else (lambda t: t)
    f = [None if t is None else t.detach().double() for t in (u, delta, A, B, C, D, z, bias, h0, dy, dstate)]
    u, delta, A, B, C, D, z, bias, h0, dy, dstate = f
    b, n, e = u.shape
    m = A.shape[1]
    if B.dim() == 3:
        B, C = B.unsqueeze(2), C.unsqueeze(2)
    g = B.shape[2]
    keep = valid(lengths, b, n, u.device)
    k1, k2 = keep.unsqueeze(-1), keep[..., None, None]
    zero = torch.zeros((), dtype=torch.float64, device=u.device)
    raw = delta if bias is None else delta + bias
    dt = torch.nn.functional.softplus(raw, threshold=100.0) if softplus else raw
    dt, uv = torch.where(k1, dt, zero), mag(torch.where(k1, u, zero))
    Bv, Cv = mag(torch.where(k2, B, zero)), mag(torch.where(k2, C, zero))
    Be = Bv.repeat_interleave(e // g, 2) if g > 1 else Bv
    Ce = Cv.repeat_interleave(e // g, 2) if g > 1 else Cv
    a = torch.exp(dt.unsqueeze(-1) * A)
    h = torch.zeros(b, e, m, dtype=torch.float64, device=u.device) if h0 is None else mag(h0)
    hs = [h]
    for t in range(n):
        h = a[:, t] * h + mag(dt[:, t] * uv[:, t]).unsqueeze(-1) * Be[:, t]
        hs.append(h)
    H = torch.stack(hs, 1)
    Dv = zero if D is None else mag(D)
    pre = (Ce * H[:, 1:]).sum(-1) + Dv * uv
    gate = torch.ones_like(pre) if z is None else mag(silu(torch.where(k1, z, zero)))
    out = {"y": torch.where(k1, pre * gate, zero), "state": h}
    if dy is None:
        return out
    dout = mag(torch.where(k1, dy, zero))
    dp = dout * gate
    G = torch.zeros(b, e, m, dtype=torch.float64, device=u.device) if dstate is None else mag(dstate)
    du, ddt = torch.zeros_like(uv), torch.zeros_like(uv)
    dB, dC = torch.zeros_like(B), torch.zeros_like(C)
    dA = torch.zeros_like(A)
    for t in range(n - 1, -1, -1):
        G = G + Ce[:, t] * dp[:, t].unsqueeze(-1)
        into = (G * Be[:, t]).sum(-1)
        w = G * a[:, t] * H[:, t]
        du[:, t] = into * mag(dt[:, t]) + Dv * dp[:, t]
        ddt[:, t] = into * uv[:, t] + (w * mag(A)).sum(-1)
        dA += (w * mag(dt[:, t]).unsqueeze(-1)).sum(0)
        dB[:, t] = (G * mag(dt[:, t] * uv[:, t]).unsqueeze(-1)).view(b, g, e // g, m).sum(2)
        dC[:, t] = (H[:, t + 1] * dp[:, t].unsqueeze(-1)).view(b, g, e // g, m).sum(2)
        G = G * a[:, t]
    draw = ddt * torch.sigmoid(raw) if softplus else ddt
    draw = torch.where(k1, draw, zero)
    out.update(u=torch.where(k1, du, zero), delta=draw, A=dA, B=torch.where(k2, dB, zero), C=torch.where(k2, dC, zero),
               D=(dp * uv).sum((0, 1)), bias=draw.sum((0, 1)), h0=G)
    if z is not None:
        out["z"] = torch.where(k1, dout * pre * (silu_slope_terms(z) if magnitudes else silu_slope(z)), zero)
    return out


def conv(x, w, bias=None, act=False, init=None, lengths=None, dy=None, dlast=None, magnitudes=False):
    """y and the last rows, and with dy the gradients, as a dict."""
    mag = (lambda t: t.abs()) if magnitudes else (lambda t: t)
    x, w, bias, init, dy, dlast = [None if t is None else t.detach().double() for t in (x, w, bias, init, dy, dlast)]
    b, n, e = x.shape
    k = w.shape[1]
    keep = valid(lengths, b, n, x.device).unsqueeze(-1)
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    xv = torch.where(keep, x, zero)
    front = torch.zeros(b, k - 1, e, dtype=torch.float64, device=x.device) if init is None else init
    whole = torch.cat([front, xv], 1)
    pre, size = torch.zeros_like(xv), torch.zeros_like(xv)
    for i in range(k):
        pre += whole[:, i:i + n] * w[:, i]
        size += (whole[:, i:i + n] * w[:, i]).abs()
    if bias is not None:
        pre, size = pre + bias, size + bias.abs()
    y = (silu(pre) if act else pre) if not magnitudes else size
    out = {"y": torch.where(keep, y, zero)}
    count = (torch.full((b,), n, device=x.device) if lengths is None else lengths.clamp(0, n)).long()
    rows = (count[:, None] + torch.arange(k - 1, device=x.device)).unsqueeze(-1).expand(b, k - 1, e)
    out["state"] = whole.gather(1, rows)
    if dy is None:
        return out
    # the slope's own error follows that of pre: its derivative is at most 1/2 in magnitude
    slope = silu_slope(pre) if act else torch.ones_like(pre)
    if magnitudes:
        slope = slope.abs() + (0.5 * size if act else 0.0) + (1.0 if act else 0.0)
    d = torch.where(keep, mag(dy) * slope, zero)
    dw, dwhole = torch.zeros_like(w), torch.zeros_like(whole)
    for i in range(k):
        dwhole[:, i:i + n] += d * mag(w[:, i])
        dw[:, i] = (d * mag(whole[:, i:i + n])).sum((0, 1))
    if dlast is not None:
        dwhole.scatter_add_(1, rows, mag(dlast))
    out.update(x=torch.where(keep, dwhole[:, k - 1:], zero), weight=dw, bias=d.sum((0, 1)), init=dwhole[:, :k - 1])
    return out
