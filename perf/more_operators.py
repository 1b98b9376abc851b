"""Selective scans of a diagonal state space and beam search over their states, as measured cases.

causal_conv, causal_conv_step_           short depthwise causal convolution, over a sequence and for one token
ssm_scan_selective, ssm_step_selective_  selective state space scan, over a sequence and for one token
beam_select                              the best continuations over beams and vocabulary
reorder_states_                          rows of many cache tensors moved to the beams that continue them

``own`` chooses between the plain form in elementary torch operations and the calls of the
package's operators. Sequences are (batch, length, channels) with contiguous channels, as views
of a projection's output; widths are those of this package's configurations.
"""

import os
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
_MOST = 8 * 2048 * 2048 * 16  # positions x channels x states of the largest listed scan


# ------------------------------------------------------------------------------ cases
def listed():
    return [
        # a padded batch of prompts through the convolution, which leaves its state for decoding
        dict(name="convolution, padded prompts", op="conv", dtype="bf16", batch=4, length=777, width=2048, taps=4, silu=True,
             bias=True, initial=False, lengths=True, state=True, grad=False),
        # the convolution of a training step, with its gradients: the largest
        dict(name="convolution, training", op="conv", dtype="bf16", batch=8, length=2048, width=2048, taps=4, silu=True,
             bias=True, initial=False, lengths=False, state=False, grad=True),
        # one token of one sequence through a small layer's convolution: latency
        dict(name="convolution, one token", op="conv_step", dtype="bf16", batch=1, width=512, taps=4, silu=True, bias=True),
        # a long prompt of one sequence, continued from a state, which it leaves for decoding
        dict(name="scan, one long prompt", op="scan", dtype="bf16", batch=1, length=8192, width=2048, states=16, groups=1,
             z=True, softplus=True, initial=True, lengths=False, state=True, grad=False),
        # training a small model in 32 bits: an odd width, an odd length, ragged sequences
        dict(name="scan, training, 32 bits", op="scan", dtype="fp32", batch=3, length=341, width=507, states=16, groups=1,
             z=True, softplus=True, initial=False, lengths=True, state=False, grad=True),
        # the scan of a training step, with its gradients: the largest
        dict(name="scan, training", op="scan", dtype="bf16", batch=8, length=2048, width=2048, states=16, groups=1, z=True,
             softplus=True, initial=False, lengths=False, state=False, grad=True),
        # one token of 256 sequences through a layer of the default width
        dict(name="scan, one token of a batch", op="scan_step", dtype="bf16", batch=256, width=5120, states=16, groups=1,
             z=True, softplus=True),
        # one prompt's beams: latency
        dict(name="beams, one prompt", op="beam", dtype="bf16", batch=1, beams=4, vocab=50000, pitch=50000, num=4,
             finished=False, first=False),
        # a serving batch with a long vocabulary: twice as many candidates as beams, some beams have ended
        dict(name="beams, a large batch", op="beam", dtype="bf16", batch=64, beams=8, vocab=131072, pitch=131072, num=16,
             finished=True, first=False),
        # the cache of a small model with three tensors a layer, one prompt's beams in place: latency
        dict(name="reorder a small cache", op="reorder", batch=1, beams=4, source=4, layers=4, heads=16, headdim=32,
             states=64, mimo=True, dtype="fp32", in_place=True),
        # prompts' caches forked into their beams' caches
        dict(name="fork prompts to beams", op="reorder", batch=4, beams=8, source=1, layers=16, heads=32, headdim=64,
             states=64, mimo=False, dtype="fp32", in_place=False),
        # a model's cache after a step of beam search: most beams go on from another one
        dict(name="reorder a model's cache", op="reorder", batch=8, beams=8, source=8, layers=16, heads=32, headdim=64,
             states=64, mimo=False, dtype="fp32", in_place=True),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["conv", "conv", "conv_step", "scan", "scan", "scan", "scan_step", "beam", "beam", "reorder"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    yes = lambda p: rng.random() < p  # noqa: E731
    if op in ("conv", "scan"):
        grad = yes(0.5)
        length = _log_uniform(rng, 1, 16384)
        if op == "conv":
            most = 33_000_000 // (2 if dtype == "fp32" else 1) // length
            width = _log_uniform(rng, 64, max(64, min(5120, most)))
            batch = _log_uniform(rng, 1, max(1, min(64, most // width)))
            return dict(op=op, dtype=dtype, batch=batch, length=length, width=width, taps=rng.choice([2, 3, 4, 4]),
                        silu=yes(0.7), bias=yes(0.7), initial=yes(0.4), lengths=yes(0.4), state=yes(0.5), grad=grad)
        groups = rng.choice([1, 1, 1, 2, 4])
        states = rng.choice([4, 8, 16, 16, 16, 24, 32, 64, 128])
        most = _MOST // max(16, states) // (2 if dtype == "fp32" else 1) // length
        width = groups * _log_uniform(rng, 32, max(32, min(5120, most) // groups))
        batch = _log_uniform(rng, 1, max(1, min(64, most // width)))
        return dict(op=op, dtype=dtype, batch=batch, length=length, width=width, states=states, groups=groups, z=yes(0.7),
                    softplus=yes(0.8), initial=yes(0.4), lengths=yes(0.4), state=yes(0.5), grad=grad)
    batch = _log_uniform(rng, 1, 256)
    if op == "conv_step":
        return dict(op=op, dtype=dtype, batch=batch, width=_log_uniform(rng, 64, 5120), taps=rng.choice([2, 3, 4, 4]),
                    silu=yes(0.7), bias=yes(0.7))
    if op == "scan_step":
        groups = rng.choice([1, 1, 2, 4])
        states = rng.choice([4, 8, 16, 16, 24, 32, 64, 128])
        width = groups * _log_uniform(rng, 32, 5120 // groups)
        return dict(op=op, dtype=dtype, batch=min(batch, max(1, 20_000_000 // (width * states))), width=width, states=states,
                    groups=groups, z=yes(0.7), softplus=yes(0.8))
    if op == "beam":
        beams = rng.choice([1, 2, 3, 4, 5, 8, 16])
        vocab = _log_uniform(rng, 300, 131072)
        most = 50_000_000 // (2 if dtype == "fp32" else 1) // (vocab * beams)
        return dict(op=op, dtype=dtype, batch=_log_uniform(rng, 1, max(1, min(128, most))), beams=beams, vocab=vocab,
                    pitch=vocab + rng.choice([0, 0, 3, 8]), num=beams * rng.choice([1, 2]), finished=yes(0.5),
                    first=yes(0.2))
    beams = rng.choice([2, 3, 4, 5, 8, 16])
    in_place = yes(0.7)
    mimo = yes(0.5)
    heads, headdim = rng.choice([4, 16, 32, 48]), rng.choice([32, 64])
    states = rng.choice([32, 64, 128])
    row = 4 * heads * (2 * states * (1 if mimo else headdim) + states // 4)
    layers = _log_uniform(rng, 1, 20)
    most = max(1, 1_000_000_000 // (row * layers * beams))
    return dict(op=op, batch=_log_uniform(rng, 1, min(32, most)), beams=beams, source=beams if in_place else rng.choice([1, beams + 1]),
                layers=layers, heads=heads, headdim=headdim, states=states, mimo=mimo, dtype="fp32", in_place=in_place)


# ----------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, dtype, *shape):
    return torch.empty(*shape, dtype=dtype, device="cuda").normal_(0.0, 1.0, generator=g)


def _lengths(case, g):
    """Sequences of a padded batch fill between a third and all of it."""
    full = case["length"]
    n = (full * (0.34 + 0.66 * torch.rand(case["batch"], device="cuda", generator=g))).ceil().long()
    return n.clamp(max=full)


def _leaf(case, t):
    return t.detach().requires_grad_(case.get("grad", False))


def _scan_inputs(case, g, lead):
    """Operands as the projections of a layer leave them: u and z are halves of one output, delta,
    B and C come from another."""
    e, n, k = case["width"], case["states"], case["groups"]
    dtype = _DTYPES[case["dtype"]]
    uz = _normal(g, dtype, *lead, 2 * e)
    s = dict(u=uz[..., :e], z=uz[..., e:] if case["z"] else None)
    s["delta"] = _normal(g, dtype, *lead, e) * 0.5
    bc = _normal(g, dtype, *lead, 2 * k * n)
    shape = (*lead, k, n) if k > 1 else (*lead, n)
    s["B"], s["C"] = bc[..., :k * n].reshape(shape), bc[..., k * n:].reshape(shape)
    # step sizes between 0.001 and 0.1, decay rates 1 .. N with some spread
    dt = torch.exp(torch.rand(e, device="cuda", generator=g) * 4.6 - 6.9)
    if case["softplus"]:
        s["bias"] = dt + torch.log(-torch.expm1(-dt))
    else:
        s["bias"] = None
        s["delta"] = (dt * torch.exp(s["delta"].float())).to(dtype)
    s["A"] = -torch.arange(1, n + 1, device="cuda").float() * torch.exp(0.1 * _normal(g, torch.float32, e, n))
    s["D"] = 1.0 + 0.1 * _normal(g, torch.float32, e)
    return s


def _cache(case, rows, g):
    """A decode cache (angles and two state tensors a layer) in one buffer."""
    h, p, n = case["heads"], case["headdim"], case["states"]
    state = (rows, h, n) if case["mimo"] else (rows, h, p, n)
    shapes = [(rows, h, n // 4), state, state] * case["layers"]
    sizes = [torch.Size(x).numel() for x in shapes]
    flat = torch.zeros(sum(sizes), dtype=_DTYPES[case["dtype"]], device="cuda")
    if g is not None:
        flat.normal_(0.0, 1.0, generator=g)
    return flat, [t.view(x) for t, x in zip(flat.split(sizes), shapes)]


def prepare(case, seed):
    g = _generator(seed)
    op, dtype = case["op"], _DTYPES[case["dtype"]]
    s = dict(case=case)
    if op in ("conv", "conv_step"):
        e, k = case["width"], case["taps"]
        lead = (case["batch"], case["length"]) if op == "conv" else (case["batch"],)
        s["x"] = _leaf(case, _normal(g, dtype, *lead, 2 * e)[..., :e])
        s["weight"] = _leaf(case, (_normal(g, torch.float32, e, k) * k ** -0.5).to(dtype))
        s["bias"] = _leaf(case, (0.3 * _normal(g, torch.float32, e)).to(dtype)) if case["bias"] else None
        s["initial"] = None
        if op == "conv_step" or case["initial"]:
            s["initial"] = _leaf(case, _normal(g, dtype, case["batch"], k - 1, e))
    elif op in ("scan", "scan_step"):
        lead = (case["batch"], case["length"]) if op == "scan" else (case["batch"],)
        x = _scan_inputs(case, g, lead)
        s.update({n: None if t is None else _leaf(case, t) for n, t in x.items()})
        s["initial"] = None
        if op == "scan_step" or case["initial"]:
            s["initial"] = _leaf(case, 0.3 * _normal(g, torch.float32, case["batch"], case["width"], case["states"]))
    elif op == "beam":
        b, k = case["batch"], case["beams"]
        logits = torch.empty(b, k, case["pitch"], dtype=dtype, device="cuda").normal_(0.0, 2.5, generator=g)
        # a few tokens that the model finds likely, apart from one another
        likely = torch.randint(0, case["vocab"], (b, k, 1), device="cuda", generator=g)
        likely = (likely + torch.arange(24, device="cuda") * (case["vocab"] // 24)) % case["vocab"]
        logits.scatter_(2, likely, (5.0 + 5.0 * torch.rand(b, k, 24, device="cuda", generator=g)).to(dtype))
        s["logits"] = logits[..., :case["vocab"]]
        # scores of the beams so far, the best first; in the first step all but one are empty
        gaps = torch.rand(b, k, device="cuda", generator=g)
        s["scores"] = -8.0 - gaps.cumsum(1)
        if case["first"]:
            s["scores"][:, 1:] = float("-inf")
        s["finished"] = torch.rand(b, k, device="cuda", generator=g) < 0.25 if case["finished"] else None
    else:
        b, k, src = case["batch"], case["beams"], case["source"]
        s["flat"], s["states"] = _cache(case, b * src, g)
        s["out_flat"], s["out"] = (None, None) if case["in_place"] else _cache(case, b * k, None)
        # the better beams are continued more often, as their candidates are sorted by score
        r = torch.rand(b, k, device="cuda", generator=g)
        s["parents"] = (src * r * r).long().clamp(max=src - 1)
    if op in ("conv", "scan"):
        s["lengths"] = _lengths(case, g) if case["lengths"] else None
        if case["grad"]:
            s["dy"] = _normal(g, dtype, case["batch"], case["length"], case["width"])
            if case["state"]:
                last = (case["taps"] - 1, case["width"]) if op == "conv" else (case["width"], case["states"])
                s["dstate"] = _normal(g, dtype if op == "conv" else torch.float32, case["batch"], *last)
    return s


# ------------------------------------------------------------------------ plain forms
def _silu_and_slope(v):
    """silu(v) and its derivative."""
    p = torch.sigmoid(v)
    return v * p, p * (1 + v * (1 - p))


def _padding(s, length):
    """(batch, length, 1), 1 where a position counts; None where all do."""
    if s.get("lengths") is None:
        return None
    return (torch.arange(length, device="cuda") < s["lengths"][:, None]).unsqueeze(-1)


def _plain_conv(s):
    c, x, k = s["case"], s["x"].detach(), s["case"]["taps"]
    b, n, e = x.shape
    keep = _padding(s, n)
    xf = x.float() if keep is None else torch.where(keep, x.float(), 0.0)
    before = torch.zeros(b, k - 1, e, device="cuda") if s["initial"] is None else s["initial"].detach().float()
    whole = torch.cat([before, xf], 1)
    w = s["weight"].detach().float()
    pre = sum([whole[:, i:i + n] * w[:, i] for i in range(k)])
    if s["bias"] is not None:
        pre = pre + s["bias"].detach().float()
    y, slope = _silu_and_slope(pre) if c["silu"] else (pre, 1.0)
    y = y if keep is None else torch.where(keep, y, 0.0)
    out = [y.to(x.dtype)]
    # the last k - 1 rows in front of each sequence's end
    count = torch.full((b,), n, device="cuda") if keep is None else s["lengths"]
    rows = (count[:, None] + torch.arange(k - 1, device="cuda")).unsqueeze(-1).expand(b, k - 1, e)
    if c["state"]:
        out.append(whole.gather(1, rows).to(x.dtype))
    if not c["grad"]:
        return out
    d = s["dy"].float() * slope
    d = d if keep is None else torch.where(keep, d, 0.0)
    dwhole = sum([torch.nn.functional.pad(d * w[:, i], (0, 0, i, k - 1 - i)) for i in range(k)])
    if c["state"]:
        dwhole = dwhole.scatter_add(1, rows, s["dstate"].float())
    dw = torch.stack([(d * whole[:, i:i + n]).sum((0, 1)) for i in range(k)], 1)
    dx = dwhole[:, k - 1:] if keep is None else torch.where(keep, dwhole[:, k - 1:], 0.0)
    out += [dx.to(x.dtype), dw.to(x.dtype)]
    if s["bias"] is not None:
        out.append(d.sum((0, 1)).to(x.dtype))
    if s["initial"] is not None:
        out.append(dwhole[:, :k - 1].to(x.dtype))
    return out


def _plain_conv_step(s):
    c, x, state = s["case"], s["x"], s["initial"]
    window = torch.cat([state, x.unsqueeze(1)], 1)
    pre = (window.float() * s["weight"].float().t()).sum(1)
    if s["bias"] is not None:
        pre = pre + s["bias"].float()
    state.copy_(window[:, 1:])
    return [(_silu_and_slope(pre)[0] if c["silu"] else pre).to(x.dtype), state]


def _linear_scan(a, v):
    """h[t] = a[t] h[t - 1] + v[t] along dimension 1 from h[-1] = 0, by doubling; uses up both."""
    step, n = 1, a.shape[1]
    while step < n:
        v[:, step:] += a[:, step:] * v[:, :-step]
        a[:, step:] *= a[:, :-step].clone()
        step *= 2
    return v


def _per_channel(t, width):
    """B or C as (..., groups, 1, states), to be spread over the channels of each group."""
    t = t.detach().float()
    return (t if t.dim() == 4 else t.unsqueeze(-2)).unsqueeze(-2)


def _step_sizes(s):
    raw = s["delta"].detach().float()
    if s["bias"] is None:
        return raw, torch.ones_like(raw)
    raw = raw + s["bias"].detach()
    return torch.nn.functional.softplus(raw), torch.sigmoid(raw)


def _plain_scan(s):
    c, u = s["case"], s["u"].detach()
    b, n, e = u.shape
    k, m = c["groups"], c["states"]
    keep = _padding(s, n)
    dt, dt_slope = _step_sizes(s)
    uf = u.float()
    B, C, D = _per_channel(s["B"], e), _per_channel(s["C"], e), s["D"].detach()
    if keep is not None:
        # padding neither decays the state nor adds to it
        dt, uf = torch.where(keep, dt, 0.0), torch.where(keep, uf, 0.0)
        B, C = torch.where(keep[..., None, None], B, 0.0), torch.where(keep[..., None, None], C, 0.0)
    A = s["A"].detach()
    a = torch.exp(dt.unsqueeze(-1) * A)
    v = ((dt * uf).view(b, n, k, e // k, 1) * B).view(b, n, e, m)
    start = torch.zeros(b, e, m, device="cuda") if s["initial"] is None else s["initial"].detach()
    v[:, 0] += a[:, 0] * start
    h = _linear_scan(a.clone() if c["grad"] else a, v)
    y = (h.view(b, n, k, e // k, m) * C).sum(-1).view(b, n, e) + D * uf
    gate, gate_slope = (1.0, 0.0) if s["z"] is None else _silu_and_slope(s["z"].detach().float())
    out = y * gate
    outs = [(out if keep is None else torch.where(keep, out, 0.0)).to(u.dtype)]
    if c["state"]:
        outs.append(h[:, -1].clone())
    if not c["grad"]:
        return outs
    dout = s["dy"].float() if keep is None else torch.where(keep, s["dy"].float(), 0.0)
    dy = dout * gate
    # the gradient of each state: from its output and from the next state
    gr = (dy.view(b, n, k, e // k, 1) * C).view(b, n, e, m)
    if c["state"]:
        gr[:, -1] += s["dstate"]
    later = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1).flip(1)
    gr = _linear_scan(later, gr.flip(1)).flip(1)
    dC = (dy.view(b, n, k, e // k, 1) * h.view(b, n, k, e // k, m)).sum(3)
    dB = ((dt * uf).view(b, n, k, e // k, 1) * gr.view(b, n, k, e // k, m)).sum(3)
    into = (gr.view(b, n, k, e // k, m) * B).sum(-1).view(b, n, e)
    before = torch.cat([start.unsqueeze(1), h[:, :-1]], 1)
    through = gr * before * a
    dA = (through * dt.unsqueeze(-1)).sum((0, 1))
    ddt = (into * uf + (through * A).sum(-1)) * dt_slope
    if keep is not None:
        ddt = torch.where(keep, ddt, 0.0)
        dB, dC = torch.where(keep[..., None], dB, 0.0), torch.where(keep[..., None], dC, 0.0)
    du = into * dt + D * dy
    outs += [du.to(u.dtype), ddt.to(s["delta"].dtype), dA, dB.view_as(s["B"]).to(s["B"].dtype),
             dC.view_as(s["C"]).to(s["C"].dtype), (dy * uf).sum((0, 1))]
    if s["z"] is not None:
        dz = dout * y * gate_slope
        outs.append(dz.to(u.dtype))
    if s["bias"] is not None:
        outs.append(ddt.sum((0, 1)))
    if s["initial"] is not None:
        outs.append(gr[:, 0] * a[:, 0])
    return outs


def _plain_scan_step(s):
    c, u, state = s["case"], s["u"], s["initial"]
    b, e = u.shape
    k, m = c["groups"], c["states"]
    dt, _ = _step_sizes(s)
    B, C = [(t if t.dim() == 3 else t.unsqueeze(1)).float().unsqueeze(2) for t in (s["B"], s["C"])]
    v = ((dt * u.float()).view(b, k, e // k, 1) * B).view(b, e, m)
    state.mul_(torch.exp(dt.unsqueeze(-1) * s["A"])).add_(v)
    y = (state.view(b, k, e // k, m) * C).sum(-1).view(b, e) + s["D"] * u.float()
    if s["z"] is not None:
        y = y * _silu_and_slope(s["z"].float())[0]
    return [y.to(u.dtype), state]


_END = 2


def _plain_beam(s):
    c, logits = s["case"], s["logits"]
    b, k, v = logits.shape
    x = logits.double()
    peak = x.amax(-1, keepdim=True)
    logp = x - peak - torch.log(torch.exp(x - peak).sum(-1, keepdim=True))
    if s["finished"] is not None:
        # a beam that has ended goes on with the end token alone, at no cost
        only = torch.where(torch.arange(v, device="cuda") == _END, 0.0, float("-inf")).double()
        logp = torch.where(s["finished"].unsqueeze(-1), only, logp)
    total = (s["scores"].double().unsqueeze(-1) + logp).view(b, k * v)
    best, at = total.sort(dim=1, descending=True, stable=True)
    best, at = best[:, :c["num"]], at[:, :c["num"]]
    return [best.float(), at // v, at % v]


def _plain_reorder(s):
    c = s["case"]
    rows = (s["parents"] + c["source"] * torch.arange(c["batch"], device="cuda")[:, None]).flatten()
    [o.copy_(t[rows]) for o, t in zip(s["out"] or s["states"], s["states"])]
    return [s["out_flat"] if s["out"] else s["flat"]]


# -------------------------------------------------------------------- the package's calls
def _package():
    if "mamba3_ssm" not in sys.modules:
        sys.path.insert(0, os.path.join(os.getcwd(), "mamba3-ssm_b200"))
    import mamba3_ssm
    return mamba3_ssm


def _own(s):
    m, c = _package(), s["case"]
    op = c["op"]
    if op == "conv_step":
        y = m.causal_conv_step_(s["initial"], s["x"], s["weight"], s["bias"], activation="silu" if c["silu"] else None)
        return [y, s["initial"]]
    if op == "scan_step":
        y = m.ssm_step_selective_(s["initial"], s["u"], s["delta"], s["A"], s["B"], s["C"], s["D"], z=s["z"],
                                  delta_bias=s["bias"], delta_softplus=c["softplus"])
        return [y, s["initial"]]
    if op == "beam":
        return list(m.beam_select(s["logits"], s["scores"], c["num"], finished=s["finished"], end_token=_END))
    if op == "reorder":
        m.reorder_states_(s["states"], s["parents"], out=s["out"])
        return [s["out_flat"] if s["out"] else s["flat"]]
    if op == "conv":
        r = m.causal_conv(s["x"], s["weight"], s["bias"], activation="silu" if c["silu"] else None,
                          initial_state=s["initial"], lengths=s["lengths"], return_state=c["state"])
        leaves = [s["x"], s["weight"], s["bias"], s["initial"]]
    else:
        r = m.ssm_scan_selective(s["u"], s["delta"], s["A"], s["B"], s["C"], s["D"], z=s["z"], delta_bias=s["bias"],
                                 delta_softplus=c["softplus"], initial_state=s["initial"], lengths=s["lengths"],
                                 return_state=c["state"])
        leaves = [s["u"], s["delta"], s["A"], s["B"], s["C"], s["D"], s["z"], s["bias"], s["initial"]]
    r = list(r) if c["state"] else [r]
    if not c["grad"]:
        return r
    up = [s["dy"], s["dstate"]] if c["state"] else [s["dy"]]
    grads = torch.autograd.grad(r, [t for t in leaves if t is not None], up)
    return [t.detach() for t in r] + list(grads)


def run(state):
    if own:
        return _own(state)
    return {"conv": _plain_conv, "conv_step": _plain_conv_step, "scan": _plain_scan, "scan_step": _plain_scan_step,
            "beam": _plain_beam, "reorder": _plain_reorder}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------- work
def work(case):
    op, size = case["op"], _SIZE[case["dtype"]]
    if op == "reorder":
        rows = case["batch"] * case["beams"]
        h, n = case["heads"], case["states"]
        row = _SIZE[case["dtype"]] * case["layers"] * h * (n // 4 + 2 * n * (1 if case["mimo"] else case["headdim"]))
        if case["source"] == 1:
            return {"bytes": row * (case["batch"] + rows), "flops": 0.0}
        # with r uniform, beam j goes on from its own place with probability sqrt((j + 1) / k) - sqrt(j / k);
        # the parents of the others that differ from one another are read once
        k, src = case["beams"], case["source"]
        own_place = sum(((j + 1) / src) ** 0.5 - (j / src) ** 0.5 for j in range(min(k, src))) if case["in_place"] else 0.0
        read = sum(1 - (1 - (((j + 1) / src) ** 0.5 - (j / src) ** 0.5)) ** k for j in range(src))
        if case["in_place"]:
            read *= 1 - own_place / k
        return {"bytes": row * case["batch"] * (read + k - own_place), "flops": 0.0}
    if op == "beam":
        n = case["batch"] * case["beams"]
        return {"bytes": n * (0.75 if case["finished"] else 1.0) * case["vocab"] * size + 4 * n + 20 * case["batch"] * case["num"],
                "flops": 4.0 * n * case["vocab"]}
    e = case["width"]
    # three quarters of a padded batch count on average; outputs are written whole
    count = case["batch"] * case.get("length", 1)
    used = count * (0.67 if case.get("lengths") else 1.0)
    if op in ("conv", "conv_step"):
        state = case["batch"] * (case["taps"] - 1) * e * size
        if op == "conv_step":
            return {"bytes": 2 * state + e * size * (2 * count + case["taps"] + 1), "flops": count * e * (2.0 * case["taps"] + 5)}
        state = state * (case["initial"] + case["state"])
        if case["grad"]:  # forward: x, y; backward: x, dy, dx
            return {"bytes": e * size * (3 * used + 2 * count) + 2 * state, "flops": used * e * (8.0 * case["taps"] + 14)}
        return {"bytes": e * size * (used + count) + state, "flops": used * e * (2.0 * case["taps"] + 5)}
    n, z = case["states"], int(case["z"])
    bc = 2 * case["groups"] * n * size
    if op == "scan_step":
        return {"bytes": count * (8 * e * n + e * size * (3 + z) + bc) + 4 * e * (n + 2), "flops": count * e * n * 7.0}
    state = 4 * case["batch"] * e * n * (case["initial"] + case["state"])
    fwd = used * (e * size * (2 + z) + bc) + count * e * size + state + 4 * e * (n + 2)
    if not case["grad"]:
        return {"bytes": fwd, "flops": used * e * n * 7.0}
    bwd = used * (e * size * (3 + z) + bc) + count * (e * size * (2 + z) + bc) + state + 8 * e * (n + 2)
    return {"bytes": fwd + bwd, "flops": used * e * n * 30.0}


# ------------------------------------------------------------- the definition in 64 bits
def _exact_leaf(t):
    return None if t is None else t.detach().double().requires_grad_(True)


def _exact_grads(outs, ups, leaves):
    """Differentiates the definition; a leaf that nothing depends on has a gradient of zeros."""
    leaves = [t for t in leaves if t is not None]
    got = torch.autograd.grad(outs, leaves, [u.double() for u in ups], allow_unused=True)
    return [torch.zeros_like(t) if g is None else g for t, g in zip(leaves, got)]


def _exact_conv(s):
    c, f = s["case"], torch.nn.functional
    x, w, bias, init = (_exact_leaf(s[n]) for n in ("x", "weight", "bias", "initial"))
    b, n, e = x.shape
    k = c["taps"]
    outs, lasts = [], []
    for i in range(b):
        m = n if s["lengths"] is None else int(s["lengths"][i])
        head = torch.zeros(k - 1, e, dtype=torch.float64, device="cuda") if init is None else init[i]
        row = torch.cat([head, x[i, :m]])
        lasts.append(row[m:])
        y = f.conv1d(row.t().unsqueeze(0), w.unsqueeze(1), bias, groups=e)[0].t()
        outs.append(f.pad(f.silu(y) if c["silu"] else y, (0, 0, 0, n - m)))
    y, last = torch.stack(outs), torch.stack(lasts)
    if not c["grad"]:
        return [y.detach()] + ([last.detach()] if c["state"] else [])
    d = _exact_grads([y, last] if c["state"] else [y], [s["dy"], s["dstate"]] if c["state"] else [s["dy"]], [x, w, bias, init])
    return [y.detach()] + ([last.detach()] if c["state"] else []) + d


def _exact_scan(s):
    c, f = s["case"], torch.nn.functional
    names = ("u", "delta", "A", "B", "C", "D", "z", "bias", "initial")
    u, delta, A, B, C, D, z, bias, init = leaves = [_exact_leaf(s[n]) for n in names]
    if not c.get("grad"):
        leaves = [None if t is None else t.detach() for t in leaves]
        u, delta, A, B, C, D, z, bias, init = leaves
    step = s["case"]["op"] == "scan_step"
    add = (lambda t: t.unsqueeze(1)) if step else (lambda t: t)
    n = 1 if step else c["length"]
    h = torch.zeros(c["batch"], c["width"], c["states"], dtype=torch.float64, device="cuda") if init is None else init
    each = c["width"] // c["groups"]
    ys = []
    parts = [add(t).unbind(1) for t in (u, delta, B, C)]
    for t, (ut, dt, Bt, Ct) in enumerate(zip(*parts)):
        if c["groups"] > 1:
            Bt, Ct = Bt.repeat_interleave(each, 1), Ct.repeat_interleave(each, 1)
        else:
            Bt, Ct = Bt.unsqueeze(1), Ct.unsqueeze(1)
        dt = dt if bias is None else f.softplus(dt + bias, threshold=100.0)
        new = torch.exp(dt.unsqueeze(2) * A) * h + (dt * ut).unsqueeze(2) * Bt
        y = (new * Ct).sum(2) + D * ut
        if s.get("lengths") is not None:
            live = (t < s["lengths"])[:, None]
            new, y = torch.where(live.unsqueeze(2), new, h), torch.where(live, y, 0.0)
        h = new
        ys.append(y)
    y = torch.stack(ys, 1)
    if z is not None:
        y = y * f.silu(add(z))
    if step:
        return [y[:, 0], h]
    if not c["grad"]:
        return [y] + ([h] if c["state"] else [])
    d = _exact_grads([y, h] if c["state"] else [y], [s["dy"], s["dstate"]] if c["state"] else [s["dy"]], leaves)
    return [y.detach()] + ([h.detach()] if c["state"] else []) + d


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "conv":
        return _exact_conv(s)
    if op == "conv_step":
        window = torch.cat([s["initial"], s["x"][:, None]], 1).double()
        y = torch.einsum("bke,ek->be", window, s["weight"].double())
        y = y if s["bias"] is None else y + s["bias"]
        return [torch.nn.functional.silu(y) if case["silu"] else y, window[:, 1:]]
    if op in ("scan", "scan_step"):
        if case.get("grad") and case["batch"] * case["length"] * case["width"] * case["states"] > 2 ** 29:
            return None  # the states of all positions in 64 bits
        return _exact_scan(s)
    if op == "beam":
        every = s["scores"].double()[..., None] + torch.log_softmax(s["logits"].double(), -1)
        if s["finished"] is not None:
            ended = torch.full_like(every, float("-inf"))
            ended[..., _END] = s["scores"].double()
            every = torch.where(s["finished"][..., None], ended, every)
        return [every.flatten(1).topk(case["num"], dim=1).values, None, None]
    k, src = case["beams"], case["source"]
    at = (s["parents"] + src * torch.arange(case["batch"], device="cuda")[:, None]).flatten()
    moved = [t.double().index_select(0, at).flatten() for t in s["states"]]
    return [torch.cat(moved)]
