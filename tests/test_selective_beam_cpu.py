"""Without a GPU: the tests' float64 adjoints against autograd and differences, and what the selective scan's,
the convolution's and the beam search's entry points refuse, in Python and at the C boundary."""

import ctypes

import pytest
import torch

import selective_ref as R
from test_capi_cpu import _view


@pytest.fixture(scope="module")
def lib():
    from mamba3_ssm import _lib
    return _lib.load()


# ------------------------------------------------------------------- the float64 formulas
def _scan_case(g=2, softplus=True):
    torch.manual_seed(0)
    b, n, e, m = 2, 9, 6, 5
    mk = lambda *s: torch.randn(*s, dtype=torch.float64)  # noqa: E731
    x = dict(u=mk(b, n, e), delta=mk(b, n, e) if softplus else mk(b, n, e).abs() * 0.3, A=-torch.rand(e, m, dtype=torch.float64),
             B=mk(b, n, g, m), C=mk(b, n, g, m), D=mk(e), z=mk(b, n, e), bias=mk(e) if softplus else None, h0=mk(b, e, m))
    return x, mk(b, n, e), mk(b, e, m), torch.tensor([9, 4])


def _forward(x, softplus, lengths):
    """Written apart from selective_ref, for autograd."""
    b, n, e = x["u"].shape
    g = x["B"].shape[2]
    keep, h, ys = R.valid(lengths, b, n, "cpu"), x["h0"], []
    for t in range(n):
        raw = x["delta"][:, t] if x["bias"] is None else x["delta"][:, t] + x["bias"]
        dt = torch.nn.functional.softplus(raw, threshold=100.0) if softplus else raw
        Be, Ce = x["B"][:, t].repeat_interleave(e // g, 1), x["C"][:, t].repeat_interleave(e // g, 1)
        new = torch.exp(dt[..., None] * x["A"]) * h + (dt * x["u"][:, t])[..., None] * Be
        k = keep[:, t]
        h = torch.where(k[:, None, None], new, h)
        y = ((Ce * h).sum(-1) + x["D"] * x["u"][:, t]) * R.silu(x["z"][:, t])
        ys.append(torch.where(k[:, None], y, 0.0))
    return torch.stack(ys, 1), h


@pytest.mark.parametrize("g,softplus", [(1, True), (2, True), (3, False)])
def test_scan_formulas_against_autograd(g, softplus):
    x, dy, ds, lengths = _scan_case(g, softplus)
    leaves = {k: v.requires_grad_(True) for k, v in x.items() if v is not None}
    y, h = _forward(x, softplus, lengths)
    want = dict(zip(leaves, torch.autograd.grad([y, h], list(leaves.values()), [dy, ds])))
    args = [x[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "bias")]
    got = R.scan(*args, softplus, x["h0"], lengths, dy, ds)
    size = R.scan(*args, softplus, x["h0"], lengths, dy, ds, magnitudes=True)
    assert (got["y"] - y).abs().max() < 1e-13 and (got["state"] - h).abs().max() < 1e-13
    for k in leaves:
        assert (got[k] - want[k]).abs().max() < 1e-12, k
        assert (size[k] >= got[k].abs() - 1e-12).all(), k
    # along one direction, against a central difference
    v = {k: torch.randn_like(t) for k, t in leaves.items()}
    step = 1e-5
    loss = lambda s: sum((o * w).sum() for o, w in zip(  # noqa: E731
        _forward({k: None if t is None else t + s * v[k] for k, t in x.items()}, softplus, lengths), (dy, ds)))
    slope = sum((want[k] * v[k]).sum() for k in leaves)
    assert abs((loss(step) - loss(-step)) / (2 * step) - slope) < 1e-6 * abs(slope) + 1e-6


@pytest.mark.parametrize("k", [2, 3, 4])
@pytest.mark.parametrize("act", [False, True])
def test_convolution_formulas_against_autograd(k, act):
    torch.manual_seed(1)
    b, n, e = 3, 6, 4
    mk = lambda *s: torch.randn(*s, dtype=torch.float64, requires_grad=True)  # noqa: E731
    x, w, bias, init = mk(b, n, e), mk(e, k), mk(e), mk(b, k - 1, e)
    lengths = torch.tensor([6, 0, 2])
    dy, dl = torch.randn(b, n, e, dtype=torch.float64), torch.randn(b, k - 1, e, dtype=torch.float64)
    ys, last = [], []
    for i in range(b):
        row = torch.cat([init[i], x[i, :int(lengths[i])]])
        y = torch.nn.functional.conv1d(row.t()[None], w[:, None], bias, groups=e)[0].t() if lengths[i] else row[:0]
        ys.append(torch.nn.functional.pad(R.silu(y) if act else y, (0, 0, 0, n - y.shape[0])))
        last.append(row[-(k - 1):])
    y, last = torch.stack(ys), torch.stack(last)
    want = torch.autograd.grad([y, last], [x, w, bias, init], [dy, dl])
    got = R.conv(x, w, bias, act, init, lengths, dy, dl)
    assert (got["y"] - y).abs().max() < 1e-13 and torch.equal(got["state"], last)
    for a, name in zip(want, ("x", "weight", "bias", "init")):
        assert (got[name] - a).abs().max() < 1e-12, name


# --------------------------------------------------------------------------- refusals, Python
def test_cpu_tensors_are_refused():
    import mamba3_ssm as M
    x = torch.zeros(2, 3, 8)
    s = torch.zeros(2, 8, 4)
    bc = torch.zeros(2, 3, 4)
    for call in (lambda: M.causal_conv(x, torch.zeros(8, 4)), lambda: M.causal_conv_step_(torch.zeros(2, 3, 8), x[:, 0], torch.zeros(8, 4)),
                 lambda: M.ssm_scan_selective(x, x, s[0], bc, bc), lambda: M.ssm_step_selective_(s, x[:, 0], x[:, 0], s[0], bc[:, 0], bc[:, 0]),
                 lambda: M.beam_select(x, torch.zeros(2, 3)), lambda: M.reorder_states_(x, torch.zeros(1, 2, dtype=torch.long))):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()
    for call in (lambda: M.causal_conv(3, x), lambda: M.beam_select(x, 3), lambda: M.reorder_states_(x, [0, 1])):
        with pytest.raises(TypeError):
            call()


# ----------------------------------------------------------------------- refusals, C boundary
F32, BF16, F16, I64, U8 = 0, 1, 2, 3, 4


def _refs(*ts):
    return [None if t is None else ctypes.byref(t) for t in ts]


def _says(lib, rc, code, text):
    assert rc == code and text in lib.m3_last_error_string(), (rc, lib.m3_last_error_string())


def test_convolution_refusals(lib):
    def call(x=(2, 0, 8), w=(8, 4), bias=None, init=None, lengths=None, silu=1, y=None, last=None, xt=BF16, wt=BF16):
        args = [_view(x, xt), _view(w, wt), bias, init, lengths]
        return lib.m3_causal_conv(*_refs(*args), silu, *_refs(y or _view(x, xt), last), None)
    _says(lib, call(x=(2, 8)), 1, b"x: expected")
    _says(lib, call(x=(0, 0, 8), w=(8, 5)), 2, b"2, 3 or 4 taps")
    _says(lib, call(x=(0, 3, 8), w=(8, 1)), 2, b"taps")
    _says(lib, call(x=(0, 3, 0), w=(1, 4)), 1, b"weight: shape")
    _says(lib, call(x=(0, 3, 0), w=(0, 4), wt=F16), 1, b"weight: unsupported dtype")
    _says(lib, call(x=(0, 3, 0), w=(0, 4), bias=_view((0,), F32)), 1, b"bias: unsupported dtype")
    _says(lib, call(x=(0, 3, 0), w=(0, 4), silu=2), 1, b"silu: expected 0 or 1")
    _says(lib, call(x=(0, 3, 0), w=(0, 4), init=_view((0, 2, 0), BF16)), 1, b"initial: shape")
    _says(lib, call(x=(0, 3, 0), w=(0, 4), init=_view((0, 3, 0), F32)), 1, b"initial: unsupported dtype")
    _says(lib, call(x=(0, 3, 0), w=(0, 4), lengths=_view((1,), I64)), 1, b"lengths")
    _says(lib, call(x=(0, 3, 0), w=(0, 4), lengths=_view((0,), F32)), 1, b"lengths")
    _says(lib, call(x=(0, 3, 0), w=(0, 4), y=_view((0, 3, 0), F32)), 1, b"y: unsupported dtype")
    assert call(x=(0, 3, 0), w=(0, 4)) == 0
    bw = lambda **k: lib.m3_causal_conv_bwd(*_refs(_view((0, 3, 0), BF16), _view((0, 4), BF16), None, None, None), 1, *_refs(  # noqa: E731
        k.get("dy", _view((0, 3, 0), BF16)), None, _view((0, 3, 0), BF16), k.get("dw", _view((0, 4), BF16)), None, None), None, 0, None)
    _says(lib, bw(dy=_view((0, 3, 0), F32)), 1, b"dy: unsupported dtype")
    _says(lib, bw(dw=_view((0, 3), BF16)), 1, b"dweight: shape")
    assert bw() == 0
    step = lambda x, s, w=(0, 4): lib.m3_causal_conv_step(*_refs(_view(s, BF16), _view(x, BF16), _view(w, BF16), None), 0,  # noqa: E731
                                                          *_refs(_view(x, BF16)), None)
    _says(lib, step((2, 3, 0), (2, 3, 0)), 1, b"x: expected")
    _says(lib, step((2, 0), (2, 2, 0)), 1, b"state: shape")
    assert step((2, 0), (2, 3, 0)) == 0
    assert lib.m3_causal_conv_bwd_workspace_size(2, 100, 8, 5) == 0
    # parts of (taps + 1, channels) floats for every sequence: a whole number of them, more for a long one
    sizes = [lib.m3_causal_conv_bwd_workspace_size(2, n, 8, 4) for n in (0, 64, 65, 100000)]
    assert all(v > 0 and v % (2 * 8 * 5 * 4) == 0 for v in sizes) and sizes[0] == sizes[1] < sizes[2] < sizes[3]


def test_scan_refusals(lib):
    def call(u=(2, 0, 8), A=(8, 16), B=(2, 0, 1, 16), C=None, delta=None, D=None, z=None, bias=None, init=None, lengths=None,
             sp=1, last=None, ut=BF16, bt=BF16, ct=None, states=None):
        ts = [_view(u, ut), _view(*delta) if delta else _view(u, F32), _view(A, F32), _view(B, bt),
              _view(C or B, bt if ct is None else ct), D, z, bias, init, lengths]
        return lib.m3_selective_scan(*_refs(*ts), sp, *_refs(_view(u, ut), last), states, 0, None, 0, None)
    e0 = dict(u=(0, 3, 0), A=(0, 16), B=(0, 3, 1, 16))
    assert call(**e0) == 0
    _says(lib, call(**{**e0, "u": (3, 0)}), 1, b"u: expected")
    _says(lib, call(**{**e0, "A": (0, 129), "B": (0, 3, 1, 129)}), 2, b"d_state above 128")
    _says(lib, call(**{**e0, "A": (0, 0), "B": (0, 3, 1, 0)}), 1, b"d_state must be positive")
    _says(lib, call(**{**e0, "A": (1, 16)}), 1, b"A: shape")
    _says(lib, call(**{**e0, "B": (0, 3, 16)}), 1, b"B: expected")
    _says(lib, call(u=(0, 3, 8), A=(8, 16), B=(0, 3, 3, 16)), 1, b"A: ")  # an address of no device
    _says(lib, call(**{**e0, "B": (0, 3, 0, 16)}), 1, b"divide into its groups")
    _says(lib, call(**e0, C=(0, 3, 2, 16)), 1, b"C: shape")
    _says(lib, call(**e0, ct=F32), 1, b"C: unsupported dtype")
    _says(lib, call(**e0, delta=((0, 3, 0), F16)), 1, b"delta: unsupported dtype")
    _says(lib, call(**e0, z=_view((0, 3, 0), F32)), 1, b"z: unsupported dtype")
    _says(lib, call(**e0, D=_view((0,), BF16)), 1, b"D: unsupported dtype")
    _says(lib, call(**e0, bias=_view((1,), F32)), 1, b"delta_bias: shape")
    _says(lib, call(**e0, init=_view((0, 0, 8), F32)), 1, b"initial: shape")
    _says(lib, call(**e0, lengths=_view((2,), I64)), 1, b"lengths")
    _says(lib, call(**e0, sp=3), 1, b"softplus: expected 0 or 1")
    _says(lib, call(**e0, last=_view((0, 0, 16), BF16)), 1, b"last: unsupported dtype")
    step = lambda s, u=(2, 0), B=(2, 1, 16): lib.m3_selective_step(*_refs(  # noqa: E731
        _view(s, F32), _view(u, BF16), _view(u, BF16), _view((0, 16), F32), _view(B, BF16), _view(B, BF16), None, None, None), 1,
        *_refs(_view(u, BF16)), None)
    assert step((2, 0, 16)) == 0
    _says(lib, step((2, 0, 8)), 1, b"state: shape")
    _says(lib, step((2, 0, 16), B=(2, 16)), 1, b"B: expected")
    # sizes: the state in front of every eighth step, d_state rounded up to a power of two
    assert lib.m3_selective_scan_states_size(2, 17, 5, 20) == 2 * 3 * 5 * 32 * 4
    assert lib.m3_selective_scan_states_size(2, 17, 5, 129) == 0
    assert lib.m3_selective_scan_workspace_size(64, 100, 4096, 16, 1) == 0
    assert lib.m3_selective_scan_workspace_size(1, 100000, 8, 16, 1) > 0
    assert lib.m3_selective_scan_bwd_workspace_size(2, 100, 64, 16, 1) > 0


def test_beam_refusals(lib):
    def select(l=(0, 2, 10), s=None, f=None, end=0, num=2, st=F32, pt=I64):
        o = (l[0], num)
        return lib.m3_beam_select(*_refs(_view(l, BF16), s or _view(l[:2], st), f), end,
                                  *_refs(_view(o, F32), _view(o, pt), _view(o, I64)), None, 0, None)
    assert select() == 0
    _says(lib, select(l=(0, 20)), 1, b"logits: expected")
    _says(lib, select(l=(0, 33, 10)), 2, b"more than 32 beams")
    _says(lib, select(l=(0, 2, 0)), 1, b"no beam or no token")
    _says(lib, select(l=(0, 2, (1 << 24) + 1)), 2, b"dimension too large")
    _says(lib, select(s=_view((0, 3), F32)), 1, b"scores")
    _says(lib, select(st=BF16), 1, b"scores")
    _says(lib, select(f=_view((0, 2), I64)), 1, b"finished")
    _says(lib, select(end=10), 1, b"end_token")
    _says(lib, select(end=-1), 1, b"end_token")
    _says(lib, select(num=21), 1, b"candidates")
    _says(lib, select(num=0), 1, b"candidates")
    _says(lib, select(l=(0, 2, 100), num=65), 2, b"more than 64")
    _says(lib, select(pt=F32), 1, b"parents")
    assert lib.m3_beam_select_workspace_size(64, 8, 50000, 4, BF16) > 0
    assert lib.m3_beam_select_workspace_size(1, 4, 50000, 4, BF16) == 0  # one launch, which needs none
    assert lib.m3_beam_select_workspace_size(1, 33, 50000, 4, BF16) == 0


def _reorder(lib, parents, tensors, outs=None, source=None):
    """tensors: (address, row bytes, pitch)."""
    n = len(tensors)
    i64 = ctypes.c_int64 * max(n, 1)
    ptr = ctypes.c_void_p * max(n, 1)
    src, rb, sp = ptr(*[t[0] for t in tensors]), i64(*[t[1] for t in tensors]), i64(*[t[2] for t in tensors])
    dst = ptr(*[t[0] for t in outs]) if outs else None
    dp = i64(*[t[1] for t in outs]) if outs else None
    return lib.m3_reorder_states(n, src, dst, rb, sp, dp, parents.shape[1] if source is None else source, ctypes.byref(parents), None)


def test_reorder_refusals(lib):
    par = _view((2, 4), I64)
    at = 1 << 20
    _says(lib, _reorder(lib, _view((8,), I64), [(at, 64, 64)]), 1, b"parents: expected")
    _says(lib, _reorder(lib, _view((2, 4), F32), [(at, 64, 64)]), 1, b"parents: expected")
    _says(lib, _reorder(lib, par, [(at, 64, 64)], source=3), 1, b"in place")
    _says(lib, _reorder(lib, _view((1, 33), I64), [(at, 64, 64)]), 2, b"in place")
    _says(lib, _reorder(lib, par, [(at, 64, 32)]), 1, b"rows overlap")
    _says(lib, _reorder(lib, par, [(at, -1, 32)]), 1, b"negative")
    _says(lib, _reorder(lib, par, [(None, 64, 64)]), 1, b"missing")
    shared = b"shares memory"
    _says(lib, _reorder(lib, par, [(at, 64, 64), (at, 64, 64)]), 1, shared)
    _says(lib, _reorder(lib, par, [(at, 64, 64), (at + 7 * 64 + 63, 64, 64)]), 1, shared)
    _says(lib, _reorder(lib, par, [(at, 64, 128), (at + 32, 64, 128)]), 1, shared)
    _says(lib, _reorder(lib, par, [(at, 64, 128), (at + 64, 64, 256)]), 1, shared)
    _says(lib, _reorder(lib, par, [(at, 64, 64)], [(at + 64, 64)]), 1, shared)
    _says(lib, _reorder(lib, par, [(at, 64, 64)], [(at, 64)]), 1, shared)
    # between each other's rows, and behind each other: refused only for their addresses, which no device has
    for ts, outs in (([(at, 64, 128), (at + 64, 64, 128)], None), ([(at, 64, 64), (at + 512, 64, 64)], None),
                     ([(at, 64, 128)], [(at + 64, 128)]), ([(at, 64, 64), (at, 64, 64)], [(at + 512, 64), (at + 1024, 64)])):
        rc = _reorder(lib, par, ts, outs)
        assert rc in (1, 3) and shared not in lib.m3_last_error_string()
    assert _reorder(lib, par, []) == 0 and _reorder(lib, par, [(at, 0, 0)]) == 0
    assert _reorder(lib, _view((0, 4), I64), [(at, 64, 64)]) == 0
