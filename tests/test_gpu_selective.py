"""causal_conv, ssm_scan_selective and their steps against float64.

Error bounds, before any run. u = 2^-24 is half a step of fp32.
* A decay exp(dt A): the hardware's 2^x is off by at most 2^-22 relative, its argument by three
  roundings and the step size's own error (below 8 u by the series and one division), times |dt A| <= 1.5 in
  these inputs: below 2^-20 in all. A term of a result passes at most `length` decays
  and a few dozen further roundings and additions (lanes, warps, tiles), so a result is off by at most
  (length + 64) 2^-20 of the sum of its terms' magnitudes, which selective_ref gives, and by the
  rounding to its own dtype.
* The convolution: at most 4 products and additions, the logistic function's few u, and sums of
  gradients over runs of 16 rows, 8 warps and (in 64 bits) the rest: 64 u of the magnitudes."""

import pytest
import torch

import selective_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SMALLEST = {torch.float32: 1e-44, torch.bfloat16: 1e-40, torch.float16: 2.0 ** -25}


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _near(got, ref, size, unit, what=""):
    """|got - ref| within unit * size, the rounding to got's dtype and half its smallest subnormal."""
    ref, size = ref.reshape(got.shape), size.reshape(got.shape)
    half = torch.finfo(got.dtype).eps / 2 * 1.01 if got.dtype is not torch.float32 else 2.0 ** -24
    tol = unit * size + half * (ref.abs() + unit * size) + SMALLEST[got.dtype]
    bad = ~((got.double() - ref).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {float(((got.double() - ref).abs() / tol).nan_to_num(1e9).max()):.3g} of the bound"


def scan_inputs(b, n, e, m, g=1, dtype=torch.float32, seed=0, strided=True, softplus=True):
    gen = _gen(seed)
    r = lambda *s: torch.randn(*s, device=DEV, generator=gen)  # noqa: E731
    uz = r(b, n, 2 * e).to(dtype)
    u, z = (uz[..., :e], uz[..., e:]) if strided else (uz[..., :e].contiguous(), uz[..., e:].contiguous())
    bc = r(b, n, 2 * g * m).to(dtype)
    B, C = bc[..., :g * m].unflatten(-1, (g, m)), bc[..., g * m:].unflatten(-1, (g, m))
    if g == 1:
        B, C = B[:, :, 0], C[:, :, 0]
    # step sizes up to about 0.3, decay rates up to 5
    delta = (0.7 * r(b, n, e)).clamp(-2, 2).to(dtype)
    bias = -4.0 + 0.5 * r(e).clamp(-2, 2)
    if not softplus:
        delta, bias = (0.3 * torch.rand(b, n, e, device=DEV, generator=gen)).to(dtype), None
    A = -5.0 * torch.rand(e, m, device=DEV, generator=gen)
    return dict(u=u, delta=delta, A=A, B=B, C=C, D=r(e), z=z, bias=bias)


def check_scan(x, softplus=True, h0=None, lengths=None, grad=True, dstate=None, seed=9):
    from mamba3_ssm import ssm_scan_selective
    b, n, e = x["u"].shape
    leaves = {k: v.detach().requires_grad_(True) for k, v in {**x, "h0": h0}.items() if v is not None and grad}
    ops = {k: leaves.get(k, v) for k, v in {**x, "h0": h0}.items()}
    y, state = ssm_scan_selective(ops["u"], ops["delta"], ops["A"], ops["B"], ops["C"], ops["D"], z=ops["z"],
                                  delta_bias=ops["bias"], delta_softplus=softplus, initial_state=ops["h0"],
                                  lengths=lengths, return_state=True)
    assert y.dtype == x["u"].dtype and y.shape == x["u"].shape and state.dtype == torch.float32
    args = (x["u"], x["delta"], x["A"], x["B"], x["C"], x["D"], x["z"], x["bias"], softplus, h0, lengths)
    dy = torch.randn(b, n, e, device=DEV, generator=_gen(seed)).to(x["u"].dtype) if grad else None
    ref, size = R.scan(*args, dy, dstate), R.scan(*args, dy, dstate, magnitudes=True)
    unit = (n + 64) * 2.0 ** -20
    _near(y.detach(), ref["y"], size["y"], unit, "y")
    _near(state.detach(), ref["state"], size["state"], unit, "state")
    if grad:
        up = [dy] + ([] if dstate is None else [dstate])
        got = torch.autograd.grad([y] + ([] if dstate is None else [state]), list(leaves.values()), up, allow_unused=True)
        for (k, leaf), d in zip(leaves.items(), got):
            assert d.dtype == leaf.dtype and d.shape == leaf.shape
            _near(d, ref[k], size[k], unit, k)
    return y, state


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("b,n,e,m,g", [
    (1, 1, 1, 1, 1), (2, 7, 5, 3, 1), (1, 33, 64, 16, 1), (2, 100, 130, 16, 1), (1, 70, 66, 4, 2), (2, 40, 24, 8, 3),
    (1, 65, 36, 24, 1), (2, 31, 20, 32, 2), (1, 50, 9, 64, 1), (1, 37, 10, 100, 1), (1, 64, 8, 128, 2), (3, 8, 257, 16, 1)])
def test_scan(b, n, e, m, g, dtype):
    x = scan_inputs(b, n, e, m, g, DTYPES[dtype], seed=b * n + e + m)
    h0 = torch.randn(b, e, m, device=DEV, generator=_gen(5))
    check_scan(x, h0=h0, dstate=torch.randn(b, e, m, device=DEV, generator=_gen(6)))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("b,n,e,m,g", [(20, 19, 513, 16, 1), (20, 9, 250, 32, 1), (21, 12, 130, 64, 2), (20, 5, 66, 100, 1)])
def test_scan_of_many_sequences(b, n, e, m, g, dtype):
    """As many as give the backward two channels a lane; the smaller ones have one."""
    x = scan_inputs(b, n, e, m, g, DTYPES[dtype], seed=m)
    lengths = torch.tensor([n - i % 3 for i in range(b)], device=DEV)
    check_scan(x, h0=torch.randn(b, e, m, device=DEV, generator=_gen(5)), lengths=lengths)


def test_steps_before_sequences_in_memory():
    """(length, batch, channels) seen as (batch, length, channels), forward, backward and in steps."""
    b, n, e, m = 3, 41, 36, 16
    x = scan_inputs(b, n, e, m, dtype=torch.bfloat16)
    turned = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    y, state = check_scan({k: turned(t) if t is not None and t.dim() > 2 else t for k, t in x.items()})
    z, again = check_scan(x)
    assert torch.equal(y, z) and torch.equal(state, again)
    cx, w, bias, init, dy, dlast = conv_inputs(b, n, e, 4, torch.bfloat16)
    check_conv(turned(cx), w, bias, turned(init), turned(dy), turned(dlast), True)


def test_steps_refuse_states_that_overlap():
    from mamba3_ssm import causal_conv_step_, ssm_step_selective_
    e, m = 24, 16
    u = torch.randn(4, e, device=DEV)
    A, w, B = torch.randn(e, m, device=DEV), torch.randn(e, 4, device=DEV), torch.randn(4, m, device=DEV)
    for state in (torch.zeros(1, e, m, device=DEV).expand(4, e, m), torch.zeros(2000, device=DEV).as_strided((4, e, m), (e * m - 4, m, 1))):
        with pytest.raises(RuntimeError, match="overlap"):
            ssm_step_selective_(state, u, u, A, B, B)
    flat = torch.zeros(2000, device=DEV)
    for strides in ((0, e, 1), (3 * e, 0, 1), (2 * e, e, 1), (3 * e, e - 1, 1), (e, 3 * e, 1)):
        with pytest.raises(RuntimeError, match="overlap"):
            causal_conv_step_(flat.as_strided((4, 3, e), strides), u, w)
    for strides in ((3 * e, e, 1), (e, 4 * e, 1), (4 * e + 1, e + 3, 1)):
        causal_conv_step_(flat.as_strided((4, 3, e), strides), u, w)


@pytest.mark.parametrize("drop", ["z", "D", "bias", "all", "softplus"])
def test_scan_without_optional_operands(drop):
    x = scan_inputs(2, 45, 48, 16, dtype=torch.bfloat16, softplus=drop != "softplus")
    for k in (["z", "D", "bias"] if drop == "all" else [drop]):
        x[k] = None
    check_scan(x, softplus=drop != "softplus")


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_scan_lengths_and_padding(dtype):
    """Padding holds NaN and infinities; empty sequences keep their state; lengths beyond the ends are cut."""
    b, n, e, m = 7, 75, 40, 16
    x = scan_inputs(b, n, e, m, dtype=DTYPES[dtype], strided=False)
    lengths = torch.tensor([75, 0, 1, 32, 33, 90, -3], device=DEV)
    pad = ~R.valid(lengths, b, n, DEV)
    for i, k in enumerate(("u", "delta", "z", "B", "C")):
        x[k][pad] = [float("nan"), float("inf"), float("-inf"), float("nan"), float("inf")][i]
    h0 = torch.randn(b, e, m, device=DEV, generator=_gen(1))
    y, state = check_scan(x, h0=h0, lengths=lengths, dstate=torch.randn(b, e, m, device=DEV, generator=_gen(2)))
    assert (y.detach()[pad] == 0).all() and torch.equal(state.detach()[1], h0[1]) and torch.equal(state.detach()[6], h0[6])
    check_scan(x, lengths=lengths.int())


@pytest.mark.parametrize("n", [2048, 4101])
def test_scan_in_pieces_along_the_sequence(n):
    """Few channels: the sequence is cut into pieces, whose states are joined."""
    x = scan_inputs(2, n, 20, 16)
    x["A"] *= 0.02  # so that states outlive the pieces
    lengths = torch.tensor([n, n // 2 + 5], device=DEV)
    h0 = torch.randn(2, 20, 16, device=DEV, generator=_gen(1))
    check_scan(x, h0=h0, lengths=lengths, dstate=torch.randn(2, 20, 16, device=DEV, generator=_gen(2)))


def test_scan_of_an_empty_sequence_and_batch():
    from mamba3_ssm import ssm_scan_selective
    x = scan_inputs(2, 0, 12, 16)
    h0 = torch.randn(2, 12, 16, device=DEV)
    check_scan(x, h0=h0, dstate=torch.ones(2, 12, 16, device=DEV))
    x = scan_inputs(0, 9, 12, 16)
    x["A"].requires_grad_(True)
    y = ssm_scan_selective(*(x[k] for k in ("u", "delta", "A", "B", "C", "D")), z=x["z"])
    assert y.shape == (0, 9, 12)
    assert (torch.autograd.grad(y.sum(), x["A"])[0] == 0).all()


def test_scan_mixed_dtypes_and_broadcast_inputs():
    """fp32 step sizes, B and C with bf16 inputs; u expanded over the batch; a gradient without strides."""
    from mamba3_ssm import ssm_scan_selective
    x = scan_inputs(3, 40, 36, 16, dtype=torch.bfloat16)
    x["delta"], x["B"], x["C"] = x["delta"].float() + 0.001, x["B"].float() * 1.001, x["C"].float() * 0.999
    check_scan(x)
    one = x["u"][:1].detach().requires_grad_(True)
    args = (x["delta"], x["A"], x["B"], x["C"], x["D"])
    y = ssm_scan_selective(one.expand(3, 40, 36), *args, delta_bias=x["bias"])
    du, = torch.autograd.grad(y.float().sum(), one)
    ones = torch.ones(3, 40, 36, device=DEV, dtype=torch.bfloat16)
    a = (one.expand(3, 40, 36), *args, None, x["bias"], True, None, None, ones)
    each = R.scan(*a)["u"]
    # each sequence's gradient is rounded, and their sum in bf16 twice more
    size = R.scan(*a, magnitudes=True)["u"].sum(0)
    _near(du[0], each.sum(0), size + each.abs().sum(0) * 2.0 ** -9 * 4 / (104 * 2.0 ** -20), 104 * 2.0 ** -20)


def test_scan_pieces_of_a_prompt_and_steps():
    """Two pieces with the state between them, then single tokens, against the sequence as a whole."""
    from mamba3_ssm import ssm_scan_selective, ssm_step_selective_
    b, n, e, m = 2, 90, 50, 16
    x = scan_inputs(b, n, e, m)
    args = (x["u"], x["delta"], x["A"], x["B"], x["C"], x["D"], x["z"], x["bias"])
    ref, size, unit = R.scan(*args), R.scan(*args, magnitudes=True), (n + 64) * 2.0 ** -20
    cut = lambda s: [x[k][:, s] if k in ("u", "delta", "B", "C", "z") else x[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "bias")]  # noqa: E731

    def call(f, state, s):
        u, delta, A, B, C, D, z, bias = cut(s)
        return f(u, delta, A, B, C, D, z=z, delta_bias=bias) if state is None else f(state, u, delta, A, B, C, D, z=z, delta_bias=bias)
    ys, state = [], None
    for s in (slice(0, 31), slice(31, 80)):
        u, delta, A, B, C, D, z, bias = cut(s)
        y, state = ssm_scan_selective(u, delta, A, B, C, D, z=z, delta_bias=bias, initial_state=state, return_state=True)
        ys.append(y)
    for t in range(80, n):
        version = state._version
        ys.append(call(ssm_step_selective_, state, t).unsqueeze(1))
        assert state._version > version
    _near(torch.cat(ys, 1), ref["y"], size["y"], unit, "y")
    _near(state, ref["state"], size["state"], unit, "state")


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("b,e,m,g", [(1, 1, 1, 1), (3, 70, 16, 1), (2, 48, 16, 4), (5, 33, 4, 1), (2, 24, 24, 2), (1, 9, 50, 1),
                                     (2, 10, 128, 1), (257, 66, 8, 3)])
def test_step(b, e, m, g, dtype):
    from mamba3_ssm import ssm_step_selective_
    x = scan_inputs(b, 1, e, m, g, DTYPES[dtype])
    h0 = torch.randn(b, e, m, device=DEV, generator=_gen(1))
    args = (x["u"], x["delta"], x["A"], x["B"], x["C"], x["D"], x["z"], x["bias"], True, h0)
    ref, size = R.scan(*args), R.scan(*args, magnitudes=True)
    pool = torch.full((b, 2, e, m), 7.0, device=DEV)
    state = pool[:, 1]  # strided over the batch
    state.copy_(h0)
    y = ssm_step_selective_(state, x["u"][:, 0], x["delta"][:, 0], x["A"], x["B"][:, 0], x["C"][:, 0], x["D"],
                            z=x["z"][:, 0], delta_bias=x["bias"])
    _near(y, ref["y"], size["y"], 65 * 2.0 ** -20, "y")
    _near(state, ref["state"], size["state"], 65 * 2.0 ** -20, "state")
    assert (pool[:, 0] == 7.0).all()


def test_scan_gradient_against_differences():
    """A directional derivative of the kernels' own outputs. The loss is a fixed weighting of y and the
    state, summed in 64 bits; the central difference of step h is off by h^2 / 6 times the third derivative along the
    direction and by the outputs' errors over 2 h: with unit directions scaled to 3e-3 of the operands both stay
    far below the 2% that are allowed."""
    from mamba3_ssm import ssm_scan_selective
    x = scan_inputs(2, 60, 30, 16)
    x["h0"] = torch.randn(2, 30, 16, device=DEV, generator=_gen(1))
    w, v = torch.randn(2, 60, 30, device=DEV, generator=_gen(2)), torch.randn(2, 30, 16, device=DEV, generator=_gen(3))

    def loss(o):
        y, s = ssm_scan_selective(o["u"], o["delta"], o["A"], o["B"], o["C"], o["D"], z=o["z"], delta_bias=o["bias"],
                                  initial_state=o["h0"], return_state=True)
        return y, s
    leaves = {k: t.detach().requires_grad_(True) for k, t in x.items()}
    grads = dict(zip(leaves, torch.autograd.grad(loss(leaves), list(leaves.values()), [w, v])))
    for i, k in enumerate(x):
        d = torch.randn(x[k].shape, device=DEV, generator=_gen(20 + i))
        d = d * grads[k].abs().clamp(min=0) / grads[k].abs().mean()  # along the larger slopes
        d = torch.where(grads[k] < 0, -d.abs(), d.abs())
        h = 3e-3 * x[k].abs().mean() / d.abs().mean()
        up, dn = ({**x, k: x[k] + s * h * d} for s in (1, -1))
        with torch.no_grad():
            (yu, su), (yd, sd) = loss(up), loss(dn)
        diff = ((yu.double() - yd.double()) * w).sum() + ((su.double() - sd.double()) * v).sum()
        want = (grads[k].double() * (up[k].double() - dn[k].double())).sum()
        assert abs(diff - want) <= 0.02 * abs(want), (k, diff.item(), want.item())


def test_scan_is_deterministic_and_backward_twice():
    from mamba3_ssm import ssm_scan_selective
    x = scan_inputs(2, 300, 200, 16, dtype=torch.bfloat16)
    leaves = {k: t.detach().requires_grad_(True) for k, t in x.items()}

    def go():
        y = ssm_scan_selective(*(leaves[k] for k in ("u", "delta", "A", "B", "C", "D")), z=leaves["z"], delta_bias=leaves["bias"])
        a = torch.autograd.grad(y, list(leaves.values()), torch.ones_like(y), retain_graph=True)
        return y, a, torch.autograd.grad(y, list(leaves.values()), torch.ones_like(y))
    (y1, a1, b1), (y2, a2, _) = go(), go()
    assert torch.equal(y1, y2)
    for p, q, r in zip(a1, b1, a2):
        assert torch.equal(p, q) and torch.equal(p, r)


# ------------------------------------------------------------------------------ convolution
def conv_inputs(b, n, e, k, dtype, seed=0, strided=True, wdtype=None):
    gen = _gen(seed)
    r = lambda *s: torch.randn(*s, device=DEV, generator=gen)  # noqa: E731
    x = r(b, n, 2 * e).to(dtype)[..., :e]
    return (x if strided else x.contiguous(), r(e, k).to(wdtype or dtype), r(e).to(wdtype or dtype),
            r(b, k - 1, e).to(dtype), r(b, n, e).to(dtype), r(b, k - 1, e).to(dtype))


def check_conv(x, w, bias, init, dy, dlast, act, lengths=None):
    from mamba3_ssm import causal_conv
    names = {"x": x, "weight": w, "bias": bias, "init": init}
    leaves = {k: t.detach().requires_grad_(True) for k, t in names.items() if t is not None}
    g = lambda k: leaves.get(k)  # noqa: E731
    y, last = causal_conv(g("x"), g("weight"), g("bias"), activation="silu" if act else None, initial_state=g("init"),
                          lengths=lengths, return_state=True)
    a = (x, w, bias, act, init, lengths, dy, dlast)
    ref, size = R.conv(*a), R.conv(*a, magnitudes=True)
    unit = 64 * 2.0 ** -24
    _near(y.detach(), ref["y"], size["y"], unit, "y")
    assert torch.equal(last.detach().double(), ref["state"])
    outs, ups = ([y, last], [dy, dlast]) if dlast is not None else ([y], [dy])
    got = torch.autograd.grad(outs, list(leaves.values()), ups)
    for (k, leaf), d in zip(leaves.items(), got):
        assert d.dtype == leaf.dtype and d.shape == leaf.shape
        _near(d, ref[k], size[k], unit, k)
    return y


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("b,n,e,k", [(1, 1, 1, 4), (2, 3, 8, 4), (2, 2, 5, 3), (1, 130, 264, 4), (3, 129, 70, 2), (2, 257, 36, 3),
                                     (1, 16, 513, 4), (2, 300, 2, 4)])
@pytest.mark.parametrize("act", [False, True])
def test_conv(b, n, e, k, act, dtype):
    x, w, bias, init, dy, dlast = conv_inputs(b, n, e, k, DTYPES[dtype])
    check_conv(x, w, bias, init, dy, dlast, act)
    check_conv(x, w, None, None, dy, None, act)


@pytest.mark.parametrize("k", [2, 4])
def test_conv_lengths_and_padding(k):
    b, n, e = 7, 140, 24
    x, w, bias, init, dy, dlast = conv_inputs(b, n, e, k, torch.bfloat16, strided=False)
    lengths = torch.tensor([140, 0, 1, 2, 129, 500, -1], device=DEV)
    pad = ~R.valid(lengths, b, n, DEV)
    x[pad] = float("nan")
    dy[pad] = float("inf")
    y = check_conv(x, w, bias, init, dy, dlast, True, lengths)
    assert (y.detach()[pad] == 0).all()


def test_conv_mixed_weights_unaligned_rows_and_odd_strides():
    x, w, bias, init, dy, dlast = conv_inputs(2, 50, 40, 4, torch.bfloat16, wdtype=torch.float32)
    check_conv(x, w, bias, init, dy, dlast, True)
    flat = torch.randn(2 * 50 * 41 + 1, device=DEV).bfloat16()
    check_conv(flat[1:].view(2, 50, 41)[..., :40], w, bias, init, dy, dlast, True)  # rows start on no vector boundary
    check_conv(flat[1:].view(2, 50, 41)[..., 1:], w.t().contiguous().t(), bias, init, dy, dlast, False)


def test_conv_of_an_empty_sequence():
    x, w, bias, init, dy, dlast = conv_inputs(2, 0, 24, 4, torch.float32)
    check_conv(x, w, bias, init, dy, dlast, True)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("b,e,k", [(1, 1, 4), (3, 40, 4), (2, 71, 3), (300, 66, 2)])
def test_conv_pieces_and_steps(b, e, k, dtype):
    from mamba3_ssm import causal_conv, causal_conv_step_
    n = 20
    x, w, bias, init, _, _ = conv_inputs(b, n, e, k, DTYPES[dtype])
    ref, size = R.conv(x, w, bias, True, init), R.conv(x, w, bias, True, init, magnitudes=True)
    y1, s = causal_conv(x[:, :1], w, bias, activation="silu", initial_state=init, return_state=True)
    y2, s = causal_conv(x[:, 1:12], w, bias, activation="silu", initial_state=s, return_state=True)
    ys = [y1, y2]
    for t in range(12, n):
        ys.append(causal_conv_step_(s, x[:, t], w, bias, activation="silu").unsqueeze(1))
    _near(torch.cat(ys, 1), ref["y"], size["y"], 64 * 2.0 ** -24, "y")
    assert torch.equal(s.double(), ref["state"])


# ----------------------------------------------------------- streams, graphs, other entry states
def test_capture_and_replay_of_forward_and_backward():
    """A convolution, a scan and both backward passes in one graph, replayed on changed inputs."""
    from mamba3_ssm import causal_conv, ssm_scan_selective
    x = scan_inputs(2, 70, 40, 16, dtype=torch.bfloat16)
    w = torch.randn(40, 4, device=DEV, generator=_gen(1))
    leaves = {**{k: t.detach().clone().requires_grad_(True) for k, t in x.items()}, "w": w.requires_grad_(True)}
    dy = torch.randn(2, 70, 40, device=DEV, generator=_gen(2)).bfloat16()

    def go():
        c = causal_conv(leaves["u"], leaves["w"], activation="silu")
        y = ssm_scan_selective(c, *(leaves[k] for k in ("delta", "A", "B", "C", "D")), z=leaves["z"], delta_bias=leaves["bias"])
        return [y.detach(), *torch.autograd.grad(y, list(leaves.values()), dy)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        go()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = go()
    for seed in (3, 4):
        with torch.no_grad():
            leaves["u"].copy_(torch.randn(2, 70, 40, device=DEV, generator=_gen(seed)))
        graph.replay()
        got = [t.clone() for t in out]
        want = go()
        for p, q in zip(got, want):
            assert torch.equal(p, q)


def test_another_stream_and_concurrent_calls():
    from mamba3_ssm import ssm_scan_selective
    xs = [scan_inputs(1, 3000, 24, 16, seed=s) for s in (1, 2)]
    call = lambda x: ssm_scan_selective(*(x[k] for k in ("u", "delta", "A", "B", "C", "D")), z=x["z"], delta_bias=x["bias"])  # noqa: E731
    want = [call(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(call(x))
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_offsets_beyond_32_bits():
    """Rows more than 2^31 elements apart, in one buffer that is not filled."""
    from mamba3_ssm import causal_conv, ssm_scan_selective
    e = 64
    big = torch.empty(2, 2 ** 31 + 64, dtype=torch.bfloat16, device=DEV)
    u = big.as_strided((2, 3, e), (2 ** 31 + 64, 2 ** 30, 1))
    x = scan_inputs(2, 3, e, 16, dtype=torch.bfloat16)
    u.copy_(x["u"])
    x["u"] = u
    check_scan(x, grad=False)
    _, w, bias, init, dy, dlast = conv_inputs(2, 3, e, 4, torch.bfloat16)
    check_conv(u, w, bias, init, dy, dlast, True)
