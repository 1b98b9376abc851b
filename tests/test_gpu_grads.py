"""clip_grads_ and clip_grad_norm_ against their definition in float64.

Tolerances: the squares of a vector (at most 8) are added in 32 bits, everything after that in
64: 8 * 2^-24 relative in the sum, half of it in the norm, and its rounding to 32 bits. A
scaled gradient: the factor's rounding to 32 bits (2^-24), the norm's error in it (2^-22),
the product's rounding (2^-24) and the result's (eps / 2 of its dtype; subnormals: half of the
smallest one)."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
TINY = {torch.float32: 1e-45, torch.bfloat16: 1e-40, torch.float16: 2.0 ** -25}
NORM_TOL = 4.5 * 2.0 ** -24


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _grads(shapes, dtypes, seed, size=1e-2):
    g = _gen(seed)
    return [(size * (1 + i % 3) * torch.randn(s, device=DEV, generator=g)).to(dtypes[i % len(dtypes)])
            for i, s in enumerate(shapes)]


def _norm64(ts, norm_type=2.0):
    v = [t.double().abs().max() if norm_type == math.inf else t.double().square().sum() for t in ts if t.numel()]
    if not v:
        return 0.0
    return torch.stack(v).max().item() if norm_type == math.inf else torch.stack(v).sum().sqrt().item()


def _assert_scaled(got, src, factor):
    for o, g in zip(got, src):
        ref = g.double() * factor
        tol = ref.abs() * (torch.finfo(o.dtype).eps / 2 * 1.01 + 2.0 ** -21) + TINY[o.dtype]
        assert ((o.double() - ref).abs() <= tol).all()


SHAPES = {
    "one": [(1,)],
    "empty": [(0,), (3, 0)],
    "layer": [(1064, 256), (32,), (32, 1, 64), (64,), (256, 512), (0, 4), (1,)],
    "odd": [(7,), (2049,), (333, 17), (1,), (4095, 3), (16385,)],
    "many": [(5,)] * 63 + [(100, 3)],
    "hundreds": [(17, 33), (64,), (3,)] * 400,
    "large": [(3000, 5001), (11,)],
}


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("dtypes", [[torch.float32], [torch.bfloat16], [torch.float16, torch.float32, torch.bfloat16]])
@pytest.mark.parametrize("name", list(SHAPES))
def test_clip_in_place(name, dtypes, norm_type):
    from mamba3_ssm import clip_grads_
    src = _grads(SHAPES[name], dtypes, 1)
    n = _norm64(src, norm_type)
    for max_norm, scale in ((0.3 * n, 1.0), (3 * n + 1, 1.0), (0.3 * n, 0.25), (3 * n + 1, 1.0 / 3), (math.inf, 1.0)):
        ts = [t.clone() for t in src]
        got = clip_grads_(ts, max_norm, norm_type, scale=scale)
        assert got.dtype == torch.float32 and got.shape == ()
        assert abs(got.item() - n * scale) <= NORM_TOL * n * scale + 1e-45
        factor = scale * (1.0 if math.isinf(max_norm) else min(1.0, max_norm / (n * scale + 1e-6)))
        _assert_scaled(ts, src, factor)
        if scale == 1.0 and max_norm > n:
            assert all(torch.equal(a, b) for a, b in zip(ts, src))


@pytest.mark.parametrize("name", ["layer", "odd", "hundreds"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("to", ["fp32", "own"])
def test_clip_into_other_tensors(name, dtype, to):
    from mamba3_ssm import clip_grads_
    src = _grads(SHAPES[name], [dtype], 2)
    keep = [t.clone() for t in src]
    out = [torch.full(t.shape, float("nan"), device=DEV, dtype=torch.float32 if to == "fp32" else dtype) for t in src]
    n = _norm64(src)
    got = clip_grads_(src, 0.5 * n, scale=0.125, out=out)
    assert abs(got.item() - n * 0.125) <= NORM_TOL * n
    _assert_scaled(out, src, 0.125)
    got = clip_grads_(src, 0.01 * n, scale=0.125, out=out)
    _assert_scaled(out, src, 0.01 * n / (0.125 * n + 1e-6) * 0.125)
    assert all(torch.equal(a, b) for a, b in zip(src, keep))
    # into the gradients themselves
    if to == "own" or dtype == torch.float32:
        clip_grads_(src, 0.5 * n, out=src)
        _assert_scaled(src, keep, 0.5 * n / (n + 1e-6))


@pytest.mark.parametrize("dtype", DTYPES)
def test_unaligned_and_permuted(dtype):
    """Views that start on no 16-byte boundary, neighbours in one buffer, transposed layouts."""
    from mamba3_ssm import clip_grads_
    flat = (1e-2 * torch.randn(40000, device=DEV, generator=_gen(3))).to(dtype)
    cuts = [0, 1, 4, 9, 2058, 20000, 20001, 39999]
    ref = flat.clone()
    ts = [flat[a:b] for a, b in zip(cuts, cuts[1:])]
    ts[4] = ts[4][:17940].view(60, 299).t()
    used = [t.clone() for t in ts]
    n = _norm64(used)
    got = clip_grads_(ts, 0.5 * n)
    assert abs(got.item() - n) <= NORM_TOL * n
    _assert_scaled(ts, used, 0.5 * n / (n + 1e-6))
    assert torch.equal(flat[39999:], ref[39999:]) and torch.equal(flat[2058 + 17940:20000], ref[2058 + 17940:20000])
    out = [torch.empty(t.numel() + 1, dtype=torch.float32, device=DEV)[1:].as_strided(t.shape, t.stride(), 1) for t in used]
    clip_grads_(used, 0.25 * _norm64(used), out=out)
    _assert_scaled(out, used, 0.25 * _norm64(used) / (_norm64(used) + 1e-6))


def test_magnitudes_beyond_32_bits_of_squares():
    from mamba3_ssm import clip_grads_
    for v in (1e30, 3e19, 1e-25, 1e-38):
        g = torch.full((5001,), v, device=DEV)
        g[::2] *= -1
        n = _norm64([g])
        assert abs(clip_grads_([g], math.inf).item() - n) <= NORM_TOL * n
    g = torch.full((100,), 1e-25, device=DEV)
    ref = g.clone()
    assert abs(clip_grads_([g], 1.0, scale=2.0 ** 60).item() - 1e-24 * 2.0 ** 60) <= NORM_TOL * 1e-24 * 2.0 ** 60
    _assert_scaled([g], [ref], 2.0 ** 60)


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
def test_nan_and_infinity(norm_type):
    from mamba3_ssm import clip_grad_norm_, clip_grads_
    for where in (0, 3000, 9998):
        g = torch.ones(9999, device=DEV)
        g[where] = float("nan")
        h = torch.ones(10, device=DEV)
        assert torch.isnan(clip_grads_([h, g], 1.0, norm_type))
        assert torch.isnan(h).all() and torch.isnan(g).all()
        g = torch.ones(9999, device=DEV)
        g[where] = float("-inf")
        assert clip_grads_([h.fill_(1.0), g], 1.0, norm_type).item() == math.inf
        assert (h == 0).all() and torch.isnan(g[where]) and (g[:where] == 0).all()
    p = torch.nn.Parameter(torch.ones(4, device=DEV))
    p.grad = torch.tensor([1.0, float("nan"), 2.0, 3.0], device=DEV)
    before = p.grad.clone()
    with pytest.raises(RuntimeError, match="nan"):
        clip_grad_norm_([p], 1.0, norm_type, error_if_nonfinite=True)
    assert torch.equal(p.grad[[0, 2, 3]], before[[0, 2, 3]])


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
def test_clip_grad_norm_like_torch(norm_type):
    from mamba3_ssm import clip_grad_norm_
    ps = [torch.nn.Parameter(torch.zeros(s, device=DEV)) for s in ((40, 30), (7,), (3, 5, 2), (9,))]
    for p, g in zip(ps[:3], _grads([p.shape for p in ps[:3]], [torch.float32], 5, 1.0)):
        p.grad = g
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    for p, q in zip(ps, qs):
        q.grad = None if p.grad is None else p.grad.clone()
    version = ps[0].grad._version
    got = clip_grad_norm_(iter(ps + ps[:1]), 0.5, norm_type, error_if_nonfinite=True)  # one of them twice
    ref = torch.nn.utils.clip_grad_norm_(qs, 0.5, norm_type)
    assert abs(got.item() - ref.item()) <= 2.0 ** -20 * ref.item()
    for p, q in zip(ps[:3], qs):
        assert ((p.grad - q.grad).abs() <= 2.0 ** -20 * q.grad.abs()).all()
    assert ps[0].grad._version > version
    assert clip_grad_norm_([ps[3]], 1.0).item() == 0.0
    assert clip_grad_norm_(ps[0], 1.0).item() > 0.0


def test_same_bits_and_captured():
    from mamba3_ssm import clip_grads_
    src = [_grads(SHAPES["odd"] * 20, [torch.bfloat16, torch.float32], s) for s in (6, 7)]
    want = []
    for s in src:
        a, b = [t.clone() for t in s], [t.clone() for t in s]
        na, nb = clip_grads_(a, 0.7, scale=0.5), clip_grads_(b, 0.7, scale=0.5)
        assert torch.equal(na, nb) and all(torch.equal(x, y) for x, y in zip(a, b))
        want.append((na.clone(), a))
    bufs = [t.clone() for t in src[0]]
    other = [t.clone() for t in src[1]]
    graphs = []
    for ts in (bufs, other):
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            n = clip_grads_(ts, 0.7, scale=0.5)
        graphs.append((g, n))
    for k in (1, 0):
        for ts, s in ((bufs, src[k]), (other, src[1 - k])):
            for t, v in zip(ts, s):
                t.copy_(v)
        for g, _ in graphs:
            g.replay()
        for (ts, (_, n)), i in zip(((bufs, graphs[0]), (other, graphs[1])), (k, 1 - k)):
            assert torch.equal(n, want[i][0]) and all(torch.equal(a, b) for a, b in zip(ts, want[i][1]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ts = [t.clone() for t in src[0]]
        n = clip_grads_(ts, 0.7, scale=0.5)
    side.synchronize()
    assert torch.equal(n, want[0][0]) and all(torch.equal(a, b) for a, b in zip(ts, want[0][1]))


def test_offsets_beyond_32_bits():
    from mamba3_ssm import clip_grads_
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    n = 2 ** 31 + 12345
    g = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    g[-3:] = 4.0
    g[0] = 1.0
    assert abs(clip_grads_([g], 3.5).item() - 7.0) <= 7 * NORM_TOL
    assert g[0].item() == 0.5 and (g[-3:] == 2.0).all() and (g[1:1000] == 0).all()


def test_refusals():
    from mamba3_ssm import clip_grad_norm_, clip_grads_
    a, b = torch.ones(10, device=DEV), torch.ones(10, device=DEV)
    with pytest.raises(RuntimeError, match="shares memory"):
        clip_grads_([a, a], 1.0)
    with pytest.raises(RuntimeError, match="shares memory"):
        clip_grads_([a[:6], b, a[5:]], 1.0)
    with pytest.raises(RuntimeError, match="shares memory"):
        clip_grads_([a, b], 1.0, out=[b, a])
    with pytest.raises(RuntimeError, match="shares memory"):
        clip_grads_([a, b], 1.0, out=[torch.empty(10, device=DEV), a])
    assert abs(clip_grads_([a, a], math.inf).item() - math.sqrt(20)) < 1e-5  # only read
    assert (a == 1).all()
    with pytest.raises(ValueError, match="dense"):
        clip_grads_([torch.ones(4, 4, device=DEV)[:, :2]], 1.0)
    with pytest.raises(ValueError, match="dense"):
        clip_grads_([torch.ones(4, 1, device=DEV).expand(4, 4)], 1.0)
    with pytest.raises(TypeError, match="float64"):
        clip_grads_([a.double()], 1.0)
    with pytest.raises(RuntimeError, match="one device"):
        clip_grads_([a, b.cpu()], 1.0)
    with pytest.raises(ValueError, match="outputs"):
        clip_grads_([a, b], 1.0, out=[a])
    with pytest.raises(ValueError, match="output of shape"):
        clip_grads_([a], 1.0, out=[torch.ones(5, 2, device=DEV)])
    with pytest.raises(RuntimeError, match="dtype"):
        clip_grads_([a], 1.0, out=[a.clone().half()])
    for bad in (dict(max_norm=-1.0), dict(max_norm=float("nan")), dict(max_norm=1.0, norm_type=3.0),
                dict(max_norm=1.0, scale=0.0), dict(max_norm=1.0, scale=math.inf)):
        with pytest.raises(ValueError):
            clip_grads_([a], **bad)
    p = torch.nn.Parameter(torch.zeros(4, 2, device=DEV))
    p.grad = torch.sparse_coo_tensor([[0], [1]], [1.0], (4, 2), device=DEV)
    with pytest.raises(TypeError, match="sparse"):
        clip_grad_norm_([p], 1.0)
    assert (a == 1).all()


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("dtype", DTYPES)
def test_without_a_bound_a_nan_still_spreads(dtype, bad, norm_type):
    """max_norm inf: min(1, inf / n) is NaN for an n that is NaN or infinite, in all that is
    written. The norm alone (in place with scale 1) writes nothing."""
    from mamba3_ssm import clip_grad_norm_, clip_grads_

    def make():
        g = torch.ones(9999, device=DEV, dtype=dtype)
        g[3000] = bad
        return [torch.ones(10, device=DEV, dtype=dtype), g]

    def same(n):
        return n.isnan() if math.isnan(bad) else n == math.inf

    a = make()
    assert same(clip_grads_(a, math.inf, norm_type, scale=0.5))
    assert all(t.isnan().all() for t in a)
    for scale in (1.0, 0.5):
        a = make()
        out = [torch.zeros(t.shape, device=DEV) for t in a]
        assert same(clip_grads_(a, math.inf, norm_type, scale=scale, out=out))
        assert all(t.isnan().all() for t in out)
        assert all(torch.equal(t, o) or math.isnan(bad) for t, o in zip(a, make()))
    a = make()
    assert same(clip_grads_(a, math.inf, norm_type))
    assert (a[0] == 1).all() and (a[1][:3000] == 1).all()
    # as torch.nn.utils.clip_grad_norm_ has it
    ps, qs = ([torch.nn.Parameter(torch.zeros(t.shape, device=DEV, dtype=dtype)) for t in a] for _ in range(2))
    for p, q, g in zip(ps, qs, a):
        p.grad, q.grad = g.clone(), g.clone()
    assert same(clip_grad_norm_(ps, math.inf, norm_type))
    torch.nn.utils.clip_grad_norm_(qs, math.inf, norm_type)
    for p, q in zip(ps, qs):
        assert torch.equal(p.grad.isnan(), q.grad.isnan()) and p.grad.isnan().all()
    with pytest.raises(RuntimeError, match="cannot be clipped"):
        clip_grad_norm_(_with_grads(make()), math.inf, norm_type, error_if_nonfinite=True)


def _with_grads(ts):
    ps = [torch.nn.Parameter(torch.zeros(t.shape, device=DEV, dtype=t.dtype)) for t in ts]
    for p, t in zip(ps, ts):
        p.grad = t
    return ps


def test_without_a_bound_nothing_changes():
    """clip_grad_norm_ with max_norm inf leaves gradients of a finite norm as they are."""
    from mamba3_ssm import clip_grad_norm_
    src = _grads(SHAPES["odd"], DTYPES, 9)
    ps = _with_grads([t.clone() for t in src])
    n = clip_grad_norm_(ps, math.inf)
    assert abs(n.item() - _norm64(src)) <= NORM_TOL * n.item()
    assert all(torch.equal(p.grad, t) for p, t in zip(ps, src))
