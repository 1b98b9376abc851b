"""token_logprobs, policy_loss and preference_loss against their definitions in float64.

Tolerances, per value (u = half a rounding step of the logits' dtype, torch.finfo(t).eps / 2):
* log-probability: the 32-bit sum of exponentials is off by the exponent's rounding and the
  exponential's own error (2^-22 each, relative), and by its additions: a thread adds at most
  V / 512 + 40 terms in a row, each addition 2^-24 of the sum. 2^-19 covers both up to V =
  131072 for errors of one sign: log-probabilities are held to 2^-19 plus the rounding to
  32 bits, 2^-24 of the value.
* gradient g (1[token] - p): p carries the same relative error, twice (its own exponential
  and the sum's): |g| (2^-18 p + 2^-23) plus the rounding of the result, u of its value (fp16:
  at least 2^-25, half the smallest subnormal).
* sums over positions (losses, rewards): the positions' tolerances added up.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
IGN = -100
LOGP_TOL = 2.0 ** -19
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _inputs(shape, dtype, seed, layout="contiguous"):
    """Logits in one of the layouts a user's program has them in, and tokens."""
    B, T, V = shape
    g = _gen(seed)

    def rand(*s):
        return (3 * torch.randn(*s, device=DEV, generator=g)).to(dtype)

    if layout == "contiguous":
        x = rand(B, T, V)
    elif layout == "cut":            # vocabulary cut from a padded one: strided rows
        x = rand(B, T, V + 3)[..., :V]
    elif layout == "wide":           # a narrow part of much wider rows
        x = rand(B, T, 3 * V + 1)[..., V:2 * V]
    elif layout == "shifted":        # logits[:, :-1]
        x = rand(B, T + 1, V)[:, :-1]
    elif layout == "transposed":     # positions before batch
        x = rand(T, B, V).transpose(0, 1)
    elif layout == "offset":         # rows that start on no 16-byte boundary
        x = rand(B * T * V + 1)[1:].view(B, T, V)
    elif layout == "expanded":       # one batch row for all
        x = rand(1, T, V).expand(B, T, V)
    tokens = torch.randint(0, V, (B, T), device=DEV, generator=g)
    return x, tokens


def _logp64(x, tokens, temperature=1.0):
    x = x.double() / temperature
    return torch.log_softmax(x, -1).gather(-1, tokens.clamp(0, x.shape[-1] - 1).unsqueeze(-1)).squeeze(-1)


def _assert_logp(got, ref):
    assert got.dtype == torch.float32
    err = (got.double() - ref).abs()
    assert (err <= LOGP_TOL + 2.0 ** -24 * ref.abs()).all(), err.max().item()


def _assert_grad(got, x, tokens, dlogp, temperature=1.0):
    """got against sum(dlogp * logp) differentiated, dlogp (B, T) in float64."""
    s = 1.0 / temperature
    p = torch.softmax(x.double() * s, -1)
    hot = torch.zeros_like(p).scatter_(-1, tokens.clamp(0, x.shape[-1] - 1).unsqueeze(-1), 1.0)
    g = (dlogp * s).unsqueeze(-1)
    ref = g * (hot - p)
    u = torch.finfo(x.dtype).eps / 2
    tol = g.abs() * (2.0 ** -18 * p + 2.0 ** -23) + u * ref.abs() * (1 + 2.0 ** -10)
    tol += 2.0 ** -25 if x.dtype == torch.float16 else 1e-37
    err = (got.double() - ref).abs()
    assert got.dtype == x.dtype and got.shape == x.shape
    assert (err <= tol).all(), (err / tol).max().item()


SHAPES = [(1, 1, 1), (1, 1, 50000), (2, 3, 7), (3, 5, 50277), (1, 48, 50000), (2, 300, 1000), (400, 1, 33), (1, 2, 131072),
          (7, 43, 515)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_token_logprobs(shape, dtype):
    from mamba3_ssm import token_logprobs
    x, tokens = _inputs(shape, dtype, 1)
    ref = _logp64(x, tokens)
    _assert_logp(token_logprobs(x, tokens), ref)
    x.requires_grad_(True)
    dout = torch.randn(tokens.shape, device=DEV, generator=_gen(2))
    out = token_logprobs(x, tokens)
    _assert_logp(out.detach(), ref)
    d, = torch.autograd.grad(out, x, dout)
    _assert_grad(d, x.detach(), tokens, dout.double())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["cut", "wide", "shifted", "transposed", "offset", "expanded"])
@pytest.mark.parametrize("shape", [(2, 5, 1001), (3, 40, 64)])
def test_token_logprobs_layouts(shape, layout, dtype):
    from mamba3_ssm import token_logprobs
    x, tokens = _inputs(shape, dtype, 3, layout)
    tokens = torch.stack([tokens, tokens], -1)[..., 0]  # strided tokens
    x = x.detach().requires_grad_(True)
    dout = torch.randn(tokens.shape[1], tokens.shape[0], device=DEV, generator=_gen(4)).t()
    out = token_logprobs(x, tokens, temperature=0.7)
    _assert_logp(out.detach(), _logp64(x.detach(), tokens, 0.7))
    d, = torch.autograd.grad(out, x, dout)
    _assert_grad(d, x.detach(), tokens, dout.double(), 0.7)


def test_token_logprobs_leading_dimensions():
    from mamba3_ssm import token_logprobs
    x, tokens = _inputs((6, 10, 77), torch.float32, 5)
    full = token_logprobs(x, tokens)
    assert torch.equal(token_logprobs(x.view(2, 3, 10, 77), tokens.view(2, 3, 10)).view(6, 10), full)
    assert torch.equal(token_logprobs(x[1], tokens[1].int()), full[1])
    one = token_logprobs(x[1, 2], tokens[1, 2])
    assert one.shape == () and torch.equal(one, full[1, 2])
    assert token_logprobs(x[:0], tokens[:0]).shape == (0, 10)
    assert token_logprobs(x[:, :0], tokens[:, :0]).shape == (6, 0)
    y = x[:0].clone().requires_grad_(True)
    d, = torch.autograd.grad(token_logprobs(y, tokens[:0]).sum(), y)
    assert d.shape == y.shape


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [50, 20000])
def test_positions_that_do_not_count_are_not_read(dtype, V):
    """Masked and ignored positions may hold anything; their results are exactly zero."""
    from mamba3_ssm import token_logprobs
    x, tokens = _inputs((3, 8, V), dtype, 6)
    mask = torch.ones(3, 8, dtype=torch.bool, device=DEV)
    mask[0, :3] = False
    tokens[1, 5:] = IGN
    mask[2] = False
    keep = mask & (tokens != IGN)
    ref = _logp64(x, tokens)
    x[0, 0] = float("nan")
    x[0, 1] = float("inf")
    x[0, 2] = float("-inf")
    x[1, 6] = torch.finfo(dtype).min
    x[2, 4] = float("nan")
    clean = torch.where(keep.unsqueeze(-1), x, torch.zeros((), dtype=dtype, device=DEV))
    for m in (mask, mask.to(torch.uint8) * 7, mask.float()):
        x = x.detach().requires_grad_(True)
        out = token_logprobs(x, tokens, mask=m)
        assert (out.detach()[~keep] == 0).all()
        _assert_logp(out.detach()[keep], ref[keep])
        d, = torch.autograd.grad(out.sum(), x)
        assert (d[~keep] == 0).all()
        _assert_grad(d, clean, tokens, keep.double())
    assert (token_logprobs(x, torch.full_like(tokens, IGN)) == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [2, 600])
@pytest.mark.parametrize("V", [40, 30011])
def test_infinite_and_extreme_logits(dtype, rows, V):
    """Excluded entries (-inf or the type's lowest value) weigh nothing; a row of -inf alone, +inf
    or NaN gives NaN; far offsets do not overflow."""
    from mamba3_ssm import token_logprobs
    if rows * V > 4_000_000:
        rows = 100
    x, tokens = _inputs((1, rows, V), dtype, 7)
    tokens[:] = torch.arange(rows, device=DEV) % 3
    x[0, :, 3:V - 1] = float("-inf")
    x[0, 1::2, 3:V - 1] = torch.finfo(dtype).min
    out = token_logprobs(x, tokens)
    few = torch.cat([x[..., :3], x[..., V - 1:]], -1)
    _assert_logp(out, _logp64(few, tokens))
    y = x.detach().requires_grad_(True)
    d, = torch.autograd.grad(token_logprobs(y, tokens).sum(), y)
    assert (d[0, :, 3:V - 1] == 0).all() and torch.isfinite(d).all()
    # rows of the lowest value alone are uniform
    low = torch.full((1, 2, V), torch.finfo(dtype).min, device=DEV, dtype=dtype)
    _assert_logp(token_logprobs(low, tokens[:, :2], temperature=0.5), torch.full((1, 2), -math.log(V), device=DEV).double())
    # a token that is excluded itself
    assert (token_logprobs(x[:, ::2], torch.full_like(tokens[:, ::2], 5)) == float("-inf")).all()
    bad = torch.full((1, 2, V), float("-inf"), device=DEV, dtype=dtype)
    assert torch.isnan(token_logprobs(bad, tokens[:, :2])).all()
    bad = x[:, :2].clone()
    bad[0, :, V // 2] = float("nan")
    assert torch.isnan(token_logprobs(bad, tokens[:, :2])).all()
    bad = x[:, :2].clone()
    bad[0, :, 1] = float("inf")
    assert torch.isnan(token_logprobs(bad, tokens[:, :2])).all()
    for offset in (-30000.0, 30000.0, -190.0):
        z = torch.full((1, 2, V), offset, device=DEV, dtype=dtype)
        z[0, 1, 0] = offset * (1 + 2.0 ** -5)
        _assert_logp(token_logprobs(z, tokens[:, :2]), _logp64(z, tokens[:, :2]))


def test_tokens_outside_the_vocabulary_give_nan():
    from mamba3_ssm import policy_loss, token_logprobs
    x, tokens = _inputs((2, 4, 100), torch.float32, 8)
    tokens[0, 1], tokens[1, 2] = 100, -1
    bad = torch.zeros(2, 4, dtype=torch.bool, device=DEV)
    bad[0, 1] = bad[1, 2] = True
    x.requires_grad_(True)
    out = token_logprobs(x, tokens)
    assert torch.equal(out.isnan(), bad)
    d, = torch.autograd.grad(out.sum(), x)
    assert torch.equal(d.isnan(), bad.unsqueeze(-1).expand_as(d))
    z = torch.zeros(2, 4, device=DEV)
    r = policy_loss(x, tokens, z, z + 1)
    assert r.loss.isnan() and torch.equal(r.logprobs.isnan(), bad)
    # a position that does not count may name any token
    r = policy_loss(x, tokens, z, z + 1, mask=~bad)
    assert r.loss.isfinite() and (r.logprobs[bad] == 0).all()


# ------------------------------------------------------------------------------- policy
def _policy64(x, tokens, old, adv, ref, keep, lo, hi, kl_coef, temperature, reduction):
    """Loss, mean KL, clipped share and d loss / d logp from the definition, and how far the
    loss may be off for the log-probabilities' tolerance."""
    logp = _logp64(x, tokens, temperature)
    logp = torch.where(keep, logp, torch.zeros_like(logp)).requires_grad_(True)
    r = (logp - old.double()).exp()
    a = adv.double()
    rc = r.clamp(1 - lo, 1 + hi)
    per = -torch.minimum(r * a, rc * a)
    clipped = (rc * a < r * a).double()
    kl = torch.zeros_like(logp)
    if ref is not None:
        d = ref.double() - logp
        kl = torch.expm1(d) - d
        per = per + kl_coef * kl
    m = keep.double()
    n = m.sum().clamp(min=1)
    if reduction == "token":
        w = m / n
    else:
        cnt = m.sum(1, keepdim=True)
        w = m / cnt.clamp(min=1) / (cnt > 0).sum().clamp(min=1)
    loss = torch.where(keep, w * per, torch.zeros_like(w)).sum()
    dlogp, = torch.autograd.grad(loss, logp)
    slack = (w * (r * a.abs() + kl_coef * (torch.expm1((ref.double() - logp) if ref is not None else logp * 0)).abs())
             * LOGP_TOL).sum() + 2.0 ** -22 * torch.where(keep, w * per.abs(), torch.zeros_like(w)).sum() + 1e-12
    return (loss.detach(), torch.where(keep, m / n * kl, 0 * m).sum().detach(), (m / n * clipped).sum(), dlogp,
            logp.detach(), slack.detach(), w)


def _off_border(x, tokens, lo, hi, temperature, g):
    """Old log-probabilities whose ratios stay 1e-3 away from the clipping borders."""
    logp = _logp64(x, tokens, temperature)
    ratio = 0.25 * torch.randn(logp.shape, device=DEV, generator=g, dtype=torch.float64)
    for edge in (math.log(max(1 - lo, 1e-9)), math.log(1 + hi)):
        ratio = torch.where((ratio - edge).abs() < 1e-3, ratio + 4e-3, ratio)
    return (logp - ratio).float()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,reduction,with_ref,masked,lo,hi,temperature", [
    ((1, 1, 3), "token", False, False, 0.2, 0.2, 1.0),
    ((2, 3, 5003), "token", True, True, 0.2, 0.3, 1.0),
    ((8, 64, 50000), "token", False, True, 0.2, 0.2, 1.0),
    ((5, 37, 1000), "sequence", True, True, 0.1, 0.1, 0.8),
    ((3, 700, 257), "sequence", True, False, 0.0, 0.5, 1.3),
    ((300, 2, 64), "sequence", False, True, 1.0, 0.2, 1.0),
    ((1, 2500, 300), "token", True, True, 0.2, 0.2, 1.0),
    ((700, 1, 600), "sequence", False, True, 0.2, 0.2, 1.0),
    ((60, 17, 520), "sequence", True, True, 0.2, 0.2, 1.0),
    ((2, 2, 900001), "token", True, True, 0.2, 0.2, 1.0),
])
def test_policy_loss(shape, reduction, with_ref, masked, lo, hi, temperature, dtype):
    from mamba3_ssm import policy_loss
    g = _gen(11)
    x, tokens = _inputs(shape, dtype, 10)
    B, T, V = shape
    old = _off_border(x, tokens, lo, hi, temperature, g)
    adv = torch.randn(B, T, device=DEV, generator=g)
    ref = (old + 0.2 * torch.randn(B, T, device=DEV, generator=g)) if with_ref else None
    keep = torch.ones(B, T, dtype=torch.bool, device=DEV)
    if masked:
        keep = torch.rand(B, T, device=DEV, generator=g) < 0.6
        keep[0] = B < 2          # a sequence without any position
        tokens[-1, -1] = IGN
    mask = keep if masked else None
    keep = keep & (tokens != IGN)
    kl_coef = 0.07 if with_ref else 0.0
    loss, kl, frac, dlogp, logp, slack, w = _policy64(x, tokens, old, adv, ref, keep, lo, hi, kl_coef, temperature, reduction)
    args = dict(ref_logprobs=ref, mask=mask, clip_low=lo, clip_high=hi, kl_coef=kl_coef, temperature=temperature,
                reduction=reduction)
    plain = policy_loss(x, tokens, old, adv, **args)
    x.requires_grad_(True)
    r = policy_loss(x, tokens, old, adv, **args)
    d, = torch.autograd.grad(r.loss, x, retain_graph=True)
    for a, b in zip(plain, r):
        assert torch.equal(a, b.detach())
    _assert_logp(r.logprobs[keep], logp[keep])
    assert (r.logprobs[~keep] == 0).all()
    assert abs(r.loss.item() - loss.item()) <= slack.item() + 2.0 ** -23 * abs(loss.item())
    assert abs(r.clip_fraction.item() - frac.item()) <= 2.0 ** -22
    # |d kl / d logp| = |1 - exp(d)|
    kslack = (keep.double() / keep.sum().clamp(min=1) * torch.expm1(ref.double() - logp).abs()).sum().item() if with_ref else 0.0
    assert abs(r.kl.item() - kl.item()) <= LOGP_TOL * kslack + 2.0 ** -20 * abs(kl.item())
    # the weights' tolerance: d(dlogp) by logp is r |A| w + k exp(d) w
    loose = 2.0 ** -17
    u = torch.finfo(dtype).eps / 2
    xs = x.detach().double() / temperature
    p = torch.softmax(xs, -1)
    hot = torch.zeros_like(p).scatter_(-1, tokens.clamp(0).unsqueeze(-1), 1.0)

    def check(got, up):
        gg = up * (dlogp / temperature).unsqueeze(-1)
        exact = gg * (hot - p)
        big = abs(up) * (w * ((logp - old.double()).exp() * adv.double().abs()
                              + kl_coef * ((ref.double() - logp).exp() if with_ref else 0.0))).unsqueeze(-1) / temperature
        tol = big * loose * (hot - p).abs() + gg.abs() * (2.0 ** -18 * p + 2.0 ** -23) + u * exact.abs() * 1.001
        tol = tol + (2.0 ** -25 if dtype == torch.float16 else 1e-37)
        err = (got.double() - exact).abs()
        assert (err <= tol).all(), (err / tol).max().item()
        assert (got[~keep] == 0).all()

    check(d, 1.0)
    # another upstream gradient, and the first one again
    up = 1024.0 * 3
    d2, = torch.autograd.grad(r.loss * up, x, retain_graph=True)
    check(d2, up)
    d.fill_(7.0)
    d3, = torch.autograd.grad(r.loss, x)
    check(d3, 1.0)


def test_policy_loss_without_a_position():
    from mamba3_ssm import policy_loss
    x, tokens = _inputs((2, 5, 64), torch.bfloat16, 12)
    x[:] = float("nan")
    x.requires_grad_(True)
    z = torch.zeros(2, 5, device=DEV)
    for reduction in ("token", "sequence"):
        r = policy_loss(x, tokens, z, z, ref_logprobs=z, mask=torch.zeros(2, 5, dtype=torch.bool, device=DEV), kl_coef=0.1,
                        reduction=reduction)
        d, = torch.autograd.grad(r.loss, x)
        assert r.loss.item() == r.kl.item() == r.clip_fraction.item() == 0.0 and (d == 0).all()
    e = x.detach()[:, :0].requires_grad_(True)
    r = policy_loss(e, tokens[:, :0], z[:, :0], z[:, :0])
    d, = torch.autograd.grad(r.loss, e)
    assert r.loss.item() == 0.0 and r.kl.item() == 0.0 and d.shape == e.shape


def test_policy_loss_broadcasts_and_clips_as_defined():
    """Advantages per sequence; ratios far outside, with both signs of the advantage."""
    from mamba3_ssm import policy_loss
    x, tokens = _inputs((4, 6, 333), torch.float32, 13)
    logp = _logp64(x, tokens)
    shift = torch.tensor([[1.0], [-1.0], [1.0], [-1.0]], device=DEV)
    adv = torch.tensor([[2.0], [2.0], [-2.0], [-2.0]], device=DEV)
    old = (logp - shift).float()        # ratios e and 1/e
    x.requires_grad_(True)
    r = policy_loss(x, tokens, old, adv, clip_low=0.2, clip_high=0.4)
    d, = torch.autograd.grad(r.loss, x)
    # clipped: ratio e with A > 0, ratio 1/e with A < 0
    exp = (-1.4 * 2 - math.exp(-1) * 2 + math.exp(1) * 2 + 0.8 * 2) / 4
    assert abs(r.loss.item() - exp) <= 1e-5 * abs(exp)
    assert r.clip_fraction.item() == 0.5
    assert (d[0] == 0).all() and (d[3] == 0).all() and (d[1] != 0).any() and (d[2] != 0).any()
    full = policy_loss(x, tokens, old, adv.expand(4, 6).contiguous(), clip_low=0.2, clip_high=0.4)
    assert torch.equal(full.loss, r.loss)
    # per position, from one-dimensional calls
    one = policy_loss(x[1], tokens[1], old[1], adv[1], clip_low=0.2, clip_high=0.4)
    assert one.logprobs.shape == (6,) and torch.equal(one.logprobs, r.logprobs[1])


def test_policy_gradient_against_differences():
    """(L(x + h u) - L(x - h u)) / 2h = <dL/dx, u> + O(h^2): inside the clipping range the loss
    is smooth; with h = 2^-7 the third derivative's term is below h^2 |u|^3 and L's rounding
    2^-24 |L| / h."""
    from mamba3_ssm import policy_loss
    x, tokens = _inputs((2, 9, 120), torch.float32, 14)
    old = (_logp64(x, tokens) + 0.02).float()
    ref = old - 0.1
    adv = torch.randn(2, 9, device=DEV, generator=_gen(15))
    u = torch.randn(x.shape, device=DEV, generator=_gen(16))
    u /= u.norm()
    h = 2.0 ** -7

    def loss(v):
        return policy_loss(v, tokens, old, adv, ref_logprobs=ref, clip_low=0.5, clip_high=0.5, kl_coef=0.3).loss

    y = x.clone().requires_grad_(True)
    d, = torch.autograd.grad(loss(y), y)
    num = (loss(x + h * u).double() - loss(x - h * u).double()) / (2 * h)
    assert abs(num.item() - (d.double() * u.double()).sum().item()) <= h * h + 2.0 ** -23 * abs(loss(x).item()) / h


# ---------------------------------------------------------------------------- preference
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,T,V,with_ref,masked,smoothing,temperature", [
    (1, 1, 5, False, False, 0.0, 1.0),
    (1, 96, 50000, True, True, 0.0, 1.0),
    (3, 70, 1003, True, True, 0.1, 1.0),
    (300, 4, 40, True, False, 0.0, 0.9),
    (2, 3000, 64, True, True, 0.5, 1.0),
])
def test_preference_loss(N, T, V, with_ref, masked, smoothing, temperature, dtype):
    from mamba3_ssm import preference_loss
    g = _gen(21)
    x, tokens = _inputs((2 * N, T, V), dtype, 20)
    logp = _logp64(x, tokens, temperature)
    ref = (logp + 0.3 * torch.randn(logp.shape, device=DEV, generator=g)).float() if with_ref else None
    keep = torch.ones(2 * N, T, dtype=torch.bool, device=DEV)
    if masked:
        keep = torch.rand(2 * N, T, device=DEV, generator=g) < 0.7
        keep[0] = False          # an answer without any position
    beta = 0.3
    z = torch.where(keep, logp - (ref.double() if with_ref else 0.0), torch.zeros_like(logp))
    count = keep.sum(1).double()
    rewards = beta * z.sum(1)
    zz = (rewards[:N] - rewards[N:]).requires_grad_(True)
    f = torch.nn.functional.logsigmoid
    loss = -((1 - smoothing) * f(zz) + smoothing * f(-zz)).mean()
    dz, = torch.autograd.grad(loss, zz)
    x.requires_grad_(True)
    r = preference_loss(x, tokens, ref, mask=keep if masked else None, beta=beta, label_smoothing=smoothing,
                        temperature=temperature)
    d, = torch.autograd.grad(r.loss, x, retain_graph=True)
    tol_r = beta * count * LOGP_TOL + 2.0 ** -23 * rewards.abs() + 1e-12
    assert ((r.rewards.double() - rewards).abs() <= tol_r).all()
    # |d loss / d z| <= 1 / N a pair
    assert abs(r.loss.item() - loss.item()) <= (tol_r[:N] + tol_r[N:]).mean().item() + 2.0 ** -23 * abs(loss.item())
    _assert_logp(r.logprobs[keep], logp[keep])
    assert (r.logprobs[~keep] == 0).all()
    dlogp = torch.where(keep, beta * torch.cat([dz, -dz]).unsqueeze(1), torch.zeros_like(logp))
    # d^2 loss / d z^2 <= 1 / (4 N): what the rewards' tolerance moves the gradient by
    loose = (beta / (4 * N) * (tol_r[:N] + tol_r[N:])).repeat(2)[:, None, None] / temperature + 2.0 ** -23 * dlogp.abs().unsqueeze(-1)
    xs = x.detach().double() / temperature
    p = torch.softmax(xs, -1)
    hot = torch.zeros_like(p).scatter_(-1, tokens.unsqueeze(-1), 1.0)
    for up, got in ((1.0, d), (-96.0, torch.autograd.grad(r.loss * -96.0, x)[0])):
        gg = up * (dlogp / temperature).unsqueeze(-1)
        exact = gg * (hot - p)
        tol = abs(up) * loose * (hot - p).abs() + gg.abs() * (2.0 ** -18 * p + 2.0 ** -23) \
            + torch.finfo(dtype).eps / 2 * exact.abs() * 1.001 + (2.0 ** -25 if dtype == torch.float16 else 1e-37)
        err = (got.double() - exact).abs()
        assert (err <= tol).all(), (err / tol).max().item()
        assert (got[~keep] == 0).all()


def test_preference_loss_far_apart():
    """Rewards hundreds apart: the loss grows linearly on the wrong side and vanishes on the
    right one, without overflow."""
    from mamba3_ssm import preference_loss
    x, tokens = _inputs((4, 50, 30), torch.float32, 22)
    ref = torch.zeros(4, 50, device=DEV)
    ref[0], ref[3] = 100.0, 100.0  # chosen 0 far worse, rejected 1 far worse
    x.requires_grad_(True)
    r = preference_loss(x, tokens, ref, beta=1.0)
    d, = torch.autograd.grad(r.loss, x)
    z = (r.rewards[:2] - r.rewards[2:]).double()
    assert z[0] < -3000 and z[1] > 3000
    assert abs(r.loss.item() + z[0].item() / 2) <= 2.0 ** -20 * r.loss.item()
    assert torch.isfinite(d).all() and (d[1] == 0).all() and (d[0] != 0).any()
    e = x.detach()[:, :0].requires_grad_(True)
    r = preference_loss(e, tokens[:, :0], beta=1.0)
    assert abs(r.loss.item() - math.log(2)) <= 2.0 ** -23 and (r.rewards == 0).all()
    assert torch.autograd.grad(r.loss, e)[0].shape == e.shape


# ------------------------------------------------------------------------ use and refusals
def test_same_inputs_same_bits():
    from mamba3_ssm import policy_loss
    x, tokens = _inputs((6, 200, 3001), torch.bfloat16, 23)
    x.requires_grad_(True)
    old = _off_border(x.detach(), tokens, 0.2, 0.2, 1.0, _gen(24))
    adv = torch.randn(6, 200, device=DEV, generator=_gen(25))
    first = None
    for _ in range(3):
        r = policy_loss(x, tokens, old, adv, ref_logprobs=old, kl_coef=0.1)
        now = [t.detach() for t in r] + [torch.autograd.grad(r.loss, x)[0]]
        if first is not None:
            assert all(torch.equal(a, b) for a, b in zip(first, now))
        first = now


def test_without_grad_no_gradient_is_formed():
    from mamba3_ssm import policy_loss
    x, tokens = _inputs((4, 256, 8192), torch.bfloat16, 26)
    x.requires_grad_(True)
    z = torch.zeros(4, 256, device=DEV)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    with torch.no_grad():
        r = policy_loss(x, tokens, z, z + 1)
    assert not r.loss.requires_grad
    assert torch.cuda.max_memory_allocated() - before < x.numel()  # half the gradient's bytes


def test_on_another_stream_and_captured():
    """The step on a side stream, then as a captured graph replayed on new inputs beside a
    second graph, with the eager result of the same inputs as the reference."""
    from mamba3_ssm import policy_loss, preference_loss
    shape = (4, 33, 5001)
    data = [(_inputs(shape, torch.bfloat16, 30 + i)) for i in range(3)]
    adv = torch.randn(4, 33, device=DEV, generator=_gen(40))
    old = torch.full((4, 33), -7.0, device=DEV)

    def policy(x, tokens):
        r = policy_loss(x, tokens, old, adv, ref_logprobs=old, kl_coef=0.1, clip_low=0.9, clip_high=50.0)
        return r.loss, r.logprobs, torch.autograd.grad(r.loss, x)[0]

    def preference(x, tokens):
        r = preference_loss(x, tokens, old, beta=0.2)
        return r.loss, r.rewards, torch.autograd.grad(r.loss, x)[0]

    want = {}
    for f in (policy, preference):
        for i, (x, t) in enumerate(data):
            want[f, i] = [v.detach().clone() for v in f(x.clone().requires_grad_(True), t)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [v.detach() for v in policy(data[1][0].clone().requires_grad_(True), data[1][1])]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[policy, 1]))

    graphs = []
    for f in (policy, preference):
        x, t = data[0][0].clone().requires_grad_(True), data[0][1].clone()
        with torch.cuda.stream(side):
            for _ in range(2):
                f(x, t)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = [v.detach() for v in f(x, t)]
        graphs.append((f, graph, x, t, out))
    for i in (2, 1, 0):
        for f, graph, x, t, out in graphs:
            with torch.no_grad():
                x.copy_(data[i][0])
            t.copy_(data[i][1])
        for f, graph, x, t, out in graphs:
            graph.replay()
        for f, graph, x, t, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want[f, i])), (f.__name__, i)


def test_offsets_beyond_32_bits():
    """More than 2^31 logits: the last rows, which lie beyond, against their definition."""
    from mamba3_ssm import policy_loss, token_logprobs
    T, V = 33000, 66000
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    x = torch.zeros(1, T, V, dtype=torch.bfloat16, device=DEV)
    last = 50
    x[:, -last:].normal_(generator=_gen(41))
    tokens = torch.randint(0, V, (1, T), device=DEV, generator=_gen(42))
    _assert_logp(token_logprobs(x, tokens)[:, -last:], _logp64(x[:, -last:], tokens[:, -last:]))
    x.requires_grad_(True)
    mask = torch.zeros(1, T, dtype=torch.bool, device=DEV)
    mask[:, -last:] = True
    old = torch.full((1, T), -11.0, device=DEV)
    adv = torch.ones(1, T, device=DEV)
    r = policy_loss(x, tokens, old, adv, mask=mask, clip_high=1e9)
    d, = torch.autograd.grad(r.loss, x)
    logp = _logp64(x[:, -last:].detach(), tokens[:, -last:])
    _assert_logp(r.logprobs[:, -last:], logp)
    xs = x.detach()[:, -last:].contiguous()
    ratio = (logp + 11.0).exp()
    # the ratio's own tolerance is that of the log-probability
    p = torch.softmax(xs.double(), -1)
    hot = torch.zeros_like(p).scatter_(-1, tokens[:, -last:].unsqueeze(-1), 1.0)
    exact = (-ratio / last).unsqueeze(-1) * (hot - p)
    err = (d[:, -last:].double() - exact).abs()
    u = torch.finfo(torch.bfloat16).eps / 2  # 2^-8: eight significant bits
    assert (err <= exact.abs() * (u + 2.0 ** -17) * 1.01 + (ratio / last).unsqueeze(-1) * 2.0 ** -23).all()
    assert (d[:, :100] == 0).all()


def test_model_scores_its_inputs():
    """MambaLMHeadModel.token_logprobs, then a policy step and the clipping on its logits: a
    whole fine-tuning step through the public entry points."""
    from mamba3_ssm import MambaConfig, MambaLMHeadModel, clip_grad_norm_, policy_loss
    torch.manual_seed(0)
    cfg = MambaConfig(d_model=64, n_layer=2, vocab_size=101, ssm_cfg=dict(d_state=32, headdim=32))
    model = MambaLMHeadModel(cfg).to(DEV)
    ids = torch.randint(0, 101, (4, 20), device=DEV, generator=_gen(50))
    mask = torch.ones(4, 19, dtype=torch.bool, device=DEV)
    mask[:, :5] = False
    with torch.no_grad():
        old = model.token_logprobs(ids, mask=mask)
        logits = model(ids)
    _assert_logp(old[mask], _logp64(logits[:, :-1], ids[:, 1:])[mask])
    assert (old[~mask] == 0).all()
    adv = torch.randn(4, 1, device=DEV, generator=_gen(51))
    # whole logits; the last position is ignored
    targets = torch.cat([ids[:, 1:], torch.full_like(ids[:, :1], IGN)], 1)
    pad = torch.nn.functional.pad
    logits = model(ids)
    r = policy_loss(logits, targets, pad(old, (0, 1)), adv, ref_logprobs=pad(old - 0.1, (0, 1)), kl_coef=0.1,
                    mask=pad(mask, (0, 1)))
    r.loss.backward()
    # the same loss in torch's operations, differentiated by torch
    grads = [p.grad.clone() for p in model.parameters() if p.grad is not None]
    model.zero_grad()
    lp = torch.log_softmax(model(ids)[:, :-1].double(), -1).gather(-1, ids[:, 1:, None]).squeeze(-1)
    d = old.double() - 0.1 - lp
    rt = (lp - old.double()).exp()
    per = -torch.minimum(rt * adv, rt.clamp(0.8, 1.2) * adv) + 0.1 * (torch.expm1(d) - d)
    loss = per[mask].mean()
    loss.backward()
    assert abs(r.loss.item() - loss.item()) <= 1e-5 + 1e-5 * abs(loss.item())
    ref = [p.grad for p in model.parameters() if p.grad is not None]
    assert len(ref) == len(grads)
    for a, b in zip(grads, ref):
        # 32-bit gradients through the same layers: their own summation error dominates
        assert (a - b).abs().max() <= 1e-4 * b.abs().max() + 1e-7
    norm = torch.cat([g.flatten().double() for g in ref]).norm()
    got = clip_grad_norm_(model.parameters(), 0.1 * norm.item())
    assert abs(got.item() - norm.item()) <= 1e-6 * norm.item()
    after = torch.cat([g.flatten().double() for g in ref]).norm()
    assert abs(after.item() - 0.1 * norm.item()) <= 1e-5 * norm.item()


def test_refusals():
    from mamba3_ssm import policy_loss, preference_loss, token_logprobs
    x, tokens = _inputs((2, 4, 16), torch.float32, 60)
    z = torch.zeros(2, 4, device=DEV)
    with pytest.raises(ValueError, match="tokens"):
        token_logprobs(x, tokens[:, :3])
    with pytest.raises(TypeError, match="logits"):
        token_logprobs(x.double(), tokens)
    with pytest.raises(TypeError, match="integers"):
        token_logprobs(x, z)
    with pytest.raises(ValueError, match="empty vocabulary"):
        token_logprobs(x[..., :0], tokens)
    with pytest.raises(RuntimeError, match="no CPU path"):
        token_logprobs(x, tokens.cpu())
    with pytest.raises(RuntimeError, match="mask is on"):
        token_logprobs(x, tokens, mask=torch.ones(2, 4))
    with pytest.raises(ValueError, match="broadcast"):
        token_logprobs(x, tokens, mask=torch.ones(3, 4, device=DEV))
    for t in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(RuntimeError, match="temperature"):
            token_logprobs(x, tokens, temperature=t)
    with pytest.raises(ValueError, match="reduction"):
        policy_loss(x, tokens, z, z, reduction="mean")
    with pytest.raises(ValueError, match="ref_logprobs"):
        policy_loss(x, tokens, z, z, kl_coef=0.1)
    with pytest.raises(RuntimeError, match="clip_low"):
        policy_loss(x, tokens, z, z, clip_low=1.5)
    with pytest.raises(RuntimeError, match="clip_high"):
        policy_loss(x, tokens, z, z, clip_high=-0.1)
    with pytest.raises(RuntimeError, match="kl_coef"):
        policy_loss(x, tokens, z, z, ref_logprobs=z, kl_coef=-1.0)
    with pytest.raises(ValueError, match="2 N"):
        preference_loss(x[:1], tokens[:1])
    with pytest.raises(ValueError, match="2 N"):
        preference_loss(x[0], tokens[0])
    with pytest.raises(RuntimeError, match="beta"):
        preference_loss(x, tokens, beta=-1.0)
    with pytest.raises(RuntimeError, match="label_smoothing"):
        preference_loss(x, tokens, label_smoothing=1.5)
    # a second derivative
    x.requires_grad_(True)
    d, = torch.autograd.grad(token_logprobs(x, tokens).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.sum(), x)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [700, 9000, 60001, 140000])
def test_rows_whose_first_elements_mislead(V, dtype):
    """Rows whose first elements and token lie far below the rest (the sum over an assumed base
    then overflows), are excluded, or are all there is; one row of each kind in turn, with
    ordinary rows between: forward, policy gradient and the gradient of log-probabilities."""
    from mamba3_ssm import policy_loss, token_logprobs
    from mamba3_ssm import _lib
    B, T = 2, 12
    x, tokens = _inputs((B, T, V), dtype, 70)
    few = min(300, V // 2)
    tokens %= few
    x[:, 1::6, :few] = -150.0
    x[:, 2::6, :few] = float("-inf")
    x[:, 2::6, 0] = -120.0
    tokens[:, 2::6] = 0
    x[:, 3::6, :] = torch.finfo(dtype).min
    x[:, 4::6, :few] = torch.finfo(dtype).min
    tokens[:, 4::6] = V - 1
    ref = _logp64(x, tokens)
    y = x.clone().requires_grad_(True)
    out = token_logprobs(y, tokens)
    _assert_logp(out.detach(), ref)
    dout = torch.randn(B, T, device=DEV, generator=_gen(71))
    d, = torch.autograd.grad(out, y, dout)
    _assert_grad(d, x, tokens, dout.double())
    old = ref.float()  # ratios of 1
    r = policy_loss(y, tokens, old, dout)
    # off by the rounding of old to 32 bits and the log-probability's tolerance
    loss = -dout.double().mean()
    slack = (dout.double().abs() * (LOGP_TOL + 2.0 ** -23 * ref.abs())).mean()
    assert abs(r.loss.item() - loss.item()) <= slack.item() + 1e-6 * abs(loss.item())
    d, = torch.autograd.grad(r.loss, y)
    p = torch.softmax(x.double(), -1)
    hot = torch.zeros_like(p).scatter_(-1, tokens.unsqueeze(-1), 1.0)
    g = (-dout.double() / (B * T)).unsqueeze(-1)
    exact = g * (hot - p)
    loose = (LOGP_TOL + 2.0 ** -22 * ref.abs()).unsqueeze(-1)
    tol = exact.abs() * (loose + torch.finfo(dtype).eps / 2 * 1.001) + g.abs() * (2.0 ** -18 * p + 2.0 ** -23) + 1e-37
    assert ((d.double() - exact).abs() <= tol).all()
    assert _lib.device_timeouts() == 0


def test_two_calls_at_once():
    """Two policy steps and two clippings on two streams beside each other: the results of each
    alone."""
    from mamba3_ssm import clip_grads_, policy_loss
    data = [_inputs((8, 100, 50001), torch.bfloat16, 80 + i) for i in range(2)]
    adv = torch.randn(8, 100, device=DEV, generator=_gen(82))
    old = torch.full((8, 100), -9.0, device=DEV)
    leaves = [x.requires_grad_(True) for x, _ in data]
    grads = [torch.randn(3000001, device=DEV, generator=_gen(83 + i)) for i in range(2)]

    def step(i):
        r = policy_loss(leaves[i], data[i][1], old, adv, clip_low=1.0, clip_high=1e6)
        g = grads[i].clone()
        return [r.loss.detach(), r.logprobs, torch.autograd.grad(r.loss, leaves[i])[0], clip_grads_([g], 1.0), g]

    want = [step(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = [None, None]
        for i in range(2):
            streams[i].wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(streams[i]):
                got[i] = step(i)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_changed_inputs_are_noticed():
    """What backward reads again must not have changed in between."""
    from mamba3_ssm import token_logprobs
    x, tokens = _inputs((2, 3, 64), torch.float32, 90)
    x = x.requires_grad_(True)
    y = x * 1.0
    out = token_logprobs(y, tokens)
    with torch.no_grad():
        y.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["cut", "wide", "shifted", "transposed", "offset", "expanded"])
@pytest.mark.parametrize("V", [513, 9001, 70003])
def test_policy_loss_layouts(V, layout, dtype):
    """Rows of every layout, whose gradient may start on other boundaries than the logits, at
    lengths that each of the kernels takes; advantages and masks broadcast."""
    from mamba3_ssm import policy_loss
    x, tokens = _inputs((3, 7, V), dtype, 95, layout)
    logp = _logp64(x, tokens)
    old = (logp - 0.1).float()
    adv = torch.tensor([[1.0], [-2.0], [0.5]], device=DEV)
    mask = torch.arange(7, device=DEV) != 2
    leaf = x.detach().requires_grad_(True)
    r = policy_loss(leaf, tokens, old, adv, mask=mask, clip_low=0.5, clip_high=0.5)
    d, = torch.autograd.grad(r.loss, leaf)
    ratio = (logp - old.double()).exp()
    keep = mask.expand(3, 7)
    dlogp = torch.where(keep, -ratio * adv.double() / 18, torch.zeros_like(ratio))
    assert torch.equal(r.logprobs == 0, ~keep)
    _assert_logp(r.logprobs[keep], logp[keep])
    # the ratio carries the log-probability's tolerance: 2^-19 of the gradient, beside p's 2^-18
    p = torch.softmax(x.double(), -1)
    hot = torch.zeros_like(p).scatter_(-1, tokens.unsqueeze(-1), 1.0)
    exact = dlogp.unsqueeze(-1) * (hot - p)
    u = torch.finfo(dtype).eps / 2
    tol = exact.abs() * (u * 1.001 + 2.0 ** -18) + dlogp.abs().unsqueeze(-1) * (2.0 ** -18 * p + 2.0 ** -23) + 1e-37
    assert ((d.double() - exact).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [12000, 60001, 140000])
def test_misleading_rows_without_grad_have_the_same_bits(V, dtype):
    """Rows that are summed a second time, over their true maximum, too."""
    from mamba3_ssm import policy_loss
    B, T = 10, 40
    x, tokens = _inputs((B, T, V), dtype, 105)
    x[..., :V // 2] = -150.0
    adv = torch.randn(B, T, device=DEV, generator=_gen(106))
    old = torch.full((B, T), -11.0, device=DEV)
    plain = policy_loss(x, tokens, old, adv)
    r = policy_loss(x.requires_grad_(True), tokens, old, adv)
    for a, b in zip(plain, r):
        assert torch.equal(a, b.detach())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["contiguous", "cut"])
@pytest.mark.parametrize("T,V", [(1000, 257), (1000, 300), (390, 1000), (154, 2500), (154, 5999), (61, 12000)])
def test_many_short_rows(T, V, layout, dtype):
    """So many rows that several share a warp and each warp takes several turns. Among them, in
    every order: positions that do not count, rows whose first elements and token lie far below
    the rest, excluded elements, a type's lowest value."""
    from mamba3_ssm import _lib, policy_loss, token_logprobs
    B = 41
    x, tokens = _inputs((B, T, V), dtype, 110, layout)
    g = _gen(111)
    few = min(300, V // 2)
    kind = torch.randint(0, 10, (B, T), device=DEV, generator=g)
    low = torch.finfo(dtype).min
    tokens = torch.where(kind < 3, tokens % few, tokens)
    x[..., :few].masked_fill_((kind == 0).unsqueeze(-1), -150.0)
    x[..., 1:].masked_fill_((kind == 1).unsqueeze(-1), float("-inf"))
    tokens.masked_fill_(kind == 1, 0)
    x.masked_fill_((kind == 2).unsqueeze(-1), low)
    x[..., :-1].masked_fill_((kind == 3).unsqueeze(-1), low)
    tokens.masked_fill_(kind == 3, V - 1)
    keep = torch.rand(B, T, device=DEV, generator=g) < 0.7
    keep[5] = False
    logp = torch.stack([_logp64(x[b], tokens[b]) for b in range(B)])
    old = (logp - 0.1).float()
    adv = torch.randn(B, 1, device=DEV, generator=g)
    dout = torch.randn(B, T, device=DEV, generator=g)
    n = keep.sum().item()
    leaf = x.detach().requires_grad_(True)
    out = token_logprobs(leaf, tokens, mask=keep)
    _assert_logp(out.detach()[keep], logp[keep])
    assert (out.detach()[~keep] == 0).all()
    d, = torch.autograd.grad(out, leaf, dout)
    r = policy_loss(leaf, tokens, old, adv, mask=keep, clip_low=0.5, clip_high=0.5)
    dp, = torch.autograd.grad(r.loss, leaf)
    plain = policy_loss(x, tokens, old, adv, mask=keep, clip_low=0.5, clip_high=0.5)
    for a, b in zip(plain, r):
        assert torch.equal(a, b.detach())
    # the scale's rounding to 32 bits, the base's and their product's: 2^-22 of a logit's distance
    loose = LOGP_TOL + 2.0 ** -22 * logp.abs()
    assert ((r.logprobs.double() - logp).abs() <= loose)[keep].all()
    ratio = (logp - old.double()).exp()
    per = torch.where(keep, ratio * adv.double(), torch.zeros_like(ratio)) / n
    assert abs(r.loss.item() + per.sum().item()) <= (per.abs() * (loose + 2.0 ** -22)).sum().item() + 1e-12
    u = torch.finfo(dtype).eps / 2
    least = 2.0 ** -25 if dtype == torch.float16 else 1e-37
    for b in range(B):
        one = slice(b, b + 1)
        _assert_grad(d[one], x[one], tokens[one], torch.where(keep, dout, torch.zeros_like(dout))[one].double())
        p = torch.softmax(x[one].double(), -1)
        hot = torch.zeros_like(p).scatter_(-1, tokens[one].unsqueeze(-1), 1.0)
        gg = -per[one].unsqueeze(-1)
        exact = gg * (hot - p)
        tol = exact.abs() * (u * 1.001 + loose[one].unsqueeze(-1) + 2.0 ** -20) + gg.abs() * (2.0 ** -18 * p + 2.0 ** -23)
        assert ((dp[one].double() - exact).abs() <= tol + least).all()
    assert (dp[~keep] == 0).all() and (d[~keep] == 0).all()
    assert _lib.device_timeouts() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [1, 2, 7, 9, 31, 70])
def test_many_rows_of_a_few_logits(V, dtype):
    """Rows with few or no whole vectors, on every boundary, several to a warp."""
    from mamba3_ssm import policy_loss, token_logprobs
    x, tokens = _inputs((41, 1000, V), dtype, 120)
    logp = _logp64(x, tokens)
    leaf = x.detach().requires_grad_(True)
    dout = torch.randn(41, 1000, device=DEV, generator=_gen(121))
    out = token_logprobs(leaf, tokens)
    _assert_logp(out.detach(), logp)
    d, = torch.autograd.grad(out, leaf, dout)
    _assert_grad(d, x, tokens, dout.double())
    old = (logp - 0.1).float()
    r = policy_loss(leaf, tokens, old, dout, clip_low=0.5, clip_high=0.5)
    _assert_logp(r.logprobs, logp)
    dp, = torch.autograd.grad(r.loss, leaf)
    p = torch.softmax(x.double(), -1)
    hot = torch.zeros_like(p).scatter_(-1, tokens.unsqueeze(-1), 1.0)
    gg = -((logp - old.double()).exp() * dout.double() / 41000).unsqueeze(-1)
    exact = gg * (hot - p)
    # the ratio carries the log-probability's tolerance, p its own
    tol = exact.abs() * (torch.finfo(dtype).eps / 2 * 1.001 + 2.0 ** -18) + gg.abs() * (2.0 ** -18 * p + 2.0 ** -23)
    tol = tol + (2.0 ** -25 if dtype == torch.float16 else 1e-37)
    assert ((dp.double() - exact).abs() <= tol).all()


@pytest.mark.parametrize("gap", [49.0, 65.0])
@pytest.mark.parametrize("V", [2000, 30000, 140000])
def test_small_gradients_of_misleading_rows(V, gap):
    """A base far below the maximum makes the sum large and the upstream gradient over it small:
    it must not leave the normal numbers (dlogp 1e-14 with the maximum 65 above the base would)."""
    from mamba3_ssm import policy_loss, token_logprobs
    x = torch.zeros(1, 3, V, device=DEV)
    tokens = torch.zeros(1, 3, dtype=torch.long, device=DEV)
    x[0, :, V - 9] = gap
    x.requires_grad_(True)
    dout = torch.full((1, 3), 1e-14, device=DEV)
    d, = torch.autograd.grad(token_logprobs(x, tokens), x, dout)
    _assert_grad(d, x.detach(), tokens, dout.double())
    r = policy_loss(x, tokens, _logp64(x.detach(), tokens).float(), dout)
    d, = torch.autograd.grad(r.loss, x)
    # ratios of 1, off by old's rounding (2^-24 of up to 65) and the tolerance of a log-probability
    exact = -dout.double() / 3
    top = -exact * torch.softmax(x.detach().double(), -1)[..., V - 9]
    assert ((d[..., V - 9].double() - top).abs() <= 2.0 ** -17 * top.abs()).all()
    assert ((d[..., 0].double() - exact).abs() <= 2.0 ** -17 * exact.abs()).all()


@pytest.mark.parametrize("V", [700, 9000, 60001, 140000])
def test_gradients_where_the_maximum_is_far_above_the_first_elements(V):
    """A low temperature spreads the scaled logits over hundreds: the first elements' maximum is
    tens below the row's, and the tolerances are those of any row."""
    from mamba3_ssm import token_logprobs
    x, tokens = _inputs((2, 40, V), torch.float32, 117)
    x.requires_grad_(True)
    dout = torch.randn(2, 40, device=DEV, generator=_gen(118))
    out = token_logprobs(x, tokens, temperature=0.1)
    _assert_logp(out.detach(), _logp64(x.detach(), tokens, 0.1))
    d, = torch.autograd.grad(out, x, dout)
    _assert_grad(d, x.detach(), tokens, dout.double(), 0.1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V", [(4096, 5001), (600, 30011)])
@pytest.mark.parametrize("temperature", [0.7, 0.8, 2.88])
def test_policy_logprobs_of_unlikely_tokens(temperature, rows, V, dtype):
    """The policy loss holds scale = log2(e) / temperature in one float, rounded to the nearest: a
    log-probability is off by that rounding times scale (l[token] - mean of l under p), the same
    way in every row. Mean error of the rows: that, the sums' (LOGP_TOL), and what is left of
    the results' own rounding, evenly spread over a step (six standard deviations)."""
    from mamba3_ssm import policy_loss
    x, tokens = _inputs((1, rows, V), dtype, 114)
    x.scatter_(-1, tokens.unsqueeze(-1), -100.0 * temperature)
    ref = _logp64(x, tokens, temperature)
    zero = torch.zeros(1, rows, device=DEV)
    got = policy_loss(x, tokens, old_logprobs=ref.float(), advantages=zero + 1, temperature=temperature).logprobs
    mean = (torch.softmax(x.double() / temperature, -1) * x.double()).sum(-1)
    c = 1.0 / math.log(2.0) / temperature
    rounding = abs(torch.tensor(c, dtype=torch.float64).float().item() / c - 1.0)
    assert rounding <= 2.0 ** -24
    moved = rounding * ((x.double().gather(-1, tokens.unsqueeze(-1)).squeeze(-1) - mean) / temperature).abs().max().item()
    step = 2.0 ** -17  # of results between 64 and 128
    assert ((ref < -64) & (ref > -128)).all()
    left = 6 * step / math.sqrt(12 * rows)
    assert abs((got.double() - ref).mean().item()) <= moved + LOGP_TOL + left


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("value", [-1e9, -1e10, 1e12, -1e20, 3e29, -726000.0, -727500.0, 43000.0])
@pytest.mark.parametrize("V", [300, 9000, 60001, 140000, 900001])
def test_rows_far_from_zero(V, value, dtype):
    """Rows that hold one mask's constant alone, two of them, or a spread around it, at scaled
    magnitudes where the rounding of base times scale leaves the exponents' range (and on either
    side of 2^20, from which the difference to the base is formed first), beside ordinary ones.
    Tolerances as in test_rows_whose_first_elements_mislead; the policy's scale is one float,
    2^-24 of the log-probability. LOGP_TOL and 2^-18 of p are of up to 131072 logits: beyond, a
    thread's chains of additions, and with them their bound, grow with V."""
    from mamba3_ssm import _lib, policy_loss, preference_loss, token_logprobs
    B, T = 2, 4
    x, tokens = _inputs((B, T, V), dtype, 110)
    x[:, 0] = value
    x[:, 1] = value
    x[:, 1, V // 2:] = value - abs(value) / 32
    tokens[:, 1] %= V // 2
    x[:, 2] += value
    dout = torch.randn(B, T, device=DEV, generator=_gen(111))
    leaf = x.clone().requires_grad_(True)
    long = max(1.0, V / 131072)
    sums, u = LOGP_TOL * long, torch.finfo(dtype).eps / 2
    for temperature in (1.0, 0.7, 0.6, 0.1):
        ref = _logp64(x, tokens, temperature)
        p = torch.softmax(x.double() / temperature, -1)
        hot = torch.zeros_like(p).scatter_(-1, tokens.unsqueeze(-1), 1.0)
        out = token_logprobs(leaf, tokens, temperature=temperature)
        assert ((out.double() - ref).abs() <= sums + 2.0 ** -24 * ref.abs()).all()
        d, = torch.autograd.grad(out, leaf, dout)
        g = (dout.double() / temperature).unsqueeze(-1)
        exact = g * (hot - p)
        of_p = long * 2.0 ** -18 * p + 2.0 ** -23
        assert ((d.double() - exact).abs() <= g.abs() * of_p + u * exact.abs() * (1 + 2.0 ** -10) + 1e-37).all()
        old = ref.float()  # ratios of 1
        r = policy_loss(leaf, tokens, old, dout, temperature=temperature)
        bare = policy_loss(x, tokens, old, dout, temperature=temperature)
        assert torch.equal(r.loss.detach(), bare.loss) and torch.equal(r.logprobs, bare.logprobs)
        slack = (dout.double().abs() * (sums + 2.0 ** -22 * ref.abs())).mean()
        assert abs(r.loss.item() + dout.double().mean().item()) <= slack.item() + 1e-6 * abs(dout.double().mean().item())
        g, exact = -g / (B * T), -exact / (B * T)
        tol = exact.abs() * ((sums + 2.0 ** -22 * ref.abs()).unsqueeze(-1) + u * 1.001) + g.abs() * of_p + 1e-37
        for up in (1.0, 3.0):
            d, = torch.autograd.grad(r.loss * up, leaf, retain_graph=True)
            assert ((d.double() - up * exact).abs() <= up * tol).all()
        q = preference_loss(leaf, tokens, old, temperature=temperature)
        reward_tol = 0.1 * (sums + 2.0 ** -24 * ref.abs()).sum(1) + 1e-12  # old's rounding
        assert (q.rewards.double().abs() <= reward_tol).all()
        assert abs(q.loss.item() - math.log(2.0)) <= reward_tol.sum().item() + 2.0 ** -23
        assert torch.isfinite(torch.autograd.grad(q.loss, leaf)[0]).all()
    assert _lib.device_timeouts() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [50, 30000])
def test_kl_that_is_only_reported(V, dtype):
    """kl_coef 0 with reference log-probabilities: the loss and its gradient are those of the call
    without them, also where the KL term overflows (a token that is excluded or all but)."""
    from mamba3_ssm import policy_loss
    x, tokens = _inputs((2, 40, V), dtype, 112)
    old = _logp64(x, tokens).float()
    x[0, 3, int(tokens[0, 3])] = float("-inf")
    x[1, 5, int(tokens[1, 5])] = -200.0
    adv = torch.randn(2, 40, device=DEV, generator=_gen(113))
    leaf = x.requires_grad_(True)
    want = policy_loss(leaf, tokens, old, adv)
    r = policy_loss(leaf, tokens, old, adv, ref_logprobs=old - 0.1)
    assert r.loss.isfinite() and torch.equal(r.loss, want.loss) and torch.equal(r.logprobs, want.logprobs)
    assert r.kl.item() == math.inf and want.kl.item() == 0.0
    for up in (1.0, 2.0):
        d, = torch.autograd.grad(r.loss * up, leaf, retain_graph=True)
        assert d.isfinite().all() and torch.equal(d, torch.autograd.grad(want.loss * up, leaf, retain_graph=True)[0])
    assert (d[0, 3] == 0).all() and (d[1, 4] != 0).any()


@pytest.mark.parametrize("smoothing", [0.0, 0.1])
def test_preference_gradient_of_pairs_that_are_told_apart(smoothing):
    """-(1 - e) sigma(-z) + e sigma(z), also where sigma(z) is 1 to the last bit: a margin's error
    is a relative one of sigma(-z); 4 tokens an answer, each with LOGP_TOL."""
    from mamba3_ssm import preference_loss
    N, T, V = 6, 4, 50
    x, tokens = _inputs((2 * N, T, V), torch.float32, 115)
    logp = _logp64(x, tokens)
    margin = torch.tensor([5.0, 20.0, 30.0, 45.0, 60.0, 70.0], device=DEV, dtype=torch.float64)
    ref = logp.clone()
    ref[:N] -= margin[:, None] / T
    ref = ref.float()
    z = (logp - ref.double()).sum(1)
    z = z[:N] - z[N:]
    x.requires_grad_(True)
    r = preference_loss(x, tokens, ref, beta=1.0, label_smoothing=smoothing)
    d, = torch.autograd.grad(r.loss, x)
    dz = (smoothing * torch.sigmoid(z) - (1 - smoothing) * torch.sigmoid(-z)) / N
    dz = torch.cat([dz, -dz])[:, None, None]
    p = torch.softmax(x.detach().double(), -1)
    hot = torch.zeros_like(p).scatter_(-1, tokens.unsqueeze(-1), 1.0)
    exact = dz * (hot - p)
    moved = 2 * T * LOGP_TOL * (torch.sigmoid(-z) / N)  # d^2 loss / d z^2 <= sigma(-z) / N
    tol = moved.repeat(2)[:, None, None] * (hot - p).abs() + dz.abs() * (2.0 ** -18 * p + 2.0 ** -22) + 1e-37
    assert ((d.double() - exact).abs() <= tol).all()
    assert (d != 0).all()


def test_preference_loss_with_an_excluded_token():
    """A rejected answer with a token of logit -inf has the reward -inf: the pair costs nothing and
    has no gradient, whatever the other pairs; with smoothing, or as the chosen one, it costs
    infinitely much."""
    from mamba3_ssm import preference_loss
    x, tokens = _inputs((4, 6, 50), torch.float32, 119)
    want = preference_loss(x[1::2], tokens[1::2], beta=1.0)
    x[2, 3, int(tokens[2, 3])] = float("-inf")
    x.requires_grad_(True)
    r = preference_loss(x, tokens, beta=1.0)
    assert r.rewards[2].item() == -math.inf
    assert abs(r.loss.item() - want.loss.item() / 2) <= 2.0 ** -23 * want.loss.item()
    d, = torch.autograd.grad(r.loss, x)
    assert (d[::2] == 0).all() and d.isfinite().all() and (d[1::2] != 0).any()
    assert preference_loss(x, tokens, beta=1.0, label_smoothing=0.1).loss.item() == math.inf
    swapped = torch.cat([x[2:], x[:2]]), torch.cat([tokens[2:], tokens[:2]])
    assert preference_loss(*swapped, beta=1.0).loss.item() == math.inf
    assert preference_loss(*swapped, beta=1.0, label_smoothing=1.0).loss.isfinite()


def test_forward_mode_tangents_are_refused():
    """There is no forward-mode derivative: a tangent of the logits must not be lost silently,
    with or without a gradient."""
    import torch.autograd.forward_ad as fwd
    from mamba3_ssm import policy_loss, preference_loss, token_logprobs
    x, tokens = _inputs((2, 4, 100), torch.float32, 116)
    z = torch.zeros(2, 4, device=DEV)
    calls = (lambda y: token_logprobs(y, tokens), lambda y: policy_loss(y, tokens, z, z + 1),
             lambda y: preference_loss(y, tokens))
    with fwd.dual_level():
        for leaf in (x, x.clone().requires_grad_(True)):
            dual = fwd.make_dual(leaf, torch.ones_like(x))
            for call in calls:
                with pytest.raises(NotImplementedError):
                    call(dual)
                with torch.no_grad(), pytest.raises(NotImplementedError):
                    call(dual)
        for call in calls:
            call(x)  # no tangent: as ever
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(calls[0], (x,), (torch.ones_like(x),))
