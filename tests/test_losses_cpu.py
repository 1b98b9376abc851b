"""Token losses and gradient clipping without a GPU: the checks that the C entries make on the
host, the Python entry points' refusals, and the arithmetic that the kernels rely on, restated
in numpy (assumed base of a row, split logarithm, series of the KL term, rounding by addition)."""

import ctypes
import math

import numpy as np
import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from mamba3_ssm import _lib
    return _lib.load()


def _view(shape, code, data=4096, stride=None):
    """A descriptor at a fake address: every call below ends on the host."""
    from mamba3_ssm import _lib
    m = _lib.M3Tensor()
    m.data, m.dtype, m.ndim = data, code, len(shape)
    st = 1
    for i in range(len(shape) - 1, -1, -1):
        m.shape[i], m.stride[i] = shape[i], st
        st *= max(shape[i], 1)
    if stride is not None:
        m.stride[:len(stride)] = stride
    return m


def _codes():
    from mamba3_ssm import _lib
    return _lib.M3_FLOAT32, _lib.M3_BFLOAT16, _lib.M3_INT64, _lib.M3_UINT8


class _Policy:
    """A call of m3_policy_loss on an empty batch (2 sequences of no position)."""

    def __init__(self, lib):
        f32, bf, i64, u8 = _codes()
        self.lib = lib
        self.t = dict(logits=_view((2, 0, 7), bf), tokens=_view((2, 0), i64), mask=_view((2, 0), u8),
                      old=_view((2, 0), f32), adv=_view((2, 0), f32), ref=_view((2, 0), f32))
        self.out = dict(loss=None, kl_out=None, clip=None, logp=_view((2, 0), f32), dlogits=_view((2, 0, 7), bf))
        self.n = dict(temperature=1.0, ignore=-100, lo=0.2, hi=0.2, kl=0.1, seq=0)

    def __call__(self, **change):
        for k, v in change.items():
            for d in (self.t, self.out, self.n):
                if k in d:
                    d[k] = v
        ref = [None if v is None else ctypes.byref(v) for v in self.t.values()]
        out = [None if v is None else ctypes.byref(v) for v in self.out.values()]
        rc = self.lib.m3_policy_loss(*ref, *self.n.values(), *out, None, 0, None)
        return rc, self.lib.m3_last_error_string().decode()


@pytest.mark.parametrize("change,word", [
    (dict(logits=None), "logits: missing"),
    (dict(logits="2d"), "logits: expected"),
    (dict(logits="novocab"), "empty vocabulary"),
    (dict(logits="int"), "logits: unsupported dtype"),
    (dict(logits="large"), "dimension too large"),
    (dict(temperature=0.0), "temperature"),
    (dict(temperature=-1.0), "temperature"),
    (dict(temperature=math.nan), "temperature"),
    (dict(temperature=math.inf), "temperature"),
    (dict(tokens="f32"), "tokens: unsupported dtype"),
    (dict(tokens=None), "tokens: missing"),
    (dict(tokens="short"), "tokens: expected"),
    (dict(mask="f32"), "mask: unsupported dtype"),
    (dict(lo=-0.1), "clip_low"),
    (dict(lo=1.1), "clip_low"),
    (dict(lo=math.nan), "clip_low"),
    (dict(hi=-0.1), "clip_high"),
    (dict(hi=math.nan), "clip_high"),
    (dict(kl=-0.1), "kl_coef"),
    (dict(kl=math.inf), "kl_coef"),
    (dict(seq=2), "by_sequence"),
    (dict(old=None), "old_logprobs: missing"),
    (dict(adv="short"), "advantages: expected"),
    (dict(ref="u8"), "ref_logprobs: unsupported dtype"),
    (dict(dlogits="f32"), "dlogits: unsupported dtype"),
    (dict(loss=None), "loss: missing"),
])
def test_policy_loss_refusals(lib, change, word):
    f32, bf, i64, u8 = _codes()
    made = {"2d": _view((2, 7), bf), "novocab": _view((2, 0, 0), bf), "int": _view((2, 0, 7), i64),
            "large": _view((1 << 20, 1 << 20, 7), bf), "f32": _view((2, 0), f32), "short": _view((1, 0), f32),
            "u8": _view((2, 0), u8)}
    key, value = next(iter(change.items()))
    if key == "dlogits":
        value = _view((2, 0, 7), f32)
    elif key == "tokens" and value == "short":
        value = _view((1, 0), i64)
    elif isinstance(value, str):
        value = made[value]
    rc, msg = _Policy(lib)(**{key: value})
    assert rc in (1, 2) and word in msg, msg


def test_other_refusals(lib):
    f32, bf, i64, u8 = _codes()
    b = ctypes.byref
    logits, tokens = _view((2, 0, 7), bf), _view((2, 0), i64)
    assert lib.m3_token_logprobs(b(logits), b(tokens), None, 1.0, -100, None, None, None) == 1
    assert b"logprobs: missing" in lib.m3_last_error_string()
    assert lib.m3_token_logprobs(b(logits), b(tokens), None, 1.0, -100, b(_view((2, 0), f32)), None, None) == 0
    # not a multiple of the element's size
    odd = _view((2, 1, 7), bf, data=4097)
    assert lib.m3_token_logprobs(b(odd), b(_view((2, 1), i64)), None, 1.0, -100, b(_view((2, 1), f32)), None, None) == 1
    # a vocabulary that is not the innermost run of memory
    strided = _view((2, 3, 7), bf, stride=(21, 1, 3))
    assert lib.m3_token_logprobs(b(strided), b(_view((2, 3), i64)), None, 1.0, -100, b(_view((2, 3), f32)), None, None) == 1
    assert b"contiguous" in lib.m3_last_error_string()
    # an odd number of sequences, numbers outside their range
    one = _view((1, 0, 7), bf)
    for args, word in (((one, 0.1, 0.0), b"even number"), ((logits, -1.0, 0.0), b"beta"), ((logits, math.inf, 0.0), b"beta"),
                       ((logits, 0.1, 1.5), b"label_smoothing"), ((logits, 0.1, math.nan), b"label_smoothing")):
        x, beta, soft = args
        t = _view((x.shape[0], 0), i64)
        rc = lib.m3_preference_loss(b(x), b(t), None, None, 1.0, -100, beta, soft, None, None, None, None, 0, None)
        assert rc == 1 and word in lib.m3_last_error_string()
    rc = lib.m3_policy_loss_grad(b(logits), b(tokens), None, None, 1.0, -100, 2, b(logits), None, 0, None)
    assert rc == 1 and b"keep_if_one" in lib.m3_last_error_string()
    assert lib.m3_policy_loss_grad(b(logits), b(tokens), None, None, 1.0, -100, 1, b(logits), None, 0, None) == 0
    assert lib.m3_preference_loss_grad(b(logits), b(tokens), None, None, 1.0, -100, b(logits), None, 0, None) == 0


def test_workspace_sizes(lib):
    assert lib.m3_policy_loss_workspace_size(-1, 5) == 0 and lib.m3_preference_loss_workspace_size(5, -1) == 0
    # stats, coefficients, order and results of each row; counts of each sequence
    n = lib.m3_policy_loss_workspace_size(3, 1000)
    assert 3000 * (8 + 4 + 4 + 12) <= n <= 3000 * (8 + 4 + 4 + 12) + 1024
    n = lib.m3_preference_loss_workspace_size(4, 1000)
    assert 4000 * (8 + 8) <= n <= 4000 * (8 + 8) + 1024
    assert lib.m3_clip_grads_workspace_size(-1) == 0 and lib.m3_clip_grads_workspace_size(5000) > 0


def _clip(lib, tensors, outs=None, max_norm=1.0, scale=1.0, largest=0, norm=None):
    """m3_clip_grads on (address, elements, dtype) triples."""
    n = len(tensors)
    arr = lambda t, v: (t * max(n, 1))(*v) if v is not None else None  # noqa: E731
    rc = lib.m3_clip_grads(n, arr(ctypes.c_void_p, [t[0] for t in tensors]), arr(ctypes.c_int64, [t[1] for t in tensors]),
                           arr(ctypes.c_int32, [t[2] for t in tensors]),
                           arr(ctypes.c_void_p, [t[0] for t in outs]) if outs else None,
                           arr(ctypes.c_int32, [t[2] for t in outs]) if outs else None, largest, max_norm, scale,
                           norm, None, 0, None)
    return rc, lib.m3_last_error_string().decode()


def test_clip_grads_refusals(lib):
    f32, bf, i64, u8 = _codes()
    a, c = (4096, 100, f32), (8192, 100, bf)
    for call, word in (
            (dict(tensors=[a], max_norm=-1.0), "max_norm"),
            (dict(tensors=[a], max_norm=math.nan), "max_norm"),
            (dict(tensors=[a], scale=0.0), "scale"),
            (dict(tensors=[a], scale=math.inf), "scale"),
            (dict(tensors=[a], largest=2), "largest"),
            (dict(tensors=[(4096, -1, f32)]), "negative"),
            (dict(tensors=[(4096, 5, i64)]), "unsupported dtype"),
            (dict(tensors=[(0, 5, f32)]), "missing"),
            (dict(tensors=[(4098, 5, f32)]), "aligned"),
            (dict(tensors=[a], outs=[(8192, 100, bf)]), "dtype must be"),
            (dict(tensors=[c], outs=[(4096, 100, i64)]), "dtype must be"),
            # shared memory: the same twice, the end of one in the next, an output over a gradient
            (dict(tensors=[a, a]), "shares memory"),
            (dict(tensors=[a, (4096 + 396, 100, f32)]), "shares memory"),
            (dict(tensors=[(4096, 1000, f32), (5000, 1, f32), (12000, 5, f32)]), "shares memory"),
            (dict(tensors=[a, c], outs=[(16384, 100, f32), (4096, 100, f32)]), "shares memory"),
            (dict(tensors=[a, c], outs=[(16384, 100, f32), (16384 + 399, 100, bf)]), "aligned"),
            (dict(tensors=[a, c], outs=[(16384, 100, f32), (16384 + 398, 100, bf)]), "shares memory")):
        rc, msg = _clip(lib, **call)
        assert rc == 1 and word in msg, (call, msg)
    # side by side, in place and into themselves: past the host's checks, to the device's
    for call in (dict(tensors=[a, (4096 + 400, 100, f32)]), dict(tensors=[a, c], outs=[a, c]),
                 dict(tensors=[a, a], max_norm=math.inf)):
        rc, msg = _clip(lib, **call)
        assert rc != 0 and "shares" not in msg and ("CUDA" in msg or "norm" in msg), msg


def test_python_refusals_without_a_device():
    from mamba3_ssm import clip_grad_norm_, clip_grads_, policy_loss, preference_loss, token_logprobs
    x, t, z = torch.randn(2, 3, 8), torch.zeros(2, 3, dtype=torch.long), torch.zeros(2, 3)
    for f in (lambda: token_logprobs(x, t), lambda: policy_loss(x, t, z, z), lambda: preference_loss(x, t)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            f()
    with pytest.raises(RuntimeError, match="no CPU path"):
        clip_grads_([z], 1.0)
    with pytest.raises(ValueError, match="norm_type"):
        clip_grads_([z], 1.0, 1.0)
    with pytest.raises(ValueError, match="max_norm"):
        clip_grads_([z], -1.0)
    with pytest.raises(ValueError, match="scale"):
        clip_grads_([z], 1.0, scale=0.0)
    with pytest.raises(ValueError, match="outputs"):
        clip_grads_([z], 1.0, out=[z, z])
    assert clip_grads_([], 1.0).item() == 0.0
    assert clip_grad_norm_([torch.nn.Parameter(z)], 1.0).item() == 0.0  # no gradient yet
    with pytest.raises(ValueError, match="reduction"):
        policy_loss(x, t, z, z, reduction="mean")
    with pytest.raises(ValueError, match="ref_logprobs"):
        policy_loss(x, t, z, z, kl_coef=0.1)


# ------------------------------------------------------------------- the kernels' arithmetic
def test_row_sum_with_an_assumed_base():
    """A base that is not the maximum, sums of parts joined by addition: the same log-softmax, and
    the range in which the kernels trust the sum covers bases 40 away from the maximum."""
    rng = np.random.default_rng(0)
    for shift in (-40.0, 0.0, 40.0):
        l = rng.normal(0, 3, 5000)
        m = l[:256].max() + shift
        c = 1.0 / np.log(2.0)
        parts = np.exp2((l - m) * c).reshape(10, 500).sum(1)
        S = parts.sum()
        assert 2.0 ** -60 < S < 2.0 ** 100
        ref = l[7] - np.log(np.exp(l - l.max()).sum()) - l.max()
        assert abs((l[7] - m) - np.log(S) - ref) < 1e-12


def test_two_float_scale_keeps_minus_infinity():
    """c in two floats with a positive lower one: l = -inf stays -inf, and the sum of the two
    products is c l to 2^-45."""
    for t in (1.0, 0.7, 2.0, 1e-3, math.log2(math.e)):
        c = 1.4426950408889634 / t
        hi = np.float32(c)
        if float(hi) >= c:
            hi = np.nextafter(hi, np.float32(0))
        lo = np.float32(c - float(hi))
        assert lo > 0
        with np.errstate(invalid="ignore"):
            assert np.float32(-np.inf) * lo + np.float32(-np.inf) * hi == -np.inf
        assert abs(float(hi) + float(lo) - c) <= 2.0 ** -45 * c


def test_split_logarithm():
    """log S = e log 2 (64 bits) + log1p(m - 1) (32 bits, m in 0.75 .. 1.5). The second term is at
    most 0.41, where a step of 32 bits is 2^-25; numpy's log1p is good to two steps."""
    S = np.float32(np.random.default_rng(1).uniform(0.5, 2e5, 20000))
    m, e = np.frexp(S)
    low = m < 0.75
    m, e = np.where(low, 2 * m, m).astype(np.float32), np.where(low, e - 1, e)
    got = e * math.log(2.0) + np.log1p(m - np.float32(1)).astype(np.float64)
    assert np.abs(got - np.log(S.astype(np.float64))).max() < 2 * 2.0 ** -25


def test_kl_series():
    """exp(d) - 1 - d below 1/2 by the series to d^9: 2^-20 of the value, which the difference of
    32-bit numbers does not reach for small d."""
    d = np.concatenate([np.linspace(-0.5, 0.5, 4001), 2.0 ** -np.arange(2, 40), -(2.0 ** -np.arange(2, 40))])
    d = d[np.abs(d) < 0.5].astype(np.float32)
    q = np.float32(1 / 362880)
    for f in (40320, 5040, 720, 120, 24, 6, 2):
        q = (q * d + np.float32(1 / f)).astype(np.float32)
    got = (q * d * d).astype(np.float64)
    D = d.astype(np.float64)
    terms = [D ** k / math.factorial(k) for k in range(2, 16)]
    ref = sum(reversed(terms))
    assert (np.abs(got - ref) <= 2.0 ** -20 * np.abs(ref) + 1e-40).all()


def test_rounding_to_bfloat16_by_addition():
    """u + 0x8000 (with the sign's bit), upper half: the nearest bf16, ties up, as near as
    rounding to even."""
    rng = np.random.default_rng(2)
    x = np.concatenate([np.exp(rng.uniform(-80, 5, 20000)), [0.0, 1.0, 1.00390625, 2.0 ** -126]]).astype(np.float32)
    for add, sign in ((0x8000, 1.0), (0x80008000, -1.0)):
        u = (x.view(np.uint32).astype(np.uint64) + add) & 0xffff0000
        got = u.astype(np.uint32).view(np.float32).astype(np.float64)
        ref = torch.from_numpy(x).to(torch.bfloat16).double().numpy()
        assert np.array_equal(np.abs(got - sign * x), np.abs(ref - x))


def test_policy_derivative_against_differences():
    """d loss / d logp as the kernel forms it, against central differences of the loss."""
    rng = np.random.default_rng(3)
    for lo, hi, k in ((0.2, 0.3, 0.0), (0.1, 0.1, 0.5), (0.0, 1e9, 0.1)):
        for _ in range(200):
            A, old, ref, lp = rng.normal(), -3.0, -3.1, -3.0 + rng.normal(0, 0.3)

            def loss(v):
                r, d = math.exp(v - old), ref - v
                return -min(r * A, min(max(r, 1 - lo), 1 + hi) * A) + k * (math.expm1(d) - d)
            r = math.exp(lp - old)
            if min(abs(r - (1 - lo)), abs(r - (1 + hi))) < 1e-3:
                continue
            clipped = (A > 0 and r > 1 + hi) or (A < 0 and r < 1 - lo)
            got = (0.0 if clipped else -r * A) - k * math.expm1(ref - lp)
            h = 1e-5
            assert abs((loss(lp + h) - loss(lp - h)) / (2 * h) - got) < 1e-6


def test_clip_grad_norm_takes_the_arguments_of_torch():
    import inspect
    from mamba3_ssm import clip_grad_norm_
    ours, theirs = (inspect.signature(f).parameters.values() for f in (clip_grad_norm_, torch.nn.utils.clip_grad_norm_))
    assert [(p.name, p.default) for p in ours] == [(p.name, p.default) for p in theirs]
    p = torch.nn.Parameter(torch.zeros(3))
    for foreach in (None, True, False):
        assert clip_grad_norm_([p], 1.0, foreach=foreach).item() == 0.0


def test_clip_grads_without_a_bound_reads_shared_memory(lib):
    """Nothing but NaN to all of them can be written then, through ``outs`` too; with a scale the
    gradients are written."""
    f32 = _codes()[0]
    a = (4096, 100, f32)
    for outs in (None, [a, a]):
        rc, msg = _clip(lib, [a, a], outs=outs, max_norm=math.inf)
        assert rc != 0 and "shares" not in msg
        rc, msg = _clip(lib, [a, a], outs=outs, max_norm=math.inf, scale=0.5)
        assert rc == 1 and "shares memory" in msg


def test_forward_mode_tangents_are_refused():
    """Before anything else: the losses have no forward-mode derivative to lose."""
    import torch.autograd.forward_ad as fwd
    from mamba3_ssm import policy_loss, preference_loss, token_logprobs
    x, t, z = torch.randn(2, 3, 8), torch.zeros(2, 3, dtype=torch.long), torch.zeros(2, 3)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for f in (lambda: token_logprobs(dual, t), lambda: policy_loss(dual, t, z, z), lambda: preference_loss(dual, t)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f()
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                f()
        with pytest.raises(RuntimeError, match="no CPU path"):
            token_logprobs(x, t)


_COPY_ROUNDS = r"""
#include "copy_rounds.cuh"
// A copying warp as in the policy loss's kernel: `rows` rows of `pieces` pieces; before row r it
// waits for a place (from the third row on), before piece k of it for the piece to be read (from
// the second row on). Wait number `fails` gives up (-1: none does). What the last copy of each
// piece is, and what is waited for at the end, as parities; -1: nothing.
extern "C" void run(int rows, int pieces, int fails, int* last, int* waited) {
  m3::CopyRounds c;
  int waits = 0;
  bool ok = true;
  for (int k = 0; k < pieces; ++k) last[k] = waited[k] = -1;
  for (int i = 0; i < rows && ok; ++i, c.next()) {
    if (c.round >= 2 && waits++ == fails) { ok = false; break; }
    for (int k = 0; k < pieces; ++k) {
      if (c.round >= 1 && waits++ == fails) { ok = false; break; }
      last[k] = i & 1;
      c.issue(k);
    }
    if (!ok) break;
  }
  for (int k = 0; k < pieces; ++k)
    if (c.copied(k)) waited[k] = (int)c.last_phase(k);
}
"""


def test_copies_in_flight_are_waited_for(tmp_path):
    """Wherever the copying warp of the policy loss gives up, and where it does not, it waits for
    the phase that each piece's last copy completes, before its CTA's shared memory is released."""
    import os
    import subprocess
    src = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mamba3-ssm_b200", "csrc")
    cpp, so = tmp_path / "rounds.cpp", tmp_path / "rounds.so"
    cpp.write_text(_COPY_ROUNDS)
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", src, str(cpp), "-o", str(so)], check=True)
    run = ctypes.CDLL(str(so)).run
    for rows in range(6):
        for pieces in range(1, 6):
            for fails in range(-1, rows * (pieces + 1)):
                last, waited = (ctypes.c_int * pieces)(), (ctypes.c_int * pieces)()
                run(rows, pieces, fails, last, waited)
                assert list(last) == list(waited), (rows, pieces, fails)
