"""Calls of the selective scan, the convolution, the beam search and the moves of states at the edge of what they allow."""

import pytest
import torch

import selective_ref as R
from test_gpu_selective import _gen, _near, check_conv, check_scan, conv_inputs, scan_inputs

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def test_complex_operands_are_refused():
    from mamba3_ssm import causal_conv, causal_conv_step_, ssm_scan_selective, ssm_step_selective_
    x = scan_inputs(2, 5, 8, 4)
    h0 = torch.zeros(2, 8, 4, device=DEV)
    c = lambda t: t.to(torch.complex64) * (1 + 1j)  # noqa: E731
    for k in ("delta", "A", "B", "C", "D", "bias", "h0"):
        y = {**x, "h0": h0}
        y[k] = c(y[k])
        with pytest.raises(TypeError, match="complex"):
            ssm_scan_selective(*(y[i] for i in ("u", "delta", "A", "B", "C", "D")), z=y["z"], delta_bias=y["bias"], initial_state=y["h0"])
        if k == "h0":
            continue
        for i in ("u", "delta", "B", "C", "z"):
            y[i] = y[i][:, 0]
        state = torch.ones_like(h0)
        with pytest.raises(TypeError, match="complex"):
            ssm_step_selective_(state, *(y[i] for i in ("u", "delta", "A", "B", "C", "D")), z=y["z"], delta_bias=y["bias"])
        assert (state == 1).all()
    w, bias = torch.randn(8, 4, device=DEV), torch.randn(8, device=DEV)
    for ww, bb in ((c(w), bias), (w, c(bias)), (c(w), None), (c(w), c(bias))):
        with pytest.raises(TypeError, match="complex"):
            causal_conv(x["u"], ww, bb)
        with pytest.raises(TypeError, match="complex"):
            causal_conv_step_(torch.zeros(2, 3, 8, device=DEV), x["u"][:, 0], ww, bb)


@pytest.mark.parametrize("xt,wt,bt", [("bf16", "bf16", "fp32"), ("fp16", "fp16", "fp32"), ("bf16", "fp32", "bf16"), ("bf16", "bf16", "fp16"),
                                      ("bf16", "fp16", "bf16"), ("fp32", "bf16", "fp32"), ("fp16", "bf16", "bf16")])
def test_convolution_keeps_the_bits_of_weight_and_bias(xt, wt, bt):
    """Each may be of any of the dtypes by itself; none is rounded to the other's."""
    from mamba3_ssm import causal_conv_step_
    x, w, bias, init, dy, dlast = conv_inputs(2, 50, 40, 4, DTYPES[xt], wdtype=torch.float32)
    w, bias = w.to(DTYPES[wt]), (4 * bias).to(DTYPES[bt])
    check_conv(x, w, bias, init, dy, dlast, False)
    check_conv(x, w, bias, init, dy, dlast, True)
    state = init.clone()
    y = causal_conv_step_(state, x[:, 0], w, bias)
    args = (x[:, :1], w, bias, False, init)
    _near(y, R.conv(*args)["y"], R.conv(*args, magnitudes=True)["y"], 64 * 2.0 ** -24)


# ------------------------------------------------------------------------------ strides
@pytest.mark.parametrize("shape,strides", [((2, 4, 8), (16, 1, 1)), ((1, 4, 8), (1, 8, 1)), ((3, 8, 12), (1, 12, 1)), ((1, 2, 4), (1, 1, 1)),
                                           ((2, 4, 6), (1, 0, 1)), ((3, 2, 4), (0, 0, 1))])
def test_rows_one_element_apart(shape, strides):
    """Windows over one buffer, and a batch of one with any stride: outputs have strides of their own."""
    b, n, e = shape
    window = lambda dtype, seed, f=lambda t: t: f(torch.randn(200, device=DEV, generator=_gen(seed))).to(dtype).as_strided(shape, strides)  # noqa: E731
    for dtype in (torch.float32, torch.bfloat16):
        x = scan_inputs(b, n, e, 16, dtype=dtype)
        x["u"], x["z"], x["delta"] = window(dtype, 1), window(dtype, 2), window(dtype, 3, lambda t: -t.abs())
        check_scan(x)
        _, w, bias, init, dy, dlast = conv_inputs(b, n, e, 4, dtype)
        check_conv(x["u"], w, bias, init, dy, dlast, True)


@pytest.mark.parametrize("shape,strides", [((4, 8), (1, 1)), ((2, 4), (1, 1)), ((3, 8), (0, 1)), ((8, 4), (1, 1))])
def test_single_steps_of_rows_one_element_apart(shape, strides):
    from mamba3_ssm import causal_conv_step_, ssm_step_selective_
    b, e = shape
    x = torch.randn(40, device=DEV, generator=_gen(1)).as_strided(shape, strides)
    w, state = torch.randn(e, 4, device=DEV, generator=_gen(2)), torch.randn(b, 3, e, device=DEV, generator=_gen(3))
    want = causal_conv_step_(state.clone(), x.contiguous(), w)
    assert torch.equal(causal_conv_step_(state, x, w), want)
    o = scan_inputs(b, 1, e, 16)
    h = torch.randn(b, e, 16, device=DEV, generator=_gen(4))
    args = (o["delta"][:, 0], o["A"], o["B"][:, 0], o["C"][:, 0])
    want = ssm_step_selective_(h.clone(), x.contiguous(), *args)
    assert torch.equal(ssm_step_selective_(h, x, *args), want)


def test_moves_of_an_empty_batch():
    from mamba3_ssm import reorder_states_
    par = torch.zeros(0, 4, dtype=torch.long, device=DEV)
    t, o = torch.zeros(0, 7, device=DEV), torch.zeros(0, 7, device=DEV)
    assert reorder_states_(t, par) is t
    assert reorder_states_([t], par, out=[o])[0] is o
    with pytest.raises(ValueError):
        reorder_states_(torch.zeros(4, 7, device=DEV), par)


def test_moves_of_conjugated_states():
    """A lazily conjugated tensor holds the other numbers in memory."""
    from mamba3_ssm import reorder_states_
    t = torch.randn(4, 6, dtype=torch.complex64, device=DEV)
    par = torch.tensor([[1, 1, 3, 0]], device=DEV)
    for src in (t, t.conj()):
        for dst in (torch.empty_like(t), torch.empty_like(t).conj()):
            if src.is_conj() == dst.is_conj():
                reorder_states_(src, par, out=dst)
                assert torch.equal(dst.resolve_conj(), src.resolve_conj()[par[0]])
            else:
                with pytest.raises(ValueError, match="conjugat"):
                    reorder_states_(src, par, out=dst)
    c = t.clone().conj()
    want = c.resolve_conj()[par[0]]
    reorder_states_(c, par)
    assert torch.equal(c.resolve_conj(), want)


def test_selection_refuses_what_carries_derivatives():
    from mamba3_ssm import beam_select
    from torch.autograd import forward_ad
    logits, scores = torch.randn(2, 3, 50, device=DEV), torch.zeros(2, 3, device=DEV)
    want = beam_select(logits, scores)
    for a, b in ((logits.clone().requires_grad_(True), scores), (logits, scores.clone().requires_grad_(True))):
        with pytest.raises(RuntimeError, match="without gradients"):
            beam_select(a, b)
        with torch.no_grad():
            assert all(torch.equal(p, q) for p, q in zip(beam_select(a, b), want))
    with forward_ad.dual_level():
        for a, b in ((forward_ad.make_dual(logits, logits), scores), (logits, forward_ad.make_dual(scores, scores))):
            with pytest.raises(NotImplementedError, match="tangent"):
                beam_select(a, b)
        assert all(torch.equal(p, q) for p, q in zip(beam_select(logits, scores), want))


@pytest.mark.parametrize("mimo", [False, True])
def test_beam_graph_starts_over(mimo):
    """reset() leaves nothing of an earlier search; what DecodeGraph does token by token is not offered."""
    from test_gpu_beam_search import lm
    g = lm(mimo).beam_graph(2, 3, end_token=5)
    prompt = torch.randint(0, 37, (2, 6), device=DEV, generator=_gen(1))
    a, sa = g.search(prompt, 10)
    g.reset()
    for t in (g.ahead, g.scores, g.parents, g.finished, g.tokens, *(t for layer in g.cache for t in layer)):
        assert not t.any()
    for name in ("feed", "prefill", "next"):
        assert not hasattr(g, name)
    b, sb = g.search(prompt, 10)
    assert torch.equal(a, b) and torch.equal(sa, sb)
