"""The selective scan in every layout of lanes and states, over padded batches and in pieces along the sequence.

Error bounds as in test_gpu_selective. In the pieces' inputs |dt A| is at most 0.031, so that the argument of a decay
adds less than a tenth to the 2^-22 of the hardware's 2^x; the decay over a whole piece is one
exponential of a sum of at most 256 step sizes, formed with 66 additions one after the other: at most 66 u of an argument
below 8, half of what its 256 decays may be off by themselves. So (length + 64) 2^-21 of the terms' magnitudes holds."""

import pytest
import torch

import selective_ref as R
from test_gpu_selective import _gen, _near, scan_inputs

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def check(x, h0, lengths, dstate, unit):
    """Outputs and gradients, which land in memory that held NaN."""
    from mamba3_ssm import ssm_scan_selective
    b, n, e = x["u"].shape
    leaves = {k: v.detach().requires_grad_(True) for k, v in {**x, "h0": h0}.items()}
    dy = torch.randn(b, n, e, device=DEV, generator=_gen(9)).to(x["u"].dtype)
    args = (*(x[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "bias")), True, h0, lengths, dy, dstate)
    ref, size = R.scan(*args), R.scan(*args, magnitudes=True)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()

    def poison(*ts):
        held = [torch.full_like(t, float("nan")) for t in ts for _ in range(2)]
        torch.cuda.synchronize()
        del held
    poison(dy, h0)
    y, state = ssm_scan_selective(*(leaves[k] for k in ("u", "delta", "A", "B", "C", "D")), z=leaves["z"],
                                  delta_bias=leaves["bias"], initial_state=leaves["h0"], lengths=lengths, return_state=True)
    _near(y.detach(), ref["y"], size["y"], unit, "y")
    _near(state.detach(), ref["state"], size["state"], unit, "state")
    poison(*x.values(), h0)
    got = dict(zip(leaves, torch.autograd.grad([y, state], list(leaves.values()), [dy, dstate])))
    pad = ~R.valid(lengths, b, n, DEV)
    for k, d in got.items():
        if d.dim() > 2 and k != "h0":
            assert (d[pad] == 0).all(), f"{k}: {int((d[pad] != 0).sum())} elements of the padding are not 0"
        _near(d, ref[k], size[k], unit, k)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("m", [3, 4, 8, 16, 24, 32, 64, 100, 128])
@pytest.mark.parametrize("many", [False, True])
def test_padding_of_a_batch(many, m, dtype):
    """Sequences of few channels, and of as many as give the backward its layout for full launches."""
    n = 300
    lengths = torch.tensor([300, 100, 0, 1, 33, 257] + ([299, 64, 31, 170] * 4 if many else []), device=DEV)
    b, e = len(lengths), (66 if m > 64 else 130 if m > 32 else 258 if m > 16 else 520) if many else 21
    x = scan_inputs(b, n, e, m, dtype=DTYPES[dtype], seed=m, strided=False)
    pad = ~R.valid(lengths, b, n, DEV)
    for i, k in enumerate(("u", "delta", "z", "B", "C")):
        x[k][pad] = [float("nan"), float("inf"), float("-inf"), float("nan"), float("inf")][i]
    r = lambda s: torch.randn(b, e, m, device=DEV, generator=_gen(s))  # noqa: E731
    check(x, r(1), lengths, r(2), (n + 64) * 2.0 ** -20)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("e,m,g,mixed", [(20, 3, 1, False), (24, 8, 2, False), (22, 16, 2, False), (12, 24, 1, False), (12, 32, 3, False),
                                         (10, 64, 2, False), (10, 100, 1, False), (6, 128, 1, False), (20, 16, 1, True), (9, 40, 1, True)])
def test_pieces_along_the_sequence(e, m, g, mixed, dtype):
    """Few channels: the sequence is cut, forward and backward. One sequence ends within a piece, one before others begin."""
    n = 1111
    x = scan_inputs(3, n, e, m, g, DTYPES[dtype], seed=m)
    x["A"] *= 0.02  # so that states outlive the pieces
    if mixed:
        x["delta"], x["B"], x["C"] = x["delta"].float() + 0.001, x["B"].float() * 1.001, x["C"].float() * 0.999
    lengths = torch.tensor([n, 601, 70], device=DEV)
    r = lambda s: torch.randn(3, e, m, device=DEV, generator=_gen(s))  # noqa: E731
    check(x, r(1), lengths, r(2), (n + 64) * 2.0 ** -21)
