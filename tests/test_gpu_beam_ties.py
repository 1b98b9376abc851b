"""The order of continuations whose scores are equal: the lower beam first, and within a beam the larger logit, then the lower token."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("b,k,v,pitch", [(1, 4, 50257, 0), (3, 4, 50257, 3), (40, 4, 4099, 0), (2, 8, 30001, 0), (1, 16, 70001, 1), (1, 3, 997, 0),
                                         (160, 4, 20011, 0)])
def test_equal_beams_go_by_their_number(b, k, v, pitch, dtype):
    """The same logits in every beam, in rows that begin at different places between two 16-byte boundaries."""
    from mamba3_ssm import beam_select
    g = torch.Generator(device=DEV).manual_seed(v)
    top = 4
    row = (2.0 * torch.randn(b, 1, v, device=DEV, generator=g)).clamp(max=6.0)
    at = torch.stack([torch.randperm(v, device=DEV, generator=g)[:top] for _ in range(b)])
    row.scatter_(2, at[:, None], torch.tensor([10.0, 9.0, 8.0, 7.0], device=DEV).expand(b, 1, top))
    logits = torch.empty(b, k, v + pitch, dtype=DTYPES[dtype], device=DEV)[..., :v]
    logits.copy_(row)
    scores = torch.full((b, k), -1.25, device=DEV)
    num = min(64, k * top)
    got = beam_select(logits, scores, num)
    want = torch.arange(num, device=DEV)
    assert torch.equal(got.parents, (want % k).expand(b, num))
    assert torch.equal(got.tokens, at.gather(1, (want // k).expand(b, num)))
    # a row's score does not depend on where it lies in memory
    assert all(torch.equal(p, q) for p, q in zip(got, beam_select(logits[:, :1].contiguous().expand(b, k, v), scores, num)))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("b,k,v,num", [(1, 2, 3000, 10), (1, 4, 131072, 16), (1, 16, 131072, 8), (1, 16, 131072, 64), (4, 32, 70000, 4),
                                       (2, 32, 100000, 33)])
def test_scores_that_swallow_the_logits(b, k, v, num, dtype):
    """Logits that differ by 1e-12 at most, beside a score of -1e30: the sum keeps no more of them than an fp32 of -log(V) does, so
    all are equal, in as many parts of a row as it is cut into."""
    from mamba3_ssm import beam_select
    g = torch.Generator(device=DEV).manual_seed(k + num)
    logits = (1e-12 * torch.rand(b, k, v, device=DEV, generator=g)).to(DTYPES[dtype])
    best = lambda j: logits[:, j].float().sort(dim=1, descending=True, stable=True).indices[:, :num]  # noqa: E731
    scores = torch.full((b, k), -1e30, device=DEV)
    got = beam_select(logits, scores, num)
    assert (got.scores == torch.tensor(-1e30)).all() and (got.parents == 0).all()
    assert torch.equal(got.tokens, best(0))
    scores[:, :2] = float("-inf")
    scores[:, -1] = -1e30
    got = beam_select(logits, scores, num)
    j = min(2, k - 1)
    assert (got.parents == j).all() and torch.equal(got.tokens, best(j))
