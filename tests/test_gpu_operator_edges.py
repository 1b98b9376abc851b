"""Calls of the selective scan, the convolution, the beam search and the moves of states at the edge of what they allow."""

import pytest
import torch

from test_gpu_selective import _gen

pytestmark = pytest.mark.gpu
DEV = "cuda"


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
