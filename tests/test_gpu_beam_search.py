"""MambaLMHeadModel.beam_search against a search written out with step(), and a small recurrent language model
made of the convolution and the selective scan searched with the same two operators: prompts through the
sequence forms, their states forked to beams, single steps, selection, states moved."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def lm(mimo, vocab=37):
    from mamba3_ssm import MambaConfig, MambaLMHeadModel
    torch.manual_seed(3)
    cfg = MambaConfig(d_model=64, n_layer=2, vocab_size=vocab,
                      ssm_cfg=dict(d_state=16, headdim=32, is_mimo=mimo, mimo_rank=2 if mimo else 4))
    m = MambaLMHeadModel(cfg, device=DEV)
    with torch.no_grad():  # predictions that differ from state to state
        m.embedding.weight.mul_(8.0)
    return m.eval()


def plain_search(step, logits, states, k, n, end, vocab):
    """Scores in float64. states: what step(tokens, states) takes and returns, beams of a prompt in a row."""
    b = logits.shape[0]
    scores = torch.full((b, k), float("-inf"), dtype=torch.float64, device=DEV)
    scores[:, 0] = 0
    done = torch.zeros(b, k, dtype=torch.bool, device=DEV)
    rows = torch.empty(b, k, 0, dtype=torch.long, device=DEV)
    logits = logits.unsqueeze(1).expand(b, k, -1)
    gaps = []
    for _ in range(n):
        logp = torch.log_softmax(logits[..., :vocab].double(), -1)
        if end is not None:
            only = torch.full((vocab,), float("-inf"), device=DEV, dtype=torch.float64)
            only[end] = 0
            logp = torch.where(done.unsqueeze(-1), only, logp)
        total = (scores.unsqueeze(-1) + logp).view(b, -1)
        best, at = total.sort(dim=1, descending=True, stable=True)
        d = best[:, :k] - best[:, 1:k + 1]
        gaps.append(d[d.isfinite()].min())
        scores, parents, tokens = best[:, :k], at[:, :k] // vocab, at[:, :k] % vocab
        rows = torch.cat([rows.gather(1, parents.unsqueeze(-1).expand_as(rows)), tokens.unsqueeze(-1)], -1)
        if end is not None:
            done = done.gather(1, parents) | (tokens == end)
        flat = (parents + k * torch.arange(b, device=DEV)[:, None]).flatten()
        states = [tuple(t[flat] for t in layer) for layer in states]
        logits, states = step(tokens.flatten(), states)
        logits = logits.view(b, k, -1)
    return rows, scores, torch.stack(gaps).min()


@pytest.mark.parametrize("mimo", [False, True])
@pytest.mark.parametrize("b,k,end", [(1, 1, None), (2, 4, None), (3, 5, 7), (1, 32, 0)])
def test_model_beam_search(mimo, b, k, end):
    m = lm(mimo)
    prompt = torch.randint(0, 37, (b, 9), device=DEV, generator=torch.Generator(device=DEV).manual_seed(b))
    n = 12
    with torch.no_grad():
        logits, cache = m.prefill(prompt)
        fork = [tuple(t.repeat_interleave(k, 0) for t in layer) for layer in cache]
        rows, scores, gap = plain_search(m.step, logits[:, -1], fork, k, n, end, 37)
        tokens, got = m.beam_search(prompt, k, n, end_token=end)
    # the graph's step and step() differ by a few fp32 roundings a layer, far below the gaps between candidates
    assert gap > 1e-4 or k == 32
    assert (got.double() - scores).abs().max() < 1e-3
    if gap > 1e-4:
        assert torch.equal(tokens, rows)


def test_beam_graph_again_and_length_penalty():
    m = lm(True)
    g = m.beam_graph(2, 4, end_token=5)
    gen = torch.Generator(device=DEV).manual_seed(1)
    p1, p2 = (torch.randint(0, 37, (2, 6), device=DEV, generator=gen) for _ in range(2))
    a, sa = g.search(p1, 10)
    g.search(p2, 10)
    c, sc = g.search(p1, 10)
    assert torch.equal(a, c) and torch.equal(sa, sc)
    d, sd = g.search(p1, 10, length_penalty=1.0)
    length = ((d == 5).cumsum(-1) == 0).sum(-1).add(1).clamp(max=10)
    for i in range(2):
        pairs = {tuple(r.tolist()): s for r, s in zip(a[i], sa[i])}
        for r, s, ln in zip(d[i], sd[i], length[i]):
            assert abs(pairs[tuple(r.tolist())] / ln - s) <= 1e-6 * abs(s)
    assert (sd[:, :-1] >= sd[:, 1:]).all()


def test_beam_graph_refusals():
    m = lm(False)
    for args in ((2, 33), (0, 2), (1, 0), (1, 2, 37), (1, 2, -1)):
        with pytest.raises(ValueError):
            m.beam_graph(*args)
    g = m.beam_graph(1, 2)
    for prompt, n in ((torch.zeros(2, 3, dtype=torch.long, device=DEV), 4), (torch.zeros(1, 0, dtype=torch.long, device=DEV), 4),
                      (torch.zeros(1, 3, dtype=torch.long, device=DEV), 0)):
        with pytest.raises(ValueError):
            g.search(prompt, n)


class Selective:
    """Two layers of convolution and selective scan around an embedding, with states (conv, ssm) a layer."""

    def __init__(self, d=48, n=16, v=41, layers=2):
        g = torch.Generator(device=DEV).manual_seed(0)
        r = lambda *s: torch.randn(*s, device=DEV, generator=g)  # noqa: E731
        self.emb = r(v, d)
        self.layers = [dict(inp=r(2 * d, d) / d ** 0.5, conv=r(d, 4), cb=r(d), proj=r(d + 2 * n, d) / d ** 0.5,
                            A=-torch.rand(d, n, device=DEV, generator=g) * 4, D=r(d), bias=r(d) - 2, out=r(d, d) / d ** 0.5)
                       for _ in range(layers)]
        self.d, self.n = d, n

    def split(self, p, x):
        return (x @ p["proj"].t()).split([self.d, self.n, self.n], -1)

    def sequence(self, ids, lengths):
        from mamba3_ssm import causal_conv, ssm_scan_selective
        x, states = self.emb[ids], []
        for p in self.layers:
            h, z = (x @ p["inp"].t()).chunk(2, -1)
            c, cs = causal_conv(h, p["conv"], p["cb"], activation="silu", lengths=lengths, return_state=True)
            dt, B, C = self.split(p, c)
            y, s = ssm_scan_selective(c, dt, p["A"], B, C, p["D"], z=z, delta_bias=p["bias"], lengths=lengths, return_state=True)
            states.append((cs, s))
            x = x + y @ p["out"].t()
        last = x.gather(1, (lengths - 1)[:, None, None].expand(-1, 1, self.d))[:, 0]
        return last @ self.emb.t(), states

    def step(self, ids, states):
        from mamba3_ssm import causal_conv_step_, ssm_step_selective_
        x = self.emb[ids]
        for p, (cs, s) in zip(self.layers, states):
            h, z = (x @ p["inp"].t()).chunk(2, -1)
            c = causal_conv_step_(cs, h, p["conv"], p["cb"], activation="silu")
            dt, B, C = self.split(p, c)
            x = x + ssm_step_selective_(s, c, dt, p["A"], B, C, p["D"], z=z, delta_bias=p["bias"]) @ p["out"].t()
        return x @ self.emb.t(), states


def test_search_over_selective_states():
    """Padded prompts through the sequence forms, then beams; against each prompt for itself by single steps."""
    from mamba3_ssm import beam_select, reorder_states_
    m, k, n = Selective(), 4, 8
    gen = torch.Generator(device=DEV).manual_seed(5)
    ids = torch.randint(0, 41, (3, 21), device=DEV, generator=gen)
    lengths = torch.tensor([21, 3, 14], device=DEV)
    logits, states = m.sequence(ids, lengths)
    beams = [tuple(torch.empty(3 * k, *t.shape[1:], device=DEV) for t in layer) for layer in states]
    reorder_states_(states, torch.zeros(3, k, dtype=torch.long, device=DEV), out=beams)
    logits = logits.unsqueeze(1).expand(3, k, -1)
    scores = torch.full((3, k), float("-inf"), device=DEV)
    scores[:, 0] = 0
    rows = torch.empty(3, k, 0, dtype=torch.long, device=DEV)
    for _ in range(n):
        sel = beam_select(logits, scores)
        scores = sel.scores
        rows = torch.cat([rows.gather(1, sel.parents.unsqueeze(-1).expand_as(rows)), sel.tokens.unsqueeze(-1)], -1)
        reorder_states_(beams, sel.parents)
        logits = m.step(sel.tokens.flatten(), beams)[0].view(3, k, -1)
    for i in range(3):
        own = [(torch.zeros(1, 3, m.d, device=DEV), torch.zeros(1, m.d, m.n, device=DEV)) for _ in m.layers]
        for t in range(int(lengths[i])):
            first, own = m.step(ids[i:i + 1, t], own)
        fork = [tuple(t.repeat_interleave(k, 0) for t in layer) for layer in own]
        want, sc, gap = plain_search(m.step, first, fork, k, n, None, 41)
        assert gap > 1e-3
        assert torch.equal(rows[i:i + 1], want)
        assert (scores[i:i + 1].double() - sc).abs().max() < 1e-3 * (1 + sc.abs().max())
