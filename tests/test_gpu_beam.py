"""beam_select and reorder_states_ against plain implementations (the selection in float64).

Scores: exp and sums in 32 bits a thread (each off by at most 2^-21 relative: the hardware's 2^x, its
argument for elements that matter, and additions), joined in two floats, so a log-sum is off by at most
2^-20 absolute; the returned score is rounded to fp32 once. Which candidates are chosen is compared exactly
where the float64 scores of neighbours are further apart than that, or equal."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
TOL = 2.0 ** -20


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def plain(logits, scores, num, finished=None, end=0):
    """Scores in float64, parents, tokens."""
    b, k, v = logits.shape
    x = logits.double()
    peak = x.amax(-1, keepdim=True)  # +inf less itself is NaN, and so is then the sum
    logp = x - peak - (x - peak).exp().sum(-1, keepdim=True).log()
    logp = torch.where((x == float("-inf")).all(-1, keepdim=True), float("-inf"), logp)
    if finished is not None:
        only = torch.full((v,), float("-inf"), device=DEV, dtype=torch.float64)
        only[end] = 0.0
        logp = torch.where(finished.unsqueeze(-1), only, logp)
    total = scores.double().unsqueeze(-1) + logp
    # a beam without a score offers nothing, whatever its logits hold
    total = torch.where((scores == float("-inf")).unsqueeze(-1), float("-inf"), total)
    total = torch.where((scores.isnan() | (scores == float("inf"))).unsqueeze(-1), float("nan"), total)
    total = torch.where(total.isnan(), float("nan"), total)  # sort() would put a NaN with a sign last
    s, at = total.reshape(b, -1).sort(dim=1, descending=True, stable=True)
    return s[:, :num + 1], at[:, :num] // v, at[:, :num] % v


def check(logits, scores, num=None, finished=None, end=0):
    from mamba3_ssm import beam_select
    got = beam_select(logits, scores, num, finished=finished, end_token=end)
    n = num or scores.shape[1]
    s, parents, tokens = plain(logits, scores, n, finished, end)
    # two candidates of different scores closer than 4 TOL may change places: each is off by TOL at most, so
    # that those further apart than 2 TOL keep their order. All others are compared exactly.
    gap = s[:, :-1] - s[:, 1:]
    close = (gap > 0) & (gap < 4 * TOL)
    clear = ~torch.nn.functional.pad(close, (0, 1))[:, :n]
    clear[:, 1:] &= ~close[:, :n - 1]
    assert clear.float().mean() > 0.9
    assert torch.equal(got.parents[clear], parents[clear]) and torch.equal(got.tokens[clear], tokens[clear])
    want = s[:, :n]
    assert torch.equal(got.scores.isnan(), want.isnan()) and torch.equal(got.scores == float("-inf"), want == float("-inf"))
    f = want.isfinite()
    assert ((got.scores.double() - want).abs()[f] <= TOL + 2.0 ** -24 * want.abs()[f]).all()
    assert got.parents.dtype == got.tokens.dtype == torch.int64 and got.scores.dtype == torch.float32
    return got


def inputs(b, k, v, dtype=torch.float32, seed=0, pitch=0):
    g = _gen(seed)
    # a permutation of distinct values in each row, beams' scores apart by odd amounts
    logits = (torch.randn(b, k, v + pitch, device=DEV, generator=g) * 2.5).to(dtype)
    scores = -torch.rand(b, k, device=DEV, generator=g).cumsum(1) * 1.7
    return logits[..., :v], scores


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("b,k,v,num,pitch", [
    (1, 1, 1, 1, 0), (1, 1, 7, 7, 0), (3, 2, 5, 10, 0), (1, 4, 50000, 4, 0), (2, 3, 257, 6, 1), (5, 5, 2049, 10, 3),
    (2, 32, 1000, 64, 0), (1, 1, 100, 64, 0), (40, 8, 8200, 16, 8), (1, 16, 131072, 32, 0), (100, 4, 300, 8, 5)])
def test_select(b, k, v, num, pitch, dtype):
    logits, scores = inputs(b, k, v, DTYPES[dtype], seed=b + k + v, pitch=pitch)
    check(logits, scores, num)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_ties_go_to_the_lowest_beam_and_token(dtype):
    logits = torch.zeros(2, 3, 9000, dtype=DTYPES[dtype], device=DEV)
    check(logits, torch.zeros(2, 3, device=DEV), 64)
    logits[0, 1, 8000:] = 1.0
    logits[1, :, ::3] = -0.0  # equal to 0
    logits[1, 2, 5:9] = 2.0
    check(logits, torch.tensor([[0.0, 0.0, 0.0], [-1.0, -2.0, -1.0]], device=DEV), 40)


@pytest.mark.parametrize("b,k,v,num,equal", [
    (1, 32, 40, 64, True), (2, 32, 3000, 64, False), (1, 8, 20000, 64, True), (1, 7, 5001, 14, False), (1, 3, 70000, 64, False),
    (38, 2, 2050, 4, False), (37, 5, 999, 8, True), (1, 6, 3, 18, False)])
def test_many_candidates_and_one_or_two_launches(b, k, v, num, equal):
    # equal: few values, so that most of what is ranked at the end differs in its beam and token alone
    logits, scores = inputs(b, k, v, torch.float32, seed=k + v)
    if equal:
        logits = (logits * 0.5).round()
        scores = torch.zeros_like(scores)
    check(logits, scores, num)
    check(logits.bfloat16(), scores, num)


@pytest.mark.parametrize("order", ["ascending", "descending", "blocks"])
def test_orders_that_pass_the_threshold_again_and_again(order):
    v = 70000
    x = torch.arange(v, device=DEV).float() * 1e-3
    x = x.flip(0) if order == "descending" else x
    if order == "blocks":
        x = x.view(7, 10000).roll(3, 0).flatten()
    logits = torch.stack([x, x * 0.999]).view(1, 2, v)
    check(logits, torch.tensor([[0.0, -0.0123]], device=DEV), 48)
    check(logits.bfloat16(), torch.tensor([[0.0, -0.0123]], device=DEV), 48)


def test_masked_logits_empty_rows_nan_and_infinities():
    inf, nan = float("inf"), float("nan")
    logits, scores = inputs(9, 3, 3000, seed=4)
    logits = logits.clone()
    logits[0, 0, 3:] = -inf                      # three tokens left
    logits[1, 1] = -inf                          # nothing left
    logits[2, 2, 2999] = nan
    logits[3, 0, 7] = inf
    logits[4] = torch.finfo(torch.float32).min   # a mask of the lowest value: all alike
    scores[4] = torch.tensor([0.0, -1.0, -2.0])
    logits[5, :, 1000:] = torch.finfo(torch.float32).min
    logits[6] = -inf
    scores[7, 1:] = -inf                         # a first step
    scores[8] = torch.tensor([nan, 0.0, inf])
    check(logits, scores, 5)
    logits = logits.clone()
    logits[7, 1:] = nan                          # of beams that do not count
    check(logits, scores, 3)
    few = torch.full((1, 2, 50), -inf, device=DEV)
    few[0, 1, 30] = 2.0
    check(few, torch.zeros(1, 2, device=DEV), 20)
    check(torch.full((1, 2, 50), -inf, device=DEV), torch.zeros(1, 2, device=DEV), 60)


@pytest.mark.parametrize("end", [0, 2, 2999])
def test_finished_beams(end):
    logits, scores = inputs(6, 4, 3000, torch.bfloat16, seed=7)
    finished = torch.tensor([[0, 1, 0, 0], [1, 1, 1, 1], [0, 0, 0, 0], [1, 0, 0, 1], [0, 0, 1, 1], [1, 1, 1, 0]], device=DEV).bool()
    logits = logits.clone()
    logits[finished] = float("nan")  # not read
    scores[5, 0] = float("-inf")
    check(logits, scores, 4, finished, end)
    got = check(logits, scores, 8, finished, end)
    assert (got.tokens[1, :4] == end).all() and torch.equal(got.scores[1, :4], scores[1].sort(descending=True).values)


def test_first_step_from_one_row_for_all_beams():
    logits, _ = inputs(3, 1, 5000, torch.bfloat16, seed=1)
    scores = torch.tensor([[0.0] + [float("-inf")] * 3], device=DEV).expand(3, 4)
    got = check(logits.expand(3, 4, 5000), scores)
    assert (got.parents == 0).all()


def test_select_strides_integers_as_finished_and_flat_logits():
    from mamba3_ssm import beam_select
    wide, _ = inputs(6, 4, 700, seed=3)
    logits = wide.transpose(0, 1)[:, ::2]  # (4, 3, 700) of other strides
    scores = torch.randn(3, 4, device=DEV, generator=_gen(1)).t()
    check(logits, scores, 5)
    fin = torch.tensor([[0, 3, 0]] * 4, device=DEV)
    check(logits, scores, 5, fin.bool())
    a, b = beam_select(logits, scores, 5, finished=fin), beam_select(logits, scores, 5, finished=fin.bool())
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    c = beam_select(logits.contiguous().flatten(0, 1), scores, 5, finished=fin)
    assert all(torch.equal(p, q) for p, q in zip(a, c))


def test_select_in_a_graph_and_on_streams():
    from mamba3_ssm import beam_select
    logits, scores = inputs(2, 4, 20000, torch.bfloat16, seed=11)
    logits = logits.clone()
    beam_select(logits, scores)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(beam_select(logits, scores))
        graphs.append(g)
    for seed in (12, 13):
        logits.copy_(inputs(2, 4, 20000, torch.bfloat16, seed=seed)[0])
        for g in graphs:
            g.replay()
        want = plain(logits, scores, 4)
        for o in outs:
            assert torch.equal(o.parents, want[1]) and torch.equal(o.tokens, want[2])


@pytest.mark.parametrize("batch,vocab", [(3, 9000), (60, 9000)])
def test_select_on_two_streams_at_once(batch, vocab):
    """In one launch and in two."""
    from mamba3_ssm import beam_select
    xs = [inputs(batch, 4, vocab, torch.bfloat16, seed=s) for s in (21, 22)]
    want = [beam_select(*x, 8) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(beam_select(*x, 8))
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for g, w in zip(got, want) for p, q in zip(g, w))


# ---------------------------------------------------------------------------------- states
def moved(t, parents, batch):
    """Rows by the definition."""
    s = t.shape[0] // batch if batch else 0
    out = torch.zeros(batch * parents.shape[1], *t.shape[1:], dtype=t.dtype, device=t.device)
    for i in range(batch):
        for j in range(parents.shape[1]):
            p = int(parents[i, j])
            if 0 <= p < s:
                out[i * parents.shape[1] + j] = t[i * s + p]
    return out


def cache(rows, seed, layers=3):
    g = _gen(seed)
    r = lambda *s: torch.randn(*s, device=DEV, generator=g)  # noqa: E731
    return [(r(rows, 4, 16), r(rows, 4, 8, 16), r(rows, 33).bfloat16(), (r(rows, 5) * 9).to(torch.int8), r(rows).double())
            for _ in range(layers)]


def same(got, want):
    for a, b in zip(got, want):
        for p, q in zip(a, b):
            assert torch.equal(p, q)


@pytest.mark.parametrize("batch,beams", [(1, 1), (1, 2), (3, 4), (2, 5), (4, 8), (1, 16), (2, 17), (1, 32)])
def test_reorder_in_place(batch, beams):
    from mamba3_ssm import reorder_states_
    parents = torch.randint(0, beams, (batch, beams), device=DEV, generator=_gen(beams))
    for par in (parents, torch.arange(beams, device=DEV).expand(batch, beams), torch.arange(beams, device=DEV).flip(0).expand(batch, beams),
                torch.zeros(batch, beams, dtype=torch.long, device=DEV), parents - 1, parents + beams // 2):
        c = cache(batch * beams, 1)
        want = [[moved(t, par, batch) for t in layer] for layer in c]
        versions = [t._version for layer in c for t in layer]
        assert reorder_states_(c, par) is c
        same(c, want)
        assert all(t._version > v for t, v in zip([t for layer in c for t in layer], versions))


@pytest.mark.parametrize("batch,source,rows", [(3, 1, 5), (2, 4, 8), (1, 10, 3), (1, 6, 70), (4, 3, 1), (2, 0, 3), (2, 3, 0)])
def test_reorder_into_other_tensors(batch, source, rows):
    from mamba3_ssm import reorder_states_
    parents = torch.randint(-1, source + 1, (batch, rows), device=DEV, generator=_gen(3))
    c, out = cache(batch * source, 1), cache(batch * rows, 2)
    keep = [[t.clone() for t in layer] for layer in c]
    assert reorder_states_(c, parents, out=out) is out
    same(out, [[moved(t, parents, batch) for t in layer] for layer in c])
    same(c, keep)


def test_reorder_views_of_a_pool_and_unaligned_rows():
    from mamba3_ssm import reorder_states_
    pool = torch.randn(6, 5, 40, device=DEV)
    before = pool.clone()
    parents = torch.tensor([[2, 0, 0], [1, 1, 2]], device=DEV)
    reorder_states_([pool[:, 1], pool[:, 3]], parents)
    for i in range(5):
        assert torch.equal(pool[:, i], moved(before[:, i], parents, 2) if i in (1, 3) else before[:, i])
    flat = torch.randn(6 * 37 + 1, device=DEV).bfloat16()
    odd = flat[1:].view(6, 37)
    want = moved(odd, parents, 2)
    reorder_states_(odd, parents)
    assert torch.equal(odd, want)
    # hundreds of tensors, and rows beyond one part
    many = [torch.randn(6, 3 + i % 5, device=DEV) for i in range(1100)] + [torch.randn(6, 70001, device=DEV)]
    want = [moved(t, parents, 2) for t in many]
    reorder_states_(many, parents)
    assert all(torch.equal(a, b) for a, b in zip(many, want))
    reorder_states_([], parents)
    reorder_states_([torch.empty(6, 0, device=DEV), odd], parents.t().contiguous().t())


def test_reorder_in_a_graph():
    from mamba3_ssm import reorder_states_
    parents = torch.zeros(2, 3, dtype=torch.long, device=DEV)
    c = cache(6, 5)
    reorder_states_(c, torch.arange(3, device=DEV).expand(2, 3))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        reorder_states_(c, parents)
    for seed in (1, 2):
        parents.copy_(torch.randint(0, 3, (2, 3), device=DEV, generator=_gen(seed)))
        want = [[moved(t, parents, 2) for t in layer] for layer in c]
        g.replay()
        same(c, want)


def test_reorder_refuses_shared_memory():
    from mamba3_ssm import reorder_states_
    t = torch.randn(8, 10, device=DEV)
    par = torch.zeros(2, 4, dtype=torch.long, device=DEV)
    for states, out in (([t, t], None), ([t[:, :5], t[:, 3:]], None), ([t], [t]), ([t[:, :5]], [t[:, 4:9]])):
        with pytest.raises(RuntimeError, match="shares memory"):
            reorder_states_(states, par, out=out)
    reorder_states_([t[:, :5], t[:, 5:]], par)
    reorder_states_([t[:, :5]], par, out=[t[:, 5:]])


def test_reorder_offsets_beyond_32_bits():
    from mamba3_ssm import reorder_states_
    big = torch.empty(4, 3 * 2 ** 29, dtype=torch.int8, device=DEV)
    rows = big[:, -64:]
    rows.copy_(torch.randint(-100, 100, (4, 64), device=DEV))
    par = torch.tensor([[3, 0, 3, 1]], device=DEV)
    want = moved(rows, par, 1)
    reorder_states_(rows, par)
    assert torch.equal(rows, want)
