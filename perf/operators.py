"""The operators of a fine-tuning step after the model's forward pass, as measured cases.

token_logprobs    log-probability of given tokens under a language model's logits, with its gradient
policy_loss       clipped policy loss with a KL term from the logits, with its gradient
preference_loss   preference loss over pairs of answers from the logits, with its gradient
clip_grads_       global gradient norm over many tensors, scaling and clipping

``own`` chooses between the plain form in elementary torch operations and the calls of the
package's operators. Logits are (batch, positions, vocabulary) as MambaLMHeadModel.forward
returns them; gradient tensors have the shapes of this package's layers and models.
"""

import os
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_IGNORE = -100


# ------------------------------------------------------------------------------ cases
def listed():
    return [
        # scoring one sampled answer: the latency of a single small call
        dict(name="score one answer", op="token_logprobs", dtype="bf16", batch=1, length=48, vocab=50000,
             width=50000, grad=False, padded=False),
        # scoring a padded batch where the padding columns of the vocabulary are cut off:
        # 50277 of 50280 columns, so rows are a strided view and end inside a vector
        dict(name="score a padded batch", op="token_logprobs", dtype="bf16", batch=4, length=500, vocab=50277,
             width=50280, grad=False, padded=True),
        # training on token log-probabilities in 32 bits with an odd vocabulary: rows that
        # start on no vector boundary
        dict(name="train on log-probabilities", op="token_logprobs", dtype="fp32", batch=3, length=341, vocab=50277,
             width=50277, grad=True, padded=True),
        # a policy step on one small group of short answers
        dict(name="policy, one small group", op="policy_loss", dtype="bf16", batch=8, length=64, vocab=50000,
             kl=0.0, clip=0.2, temperature=1.0, sequence=False),
        # an ordinary policy step with a KL term towards a reference model
        dict(name="policy, an ordinary step", op="policy_loss", dtype="bf16", batch=16, length=1000, vocab=50000,
             kl=0.05, clip=0.2, temperature=1.0, sequence=False),
        # half precision, answers sampled at a temperature, a long vocabulary, mean per answer
        dict(name="policy, long vocabulary", op="policy_loss", dtype="fp16", batch=8, length=512, vocab=131072,
             kl=0.02, clip=0.1, temperature=0.8, sequence=True),
        # the largest policy batch: 32 answers of 1024 tokens
        dict(name="policy, a large batch", op="policy_loss", dtype="bf16", batch=32, length=1024, vocab=50280,
             kl=0.05, clip=0.2, temperature=1.0, sequence=False),
        # one pair of short answers, 32 bits
        dict(name="preference, one pair", op="preference_loss", dtype="fp32", pairs=1, length=96, vocab=50000,
             beta=0.1, smoothing=0.0),
        # a batch of eight pairs, answers of different lengths
        dict(name="preference, eight pairs", op="preference_loss", dtype="bf16", pairs=8, length=700, vocab=50280,
             beta=0.1, smoothing=0.1),
        # the gradients of one small layer, whose norm is below the bound: nothing is scaled
        dict(name="clip one layer", op="clip_grads_", grads="fp32", out="", d_model=256, layers=1, d_state=64,
             headdim=32, rank=4, vocab=0, scale=1.0, clipped=False),
        # a language model's 32-bit gradients in place, norm below the bound
        dict(name="clip a model in place", op="clip_grads_", grads="fp32", out="", d_model=1024, layers=16, d_state=64,
             headdim=64, rank=1, vocab=50000, scale=1.0, clipped=False),
        # the largest: bf16 gradients summed over eight micro-batches, averaged and clipped
        # into the 32-bit gradients of the optimiser, at the default configuration
        dict(name="clip into 32-bit gradients", op="clip_grads_", grads="bf16", out="fp32", d_model=2560, layers=64,
             d_state=128, headdim=64, rank=1, vocab=50280, scale=0.125, clipped=True),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["token_logprobs", "policy_loss", "preference_loss", "clip_grads_"])
    if op == "clip_grads_":
        grads = rng.choice(["bf16", "fp16", "fp32"])
        out = rng.choice(["", "fp32"])
        return dict(op=op, grads=grads, out=out, d_model=64 * _log_uniform(rng, 2, 32), layers=_log_uniform(rng, 1, 40),
                    d_state=rng.choice([32, 64, 128]), headdim=rng.choice([32, 64]), rank=rng.choice([1, 2, 4]),
                    vocab=rng.choice([0, _log_uniform(rng, 256, 100000)]),
                    scale=rng.choice([1.0, 0.25, 1.0 / 3.0]) if out else 1.0, clipped=bool(out) and rng.random() < 0.7)
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    vocab = _log_uniform(rng, 256, 131072)
    most = min(32768, 1_600_000_000 // (2 if dtype == "fp32" else 1) // vocab)
    rows = _log_uniform(rng, 16, most)
    batch = _log_uniform(rng, 1, min(rows // 4, 64))
    length = max(2, rows // batch)
    if op == "token_logprobs":
        cut = rng.choice([0, 0, 3, 8])
        return dict(op=op, dtype=dtype, batch=batch, length=length, vocab=vocab - cut, width=vocab, padded=rng.random() < 0.5,
                    grad=rng.random() < 0.5)
    if op == "policy_loss":
        return dict(op=op, dtype=dtype, batch=batch, length=length, vocab=vocab, kl=rng.choice([0.0, 0.02, 0.1]),
                    clip=rng.choice([0.1, 0.2]), temperature=rng.choice([1.0, 1.0, 0.7]), sequence=rng.random() < 0.4)
    return dict(op=op, dtype=dtype, pairs=max(1, batch // 2), length=length, vocab=vocab, beta=rng.choice([0.05, 0.1, 0.5]),
                smoothing=rng.choice([0.0, 0.1]))


# ----------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _logits(batch, length, width, dtype, g):
    """Logits of about a trained model's spread, and tokens that the model finds likely."""
    logits = torch.empty(batch, length, width, dtype=_DTYPES[dtype], device="cuda").normal_(0.0, 2.5, generator=g)
    tokens = torch.randint(0, max(1, width - 8), (batch, length), device="cuda", generator=g)
    likely = 6.0 + 4.0 * torch.rand(batch, length, 1, device="cuda", generator=g)
    logits.scatter_(2, tokens.unsqueeze(-1), likely.to(logits.dtype))
    return logits, tokens


def _measured(logits, tokens, temperature):
    """The log-probabilities that a sampling engine would have recorded, in 32 bits."""
    flat, at, got = logits.flatten(0, 1), tokens.flatten(), []
    for r in range(0, flat.shape[0], 1024):
        x = flat[r:r + 1024].float() / temperature
        got.append(x.gather(1, at[r:r + 1024, None])[:, 0] - x.logsumexp(1))
    return torch.cat(got).view_as(tokens)


def _answers(batch, length, g):
    """Which positions are an answer's: behind a prompt, before the padding."""
    at = torch.arange(length, device="cuda")
    first = (0.4 * length * torch.rand(batch, 1, device="cuda", generator=g)).long()
    last = (length * (0.6 + 0.4 * torch.rand(batch, 1, device="cuda", generator=g))).long().clamp(min=1)
    return (at >= first) & (at < last)


def _parameter_shapes(case):
    """The parameters of this package's layers (and of the model around them, with a vocabulary)."""
    d, n, r = case["d_model"], case["d_state"], case["rank"]
    inner = 2 * d
    heads = inner // case["headdim"]
    layer = [(2 * inner + 2 * n * r + 3 * heads + n // 4, d), (heads,), (heads, r, n), (heads, r, n), (n,), (n,), (heads,),
             (d, inner), (d,)]
    if r > 1:
        layer += [(heads, r, case["headdim"])] * 2
    return ([(case["vocab"], d), (d,)] if case["vocab"] else []) + layer * case["layers"]


def _views(shapes, dtype):
    """Tensors of these shapes in one buffer, each on a boundary of 64 elements."""
    sizes = [torch.Size(s).numel() for s in shapes]
    starts, end = [], 0
    for n in sizes:
        starts.append(end)
        end += -(-n // 64) * 64
    flat = torch.zeros(end, dtype=_DTYPES[dtype], device="cuda")
    return flat, [flat[a:a + n].view(s) for a, n, s in zip(starts, sizes, shapes)]


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    state = dict(case=case)
    if op == "clip_grads_":
        shapes = _parameter_shapes(case)
        flat, grads = _views(shapes, case["grads"])
        for t in grads:
            # weights' gradients differ in size from layer to layer and from norms' and biases'
            t.normal_(0.0, 2e-4 if t.dim() == 2 else 5e-3, generator=g)
        state.update(flat=flat, grads=grads, out_flat=None, out=None)
        if case["out"]:
            state["out_flat"], state["out"] = _views(shapes, case["out"])
        # about the norm that these gradients have once scaled
        about = case["scale"] * sum(t.numel() * (4e-8 if t.dim() == 2 else 2.5e-5) for t in grads) ** 0.5
        state["max_norm"] = about * (0.4 if case["clipped"] else 2.5)
        return state
    if op == "token_logprobs":
        logits, tokens = _logits(case["batch"], case["length"], case["width"], case["dtype"], g)
        logits = logits[..., :case["vocab"]]
        if case["padded"]:
            tokens = torch.where(_answers(case["batch"], case["length"], g), tokens, _IGNORE)
        if case["grad"]:
            state["dout"] = torch.randn(tokens.shape, device="cuda", generator=g)
        state.update(logits=logits.detach().requires_grad_(case["grad"]), tokens=tokens)
        return state
    batch = 2 * case["pairs"] if op == "preference_loss" else case["batch"]
    logits, tokens = _logits(batch, case["length"], case["vocab"], case["dtype"], g)
    mask = _answers(batch, case["length"], g)
    temperature = case.get("temperature", 1.0)
    logp = _measured(logits, tokens, temperature)
    ref = logp + 0.15 * torch.randn(logp.shape, device="cuda", generator=g) - 0.02
    state.update(logits=logits.requires_grad_(True), tokens=tokens, mask=mask, ref=ref)
    if op == "policy_loss":
        # log ratios of a policy some updates after sampling; those within 1e-3 of a clipping
        # border, where either side's gradient is right, are moved off it
        ratio = 0.15 * torch.randn(logp.shape, device="cuda", generator=g)
        for border in (1.0 - case["clip"], 1.0 + case["clip"]):
            edge = float(torch.tensor(border, dtype=torch.float64).log())
            ratio = torch.where((ratio - edge).abs() < 1e-3, edge - 2e-3, ratio)
        state["old"] = logp - ratio
        # advantages of this step's tokens: one part of the answer's, one of the token's own
        state["advantages"] = 0.3 + torch.randn(batch, 1, device="cuda", generator=g) + 0.3 * torch.randn(
            logp.shape, device="cuda", generator=g)
    return state


# ------------------------------------------------------------------------ plain forms
def _plain_rows(logits, tokens, temperature):
    """exp(x - max), its sum in 64 bits and the tokens' log-probabilities in 64 bits."""
    x = logits.detach().float()
    if temperature != 1.0:
        x = x / temperature
    m = x.amax(-1, keepdim=True)
    at = x.gather(-1, tokens.unsqueeze(-1))
    e = torch.exp(x - m)
    s = e.sum(-1, keepdim=True, dtype=torch.float64)
    return e, s, (at.double() - m.double() - torch.log(s)).squeeze(-1)


def _plain_dlogits(e, s, tokens, coef, dtype):
    """coef * (one-hot - softmax), rounded once."""
    d = e * (-coef.unsqueeze(-1) / s).float()
    d.scatter_add_(-1, tokens.unsqueeze(-1), coef.float().unsqueeze(-1))
    return d.to(dtype)


def _plain_token_logprobs(s):
    keep = s["tokens"] != _IGNORE
    tokens = torch.where(keep, s["tokens"], 0)
    e, total, logp = _plain_rows(s["logits"], tokens, 1.0)
    logp = torch.where(keep, logp, 0.0).float()
    if not s["case"]["grad"]:
        return [logp]
    coef = torch.where(keep, s["dout"].double(), 0.0)
    return [logp, _plain_dlogits(e, total, tokens, coef, s["logits"].dtype)]


def _plain_policy_loss(s):
    c, mask, tokens = s["case"], s["mask"], s["tokens"]
    e, total, logp = _plain_rows(s["logits"], tokens, c["temperature"])
    a, ratio = s["advantages"].double(), torch.exp(logp - s["old"].double())
    lo, hi = 1.0 - c["clip"], 1.0 + c["clip"]
    token_loss = -torch.minimum(ratio * a, ratio.clamp(lo, hi) * a)
    clipped = ((a > 0) & (ratio > hi)) | ((a < 0) & (ratio < lo))
    coef = torch.where(clipped, 0.0, -ratio * a)
    kl = torch.zeros_like(logp)
    if c["kl"]:
        d = s["ref"].double() - logp
        kl = torch.expm1(d) - d
        token_loss = token_loss + c["kl"] * kl
        coef = coef - c["kl"] * torch.expm1(d)
    n = mask.sum().clamp(min=1).double()
    w = mask.double() / n
    if c["sequence"]:
        per = mask.sum(1, keepdim=True)
        weight = mask.double() / per.clamp(min=1) / (per > 0).sum().clamp(min=1)
    else:
        weight = w
    loss = (weight * token_loss).sum()
    d = _plain_dlogits(e, total, tokens, weight * coef / c["temperature"], s["logits"].dtype)
    return [loss.float(), torch.where(mask, logp, 0.0).float(), (w * kl).sum().float(), (w * clipped).sum().float(), d]


def _plain_preference_loss(s):
    c, mask, tokens = s["case"], s["mask"], s["tokens"]
    e, total, logp = _plain_rows(s["logits"], tokens, 1.0)
    rewards = c["beta"] * torch.where(mask, logp - s["ref"].double(), 0.0).sum(1)
    n = c["pairs"]
    z = rewards[:n] - rewards[n:]
    soft = c["smoothing"]
    # -log sigmoid(z) = log(1 + exp(-z))
    up, down = torch.log1p(torch.exp(-z.abs())) + (-z).clamp(min=0), torch.log1p(torch.exp(-z.abs())) + z.clamp(min=0)
    loss = ((1 - soft) * up + soft * down).mean()
    dz = (1 / (1 + torch.exp(-z)) - (1 - soft)) * c["beta"] / n
    coef = torch.where(mask, torch.cat([dz, -dz]).unsqueeze(1), 0.0)
    d = _plain_dlogits(e, total, tokens, coef, s["logits"].dtype)
    return [loss.float(), rewards.float(), torch.where(mask, logp, 0.0).float(), d]


def _plain_clip_grads(s):
    scale = s["case"]["scale"]
    squares = torch.stack([t.float().square().sum(dtype=torch.float64) for t in s["grads"]])
    norm = squares.sum().sqrt() * scale
    factor = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0) * scale
    to = s["out"] or s["grads"]
    [o.copy_(t.float() * factor.float()) for o, t in zip(to, s["grads"])]
    return [norm.float(), s["out_flat"] if s["out"] else s["flat"]]


# -------------------------------------------------------------------- the package's calls
def _package():
    if "mamba3_ssm" not in sys.modules:
        sys.path.insert(0, os.path.join(os.getcwd(), "mamba3-ssm_b200"))
    import mamba3_ssm
    return mamba3_ssm


def _own(s):
    m, c = _package(), s["case"]
    if c["op"] == "token_logprobs":
        logp = m.token_logprobs(s["logits"], s["tokens"], ignore_index=_IGNORE)
        if not c["grad"]:
            return [logp]
        return [logp.detach(), torch.autograd.grad(logp, s["logits"], s["dout"])[0]]
    if c["op"] == "policy_loss":
        r = m.policy_loss(s["logits"], s["tokens"], s["old"], s["advantages"], ref_logprobs=s["ref"] if c["kl"] else None,
                          mask=s["mask"], clip_low=c["clip"], clip_high=c["clip"], kl_coef=c["kl"],
                          temperature=c["temperature"], reduction="sequence" if c["sequence"] else "token")
        d, = torch.autograd.grad(r.loss, s["logits"])
        return [r.loss.detach(), r.logprobs, r.kl, r.clip_fraction, d]
    if c["op"] == "preference_loss":
        r = m.preference_loss(s["logits"], s["tokens"], s["ref"], mask=s["mask"], beta=c["beta"],
                              label_smoothing=c["smoothing"])
        d, = torch.autograd.grad(r.loss, s["logits"])
        return [r.loss.detach(), r.rewards, r.logprobs, d]
    norm = m.clip_grads_(s["grads"], s["max_norm"], scale=c["scale"], out=s["out"])
    return [norm, s["out_flat"] if s["out"] else s["flat"]]


def run(state):
    if own:
        return _own(state)
    return {"token_logprobs": _plain_token_logprobs, "policy_loss": _plain_policy_loss,
            "preference_loss": _plain_preference_loss, "clip_grads_": _plain_clip_grads}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------- work
def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    if case["op"] == "clip_grads_":
        n = sum(torch.Size(s).numel() for s in _parameter_shapes(case))
        wrote = size[case["out"]] if case["out"] else size[case["grads"]] * (case["scale"] != 1.0 or case["clipped"])
        return {"bytes": n * (size[case["grads"]] + wrote) + 4, "flops": 3.0 * n}
    batch = case["batch"] if "batch" in case else 2 * case["pairs"]
    rows = batch * case["length"]
    grad = case.get("grad", True)
    # prompts and padding take 0.2 + 0.2 of the positions on average; their logits are not needed
    read = rows * (0.6 if case["op"] != "token_logprobs" or case["padded"] else 1.0)
    per_row = 8 + 4 + 1 + (4 if case["op"] == "preference_loss" else 0) + (12 if case["op"] == "policy_loss" else 0)
    n = size[case["dtype"]] * case["vocab"]
    return {"bytes": read * n + (rows * n if grad else 0) + rows * per_row,
            "flops": read * case["vocab"] * (7.0 if grad else 4.0)}


# ------------------------------------------------------------- the definition in 64 bits
def _exact_logp(x, tokens, temperature):
    return torch.log_softmax(x / temperature, 1).gather(1, tokens[:, None])[:, 0]


def _exact_rows(logits, tokens, temperature, dlogp):
    """Log-probabilities by rows, and the gradient of sum(dlogp * logp) by differentiating them."""
    flat, at, logp, grads = logits.detach().flatten(0, 1), tokens.flatten(), [], []
    step = max(1, 40_000_000 // flat.shape[1])
    for r in range(0, flat.shape[0], step):
        x = flat[r:r + step].double().requires_grad_(dlogp is not None)
        y = _exact_logp(x, at[r:r + step], temperature)
        logp.append(y.detach())
        if dlogp is not None:
            grads.append(torch.autograd.grad(y, x, dlogp.flatten()[r:r + step])[0])
    return torch.cat(logp).view_as(tokens), torch.cat(grads).view(logits.shape) if grads else None


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "clip_grads_":
        norm = case["scale"] * torch.sqrt(sum(torch.linalg.vector_norm(t, dtype=torch.float64) ** 2 for t in s["grads"]))
        bound = float(norm) + 1e-6
        factor = case["scale"] * (s["max_norm"] / bound if s["max_norm"] < bound else 1.0)
        return [norm, s["flat"].double().mul_(factor)]
    if case["op"] == "token_logprobs":
        keep = s["tokens"] != _IGNORE
        tokens = s["tokens"].clamp(min=0)
        dlogp = s["dout"].double() * keep if case["grad"] else None
        logp, d = _exact_rows(s["logits"], tokens, 1.0, dlogp)
        return [logp * keep] + ([d] if case["grad"] else [])
    tokens, mask = s["tokens"], s["mask"].double()
    temperature = case.get("temperature", 1.0)
    logp = _exact_rows(s["logits"], tokens, temperature, None)[0].requires_grad_(True)
    if case["op"] == "policy_loss":
        a, low, high = s["advantages"].double(), 1.0 - case["clip"], 1.0 + case["clip"]
        r = (logp - s["old"].double()).exp()
        surrogate = torch.min(r * a, r.clamp(low, high) * a)
        away = (surrogate < r * a).double()
        d = s["ref"].double() - logp
        k = d.exp() - d - 1.0 if case["kl"] else 0.0 * logp
        per = -surrogate + case["kl"] * k
        if case["sequence"]:
            count = mask.sum(1)
            loss = ((per * mask).sum(1) / count.clamp(min=1.0)).sum() / (count > 0).sum().clamp(min=1)
        else:
            loss = (per * mask).sum() / mask.sum().clamp(min=1.0)
        n = mask.sum().clamp(min=1.0)
        rest = [(k * mask).sum() / n, (away * mask).sum() / n]
    else:
        rewards = case["beta"] * ((logp - s["ref"].double()) * mask).sum(1)
        chosen, rejected = rewards.chunk(2)
        f = torch.nn.functional.logsigmoid
        loss = -((1.0 - case["smoothing"]) * f(chosen - rejected) + case["smoothing"] * f(rejected - chosen)).mean()
    dlogp, = torch.autograd.grad(loss, logp)
    d = _exact_rows(s["logits"], tokens, temperature, dlogp)[1]
    logp = logp.detach() * mask
    if case["op"] == "policy_loss":
        return [loss.detach(), logp, rest[0].detach(), rest[1].detach(), d]
    return [loss.detach(), rewards.detach(), logp, d]
