"""Losses over the tokens of a language model's logits, for fine-tuning MambaLMHeadModel.

    logits = model(input_ids)                                  # (batch, length, vocabulary)
    token_logprobs(logits, tokens)                             # scoring, or a loss of one's own
    policy_loss(logits, tokens, old_logprobs, advantages).loss.backward()
    preference_loss(logits, tokens, ref_logprobs).loss.backward()

``tokens[b, t]`` is the token that ``logits[b, t]`` predicts, i.e. the input shifted by one.
``logits[:, :-1]`` with ``input_ids[:, 1:]`` is read in place; keeping the logits whole and
giving the last position ``ignore_index`` also spares autograd the padding of that slice.

Positions with mask 0 or the token ``ignore_index`` do not count: their logits are not read,
their log-probability is 0 and their gradient is 0, whatever is stored there. A token id
outside the vocabulary that is not ``ignore_index`` makes its position NaN. Gradients flow to
the logits alone, once and backwards (no second derivatives, no forward mode); old and reference
log-probabilities, advantages and masks are constants.
No counterpart in the reference's package.
"""

from typing import NamedTuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib as L
from .ops import _inner, _require_cuda

__all__ = ["PolicyLoss", "PreferenceLoss", "policy_loss", "preference_loss", "token_logprobs"]

_LOGIT_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


class PolicyLoss(NamedTuple):
    """loss: scalar, differentiable by the logits. logprobs: of the tokens, in fp32 (0 where a
    position does not count). kl, clip_fraction: means over the positions that count."""
    loss: torch.Tensor
    logprobs: torch.Tensor
    kl: torch.Tensor
    clip_fraction: torch.Tensor


class PreferenceLoss(NamedTuple):
    """loss: scalar, differentiable by the logits. rewards (2 N): beta * sum(logp - ref) of each
    sequence. logprobs: of the tokens, in fp32 (0 where a position does not count)."""
    loss: torch.Tensor
    rewards: torch.Tensor
    logprobs: torch.Tensor


def _rows(name, logits, tokens):
    """Logits as (batch, length, V) and tokens as (batch, length), without a copy where the
    strides allow."""
    if forward_ad.unpack_dual(logits).tangent is not None:
        raise NotImplementedError(f"{name}: no forward-mode derivative, but the logits carry a tangent")
    if not (logits.is_cuda and tokens.is_cuda):
        _require_cuda(name, logits, tokens)
    if logits.dtype not in _LOGIT_DTYPES:
        raise TypeError(f"{name}: logits must be float32, bfloat16 or float16, got {logits.dtype}")
    shape = tokens.shape
    if logits.dim() < 1 or logits.shape[:-1] != shape:
        raise ValueError(f"{name}: logits (..., V) and tokens (...) expected, got {tuple(logits.shape)} and "
                         f"{tuple(shape)}")
    if logits.shape[-1] == 0:
        raise ValueError(f"{name}: empty vocabulary")
    if tokens.dtype is not torch.int64:
        if tokens.dtype not in (torch.int32, torch.int16, torch.uint8):
            raise TypeError(f"{name}: tokens must be integers, got {tokens.dtype}")
        tokens = tokens.long()
    if tokens.get_device() != logits.get_device():
        raise RuntimeError(f"{name}: tokens are on {tokens.device}, logits on {logits.device}")
    n = len(shape)
    if n < 2:
        logits, tokens = logits.reshape(1, -1, logits.shape[-1]), tokens.reshape(1, -1)
    elif n > 2:
        logits, tokens = logits.flatten(0, n - 2), tokens.flatten(0, n - 2)
    return _inner(logits), tokens


def _per_token(name, what, v, logits, tokens, shape, dtype=torch.float32):
    """A constant operand as (batch, length); it may be of any shape that broadcasts to
    ``shape``, the shape the caller gave its tokens in."""
    if v is None:
        return None
    if not isinstance(v, torch.Tensor):
        raise TypeError(f"{name}: {what} must be a tensor")
    if v.get_device() != logits.get_device():
        raise RuntimeError(f"{name}: {what} is on {v.device}, logits on {logits.device}")
    if v.dtype is not dtype:
        v = v.detach()
        if dtype is not torch.bool:
            v = v.to(dtype)
        elif v.dtype is not torch.uint8:
            v = v != 0
    if v.shape != shape:
        try:
            v = v.expand(shape)
        except RuntimeError:
            raise ValueError(f"{name}: {what} of shape {tuple(v.shape)} does not broadcast to the tokens' "
                             f"{tuple(shape)}") from None
    if len(shape) == 2:
        return v
    return v.reshape(tokens.shape)


def _like_rows(logits):
    """The gradient's tensor: rows of the logits' pitch where these are cut from wider rows, so
    that both start on the same boundaries."""
    if logits.is_contiguous():
        return torch.empty_like(logits)
    B, T, V = logits.shape
    pitch = logits.stride(1)
    if V < pitch < 2 * V:
        return torch.empty(B, T, pitch, dtype=logits.dtype, device=logits.device)[..., :V]
    return torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)


def _records(logits, tokens, *per_token):
    """The records of logits, tokens and optional operands of the tokens' shape: a mask first,
    then fp32."""
    B, T, V = logits.shape
    vals = [*L.rec3(logits, L._DTYPE_CODE[logits.dtype], B, T, V), *L.rec2(tokens, L.M3_INT64, B, T)]
    code = L.M3_UINT8
    for v in per_token:
        vals += L.NO_RECORD if v is None else L.rec2(v, code, B, T)
        code = L.M3_FLOAT32
    return vals


def _apply(fn, logits, *rest):
    """fn on logits that may need a gradient; where they do not, its forward alone (autograd's
    bookkeeping would cost as much as a small call's launches)."""
    if torch.is_grad_enabled() and logits.requires_grad:
        return fn.apply(logits, (*rest, True))
    with torch.no_grad():
        return fn.forward(None, logits, (*rest, False))


# The functions take the logits and one tuple of everything else, none of which has a gradient.
# What a user could change between forward and backward (logits, tokens, mask) is saved through
# autograd, which notices it; what is made here is held by the context.
class _TokenLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, rest):
        tokens, mask, temperature, ignore_index, need = rest
        B, T = tokens.shape
        dev = logits.device
        logp = torch.empty((B, T), dtype=torch.float32, device=dev)
        stats = torch.empty((B, T, 2), dtype=torch.float32, device=dev) if need else None
        vals = _records(logits, tokens, mask, logp)
        vals += L.rec3(stats, L.M3_FLOAT32, B, T, 2) if need else L.NO_RECORD
        a = L.Records(vals)
        with L.on_device(dev):
            L.check(L.load().m3_token_logprobs(a.at(0), a.at(1), a.at(2), temperature, ignore_index, a.at(3), a.at(4),
                                               L.stream_ptr(dev)), "m3_token_logprobs")
        if need:
            ctx.save_for_backward(logits, tokens, mask)
            ctx.held = (stats, temperature, ignore_index)
        return logp

    @staticmethod
    @once_differentiable
    def backward(ctx, dlogp):
        logits, tokens, mask = ctx.saved_tensors
        stats, temperature, ignore_index = ctx.held
        dlogits = _like_rows(logits)
        B, T, V = logits.shape
        dlogp = dlogp if dlogp.dtype is torch.float32 else dlogp.float()
        vals = _records(logits, tokens, mask)
        vals += L.rec2(dlogp, L.M3_FLOAT32, B, T)
        vals += L.rec3(stats, L.M3_FLOAT32, B, T, 2)
        vals += L.rec3(dlogits, L._DTYPE_CODE[logits.dtype], B, T, V)
        a = L.Records(vals)
        dev = logits.device
        with L.on_device(dev):
            L.check(L.load().m3_token_logprobs_grad(a.at(0), a.at(1), a.at(2), a.at(4), a.at(3), temperature,
                                                    ignore_index, a.at(5), L.stream_ptr(dev)),
                    "m3_token_logprobs_grad")
        return dlogits, None


def _grad_records(logits, tokens, mask, up, dlogits):
    vals = _records(logits, tokens, mask)
    up = up if up.dtype is torch.float32 else up.float()
    B, T, V = logits.shape
    vals += L.rec0(up.data_ptr(), L.M3_FLOAT32)
    vals += L.rec3(dlogits, L._DTYPE_CODE[logits.dtype], B, T, V)
    return L.Records(vals), up


class _PolicyLossFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, rest):
        tokens, mask, old, adv, ref, temperature, ignore_index, clip_low, clip_high, kl_coef, by_sequence, need = rest
        lib = L.load()
        B, T, V = logits.shape
        dev = logits.device
        loss = torch.empty((), dtype=torch.float32, device=dev)
        means = torch.empty((2,), dtype=torch.float32, device=dev)  # KL, share of clipped positions
        logp = torch.empty((B, T), dtype=torch.float32, device=dev)
        # the gradient for an upstream gradient of 1, while each row is at hand; backward forms it
        # again only where the upstream gradient is another
        dlogits = _like_rows(logits) if need else None
        nbytes = lib.m3_policy_loss_workspace_size(B, T)
        ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev)
        f32, m = L.M3_FLOAT32, means.data_ptr()
        vals = _records(logits, tokens, mask, old, adv, ref, logp)
        vals += L.rec0(loss.data_ptr(), f32)
        vals += L.rec0(m, f32)
        vals += L.rec0(m + 4, f32)
        vals += L.rec3(dlogits, L._DTYPE_CODE[logits.dtype], B, T, V) if need else L.NO_RECORD
        a = L.Records(vals)
        with L.on_device(dev):
            L.check(lib.m3_policy_loss(a.at(0), a.at(1), a.at(2), a.at(3), a.at(4), a.at(5), temperature, ignore_index,
                                       clip_low, clip_high, kl_coef, by_sequence, a.at(7), a.at(8), a.at(9), a.at(6),
                                       a.at(10), ws.data_ptr(), nbytes, L.stream_ptr(dev)), "m3_policy_loss")
        if need:
            ctx.save_for_backward(logits, tokens, mask)
            ctx.held = (ws, temperature, ignore_index)
            ctx.dlogits = dlogits
            ctx.mark_non_differentiable(logp, means)
            ctx.set_materialize_grads(False)  # no zeros for the outputs without a gradient
        return loss, logp, means

    @staticmethod
    @once_differentiable
    def backward(ctx, up, _dlogp, _dmeans):
        logits, tokens, mask = ctx.saved_tensors
        ws, temperature, ignore_index = ctx.held
        # handed out once: what receives it may write to it
        dlogits, ctx.dlogits = ctx.dlogits, None
        keep = dlogits is not None
        if not keep:
            dlogits = _like_rows(logits)
        a, up = _grad_records(logits, tokens, mask, up, dlogits)
        dev = logits.device
        with L.on_device(dev):
            L.check(L.load().m3_policy_loss_grad(a.at(0), a.at(1), a.at(2), a.at(3), temperature, ignore_index, keep,
                                                 a.at(4), ws.data_ptr(), ws.numel(), L.stream_ptr(dev)),
                    "m3_policy_loss_grad")
        return dlogits, None


class _PreferenceLossFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, rest):
        tokens, mask, ref, temperature, ignore_index, beta, label_smoothing, need = rest
        lib = L.load()
        B, T = tokens.shape
        dev = logits.device
        loss = torch.empty((), dtype=torch.float32, device=dev)
        rewards = torch.empty((B,), dtype=torch.float32, device=dev)
        logp = torch.empty((B, T), dtype=torch.float32, device=dev)
        nbytes = lib.m3_preference_loss_workspace_size(B, T)
        ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev)
        f32 = L.M3_FLOAT32
        vals = _records(logits, tokens, mask, ref, logp)
        vals += L.rec0(loss.data_ptr(), f32)
        vals += (rewards.data_ptr(), f32, 1, B, 0, 0, 0, 0, 0, 1, 0, 0, 0, 0, 0)
        a = L.Records(vals)
        with L.on_device(dev):
            L.check(lib.m3_preference_loss(a.at(0), a.at(1), a.at(2), a.at(3), temperature, ignore_index, beta,
                                           label_smoothing, a.at(5), a.at(6), a.at(4), ws.data_ptr(), nbytes,
                                           L.stream_ptr(dev)), "m3_preference_loss")
        if need:
            ctx.save_for_backward(logits, tokens, mask)
            ctx.held = (ws, temperature, ignore_index)
            ctx.mark_non_differentiable(rewards, logp)
            ctx.set_materialize_grads(False)  # no zeros for the outputs without a gradient
        return loss, rewards, logp

    @staticmethod
    @once_differentiable
    def backward(ctx, up, _drewards, _dlogp):
        logits, tokens, mask = ctx.saved_tensors
        ws, temperature, ignore_index = ctx.held
        dlogits = _like_rows(logits)
        a, up = _grad_records(logits, tokens, mask, up, dlogits)
        dev = logits.device
        with L.on_device(dev):
            L.check(L.load().m3_preference_loss_grad(a.at(0), a.at(1), a.at(2), a.at(3), temperature, ignore_index,
                                                     a.at(4), ws.data_ptr(), ws.numel(), L.stream_ptr(dev)),
                    "m3_preference_loss_grad")
        return dlogits, None


def token_logprobs(logits, tokens, *, mask=None, temperature=1.0, ignore_index=-100):
    """log softmax(logits / temperature) at ``tokens``, in fp32: logits (..., V) in fp32, bf16 or
    fp16, tokens (...) integers, mask broadcastable to the tokens (nonzero = counts).
    Differentiable by the logits; without the (..., V) tensor of all log-probabilities."""
    x, t = _rows("token_logprobs", logits, tokens)
    m = _per_token("token_logprobs", "mask", mask, x, t, tokens.shape, torch.bool)
    logp = _apply(_TokenLogprobsFn, x, t, m, float(temperature), int(ignore_index))
    return logp if logp.shape == tokens.shape else logp.reshape(tokens.shape)


def policy_loss(logits, tokens, old_logprobs, advantages, *, ref_logprobs=None, mask=None, clip_low=0.2,
                clip_high=None, kl_coef=0.0, temperature=1.0, reduction="token", ignore_index=-100):
    """Clipped policy loss with a KL term: per position, with r = exp(logp - old_logprobs) and
    d = ref_logprobs - logp,

        -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef (exp(d) - d - 1)

    ``reduction`` "token": the mean over the positions that count; "sequence": the mean over
    the sequences (last dimension of tokens) that have any, of each one's mean. 0 where no
    position counts. ``advantages`` may be per token or broadcast (e.g. (batch, 1)).
    ``clip_high`` defaults to ``clip_low``. Without ``ref_logprobs`` there is no KL term (and
    ``kl_coef`` must be 0); with them ``kl`` is reported also for kl_coef 0, where the
    loss is the one without them.
    Where the logits need a gradient it is formed in the forward pass, so that they are read
    once; a loss that is scaled before backward() costs a second pass over them. That gradient is
    kept until backward outside of autograd's saved tensors, where their hooks do not see it.
    Returns PolicyLoss(loss, logprobs, kl, clip_fraction). ``logprobs`` are within a few roundings
    of token_logprobs' (1 / temperature is held in one float here, in two there), not its bits."""
    name = "policy_loss"
    if reduction not in ("token", "sequence"):
        raise ValueError(f"{name}: reduction is 'token' or 'sequence', got {reduction!r}")
    if ref_logprobs is None and kl_coef != 0:
        raise ValueError(f"{name}: kl_coef needs ref_logprobs")
    x, t = _rows(name, logits, tokens)
    m = _per_token(name, "mask", mask, x, t, tokens.shape, torch.bool)
    old = _per_token(name, "old_logprobs", old_logprobs, x, t, tokens.shape)
    adv = _per_token(name, "advantages", advantages, x, t, tokens.shape)
    ref = _per_token(name, "ref_logprobs", ref_logprobs, x, t, tokens.shape)
    loss, logp, means = _apply(
        _PolicyLossFn, x, t, m, old, adv, ref, float(temperature), int(ignore_index), float(clip_low),
        float(clip_low if clip_high is None else clip_high), float(kl_coef), int(reduction == "sequence"))
    return PolicyLoss(loss, logp if logp.shape == tokens.shape else logp.reshape(tokens.shape), *means.unbind(0))


def preference_loss(logits, tokens, ref_logprobs=None, *, mask=None, beta=0.1, label_smoothing=0.0, temperature=1.0,
                    ignore_index=-100):
    """Preference loss over pairs of answers: logits (2 N, T, V), tokens (2 N, T), sequence i the
    chosen and sequence N + i the rejected answer of pair i. With reward = beta * sum over
    the positions that count of (logp - ref_logprobs) and z = reward_i - reward_{N+i}:

        loss = mean_i of -(1 - label_smoothing) log sigmoid(z) - label_smoothing log sigmoid(-z)

    ``ref_logprobs`` (2 N, T): the reference model's, as token_logprobs returns them; None: 0.
    Returns PreferenceLoss(loss, rewards, logprobs)."""
    name = "preference_loss"
    if logits.dim() != 3 or logits.shape[0] == 0 or logits.shape[0] % 2:
        raise ValueError(f"{name}: logits (2 N, T, V) expected, the N chosen answers before the N rejected ones, got "
                         f"{tuple(logits.shape)}")
    x, t = _rows(name, logits, tokens)
    m = _per_token(name, "mask", mask, x, t, tokens.shape, torch.bool)
    ref = _per_token(name, "ref_logprobs", ref_logprobs, x, t, tokens.shape)
    return PreferenceLoss(*_apply(_PreferenceLossFn, x, t, m, ref, float(temperature), int(ignore_index), float(beta),
                                  float(label_smoothing)))
