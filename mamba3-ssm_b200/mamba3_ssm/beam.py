"""Beam search: the selection over beams and vocabulary, and the moves of the beams' decode states.

    sel = beam_select(logits, scores, finished=finished, end_token=end)   # scores, parents, tokens
    reorder_states_(cache, sel.parents)                                   # every state tensor, one launch
    reorder_states_(prompt_cache, zeros, out=cache)                       # a prompt's state to its beams

A recurrent model's state has one size whatever was decoded, so a beam that continues another one takes
over its rows. ``MambaLMHeadModel.beam_search`` runs both, with the model's step, in one CUDA graph. No
counterpart in the reference's package (its generate.py samples).
"""

import struct
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import _lib as L
from .ops import _require_cuda

__all__ = ["BeamSelection", "beam_select", "reorder_states_"]

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
_MAX_BEAMS, _MAX_NUM, _MAX_VOCAB = 32, 64, 1 << 24


class BeamSelection(NamedTuple):
    """(batch, num) each, the best first. scores: fp32. parents: the beam that is continued, in
    [0, beams). tokens: the token it is continued with."""
    scores: torch.Tensor
    parents: torch.Tensor
    tokens: torch.Tensor


def beam_select(logits, scores, num=None, *, finished=None, end_token=0):
    """The ``num`` (as many as beams by default, at most 64) best continuations of each prompt by
    scores[b, j] + log_softmax(logits[b, j])[v], over its beams j and tokens v, the largest first.
    The sums are formed and compared in two floats; the exponentials below the logarithm are added up in one a
    thread, so that the difference between two beams is good to about 2^-20. Of equal sums the lower beam's come
    first, and within a beam the larger logit's, then the lower token's; beams with the same logits and scores tie.
    logits (batch, beams, V), or (batch * beams, V) as a model returns them, fp32, bf16 or fp16; at most 32
    beams and 65535 rows; scores (batch, beams) fp32: the beams' sums of log-probabilities so far.

    ``finished`` (batch, beams), optional: such a beam offers ``end_token`` alone, with its score
    unchanged. A beam with score -inf (an empty place, as all but one in a search's first step), or
    all of whose logits are -inf, offers continuations of score -inf only; they are chosen where
    nothing else is left. A NaN or +inf among a beam's logits, or as its score, makes its
    continuations NaN, which rank first, as they do in torch.topk. Without gradients."""
    name = "beam_select"
    if not (isinstance(logits, torch.Tensor) and isinstance(scores, torch.Tensor)):
        raise TypeError(f"{name}: logits and scores must be tensors")
    dev = logits.device
    if not (logits.is_cuda and scores.is_cuda):
        _require_cuda(name, logits, scores, finished)
    if torch.is_grad_enabled() and (logits.requires_grad or scores.requires_grad):
        raise RuntimeError(f"{name}: works without gradients; call it under torch.no_grad()")
    if getattr(forward_ad, "_current_level", 0) >= 0:
        for k, t in (("logits", logits), ("scores", scores)):
            if forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"{name}: no forward-mode derivative, but {k} carry a tangent")
    if logits.dtype not in _FLOATS:
        raise TypeError(f"{name}: logits must be float32, bfloat16 or float16, got {logits.dtype}")
    shape = scores.shape
    if len(shape) != 2 or shape[1] == 0:
        raise ValueError(f"{name}: scores are (batch, beams), got {tuple(shape)}")
    b, k = shape
    if logits.dim() == 2 and logits.shape[0] == b * k:
        logits = logits.unflatten(0, (b, k))
    ls = logits.shape
    if len(ls) != 3 or ls[0] != b or ls[1] != k or ls[2] == 0:
        raise ValueError(f"{name}: logits are {(b, k, 'V')} or {(b * k, 'V')}, got {tuple(ls)}")
    v = ls[2]
    num = k if num is None else int(num)
    if k > _MAX_BEAMS or v > _MAX_VOCAB or not 1 <= num <= min(_MAX_NUM, k * v):
        raise ValueError(f"{name}: at most {_MAX_BEAMS} beams, {_MAX_VOCAB} tokens, and 1 to {_MAX_NUM} continuations of "
                         f"those there are; got {k}, {v}, {num}")
    end_token = int(end_token)
    if not 0 <= end_token < v:
        raise ValueError(f"{name}: end_token {end_token} is outside the vocabulary of {v}")
    if scores.get_device() != dev.index or (finished is not None and finished.get_device() != dev.index):
        raise RuntimeError(f"{name}: logits, scores and finished must be on one device")
    if scores.dtype is not torch.float32:
        raise TypeError(f"{name}: scores must be float32, got {scores.dtype}")
    if finished is not None:
        if finished.shape != shape:
            raise ValueError(f"{name}: finished of shape {tuple(finished.shape)}, expected {(b, k)}")
        if finished.dtype is not torch.bool:
            finished = finished != 0
    if logits.stride(2) != 1 and v > 1:
        logits = logits.contiguous()
    out = torch.empty((b, num), dtype=torch.float32, device=dev)
    parents = torch.empty((b, num), dtype=torch.int64, device=dev)
    tokens = torch.empty_like(parents)
    lib = L.load()
    with L.on_device(dev):
        code = L._DTYPE_CODE[logits.dtype]
        nbytes = lib.m3_beam_select_workspace_size(b, k, v, num, code)
        ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev) if nbytes else None  # none where one launch does
        vals = [*L.rec3(logits, code, b, k, v), *L.rec2(scores, L.M3_FLOAT32, b, k)]
        vals += L.NO_RECORD if finished is None else L.rec2(finished, L.M3_UINT8, b, k)
        tail = (2, b, num, 0, 0, 0, 0, num, 1, 0, 0, 0, 0)
        vals += (out.data_ptr() or 1, L.M3_FLOAT32, *tail, parents.data_ptr() or 1, L.M3_INT64, *tail,
                 tokens.data_ptr() or 1, L.M3_INT64, *tail)
        a = L.Records(vals)
        at = a.base
        rc = lib.m3_beam_select(at, at + 112, None if finished is None else at + 224, end_token, at + 336, at + 448,
                                at + 560, ws.data_ptr() if nbytes else None, nbytes, L.stream_ptr(dev))
    L.check(rc, "m3_beam_select")
    return BeamSelection(out, parents, tokens)


def _flat(states):
    """The tensors of a cache: one, or any lists and tuples of them."""
    if isinstance(states, torch.Tensor):
        return [states]
    if not isinstance(states, (list, tuple)):
        raise TypeError(f"reorder_states_: a tensor, or lists and tuples of them, expected; got {type(states).__name__}")
    return [t for s in states for t in ((s,) if isinstance(s, torch.Tensor) else _flat(s))]


def _pitches(what, ts, rows, index):
    """Addresses, row pitches and row sizes in bytes; each tensor has that many rows, each row dense."""
    if not all([t.get_device() == index for t in ts]):
        raise RuntimeError(f"reorder_states_: {what} must be CUDA tensors of the parents' device (no CPU path)")
    pitches, sizes = [], []
    for t in ts:
        if not t.dim() or t.size(0) != rows:
            raise ValueError(f"reorder_states_: {what} of {rows} rows expected, got {tuple(t.shape)}")
        if rows and t.is_contiguous():
            pitch = t.nbytes // rows
            pitches.append(pitch)
            sizes.append(pitch)
            continue
        n, es = t.numel(), t.element_size()
        if n and not t[0].is_contiguous():
            raise ValueError(f"reorder_states_: rows of {what} must be dense in memory, got strides {t.stride()} for "
                             f"{tuple(t.shape)}")
        pitches.append(t.stride(0) * es)
        sizes.append(n // rows * es if rows else 0)
    return [t.data_ptr() for t in ts], pitches, sizes


def reorder_states_(states, parents, *, out=None):
    """Row b * T + j of every tensor of ``states`` becomes its row b * S + parents[b, j], in one
    launch. ``parents`` (batch, T) int64; a parent outside [0, S) makes the row zeros. ``states``: a
    tensor or lists and tuples of them (a decode cache), of any dtypes, with their rows in
    front, each row dense in memory.

    In place S = T, at most 32; rows that stay are not touched. ``out``: as many tensors of the same
    row shapes and dtypes that receive the result instead, batch * T rows each; S is then what the
    rows of ``states`` come to for each of the batch: one for a prompt's state that is forked to T beams;
    with a batch of one, any rows in any order (compaction). Tensors that are written must not
    share memory with others. Returns ``out``, or ``states``. Without gradients."""
    name = "reorder_states_"
    if not isinstance(parents, torch.Tensor):
        raise TypeError(f"{name}: parents must be a tensor")
    _require_cuda(name, parents)
    if parents.dim() != 2 or parents.dtype is not torch.int64:
        raise ValueError(f"{name}: parents are (batch, rows) int64, got {tuple(parents.shape)} {parents.dtype}")
    batch, rows = parents.shape
    src = _flat(states)
    n = len(src)
    given = out if out is not None else states
    if not n:
        return given
    first = src[0].shape
    if not first or (batch and first[0] % batch):
        raise ValueError(f"{name}: states of {tuple(first)} for a batch of {batch}")
    source = first[0] // batch if batch else rows  # (of an empty batch nothing is moved)
    dev = parents.device
    ptrs, pitch, size = _pitches("states", src, source * batch, dev.index)
    dst = src
    if out is None:
        if source != rows:
            raise ValueError(f"{name}: in place, parents of {source} rows a group expected, got {rows}")
        if rows > _MAX_BEAMS:
            raise ValueError(f"{name}: in place at most {_MAX_BEAMS} rows a group, got {rows}")
        outs = opitch = None
    else:
        dst = _flat(out)
        if len(dst) != n:
            raise ValueError(f"{name}: {n} states but {len(dst)} outputs")
        outs, opitch, osize = _pitches("out", dst, rows * batch, dev.index)
        for t, o in zip(src, dst):
            if t.shape[1:] != o.shape[1:] or t.dtype is not o.dtype:
                raise ValueError(f"{name}: output of rows {tuple(o.shape[1:])} {o.dtype} for rows {tuple(t.shape[1:])} {t.dtype}")
            if t.dtype.is_complex and t.is_conj() != o.is_conj():  # their memory holds different numbers
                raise ValueError(f"{name}: states and out are lazily conjugated both or neither; see torch.Tensor.resolve_conj")
        if not source:
            size = osize
    if torch.is_grad_enabled() and (any([t.requires_grad for t in src]) or (out is not None and any([t.requires_grad for t in dst]))):
        raise RuntimeError(f"{name}: works without gradients; call it under torch.no_grad()")
    lib = L.load()
    # one block of host memory: addresses, row sizes and pitches
    table = struct.pack(f"={(5 if outs else 3) * n}q", *ptrs, *size, *pitch, *(outs + opitch if outs else ()))
    base = L.address(table)
    a = L.Records(L.rec2(parents, L.M3_INT64, batch, rows))
    with L.on_device(dev):
        rc = lib.m3_reorder_states(n, base, base + 24 * n if outs else None, base + 8 * n, base + 16 * n,
                                   base + 32 * n if outs else None, source, a.at(0), L.stream_ptr(dev))
    L.check(rc, "m3_reorder_states")
    try:
        torch.autograd.graph.increment_version(dst)
    except RuntimeError:  # inference tensors have no version
        torch.autograd.graph.increment_version([t for t in dst if not t.is_inference()])
    return given
