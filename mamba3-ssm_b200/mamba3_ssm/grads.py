"""Global norm of a model's gradients, and their scaling and clipping, on m3_clip_grads (two
kernel launches for up to a thousand tensors, no host synchronisation, deterministic).

``clip_grad_norm_`` takes parameters, with the arguments of torch.nn.utils.clip_grad_norm_ (norm
types, dtypes and devices: see there);
``clip_grads_`` takes the gradients themselves and can also unscale them (loss scaling,
accumulated micro-batches) and write fp32 gradients for an optimiser from 16-bit ones. No
counterpart in the reference's package.
"""

import math
import struct

import torch

from . import _lib as L

__all__ = ["clip_grad_norm_", "clip_grads_"]

_CODES = {torch.float32: L.M3_FLOAT32, torch.bfloat16: L.M3_BFLOAT16, torch.float16: L.M3_FLOAT16}


def _dense(t):
    """Whether the elements fill one run of memory, in any order of the dimensions."""
    n = 1
    for size, stride in sorted(((s, st) for s, st in zip(t.shape, t.stride()) if s != 1), key=lambda p: p[1]):
        if stride != n:
            return False
        n *= size
    return True


def _check(what, ts, device_index):
    """Addresses and dtype codes of the tensors, each dense and on the one device."""
    if not all([t.get_device() == device_index for t in ts]):
        raise RuntimeError(f"clip_grads_: {what} must be CUDA tensors of one device (no CPU path)")
    try:
        codes = [_CODES[t.dtype] for t in ts]
    except KeyError as e:
        raise TypeError(f"clip_grads_: {what} must be float32, bfloat16 or float16, got {e.args[0]}") from None
    if not all([t.is_contiguous() for t in ts]):
        for t in ts:
            if t.numel() and not _dense(t):
                raise ValueError(f"clip_grads_: {what} must be dense in memory, got strides {t.stride()} for "
                                 f"{tuple(t.shape)}")
    return [t.data_ptr() for t in ts], codes


def clip_grads_(grads, max_norm, norm_type=2.0, *, scale=1.0, out=None):
    """With n = scale * (2-norm of all gradients together, or for norm_type inf the largest
    magnitude), multiplies every gradient by scale * min(1, max_norm / (n + 1e-6)) and returns n
    (fp32, 0-d, on the device; nothing waits for it).

    ``max_norm`` inf scales without clipping; in place with scale 1 that is the norm alone, and
    nothing is written. ``out``: as
    many tensors of the same shapes and strides that receive the result in place of the
    gradients, fp32 or the gradient's dtype. The gradients may be of mixed dtypes, each
    dense in memory, and must not share memory. A NaN among them makes n and all that is written
    NaN; so does an infinite n with an infinite ``max_norm``."""
    if isinstance(grads, torch.Tensor):
        grads = [grads]
        out = [out] if isinstance(out, torch.Tensor) else out
    grads = list(grads)
    norm_type, max_norm, scale = float(norm_type), float(max_norm), float(scale)
    if norm_type not in (2.0, math.inf):
        raise ValueError(f"clip_grads_: norm_type is 2 or inf, got {norm_type}")
    if not max_norm >= 0:
        raise ValueError(f"clip_grads_: max_norm must be 0 or more, got {max_norm}")
    if not 0 < scale < math.inf:
        raise ValueError(f"clip_grads_: scale must be positive and finite, got {scale}")
    n = len(grads)
    if out is not None:
        out = list(out)
        if len(out) != n:
            raise ValueError(f"clip_grads_: {n} gradients but {len(out)} outputs")
    if not n:
        return torch.zeros(())
    dev = grads[0].device
    if dev.type != "cuda":
        raise RuntimeError("clip_grads_: the B200 build runs on CUDA tensors only (no CPU path)")
    ptrs, codes = _check("gradients", grads, dev.index)
    numel = [t.numel() for t in grads]
    outs = out_codes = None
    if out is not None:
        outs, out_codes = _check("outputs", out, dev.index)
        for g, o in zip(grads, out):
            if g.shape != o.shape or (g.numel() and g.stride() != o.stride()
                                      and not (g.is_contiguous() and o.is_contiguous())):
                raise ValueError(f"clip_grads_: output of shape {tuple(o.shape)}, strides {o.stride()} for a gradient "
                                 f"of {tuple(g.shape)}, {g.stride()}")
    # one block of host memory: addresses, counts and dtype codes
    tables = struct.pack(f"={2 * n}q{n}i", *ptrs, *numel, *codes)
    out_tables = struct.pack(f"={n}q{n}i", *outs, *out_codes) if outs is not None else None
    lib = L.load()
    norm = torch.empty((), dtype=torch.float32, device=dev)
    nbytes = lib.m3_clip_grads_workspace_size(n)
    ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev)
    a = L.Records(L.rec0(norm.data_ptr(), L.M3_FLOAT32))
    base = L.address(tables)
    obase = L.address(out_tables) if out_tables is not None else None
    with L.on_device(dev):
        rc = lib.m3_clip_grads(n, base, base + 8 * n, base + 16 * n, obase, obase + 8 * n if obase else None,
                               int(norm_type == math.inf), max_norm, scale, a.at(0), ws.data_ptr(), nbytes,
                               L.stream_ptr(dev))
    L.check(rc, "m3_clip_grads")
    if out is not None or scale != 1.0 or max_norm != math.inf:
        written = out if out is not None else grads
        try:
            torch.autograd.graph.increment_version(written)
        except RuntimeError:  # inference tensors have no version
            torch.autograd.graph.increment_version([t for t in written if not t.is_inference()])
    return norm


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False, foreach=None):
    """torch.nn.utils.clip_grad_norm_ for norm_type 2 or inf and float32, bfloat16 or float16
    gradients on one device: clips the ``.grad`` of the parameters in place to a global norm of
    ``max_norm`` and returns the norm they had. A parameter given twice counts once (torch: twice).
    ``error_if_nonfinite`` waits for the norm and raises, with the gradients as they were.
    ``foreach`` has no effect: there is one way here."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [p.grad for p in dict.fromkeys(parameters) if p.grad is not None]
    if any([g.layout is not torch.strided for g in grads]):
        raise TypeError("clip_grad_norm_: sparse gradients are not supported")
    if error_if_nonfinite:
        norm = clip_grads_(grads, math.inf, norm_type)
        if not torch.isfinite(norm):
            raise RuntimeError(f"clip_grad_norm_: the total norm of order {float(norm_type)} is {norm.item()}, so the "
                               "gradients cannot be clipped")
    # without a bound clip_grads_ would form the norm alone, and a NaN would not spread
    return clip_grads_(grads, max_norm, norm_type, out=grads if max_norm == math.inf else None)
