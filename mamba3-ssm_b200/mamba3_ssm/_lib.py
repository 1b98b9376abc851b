"""ctypes binding of libmamba3_b200.so (declared in include/mamba3_b200.h).

The library is built in-tree by ``mamba3-ssm_b200/build_lib.py`` and loaded from this
directory. There is deliberately no fallback: if the library is missing or a call fails,
a RuntimeError is raised with the library's own error text.
"""

import contextlib
import ctypes
import functools
import os
import struct

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libmamba3_b200.so")
MAX_DIMS = 6

M3_FLOAT32, M3_BFLOAT16, M3_FLOAT16 = 0, 1, 2
M3_OK, M3_ERR_INVALID_ARGUMENT, M3_ERR_UNSUPPORTED, M3_ERR_CUDA, M3_ERR_WORKSPACE = 0, 1, 2, 3, 4
M3_INT64, M3_UINT8 = 3, 4
_DTYPE_CODE = {torch.float32: M3_FLOAT32, torch.bfloat16: M3_BFLOAT16, torch.float16: M3_FLOAT16,
               torch.int64: M3_INT64}
_STATUS = {1: "invalid argument", 2: "unsupported", 3: "CUDA error", 4: "workspace"}


class M3Tensor(ctypes.Structure):
    _fields_ = [
        ("data", ctypes.c_void_p),
        ("dtype", ctypes.c_int32),
        ("ndim", ctypes.c_int32),
        ("shape", ctypes.c_int64 * MAX_DIMS),
        ("stride", ctypes.c_int64 * MAX_DIMS),
    ]


class M3LayerDims(ctypes.Structure):
    _fields_ = [
        ("d_model", ctypes.c_int32),
        ("d_inner", ctypes.c_int32),
        ("nheads", ctypes.c_int32),
        ("headdim", ctypes.c_int32),
        ("d_state", ctypes.c_int32),
        ("ngroups", ctypes.c_int32),
        ("mimo_rank", ctypes.c_int32),
        ("num_rope_angles", ctypes.c_int32),
        ("rope_split", ctypes.c_int32),
        ("A_floor", ctypes.c_float),
        ("norm_eps", ctypes.c_float),
    ]


# tensor arguments are passed as plain addresses of m3_tensor records (see pack())
_P = ctypes.c_void_p
_REC = struct.Struct("<qii" + "q" * MAX_DIMS + "q" * MAX_DIMS)
assert _REC.size == ctypes.sizeof(M3Tensor)
_SIGS = {
    "m3_abi_version": ([], ctypes.c_int),
    "m3_last_error_string": ([], ctypes.c_char_p),
    "m3_siso_scan_fwd": ([_P] * 12 + [ctypes.c_void_p], ctypes.c_int),
    "m3_siso_scan_bwd_workspace_size": ([ctypes.c_int64] * 5, ctypes.c_size_t),
    "m3_siso_scan_bwd": ([_P] * 19 + [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p], ctypes.c_int),
    "m3_siso_scan_bwd_noalloc": ([_P] * 19 + [ctypes.c_void_p], ctypes.c_int),
    "m3_siso_scan_kstates_size": ([ctypes.c_int64] * 5 + [ctypes.c_int, ctypes.c_int], ctypes.c_size_t),
    "m3_siso_scan_bwd_kstates_workspace_size": ([ctypes.c_int64] * 3, ctypes.c_size_t),
    "m3_siso_scan_fwd_kstates": ([_P] * 12 + [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p], ctypes.c_int),
    "m3_siso_scan_bwd_kstates": ([_P] * 19 + [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p, ctypes.c_size_t,
                                              ctypes.c_void_p], ctypes.c_int),
    "m3_mimo_scan_fwd": ([_P] * 14 + [ctypes.c_void_p], ctypes.c_int),
    "m3_mimo_scan_fwd_workspace_size": ([ctypes.c_int64] * 4, ctypes.c_size_t),
    "m3_mimo_scan_fwd_ws": ([_P] * 14 + [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p], ctypes.c_int),
    "m3_mimo_scan_bwd_workspace_size": ([ctypes.c_int64] * 6, ctypes.c_size_t),
    "m3_mimo_scan_bwd": ([_P] * 23 + [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p], ctypes.c_int),
    "m3_mimo_scan_bwd_ws_workspace_size": ([ctypes.c_int64] * 6, ctypes.c_size_t),
    "m3_mimo_scan_bwd_ws": ([_P] * 23 + [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p, ctypes.c_size_t,
                                         ctypes.c_void_p], ctypes.c_int),
    "m3_siso_step": ([ctypes.c_void_p] + [_P] * 14 + [ctypes.c_void_p], ctypes.c_int),
    "m3_mimo_step": ([ctypes.c_void_p] + [_P] * 16 + [ctypes.c_void_p], ctypes.c_int),
    "m3_rmsnorm": ([_P, _P, _P, ctypes.c_float, _P, _P, ctypes.c_void_p], ctypes.c_int),
    "m3_device_timeouts": ([ctypes.c_int, ctypes.POINTER(ctypes.c_int)], ctypes.c_int),
    "m3_layer_prologue": ([ctypes.c_void_p] + [_P] * 13 + [ctypes.c_void_p], ctypes.c_int),
    "m3_silu_gate": ([_P] * 3 + [ctypes.c_void_p], ctypes.c_int),
    "m3_mimo_layer_scan_fwd": ([ctypes.c_void_p] + [_P] * 14 + [ctypes.c_int32] + [_P] * 3 +
                               [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p], ctypes.c_int),
    "m3_layer_prologue_bwd_workspace_size": ([ctypes.c_void_p, ctypes.c_int64, ctypes.c_int64], ctypes.c_size_t),
    "m3_layer_prologue_bwd": ([ctypes.c_void_p] + [_P] * 19 + [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p],
                              ctypes.c_int),
    "m3_silu_gate_bwd": ([_P] * 5 + [ctypes.c_void_p], ctypes.c_int),
    "m3_argmax_rows": ([_P, _P, ctypes.c_void_p], ctypes.c_int),
    "m3_token_logprobs": ([_P] * 3 + [ctypes.c_double, ctypes.c_int64] + [_P] * 2 + [ctypes.c_void_p], ctypes.c_int),
    "m3_token_logprobs_grad": ([_P] * 5 + [ctypes.c_double, ctypes.c_int64, _P, ctypes.c_void_p], ctypes.c_int),
    "m3_policy_loss_workspace_size": ([ctypes.c_int64] * 2, ctypes.c_size_t),
    "m3_policy_loss": ([_P] * 6 + [ctypes.c_double, ctypes.c_int64] + [ctypes.c_double] * 3 + [ctypes.c_int] +
                       [_P] * 5 + [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p], ctypes.c_int),
    "m3_policy_loss_grad": ([_P] * 4 + [ctypes.c_double, ctypes.c_int64, ctypes.c_int, _P, ctypes.c_void_p,
                                       ctypes.c_size_t, ctypes.c_void_p], ctypes.c_int),
    "m3_preference_loss_workspace_size": ([ctypes.c_int64] * 2, ctypes.c_size_t),
    "m3_preference_loss": ([_P] * 4 + [ctypes.c_double, ctypes.c_int64, ctypes.c_double, ctypes.c_double] + [_P] * 3 +
                           [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p], ctypes.c_int),
    "m3_preference_loss_grad": ([_P] * 4 + [ctypes.c_double, ctypes.c_int64, _P, ctypes.c_void_p, ctypes.c_size_t,
                                           ctypes.c_void_p], ctypes.c_int),
    "m3_clip_grads_workspace_size": ([ctypes.c_int64], ctypes.c_size_t),
    "m3_clip_grads": ([ctypes.c_int64] + [ctypes.c_void_p] * 5 + [ctypes.c_int, ctypes.c_double, ctypes.c_double, _P,
                       ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p], ctypes.c_int),
}

_lib = None


def load():
    """Load the library once and attach the C signatures."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise RuntimeError(
            f"{LIB_PATH} is not built; run `python mamba3-ssm_b200/build_lib.py` (nvcc, sm_100a). "
            "There is no CPU or PyTorch fallback.")
    lib = ctypes.CDLL(LIB_PATH)
    for name, (args, res) in _SIGS.items():
        fn = getattr(lib, name)
        fn.argtypes = args
        fn.restype = res
    if lib.m3_abi_version() != 1:
        raise RuntimeError("libmamba3_b200.so ABI version mismatch")
    _lib = lib
    return lib


def exported_symbols():
    return list(_SIGS)


def tensor(t):
    """m3_tensor view of a torch tensor (None -> absent optional argument)."""
    m = M3Tensor()
    if t is None:
        m.data = None
        m.ndim = 0
        return m
    if t.dim() > MAX_DIMS:
        raise ValueError("tensor has too many dimensions for the C ABI")
    code = _DTYPE_CODE.get(t.dtype)
    if code is None:
        raise TypeError(f"dtype {t.dtype} is not supported by libmamba3_b200")
    n = t.dim()
    m.data = t.data_ptr() or (1 if t.numel() == 0 else 0)
    m.dtype = code
    m.ndim = n
    m.shape[:n] = t.shape
    m.stride[:n] = t.stride()
    return m


_PADS = tuple((0,) * (MAX_DIMS - n) for n in range(MAX_DIMS + 1))


@functools.lru_cache(maxsize=64)
def _records_struct(n):
    return struct.Struct("=" + ("qii" + "q" * (2 * MAX_DIMS)) * n)


class Packed:
    """m3_tensor records of several tensors in one buffer (built with struct, which is
    several times cheaper than filling ctypes structures). ``ptrs[i]`` is the address
    of record i, or None for an absent optional argument; the object must stay alive
    until the call returns."""

    __slots__ = ("buf", "ptrs")

    def __init__(self, ts):
        vals = []
        ptrs = []
        n = 0
        for t in ts:
            if t is None:
                ptrs.append(None)
                continue
            code = _DTYPE_CODE.get(t.dtype)
            if code is None:
                raise TypeError(f"dtype {t.dtype} is not supported by libmamba3_b200")
            shape = t.shape
            nd = len(shape)
            if nd > MAX_DIMS:
                raise ValueError("tensor has too many dimensions for the C ABI")
            pad = _PADS[nd]
            vals += (t.data_ptr() or (1 if t.numel() == 0 else 0), code, nd, *shape, *pad, *t.stride(), *pad)
            ptrs.append(n)
            n += _REC.size
        if n:
            self.buf = _records_struct(n // _REC.size).pack(*vals)
            base = address(self.buf)
            ptrs = [None if p is None else base + p for p in ptrs]
        else:
            self.buf = None
        self.ptrs = ptrs


def pack(*ts):
    return Packed(ts)


class Records:
    """Records whose fields the caller knows already (an entry point with a dozen operands of
    one shape would otherwise spend more time on packing than on its launches): ``vals`` holds
    rec2 / rec3 / NO_RECORD tuples one after the other. ``at(i)`` is the address of record i."""

    __slots__ = ("buf", "base")

    def __init__(self, vals):
        self.buf = _records_struct(len(vals) // 15).pack(*vals)
        self.base = address(self.buf)

    def at(self, i):
        return self.base + _REC.size * i


NO_RECORD = (0,) * 15  # data NULL: an absent optional argument


def rec2(t, code, a, b):
    """The record of a two-dimensional (a, b) tensor of dtype ``code``."""
    return (t.data_ptr() or 1, code, 2, a, b, 0, 0, 0, 0, *t.stride(), 0, 0, 0, 0)


def rec3(t, code, a, b, c):
    return (t.data_ptr() or 1, code, 3, a, b, c, 0, 0, 0, *t.stride(), 0, 0, 0)


def rec0(ptr, code):
    """The record of one value at an address."""
    return (ptr, code, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)


def address(b):
    """Address of a bytes object's contents; it must stay alive until the call returns."""
    return ctypes.cast(ctypes.c_char_p(b), ctypes.c_void_p).value


def ref(m):
    return ctypes.byref(m) if m is not None else None


def check(rc, what):
    if rc != 0:
        msg = load().m3_last_error_string().decode(errors="replace")
        raise RuntimeError(f"{what} failed ({_STATUS.get(rc, rc)}): {msg}")


# the current stream's handle as an integer: the public Stream object costs as much as a launch
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def stream_ptr(device):
    """Handle of the current stream of a CUDA device, as an integer."""
    if _raw_stream is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


def stream_of(t):
    return ctypes.c_void_p(stream_ptr(t.device))


_NO_SWITCH = contextlib.nullcontext()


def on_device(device):
    """The context of a call on ``device``: the switch to it, or nothing where it is current."""
    return _NO_SWITCH if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def device_timeouts(reset=False, device=None):
    """Nonzero once a bounded inter-warp wait of a kernel on this device gave up (outputs
    of that launch are invalid). Synchronises the device."""
    lib = load()
    v = ctypes.c_int(0)
    with torch.cuda.device(device if device is not None else torch.cuda.current_device()):
        check(lib.m3_device_timeouts(1 if reset else 0, ctypes.byref(v)), "m3_device_timeouts")
    return v.value
