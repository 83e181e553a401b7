"""ctypes binding of the C ABI in include/hgemm_sm100_train.h: what a non-torch
host writes against ``libhgemm_train_sm100.so``. ``load()`` only opens the
library (no GPU needed); the status codes are those of :mod:`llm_hgemm.capi`.
"""

from __future__ import annotations

import ctypes
from ctypes import c_double, c_float, c_int32, c_int64, c_uint64, c_void_p
from pathlib import Path

LIB_PATH = Path(__file__).resolve().parent / "libhgemm_train_sm100.so"

F16, BF16 = 0, 1
TILE_PAIR = 0x1000
LOSS_NONE, LOSS_MEAN, LOSS_SUM = 0, 1, 2


class Common(ctypes.Structure):
    _fields_ = [("dtype", c_int32), ("tile", c_int32), ("flags", c_int32), ("splits", c_int32),
                ("status", c_void_p), ("timeout_ns", c_uint64)]


def _struct(name: str, pointers: str, sizes: str, rest=()):
    fields = [("common", Common)] + [(p, c_void_p) for p in pointers.split()]
    for s in sizes.split():
        fields.append((s, c_uint64 if s == "workspace_bytes" else c_int64))
    return type(name, (ctypes.Structure,), {"_fields_": fields + list(rest)})


FfnForward = _struct("FfnForward", "x gate up down y h silu slope workspace",
                     "workspace_bytes tokens hidden inter out ldx")
FfnBackward = _struct("FfnBackward", "dy x gate up down silu slope h dgate_pre dup_pre dx dgate dup ddown workspace",
                      "workspace_bytes tokens hidden inter out ldx lddy")
_REDUCTION = [("reduction", c_int32), ("reserved", c_int32)]
LossForward = _struct("LossForward", "x weight target loss lse workspace",
                      "workspace_bytes tokens hidden vocab ldx ignore_index", _REDUCTION)
LossBackward = _struct("LossBackward", "x weight target lse dloss dx dweight workspace",
                       "workspace_bytes tokens hidden vocab ldx ignore_index piece", _REDUCTION)
Orthogonalize = _struct("Orthogonalize", "g out workspace", "workspace_bytes batch rows cols ldg batch_stride",
                        [("steps", c_int32), ("reserved", c_int32), ("a", c_float), ("b", c_float), ("c", c_float),
                         ("reserved2", c_float), ("eps", c_double)])

_lib: ctypes.CDLL | None = None


def load() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        lib = ctypes.CDLL(str(LIB_PATH))
        for name, struct in (("ffn_forward", FfnForward), ("ffn_backward", FfnBackward),
                             ("loss_forward", LossForward), ("loss_backward", LossBackward),
                             ("orthogonalize", Orthogonalize)):
            fn = getattr(lib, f"hgemm_sm100_{name}")
            fn.argtypes, fn.restype = [ctypes.POINTER(struct), c_void_p], ctypes.c_int
            size = getattr(lib, f"hgemm_sm100_{name}_workspace")
            size.argtypes, size.restype = [ctypes.POINTER(struct)], ctypes.c_size_t
        lib.hgemm_sm100_train_read_status.argtypes = [ctypes.POINTER(c_int32), ctypes.c_int]
        lib.hgemm_sm100_train_read_status.restype = ctypes.c_int
        _lib = lib
    return _lib


def run(name: str, args: ctypes.Structure, stream: int = 0) -> int:
    """``hgemm_sm100_<name>(&args, stream)``."""
    return getattr(load(), f"hgemm_sm100_{name}")(ctypes.byref(args), c_void_p(stream))


def workspace(name: str, args: ctypes.Structure) -> int:
    """``hgemm_sm100_<name>_workspace(&args)`` in bytes."""
    return getattr(load(), f"hgemm_sm100_{name}_workspace")(ctypes.byref(args))


def read_status(clear: bool = True) -> tuple[int, int]:
    v = c_int32(0)
    return load().hgemm_sm100_train_read_status(ctypes.byref(v), 1 if clear else 0), v.value
