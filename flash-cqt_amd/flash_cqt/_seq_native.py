"""ctypes boundary to libflashcqt_seq.so (the C ABI declared in
include/flashcqt_seq.h): the sequence operators' kernels.

A library of its own beside libflashcqt.so: the transform needs none of it and
is built in variants. As there, it is loaded after torch, binds to the HIP
runtime that torch loaded, and there is no fallback: if it is missing or does
not load, every sequence operator raises.
"""
import ctypes
import importlib.util

import torch
from torch.autograd import forward_ad

from . import _native
from ._native import NativeError, stream_handle  # noqa: F401

LIB_PATH = _native.LIB_PATH.with_name("libflashcqt_seq.so")
GLUE_PATH = LIB_PATH.with_name("_fcqt_seq_torch.so")
ABI_VERSION = 2
MAX_DIM = 256             # FCQT_SEQ_MAX_DIM
DECAY_MAX_DIM = 128       # FCQT_DECAY_MAX_DIM
ROTARY_AXES = 4           # FCQT_ROTARY_AXES
ADAMW_BLOCK = 256         # FCQT_ADAMW_BLOCK
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}

#: every symbol include/flashcqt_seq.h declares
EXPORTS = ("fcqt_seq_abi_version", "fcqt_seq_last_hip_error", "fcqt_head_norm_rotary",
           "fcqt_head_norm_rotary_partial", "fcqt_head_norm_rotary_bwd",
           "fcqt_decay_attention_workspace", "fcqt_decay_attention", "fcqt_decay_attention_bwd",
           "fcqt_decay_attention_step",
           "fcqt_adamw", "fcqt_adamw_drawn", "fcqt_adamw_read")

#: the functions that the glue is handed, in its order
GLUE_CALLS = ("fcqt_head_norm_rotary", "fcqt_head_norm_rotary_partial", "fcqt_head_norm_rotary_bwd",
              "fcqt_decay_attention_workspace", "fcqt_decay_attention", "fcqt_decay_attention_bwd",
              "fcqt_decay_attention_step", "fcqt_adamw", "fcqt_adamw_drawn", "fcqt_adamw_read")

P, I32, I64, U64, F32 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_uint64, ctypes.c_float


class Heads(ctypes.Structure):
    """Mirror of struct fcqt_heads."""
    _fields_ = [("data", P), ("batch_stride", I64), ("token_stride", I64), ("head_stride", I64), ("heads", I32)]


class Rotary(ctypes.Structure):
    """Mirror of struct fcqt_rotary."""
    _fields_ = [("positions", P), ("positions_batch", I64), ("freq", P), ("axes", I32), ("ends", I32 * ROTARY_AXES),
                ("interleaved", I32)]


class AdamwTensor(ctypes.Structure):
    """Mirror of struct fcqt_adamw_tensor."""
    _fields_ = [("p", P), ("g", P), ("m", P), ("v", P), ("m_scale", P), ("v_scale", P), ("n", I64)]


class AdamwFactors(ctypes.Structure):
    """Mirror of struct fcqt_adamw_factors."""
    _fields_ = [(n, F32) for n in ("b1", "c1", "b2", "c2", "keep", "rate", "root", "eps")]


_lib = None


def load():
    """Load and type the library once; raise NativeError if unavailable."""
    global _lib
    if _lib is not None:
        return _lib
    if not LIB_PATH.exists():
        raise NativeError(f"flash_cqt sequence library not built ({LIB_PATH}); run __graft_entry__.build()")
    try:
        lib = ctypes.CDLL(str(LIB_PATH))
    except OSError as e:
        raise NativeError(f"cannot load {LIB_PATH}: {e}") from e
    H, R = ctypes.POINTER(Heads), ctypes.POINTER(Rotary)
    sig = {
        "fcqt_seq_abi_version": ([], ctypes.c_int),
        "fcqt_seq_last_hip_error": ([], ctypes.c_char_p),
        "fcqt_head_norm_rotary": ([H, H, R, P, P, P, P, I64, I64, I32, I32, I32, F32, P], ctypes.c_int),
        "fcqt_head_norm_rotary_partial": ([I64, I64, I32, I32, I32], I64),
        "fcqt_head_norm_rotary_bwd": ([H, H, H, H, R, P, P, P, P, P, P, I64, I64, I32, I32, I32, F32, P], ctypes.c_int),
        "fcqt_decay_attention_workspace": ([I64, I64, I32, I32, I32, I32, I32, I32, I32], I64),
        "fcqt_decay_attention": ([H, H, H, P, P, P, P, P, P, I64, I64, I64, I32, I32, I32, F32, P], ctypes.c_int),
        "fcqt_decay_attention_bwd": ([H, H, H, P, P, P, P, H, P, P, P, P, P, P, P, I64, I64, I64, I32, I32, I32, F32, P],
                                     ctypes.c_int),
        "fcqt_decay_attention_step": ([H, H, H, P, P, P, P, I64, I64, I32, I32, I32, F32, P], ctypes.c_int),
        "fcqt_adamw": ([ctypes.POINTER(AdamwTensor), I64, I32, I32, ctypes.POINTER(AdamwFactors), P, P], ctypes.c_int),
        "fcqt_adamw_drawn": ([ctypes.POINTER(AdamwTensor), I64, I32, ctypes.POINTER(AdamwFactors), P, U64, I64, P], ctypes.c_int),
        "fcqt_adamw_read": ([ctypes.POINTER(AdamwTensor), I64, P], ctypes.c_int),
    }
    ver = lib.fcqt_seq_abi_version() if hasattr(lib, "fcqt_seq_abi_version") else None
    if ver != ABI_VERSION:
        raise NativeError(f"libflashcqt_seq ABI {ver}, expected {ABI_VERSION}; rebuild")
    for name, (args, res) in sig.items():
        fn = getattr(lib, name, None)
        if fn is None:
            raise NativeError(f"{LIB_PATH} lacks {name}; rebuild")
        fn.argtypes = args
        fn.restype = res
    _lib = lib
    return lib


_glue = False


def load_glue():
    """The host glue module (csrc/seq_glue.cpp): the entry points' checks,
    allocations, autograd nodes and launches of ordinary calls in one C++ call,
    or None when it was not built: the Python paths then do the same work. One
    built for another ABI version or another torch raises NativeError."""
    global _glue
    if _glue is False:
        _glue = None
        if GLUE_PATH.exists():
            try:
                spec = importlib.util.spec_from_file_location("_fcqt_seq_torch", GLUE_PATH)
                mod = importlib.util.module_from_spec(spec)
                spec.loader.exec_module(mod)
            except ImportError as e:
                raise NativeError(f"cannot load {GLUE_PATH}: {e}; rebuild") from e
            built = (getattr(mod, "abi_version", None), getattr(mod, "torch_version", None))
            if built != (ABI_VERSION, str(torch.__version__)):
                raise NativeError(f"{GLUE_PATH} was built for ABI {built[0]} and torch {built[1]}, expected "
                                  f"{ABI_VERSION} and {torch.__version__}; rebuild")
            lib = load()
            mod.attach(*[ctypes.cast(getattr(lib, name), P).value for name in GLUE_CALLS])
            _glue = mod
    return _glue


#: FCQT_E* of include/flashcqt.h
STATUS = {1: "bad argument", 2: "misaligned pointer", 3: "kernel launch failed"}


def check(status, what):
    if status != 0:
        hip = load().fcqt_seq_last_hip_error().decode() if status == 3 else ""
        raise NativeError(f"{what}: {STATUS.get(status, status)}" + (f" [{hip}]" if hip else ""))


def no_tangents(*tensors):
    """The kernels have no forward-mode derivatives: without this the outputs would have none either."""
    if any(torch.is_tensor(t) and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("the sequence operators have no forward-mode derivatives")


def heads(t):
    """The [batch, tokens, heads, dim] tensor t as struct fcqt_heads."""
    b, n, h, _ = t.stride()
    return Heads(t.data_ptr(), b, n, h, t.shape[2])
