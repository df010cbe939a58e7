"""ctypes binding of ``libvops.so`` (the C ABI in include/vops.h): beam search and distillation.

Built beside ``libvsampler.so`` by ``python -m vinfer_amd.csrc.build``. Loading never falls back to
anything: if the library is missing, ``load()`` raises.
"""

from __future__ import annotations

import ctypes
import threading
from pathlib import Path

import torch

LIB_PATH = Path(__file__).resolve().parent / "libvops.so"
ABI_VERSION = 2

VOPS_BF16 = 0
VOPS_F32 = 1
VOPS_BEAM_KEEP_SLOTS = 1
VOPS_DISTILL_TAIL = 1

MAX_VOCAB = 524288
MAX_BEAMS = 64
MAX_CONTINUATIONS = 64
MAX_REORDER_BEAMS = 32
MAX_ENTRIES = 1024
TEMPERATURES = (1e-6, 1e6)

STATUS = {0: "ok", 1: "VOPS_E_ARG", 2: "VOPS_E_DTYPE", 3: "VOPS_E_HIP", 4: "VOPS_E_WORKSPACE", 5: "VOPS_E_DEVICE"}

# Every symbol include/vops.h declares.
EXPORTS = (
    "vops_abi_version",
    "vops_query",
    "vops_beam_workspace_bytes",
    "vops_beam_select",
    "vops_state_columns",
    "vops_reorder",
    "vops_distill_workspace_bytes",
    "vops_distill",
    "vops_distill_grad",
    "vops_last_error",
)


class VopsBeamArgs(ctypes.Structure):
    """``vops_beam_args`` field for field."""

    _fields_ = [
        ("logits", ctypes.c_void_p),
        ("dtype", ctypes.c_int32),
        ("requests", ctypes.c_int32),
        ("beams", ctypes.c_int32),
        ("vocab", ctypes.c_int32),
        ("request_stride", ctypes.c_int64),
        ("beam_stride", ctypes.c_int64),
        ("scores", ctypes.c_void_p),
        ("finished", ctypes.c_void_p),
        ("n", ctypes.c_int32),
        ("pad_id", ctypes.c_int32),
        ("flags", ctypes.c_uint32),
        ("reserved", ctypes.c_uint32),
        ("out_scores", ctypes.c_void_p),
        ("out_beams", ctypes.c_void_p),
        ("out_tokens", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_size_t),
    ]


class VopsState(ctypes.Structure):
    """``vops_state`` field for field."""

    _fields_ = [
        ("data", ctypes.c_void_p),
        ("slot_stride", ctypes.c_int64),
        ("stride", ctypes.c_int64 * 3),
        ("run", ctypes.c_int64),
        ("unit", ctypes.c_int64),
        ("size", ctypes.c_int32 * 3),
        ("length_dim", ctypes.c_int32),
        ("max_length", ctypes.c_int32),
        ("reserved", ctypes.c_int32),
    ]


class VopsDistillArgs(ctypes.Structure):
    """``vops_distill_args`` field for field."""

    _fields_ = [
        ("student", ctypes.c_void_p),
        ("dtype", ctypes.c_int32),
        ("rows", ctypes.c_int32),
        ("vocab", ctypes.c_int32),
        ("entries", ctypes.c_int32),
        ("row_stride", ctypes.c_int64),
        ("ids", ctypes.c_void_p),
        ("teacher", ctypes.c_void_p),
        ("weights", ctypes.c_void_p),
        ("temperature", ctypes.c_double),
        ("flags", ctypes.c_uint32),
        ("out_loss", ctypes.c_void_p),
        ("out_grad", ctypes.c_void_p),
        ("grad_stride", ctypes.c_int64),
        ("states", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_size_t),
    ]


class VopsError(RuntimeError):
    """A failed library call; ``code`` is the VOPS_E_* status."""

    def __init__(self, code: int, message: str) -> None:
        super().__init__(f"{STATUS.get(code, code)}: {message}")
        self.code = code


_lock = threading.Lock()
_lib: ctypes.CDLL | None = None


def load() -> ctypes.CDLL:
    """The loaded library (once per process); raises if it is missing or mismatched."""
    global _lib
    with _lock:
        if _lib is not None:
            return _lib
        if not LIB_PATH.exists():
            raise FileNotFoundError(f"{LIB_PATH} is not built; run `python -m vinfer_amd.csrc.build` (needs hipcc)")
        lib = ctypes.CDLL(str(LIB_PATH))
        i32, i64, p = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p
        lib.vops_abi_version.restype = ctypes.c_int
        version = lib.vops_abi_version()
        if version != ABI_VERSION:
            raise RuntimeError(f"{LIB_PATH} has ABI version {version}, expected {ABI_VERSION}")
        lib.vops_query.argtypes = [ctypes.c_int, ctypes.c_char_p, ctypes.c_size_t]
        lib.vops_query.restype = ctypes.c_int
        lib.vops_beam_workspace_bytes.argtypes = [i32, i32, i32, i32, i32]
        lib.vops_beam_workspace_bytes.restype = ctypes.c_size_t
        lib.vops_beam_select.argtypes = [ctypes.POINTER(VopsBeamArgs), p]
        lib.vops_beam_select.restype = ctypes.c_int
        lib.vops_state_columns.argtypes = [ctypes.POINTER(VopsState)]
        lib.vops_state_columns.restype = i64
        lib.vops_reorder.argtypes = [p, i32, i64, i32, i32, p, p, p]
        lib.vops_reorder.restype = ctypes.c_int
        lib.vops_distill_workspace_bytes.argtypes = [i32, i32, i32, i32]
        lib.vops_distill_workspace_bytes.restype = ctypes.c_size_t
        lib.vops_distill.argtypes = [ctypes.POINTER(VopsDistillArgs), p]
        lib.vops_distill.restype = ctypes.c_int
        lib.vops_distill_grad.argtypes = [ctypes.POINTER(VopsDistillArgs), p]
        lib.vops_distill_grad.restype = ctypes.c_int
        lib.vops_last_error.restype = ctypes.c_char_p
        _lib = lib
        return lib


def check(code: int) -> None:
    """Raise ``VopsError`` for a non-zero status."""
    if code != 0:
        raise VopsError(code, load().vops_last_error().decode(errors="replace"))


def call(entry, device, *args) -> None:
    """``entry(*args, stream)`` with torch's current stream of ``device``, which is made the current device
    where it is not."""
    stream = torch._C._cuda_getCurrentRawStream(device.index)
    if torch._C._cuda_getDevice() == device.index:
        code = entry(*args, stream)
    else:
        with torch.cuda.device(device):
            code = entry(*args, stream)
    if code:
        check(code)


def query(device_index: int) -> str | None:
    """``None`` if the device can run the kernels, else the library's reason."""
    buf = ctypes.create_string_buffer(256)
    code = load().vops_query(device_index, buf, len(buf))
    return None if code == 0 else (buf.value.decode(errors="replace") or STATUS.get(code, str(code)))


def unsupported(device) -> str | None:
    """Why a backend over this library cannot run on ``device``, or ``None`` if it can (``supports`` of a
    registry entry: kernels/registry.py:38-43)."""
    if torch.version.hip is None:
        return "needs a ROCm build of PyTorch"
    if not torch.cuda.is_available():
        return "no HIP device is visible"
    try:
        load()
    except Exception as e:  # the reason is reported, never swallowed into a fallback
        return f"libvops.so does not load: {e}"
    return query(device.index if device.index is not None else torch.cuda.current_device())
