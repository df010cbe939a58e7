"""ctypes binding of ``libvpaged.so`` (the C ABI in include/vpaged.h): the paged cache that sequences share.

Built beside ``libvsampler.so`` by ``python -m vinfer_amd.csrc.build``. Loading never falls back to
anything: if the library is missing, ``load()`` raises.
"""

from __future__ import annotations

import ctypes
import struct
import threading
from pathlib import Path

import torch

LIB_PATH = Path(__file__).resolve().parent / "libvpaged.so"
ABI_VERSION = 1

VPAGED_BF16 = 0
VPAGED_F16 = 1

MAX_PAGE_SIZE = 4096
MAX_HEAD_DIM = 256
MAX_HEADS = 1024
MAX_SEQUENCES = 65536
MAX_QUERIES = 65536
MAX_TOKENS = (1 << 30) - 1

STATUS = {0: "ok", 1: "VPAGED_E_ARG", 2: "VPAGED_E_DTYPE", 3: "VPAGED_E_HIP", 4: "VPAGED_E_WORKSPACE", 5: "VPAGED_E_DEVICE"}

# Every symbol include/vpaged.h declares.
EXPORTS = (
    "vpaged_abi_version",
    "vpaged_query",
    "vpaged_extend_workspace_bytes",
    "vpaged_extend",
    "vpaged_shrink",
    "vpaged_rotate_store",
    "vpaged_plan_bytes",
    "vpaged_plan",
    "vpaged_attend_workspace_bytes",
    "vpaged_attend",
    "vpaged_last_error",
)

_p, _i32, _i64, _f = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float


class VpagedTables(ctypes.Structure):
    """``vpaged_tables`` field for field."""

    _fields_ = [
        ("tables", _p),
        ("lengths", _p),
        ("free_pages", _p),
        ("free_count", _p),
        ("sequences", _i32),
        ("max_pages", _i32),
        ("pages", _i32),
        ("page_size", _i32),
    ]


class VpagedRotateArgs(ctypes.Structure):
    """``vpaged_rotate_args`` field for field."""

    _fields_ = [
        ("q", _p),
        ("k", _p),
        ("v", _p),
        ("q_stride", _i64),
        ("k_stride", _i64),
        ("v_stride", _i64),
        ("q_head_stride", _i64),
        ("k_head_stride", _i64),
        ("v_head_stride", _i64),
        ("out_q", _p),
        ("k_pages", _p),
        ("v_pages", _p),
        ("page_stride", _i64),
        ("place_stride", _i64),
        ("head_stride", _i64),
        ("positions", _p),
        ("slots", _p),
        ("frequencies", _p),
        ("magnitude", _f),
        ("dtype", _i32),
        ("tokens", _i32),
        ("heads", _i32),
        ("kv_heads", _i32),
        ("head_dim", _i32),
        ("dim", _i32),
        ("interleaved", _i32),
        ("pages", _i32),
        ("page_size", _i32),
    ]


class VpagedShape(ctypes.Structure):
    """``vpaged_shape`` field for field."""

    _fields_ = [
        ("dtype", _i32),
        ("sequences", _i32),
        ("groups", _i32),
        ("queries", _i32),
        ("heads", _i32),
        ("kv_heads", _i32),
        ("head_dim", _i32),
        ("page_size", _i32),
        ("max_pages", _i32),
        ("max_prefix_pages", _i32),
    ]


class VpagedAttendArgs(ctypes.Structure):
    """``vpaged_attend_args`` field for field."""

    _fields_ = [
        ("shape", VpagedShape),
        ("pages", _i32),
        ("scale", _f),
        ("q", _p),
        ("q_stride", _i64),
        ("q_token_stride", _i64),
        ("q_head_stride", _i64),
        ("k_pages", _p),
        ("v_pages", _p),
        ("page_stride", _i64),
        ("place_stride", _i64),
        ("head_stride", _i64),
        ("tables", _p),
        ("prefix_tables", _p),
        ("table_stride", _i64),
        ("prefix_table_stride", _i64),
        ("out", _p),
        ("plan", _p),
        ("workspace", _p),
        ("workspace_bytes", ctypes.c_size_t),
    ]


# The same blocks as bytes (``struct`` formats, of their fields in order): packing one is several times as fast as filling
# a ``Structure``. They begin at multiples of 16 bytes of a bytes object, whose address the library is given.
PACK_TABLES = struct.Struct("4Q4i")
PACK_ROTATE = struct.Struct("3Q6q3Q3q3Qf9i")
PACK_SHAPE = struct.Struct("10i")
PACK_ATTEND = struct.Struct("10iifQ3q2Q3q2Q2q4Q")


class VpagedError(RuntimeError):
    """A failed library call; ``code`` is the VPAGED_E_* status."""

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
        size = ctypes.c_size_t
        lib.vpaged_abi_version.restype = ctypes.c_int
        version = lib.vpaged_abi_version()
        if version != ABI_VERSION:
            raise RuntimeError(f"{LIB_PATH} has ABI version {version}, expected {ABI_VERSION}")
        lib.vpaged_query.argtypes = [ctypes.c_int, ctypes.c_char_p, size]
        lib.vpaged_extend_workspace_bytes.argtypes = [_i32, _i32]
        lib.vpaged_extend.argtypes = [_p, _p, _i32, _p, _p, _p, _p, _p, size, _p]
        lib.vpaged_shrink.argtypes = [_p, _p, _p]
        lib.vpaged_rotate_store.argtypes = [_p, _p]
        lib.vpaged_plan_bytes.argtypes = [_p]
        lib.vpaged_plan.argtypes = [_p, _p, _p, _p, _p, size, _p]
        lib.vpaged_attend_workspace_bytes.argtypes = [_p]
        lib.vpaged_attend.argtypes = [_p, _p]
        for name in ("query", "extend", "shrink", "rotate_store", "plan", "attend"):
            getattr(lib, f"vpaged_{name}").restype = ctypes.c_int
        for name in ("extend_workspace_bytes", "plan_bytes", "attend_workspace_bytes"):
            getattr(lib, f"vpaged_{name}").restype = size
        lib.vpaged_last_error.restype = ctypes.c_char_p
        _lib = lib
        return lib


def check(code: int) -> None:
    """Raise ``VpagedError`` for a non-zero status."""
    if code != 0:
        raise VpagedError(code, load().vpaged_last_error().decode(errors="replace"))


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
    code = load().vpaged_query(device_index, buf, len(buf))
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
        return f"libvpaged.so does not load: {e}"
    return query(device.index if device.index is not None else torch.cuda.current_device())
