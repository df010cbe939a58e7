"""libvops.so: it loads, exports exactly what include/vops.h declares, and its structs are the binding's."""

from __future__ import annotations

import ctypes
import re
import shutil
import subprocess
from pathlib import Path

import pytest

from vinfer_amd import _vops

HEADER = Path(__file__).resolve().parents[1] / "include" / "vops.h"
STRUCTS = {"vops_beam_args": _vops.VopsBeamArgs, "vops_state": _vops.VopsState, "vops_distill_args": _vops.VopsDistillArgs}


def test_symbols_version_and_limits_are_the_headers():
    text = HEADER.read_text()
    names = sorted(set(re.findall(r"^\s*(?:int|int64_t|size_t|const char\*)\s+(vops_\w+)\s*\(", text, re.M)))
    assert names == sorted(_vops.EXPORTS)
    lib = _vops.load()
    for n in names:
        assert hasattr(lib, n), n
    define = lambda n: int(re.search(rf"#define VOPS_{n} (\d+)", text).group(1))  # noqa: E731
    assert lib.vops_abi_version() == _vops.ABI_VERSION == define("ABI_VERSION")
    for n in ("MAX_VOCAB", "MAX_BEAMS", "MAX_CONTINUATIONS", "MAX_REORDER_BEAMS", "MAX_ENTRIES"):
        assert define(n) == getattr(_vops, n)


@pytest.mark.parametrize("name", STRUCTS)
def test_structs_match_the_binding(tmp_path, name):
    text = HEADER.read_text()
    body = text[text.index(f"typedef struct {name} ") : text.index(f"}} {name};")]
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    fields = re.findall(r"\b(\w+)(?:\[\d\])?;", body)
    struct = STRUCTS[name]
    assert fields == [f for f, _ in struct._fields_]
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not available")
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "vops.h"\nint main(void){'
                   + "".join(f'printf("%zu\\n", offsetof({name}, {f}));' for f in fields)
                   + f'printf("%zu\\n", sizeof({name}));return 0;}}\n')
    exe = tmp_path / "layout"
    subprocess.run([gcc, f"-I{HEADER.parent}", str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [getattr(struct, f).offset for f in fields] + [ctypes.sizeof(struct)]


def test_workspaces_hold_the_segments():
    lib = _vops.load()
    assert lib.vops_beam_workspace_bytes(0, 2, 4, 151936, 8) >= 2 * 4 * 10 * (8 * 8 + 12)
    assert lib.vops_beam_workspace_bytes(0, -1, 4, 100, 8) == 0
    assert lib.vops_beam_workspace_bytes(0, 2, 4, 100, 65) == 0
    assert lib.vops_distill_workspace_bytes(1, 5, 151936, 64) >= 5 * 66 * 4
    assert lib.vops_distill_workspace_bytes(3, 5, 100, 8) == 0
