"""libvpaged.so: it loads, exports exactly what include/vpaged.h declares, its structs are the binding's, and its entry
points refuse what does not fit before anything is launched."""

from __future__ import annotations

import ctypes
import re
import shutil
import subprocess
from pathlib import Path

import pytest

from vinfer_amd import _vpaged

HEADER = Path(__file__).resolve().parents[1] / "include" / "vpaged.h"
STRUCTS = {"vpaged_tables": _vpaged.VpagedTables, "vpaged_rotate_args": _vpaged.VpagedRotateArgs,
           "vpaged_shape": _vpaged.VpagedShape, "vpaged_attend_args": _vpaged.VpagedAttendArgs}


def test_symbols_version_and_limits_are_the_headers():
    text = HEADER.read_text()
    names = sorted(set(re.findall(r"^\s*(?:int|size_t|const char\*)\s+(vpaged_\w+)\s*\(", text, re.M)))
    assert names == sorted(_vpaged.EXPORTS)
    lib = _vpaged.load()
    for n in names:
        assert hasattr(lib, n), n
    define = lambda n: int(re.search(rf"#define VPAGED_{n} (\d+)", text).group(1))  # noqa: E731
    assert lib.vpaged_abi_version() == _vpaged.ABI_VERSION == define("ABI_VERSION")
    for n in ("MAX_PAGE_SIZE", "MAX_HEAD_DIM", "MAX_HEADS", "MAX_SEQUENCES", "MAX_QUERIES", "MAX_TOKENS"):
        assert define(n) == getattr(_vpaged, n)


@pytest.mark.parametrize("name", STRUCTS)
def test_structs_match_the_binding(tmp_path, name):
    text = HEADER.read_text()
    body = text[text.index(f"typedef struct {name} ") : text.index(f"}} {name};")]
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    fields = re.findall(r"\b(\w+)\s*[;,]", body)
    struct = STRUCTS[name]
    assert fields == [f for f, _ in struct._fields_]
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not available")
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "vpaged.h"\nint main(void){'
                   + "".join(f'printf("%zu\\n", offsetof({name}, {f}));' for f in fields)
                   + f'printf("%zu\\n", sizeof({name}));return 0;}}\n')
    exe = tmp_path / "layout"
    subprocess.run([gcc, f"-I{HEADER.parent}", str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [getattr(struct, f).offset for f in fields] + [ctypes.sizeof(struct)]


@pytest.mark.parametrize("name", STRUCTS)
def test_packed_blocks_are_the_structs(name):
    struct = STRUCTS[name]
    pack = {"vpaged_tables": _vpaged.PACK_TABLES, "vpaged_rotate_args": _vpaged.PACK_ROTATE, "vpaged_shape": _vpaged.PACK_SHAPE,
            "vpaged_attend_args": _vpaged.PACK_ATTEND}[name]
    flat = [f for f, t in struct._fields_ for f in ([f] if t is not _vpaged.VpagedShape else [f"shape.{g}" for g, _ in t._fields_])]
    values = [i + 1 for i in range(len(flat))]
    block = struct.from_buffer_copy(pack.pack(*values))
    assert ctypes.sizeof(struct) == pack.size
    got = [getattr(block.shape, f[6:]) if f.startswith("shape.") else getattr(block, f) for f in flat]
    assert got == values


def shape(**changes):
    s = dict(dtype=0, sequences=8, groups=2, queries=1, heads=8, kv_heads=2, head_dim=128, page_size=16, max_pages=10,
             max_prefix_pages=20)
    return _vpaged.VpagedShape(*{**s, **changes}.values())


@pytest.mark.parametrize("bad", [dict(sequences=-1), dict(queries=0), dict(heads=7), dict(head_dim=12), dict(head_dim=264),
                                 dict(page_size=24), dict(page_size=0), dict(max_pages=0), dict(max_prefix_pages=0),
                                 dict(groups=-1), dict(sequences=1 << 17), dict(max_pages=(1 << 31) - 1, page_size=4096)], ids=str)
def test_shapes_that_are_refused(bad):
    lib = _vpaged.load()
    assert lib.vpaged_plan_bytes(ctypes.byref(shape())) > 0 < lib.vpaged_attend_workspace_bytes(ctypes.byref(shape()))
    s = shape(**bad)
    assert lib.vpaged_plan_bytes(ctypes.byref(s)) == 0 == lib.vpaged_attend_workspace_bytes(ctypes.byref(s))
    assert lib.vpaged_plan(ctypes.byref(s), None, None, None, None, 0, None) == 1
    assert b"refused" in lib.vpaged_last_error()


def test_calls_that_are_refused():
    lib, one = _vpaged.load(), ctypes.c_void_p(256)  # (never followed: every call here is refused before)
    error = lambda: lib.vpaged_last_error().decode()  # noqa: E731
    assert lib.vpaged_plan(ctypes.byref(shape()), None, one, one, one, 1 << 20, None) == 1 and "lengths" in error()
    assert lib.vpaged_plan(ctypes.byref(shape()), one, one, one, one, 16, None) == 4 and "plan" in error()
    assert lib.vpaged_plan(ctypes.byref(shape()), one, one, one, ctypes.c_void_p(8), 1 << 20, None) == 4 and "aligned" in error()
    a = lambda **c: ctypes.byref(_vpaged.VpagedAttendArgs(  # noqa: E731
        shape=c.pop("shape", shape()), **{**dict(pages=9, scale=1.0, q=256, k_pages=256, v_pages=256, tables=256,
                                                 prefix_tables=256, out=256, plan=256, workspace=256, workspace_bytes=1 << 40), **c}))
    for code, change, text in ((2, dict(shape=shape(dtype=2)), "dtype"), (1, dict(scale=0.0), "scale"), (1, dict(scale=float("inf")), "scale"),
                               (1, dict(pages=0), "pages"), (1, dict(q=None), "set"), (1, dict(prefix_tables=None), "set"),
                               (1, dict(q=264), "aligned"), (1, dict(page_stride=4), "multiples"), (1, dict(table_stride=-1), "strides"),
                               (4, dict(plan=None), "plan"), (4, dict(workspace_bytes=5), "workspace"), (4, dict(workspace=264), "aligned")):
        assert lib.vpaged_attend(a(**change), None) == code and text in error(), change
    t = lambda **c: ctypes.byref(_vpaged.VpagedTables(**{**dict(tables=256, lengths=256, free_pages=256, free_count=256,  # noqa: E731
                                                              sequences=2, max_pages=3, pages=4, page_size=16), **c}))
    for change in (dict(sequences=-1), dict(max_pages=0), dict(pages=0), dict(page_size=3), dict(page_size=8192), dict(lengths=None),
                   dict(sequences=65536, max_pages=32768), dict(pages=1 << 30)):
        assert lib.vpaged_extend(t(**change), one, 4, one, one, one, one, None, 0, None) == 1, change
        assert lib.vpaged_shrink(t(**change), one, None) == 1
    assert lib.vpaged_extend(t(), one, -1, one, one, one, one, None, 0, None) == 1 and "tokens" in error()
    assert lib.vpaged_extend(t(), None, 4, one, one, one, one, None, 0, None) == 1 and "counts" in error()
    assert lib.vpaged_extend(t(), one, 9000, one, one, one, one, None, 0, None) == 4
    assert lib.vpaged_extend(t(sequences=0), one, 4, one, one, one, one, None, 0, None) == 1 and "without sequences" in error()
    r = lambda **c: ctypes.byref(_vpaged.VpagedRotateArgs(**{**dict(  # noqa: E731
        q=256, k=256, v=256, out_q=256, k_pages=256, v_pages=256, positions=256, slots=256, frequencies=256, magnitude=1.0, tokens=3,
        heads=2, kv_heads=1, head_dim=64, dim=64, pages=4, page_size=16), **c}))
    for code, change in ((2, dict(dtype=7)), (1, dict(tokens=-1)), (1, dict(heads=2000)), (1, dict(head_dim=0)), (1, dict(head_dim=300)),
                         (1, dict(dim=3)), (1, dict(dim=66)), (1, dict(page_size=5)), (1, dict(magnitude=float("nan"))),
                         (1, dict(frequencies=None)), (1, dict(k_pages=None)), (1, dict(pages=1 << 30))):
        assert lib.vpaged_rotate_store(r(**change), None) == code, change
