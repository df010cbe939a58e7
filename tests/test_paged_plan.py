"""The plan of a step's attention at sizes that its products do not reach: where the stretches of a line begin, on the
host for lines around 2^29 to 2^31 tiles, and what the GPU writes for such lines."""

from __future__ import annotations

import ctypes
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from vinfer_amd import _vpaged
from vinfer_amd.paged import PAGED
from vinfer_amd.registry import BackendContext

GPU = torch.device("cuda", 0)
CSRC = Path(_vpaged.__file__).resolve().parent / "csrc"

# 1024 threads ask for the stretches as the plan's do: each one below `count` that begins within the line is found once,
# where it begins, and no other is found.
ASK = """
#include <cstdio>
#include <vector>
#define __host__
#define __device__
#include "stretches.cuh"
template <class Index> bool right(const vpg::Stretches& s) {
  const __int128 all = static_cast<__int128>(s.units) * s.heads;
  if (static_cast<__int128>(s.per) * s.count < all) return false;
  std::vector<int> found(s.count);
  for (int t = 0; t < 1024; ++t)
    for (int w = t; vpg::begins<Index>(s, w); w += 1024) {
      if (w >= s.count || static_cast<__int128>(static_cast<Index>(w) * s.per) != static_cast<__int128>(w) * s.per) return false;
      ++found[w];
    }
  for (int w = 0; w < s.count; ++w)
    if (found[w] != (static_cast<__int128>(w) * s.per < all)) return false;
  return true;
}
int main() {
  long long units, heads, count, least;
  while (scanf("%lld %lld %lld %lld", &units, &heads, &count, &least) == 4) {
    const vpg::Stretches s = vpg::cut(units, heads, count, least);
    puts((vpg::small(s) ? right<int>(s) : right<int64_t>(s)) ? "right" : "wrong");
  }
}
"""


def test_where_stretches_begin(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    (tmp_path / "ask.cpp").write_text(ASK)
    subprocess.run([gxx, "-std=c++17", "-O1", "-fwrapv", f"-I{CSRC}", str(tmp_path / "ask.cpp"), "-o", str(tmp_path / "ask")], check=True)
    lines = [(u + d, h, c, least) for c, least in ((256, 1), (512, 1), (1024, 2), (2048, 2)) for h in (1, 3, 8, 1024)
             for u in (0, 3, c // h, *(int(f * 2**30) // h for f in (0.4, 0.5, 0.7, 0.99, 1, 1.5, 2, 2.5, 7))) for d in (0, 1)
             if u + d < 1 << 31]
    text = "\n".join(" ".join(map(str, x)) for x in lines)
    got = subprocess.run([str(tmp_path / "ask")], input=text, capture_output=True, text=True, check=True).stdout.split()
    assert len(got) == len(lines) and [x for x, g in zip(lines, got) if g != "right"] == []


@pytest.mark.gpu
@pytest.mark.parametrize("D, heads, length", [(256, 128, 1048576), (256, 64, 1200000), (128, 64, 1500000), (128, 128, 1500000)], ids=str)
def test_lines_of_half_a_billion_tiles(D, heads, length):
    # one sequence of 65536 new tokens, 8 key heads: each starts where its line's tiles say, and nothing is written behind
    lib, kv_heads, page, T = _vpaged.load(), 8, 4096, 65536
    shape = _vpaged.VpagedShape(0, 1, 0, T, heads, kv_heads, D, page, -(-length // page), 0)
    need = lib.vpaged_plan_bytes(ctypes.byref(shape))
    words, guard = need // 4, 1 << 20
    plan = torch.full((words + guard,), -7, dtype=torch.int32, device=GPU)
    lengths = torch.tensor([length], dtype=torch.int32, device=GPU)
    _vpaged.call(lib.vpaged_plan, GPU, ctypes.byref(shape), lengths.data_ptr(), None, None, plan.data_ptr(), need)
    got = plan.cpu().numpy().astype(np.int64)
    assert (got[words:] == -7).all()
    # the segments: 128 rows each, the tiles of 64 keys that their last token sees, two places before each
    G, wgs = heads // kv_heads, 256 if D > 128 else 512
    last = length - T + 1 + (np.minimum(np.arange(0, T * G, 128) + 128, T * G) - 1) // G
    tiles = -(-last // 64)
    first = np.cumsum(tiles + 2) - tiles
    units = int((tiles + 2).sum())
    per = -(-units * kv_heads // wgs)
    assert got[:3].tolist() == [units, len(tiles), per] and (got[3:5] == 0).all()
    u = np.arange(wgs) * per
    u = u[u < units * kv_heads]
    at = u % units
    seg = np.searchsorted(first, at + 2, side="right") - 1
    starts = got[64 : 64 + 12 * wgs].reshape(wgs, 12)
    want = np.stack([seg, np.maximum(at - first[seg], 0), u // units, np.maximum(first[seg] - at, 0)], 1)
    np.testing.assert_array_equal(starts[: len(u), :4], want)
    np.testing.assert_array_equal(starts[: len(u), 9:11], np.stack([tiles[seg], first[seg]], 1))
    behind = 64 + (12 * wgs + 63) // 64 * 64
    assert (starts[len(u) :] == -7).all()
    assert (got[behind : behind + 12 * 4 * wgs] == -7).all()  # (no narrow segment: their starts stay)


def test_stretches_of_2_31_tiles_are_refused():
    # 512 segments of 65536 x 1 rows on 1024 key heads: more than 2^31 tiles for each of the 256 workgroups of wide heads
    lib = _vpaged.load()
    shape = lambda pages, D=256: ctypes.byref(_vpaged.VpagedShape(0, 1, 0, 65536, 1024, 1024, D, 4096, pages, 0))  # noqa: E731
    for D, least in ((256, 8192), (128, 16384)):
        # (pages * 4096 / 32 + 3 tiles of 512 segments and a head each)
        assert 512 * (least * 128 + 3) * 1024 >= (2**31 - 1) * (256 if D > 128 else 512) > 512 * ((least - 1) * 128 + 3) * 1024
        assert lib.vpaged_plan_bytes(shape(least, D)) == 0 < lib.vpaged_plan_bytes(shape(least - 1, D))


@pytest.mark.gpu
def test_a_plan_serves_layers_of_either_type():
    types = torch.bfloat16, torch.float16
    backends = [PAGED.resolve("hip", BackendContext(GPU, t)) for t in types]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=GPU)  # noqa: E731
    plans = [b.plan(i32([40, 7, 65]), queries=1, heads=4, kv_heads=2, head_dim=64, page_size=16, max_pages=5, prefix_lengths=i32([50]),
                    group_starts=i32([0, 3]), max_prefix_pages=4) for b in backends]
    tables, prefix_tables = i32(np.arange(15).reshape(3, 5)), i32([[15, 16, 17, 18]])
    for t, b, own in zip(types, backends, plans):
        q, k, v = (torch.randn(*s, device=GPU).to(t) for s in ((3, 1, 4, 64), (19, 16, 2, 64), (19, 16, 2, 64)))
        got = [b.attend(q, k, v, tables, p, prefix_tables=prefix_tables) for p in plans]
        assert torch.equal(got[0], got[1])
        with pytest.raises(ValueError, match="made for"):
            backends[t == types[0]].attend(q, k, v, tables, own, prefix_tables=prefix_tables)
