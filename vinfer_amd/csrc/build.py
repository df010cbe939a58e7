"""Compile the HIP sources (gfx950 only): the sampler into ``vinfer_amd/libvsampler.so``, the operators
around it into ``vinfer_amd/libvops.so``, the paged cache into ``vinfer_amd/libvpaged.so``.

Run as ``python -m vinfer_amd.csrc.build``. The build is in-tree so the library travels with
the source tree; there is no JIT cache.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parents[1]
ROOT = PKG.parent
LIB = PKG / "libvsampler.so"
SOURCES = [PKG / "csrc" / "capi.hip"]
OPS_LIB = PKG / "libvops.so"
OPS_SOURCES = [PKG / "csrc" / "vops.hip"]
PAGED_LIB = PKG / "libvpaged.so"
PAGED_SOURCES = [PKG / "csrc" / "vpaged.hip"]

# -ffp-contract=off: the penalty arithmetic rounds every operation on its own.
# -fhip-fp32-correctly-rounded-divide-sqrt: x / T is IEEE division, as on the CPU.
# -packed-fp32-ops is disabled for every kernel (no v_pk_*_f32 code).
FLAGS = [
    "--offload-arch=gfx950",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-shared",
    "-ffp-contract=off",
    "-fhip-fp32-correctly-rounded-divide-sqrt",
    "-Xclang",
    "-target-feature",
    "-Xclang",
    "-packed-fp32-ops",
    "-Wno-unused-command-line-argument",
]
# The operators keep rows in registers across loops: constants that were kept in registers beside them would not fit
# (the compiler moves each one's load out of the loop, fp64 polynomials' coefficients above all).
OPS_FLAGS = [*FLAGS, "-mllvm", "-disable-machine-licm"]
# The paged cache's products and sums are held in fp32 with one rounding fewer where the compiler fuses them.
PAGED_FLAGS = [f for f in FLAGS if f != "-ffp-contract=off"]


def hipcc() -> str:
    for c in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if c and Path(c).exists():
            return c
    raise RuntimeError("hipcc not found (ROCm is required to build the libraries)")


def _compile(lib: Path, sources: list[Path], flags: list[str], verbose: bool) -> None:
    tmp = lib.with_suffix(".so.tmp")
    cmd = [hipcc(), *flags, f"-I{ROOT / 'include'}", "-o", str(tmp), *map(str, sources)]
    if verbose:
        print(" ".join(cmd), flush=True)
    proc = subprocess.run(cmd, capture_output=True, text=True)
    out = "\n".join(
        line
        for line in (proc.stdout + proc.stderr).splitlines()
        if "packed-fp32-ops" not in line  # the host pass does not know the feature: harmless
    )
    if proc.returncode != 0:
        raise RuntimeError(f"hipcc failed ({proc.returncode}):\n{out}")
    if verbose and out.strip():
        print(out)
    os.replace(tmp, lib)


def build(verbose: bool = False) -> Path:
    libraries = (LIB, SOURCES, FLAGS), (OPS_LIB, OPS_SOURCES, OPS_FLAGS), (PAGED_LIB, PAGED_SOURCES, PAGED_FLAGS)
    with ThreadPoolExecutor(3) as pool:
        jobs = [pool.submit(_compile, *job, verbose) for job in libraries]
    for job in jobs:
        job.result()
    return LIB


if __name__ == "__main__":
    build(verbose="-v" in sys.argv)
    print(LIB)
    print(OPS_LIB)
    print(PAGED_LIB)
