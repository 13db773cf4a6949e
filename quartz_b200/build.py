"""Build the sm_100a shared library ``quartz_b200/libquartz_b200.so`` in-tree.

    python -m quartz_b200.build

nvcc cross-compiles for sm_100a on a host without a GPU. The library exports
the C ABI declared in include/quartz_b200.h. ``quartz_b200/_fastcall.so``, a
CPython extension over the same entry points (csrc/fastcall.cpp), is built with
the host compiler against the installed torch; without it the calls take their
checked way through Python, so a failure to build it is a warning. It reads
tensors by the layout of one torch's headers: a stamp in it names that torch and
Python, and one of another is neither kept by build() nor loaded.
"""

from __future__ import annotations

import os
import re
import shutil
import subprocess
import sys
import warnings
from pathlib import Path

PKG = Path(__file__).resolve().parent
REPO = PKG.parent
SRC = PKG / "csrc"
OUT = PKG / "libquartz_b200.so"

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "-shared",
    "--expt-relaxed-constexpr",
]


def nvcc() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found")
    return cand


FAST_SRC = SRC / "fastcall.cpp"
FAST_OUT = PKG / "_fastcall.so"


def fast_tag() -> str:
    """The torch and the Python that a _fastcall.so has to be built for."""
    import sysconfig

    import torch

    return (f"torch={torch.__version__};python={sysconfig.get_config_var('SOABI')};"
            f"cxx11={int(torch._C._GLIBCXX_USE_CXX11_ABI)}")


def fast_stamp(path: Path = FAST_OUT) -> str:
    """The stamp of a built _fastcall.so ("" without one that can be read)."""
    import ctypes

    try:
        return ctypes.c_char_p(ctypes.addressof(
            ctypes.c_char.in_dll(ctypes.CDLL(str(path)), "qz_fastcall_stamp"))).value.decode()
    except (OSError, ValueError):
        return ""


def fast_up_to_date() -> bool:
    header = REPO / "include" / "quartz_b200.h"
    return (FAST_OUT.exists()
            and all(p.stat().st_mtime <= FAST_OUT.stat().st_mtime for p in (FAST_SRC, header, Path(__file__)))
            and fast_stamp() == fast_tag())


def build_fastcall(force: bool = False) -> Path:
    """The extension module quartz_b200._fastcall."""
    import sysconfig

    import torch

    if not force and fast_up_to_date():
        return FAST_OUT
    root = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc()).resolve().parent.parent
    inc = [root / "include", root / "include" / "torch" / "csrc" / "api" / "include",
           cuda / "include", REPO / "include", sysconfig.get_paths()["include"]]
    lib = root / "lib"
    cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f'-DQZ_FASTCALL_STAMP="{fast_tag()}"',
           *[f"-I{p}" for p in inc], str(FAST_SRC), "-o", str(FAST_OUT), f"-L{lib}",
           f"-L{cuda / 'lib64'}", "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10_cuda", "-lc10",
           "-lcudart", f"-Wl,-rpath,{lib}"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise subprocess.CalledProcessError(r.returncode, cmd)
    return FAST_OUT


def sources() -> list[Path]:
    return sorted(SRC.glob("*.cu")) + sorted(SRC.glob("*.cuh")) + [REPO / "include" / "quartz_b200.h"]


def up_to_date() -> bool:
    if not OUT.exists():
        return False
    t = OUT.stat().st_mtime
    return all(p.stat().st_mtime <= t for p in sources())


RESOURCES = PKG / "libquartz_b200.resources.txt"


def parse_ptxas(log: str) -> dict[str, dict]:
    """Per kernel: registers, static shared memory bytes, spill bytes (from
    ptxas -v)."""
    out: dict[str, dict] = {}
    cur = None
    for line in log.splitlines():
        m = re.search(r"Compiling entry function '([^']+)'", line)
        if m:
            cur = m.group(1)
            out[cur] = {"registers": 0, "smem": 0, "spill": 0}
            continue
        if cur is None:
            continue
        m = re.search(r"(\d+) bytes spill stores", line)
        if m:
            out[cur]["spill"] = int(m.group(1))
        m = re.search(r"Used (\d+) registers", line)
        if m:
            out[cur]["registers"] = int(m.group(1))
            m2 = re.search(r"(\d+) bytes smem", line)
            out[cur]["smem"] = int(m2.group(1)) if m2 else 0
    return out


def build(force: bool = False, verbose: bool = False) -> Path:
    build_library(force, verbose)
    try:
        build_fastcall(force)
    except (OSError, ImportError, RuntimeError, subprocess.CalledProcessError) as e:
        warnings.warn(f"{FAST_OUT.name} is not built, paged-cache calls take longer: {e}",
                      RuntimeWarning, stacklevel=2)
    return OUT


def build_library(force: bool = False, verbose: bool = False) -> Path:
    """libquartz_b200.so."""
    if not force and up_to_date():
        return OUT
    cmd = [nvcc(), "-Xptxas=-v", *NVCC_FLAGS, f"-I{REPO / 'include'}", f"-I{SRC}",
           "-o", str(OUT), str(SRC / "qz_api.cu")]
    if verbose:
        print(" ".join(cmd))
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise subprocess.CalledProcessError(r.returncode, cmd)
    if verbose:
        sys.stderr.write(r.stderr)
    res = parse_ptxas(r.stderr)
    RESOURCES.write_text("".join(f"{k} registers={v['registers']} smem={v['smem']} "
                                 f"spill={v['spill']}\n" for k, v in sorted(res.items())))
    return OUT


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(OUT)
