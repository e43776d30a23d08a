"""In-tree build of the CUDA library (sm_100a) -- no JIT cache, the .so sits next to the
package so it travels with the source tree."""
from __future__ import annotations

import os
import shutil
import subprocess
import tempfile
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libbitdance_b200.so")
SOURCES = [os.path.join(CSRC, f) for f in ("bitdance.cu", "fp4.cu", "moe.cu")]
HEADERS = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-lineinfo", "-std=c++17",
              "-Xcompiler", "-fPIC", "-shared"]


def nvcc() -> str:
    for c in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if c and os.path.exists(c):
            return c
    raise RuntimeError("nvcc not found")


def _newest_header() -> float:
    inc = os.path.join(os.path.dirname(HERE), "include", "bitdance_b200.h")
    return max(os.path.getmtime(f) for f in HEADERS + [inc])


def stale() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    return _newest_header() > t or any(os.path.getmtime(f) > t for f in SOURCES)


def _run(cmd) -> str:
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed:\n{r.stdout}\n{r.stderr}")
    return r.stderr


def build_library(force: bool = False, verbose: bool = False) -> str:
    if force or stale():
        flags = [f for f in NVCC_FLAGS if f != "-shared"] + (["-Xptxas=-v"] if verbose else [])
        # objects and the new library beside no one else's: processes may build at the same time, and
        # one may have the old library open
        with tempfile.TemporaryDirectory() as tmp:
            objs = [os.path.join(tmp, os.path.basename(f)[:-3] + ".o") for f in SOURCES]
            with ThreadPoolExecutor(len(SOURCES)) as pool:  # one nvcc per source
                logs = list(pool.map(lambda so: _run([nvcc(), *flags, "-c", "-o", so[1], so[0]]),
                                     zip(SOURCES, objs)))
            new = f"{LIB[:-3]}.{os.getpid()}.so"
            _run([nvcc(), *NVCC_FLAGS, "-o", new, *objs])
            os.replace(new, LIB)
        if verbose:
            print("".join(logs))
    return LIB
