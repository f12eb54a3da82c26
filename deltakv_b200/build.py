"""Build libdkv_b200.so (sm_100a) in-tree with nvcc, and the extension module _step.so with g++.

Each ``csrc/*.cu`` is compiled to an object under ``deltakv_b200/_build`` (skipped when
it is newer than its source and every header), then linked into
``deltakv_b200/libdkv_b200.so``.  ``csrc/step_binding.cpp`` (host side of the paged step
operators, against the installed torch and Python) becomes ``deltakv_b200/_step.so``.  ``python -m deltakv_b200.build`` rebuilds; ``--ptxas``
prints register / spill / shared-memory usage per kernel.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
BUILD = PKG / "_build"
LIB = PKG / "libdkv_b200.so"
STEP_SRC, STEP = CSRC / "step_binding.cpp", PKG / "_step.so"
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found: set NVCC or put the CUDA toolkit on PATH")


def _headers() -> list[Path]:
    return sorted(CSRC.glob("*.cuh")) + sorted((ROOT / "include").glob("*.h"))


def _flags() -> list[str]:
    return [
        *ARCH,
        "-O3",
        "-lineinfo",
        "-std=c++17",
        "-Xcompiler",
        "-fPIC",
        "-I",
        str(ROOT / "include"),
        "--expt-relaxed-constexpr",
    ]


def _compile(src: Path, ptxas: bool) -> tuple[Path, str]:
    obj = BUILD / (src.stem + ".o")
    newest_dep = max([src.stat().st_mtime] + [h.stat().st_mtime for h in _headers()])
    if not ptxas and obj.exists() and obj.stat().st_mtime >= newest_dep:
        return obj, ""
    cmd = [_nvcc(), *_flags(), "-c", str(src), "-o", str(obj)]
    if ptxas:
        cmd += ["-Xptxas", "-v"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src.name}:\n{res.stdout}\n{res.stderr}")
    return obj, res.stderr


def _step_stamp() -> str:
    import torch

    return f"{sys.version} torch {torch.__version__}"


def build_step() -> Path | None:
    """The extension module; rebuilt when its source, the C header, Python or torch changed.

    Against a torch without CUDA there is nothing to build it with (and no GPU tensor to call it on): None."""
    import torch

    if torch.version.cuda is None:
        print(f"{STEP.name} not built: torch {torch.__version__} has no CUDA", file=sys.stderr)
        return None
    stamp = BUILD / "step.stamp"
    newest = max(STEP_SRC.stat().st_mtime, *(h.stat().st_mtime for h in (ROOT / "include").glob("*.h")))
    if STEP.exists() and STEP.stat().st_mtime >= newest and stamp.exists() and stamp.read_text() == _step_stamp():
        return STEP
    root = Path(torch.__file__).resolve().parent
    cuda = Path(_nvcc()).resolve().parent.parent
    tmp = STEP.with_suffix(".so.tmp")
    # the system's g++, whose libstdc++ is the one that torch loads
    cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-shared", "-fPIC",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           "-I", sysconfig.get_paths()["include"], "-isystem", str(root / "include"),
           "-isystem", str(root / "include/torch/csrc/api/include"), "-isystem", str(cuda / "include"),
           str(STEP_SRC), "-o", str(tmp), "-L", str(root / "lib"),
           "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch", "-ltorch_python"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed for {STEP_SRC.name}:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, STEP)
    stamp.write_text(_step_stamp())
    return STEP


def build(ptxas: bool = False, verbose: bool = False) -> Path:
    """Both; the library does not depend on torch, so it is linked even where the module's build raises."""
    BUILD.mkdir(exist_ok=True)
    srcs = sorted(CSRC.glob("*.cu"))
    with ThreadPoolExecutor(max_workers=min(8, len(srcs) + 1)) as ex:
        step = ex.submit(build_step)
        results = list(ex.map(lambda s: _compile(s, ptxas), srcs))
        out = _link(results, ptxas, verbose)
        step.result()
    return out


def _link(results: list[tuple[Path, str]], ptxas: bool, verbose: bool) -> Path:
    if ptxas or verbose:
        for _, log in results:
            if log:
                print(log, file=sys.stderr)
    objs = [o for o, _ in results]
    newest = max(o.stat().st_mtime for o in objs)
    if LIB.exists() and LIB.stat().st_mtime >= newest and not ptxas:
        return LIB
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [_nvcc(), *ARCH, "-shared", "-o", str(tmp), *map(str, objs)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    out = build(ptxas="--ptxas" in sys.argv, verbose=True)
    print(out)
