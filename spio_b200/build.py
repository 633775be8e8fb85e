"""Build libspio_b200.so (the C-ABI library with the sm_100a kernels) in-tree with nvcc, and
libspio_b200_torch.so (PyTorch operators on top of it, see csrc/torch_ops.cpp) with the host compiler.

Run as ``python -m spio_b200.build`` or call :func:`build`.  nvcc cross-compiles for
sm_100a, so no GPU is needed to build.  Plays the role of the reference's Cython build
of its driver shim (setup.py:27-51); the kernels themselves were JIT-only there.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path
from typing import Optional

from ._clib import TORCH_LIB_PATH, TORCH_STAMP_PATH, torch_stamp

PKG_DIR = Path(__file__).resolve().parent
CSRC = PKG_DIR / "csrc"
LIB_DIR = PKG_DIR / "lib"
OBJ_DIR = PKG_DIR / "lib" / "obj"
LIB_PATH = LIB_DIR / "libspio_b200.so"
TORCH_SOURCE = CSRC / "torch_ops.cpp"

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMMON_FLAGS = ["-std=c++17", "-O3", "-lineinfo", "-Xcompiler", "-fPIC", "-diag-suppress", "177"]


def find_nvcc() -> str:
    """Locate nvcc: $CUDA_HOME, then PATH, then /usr/local/cuda."""
    cands = []
    if os.environ.get("CUDA_HOME"):
        cands.append(Path(os.environ["CUDA_HOME"]) / "bin" / "nvcc")
    which = shutil.which("nvcc")
    if which:
        cands.append(Path(which))
    cands.append(Path("/usr/local/cuda/bin/nvcc"))
    for c in cands:
        if c.exists():
            return str(c)
    raise RuntimeError("nvcc not found; set CUDA_HOME")


def _sources():
    """(source, object, extra flags) for every translation unit."""
    units = [(CSRC / "gw8_capi.cu", OBJ_DIR / "gw8_capi.o", [])]
    for r in range(1, 6):
        units.append((CSRC / "gw8_inst.cu", OBJ_DIR / f"gw8_inst_r{r}.o", [f"-DGW8_R={r}"]))
    units.append((CSRC / "gw8_tc_inst.cu", OBJ_DIR / "gw8_tc_inst.o", []))
    units.append((CSRC / "jit_driver.cpp", OBJ_DIR / "jit_driver.o", []))
    units.append((CSRC / "layernorm_2d.cu", OBJ_DIR / "layernorm_2d.o", []))
    units.append((CSRC / "dp_exchange.cu", OBJ_DIR / "dp_exchange.o", []))
    for data_type in range(3):
        for threads in (128, 256):
            units.append((CSRC / "groupnorm_2d_inst.cu", OBJ_DIR / f"groupnorm_2d_{data_type}_{threads}.o",
                          [f"-DGN_TYPE={data_type}", f"-DGN_THREADS={threads}"]))
    units.append((CSRC / "groupnorm_2d.cu", OBJ_DIR / "groupnorm_2d.o", []))
    units.append((CSRC / "checkpoint8.cu", OBJ_DIR / "checkpoint8.o", []))
    return units


def _newest_input() -> float:
    deps = list(CSRC.glob("*.cu")) + list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h"))
    deps += [p for p in CSRC.glob("*.cpp") if p != TORCH_SOURCE] + [PKG_DIR.parent / "include" / "spio_b200.h"]
    return max(p.stat().st_mtime for p in deps if p.exists())


def is_current() -> bool:
    """True when the library exists and is newer than every source."""
    return LIB_PATH.exists() and LIB_PATH.stat().st_mtime >= _newest_input()


def torch_lib_is_current() -> bool:
    """Whether it is newer than what it is made from, and made for the installed torch."""
    header = PKG_DIR.parent / "include" / "spio_b200.h"
    newest = max(p.stat().st_mtime for p in (TORCH_SOURCE, header))
    return (TORCH_LIB_PATH.exists() and TORCH_LIB_PATH.stat().st_mtime >= newest
            and TORCH_STAMP_PATH.exists() and TORCH_STAMP_PATH.read_text().strip() == torch_stamp())


def _run(cmd, verbose):
    if verbose:
        print(" ".join(map(str, cmd)), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"command failed: {' '.join(map(str, cmd))}\n{res.stdout}\n{res.stderr}")
    return res.stdout + res.stderr


def build_torch_lib(force: bool = False, verbose: bool = False) -> Optional[Path]:
    """Compile the operators implemented in C++ against the installed torch; they call libspio_b200, which lies
    beside them.  Without a torch that has CUDA libraries there is nothing to link them with: the C-ABI library is
    then all that is built, and the operators' calls say that theirs is missing."""
    try:
        import torch
    except ImportError:
        torch = None
    if torch is None or torch.version.cuda is None:
        print("torch with CUDA is not installed: the PyTorch operators in C++ are not built", file=sys.stderr)
        return None
    if not force and torch_lib_is_current():
        return TORCH_LIB_PATH
    root = Path(torch.__file__).resolve().parent
    cuda = Path(find_nvcc()).resolve().parent.parent
    _run([os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-w",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
          f"-I{root / 'include'}", f"-I{root / 'include' / 'torch' / 'csrc' / 'api' / 'include'}",
          f"-I{cuda / 'include'}", str(TORCH_SOURCE), "-o", str(TORCH_LIB_PATH),
          f"-L{LIB_DIR}", "-lspio_b200", "-Wl,-rpath,$ORIGIN",
          f"-L{root / 'lib'}", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch"], verbose)
    TORCH_STAMP_PATH.write_text(torch_stamp() + "\n")
    return TORCH_LIB_PATH


def build(force: bool = False, verbose: bool = False, ptxas_info: bool = False) -> Path:
    """Compile every translation unit (in parallel) and link the shared libraries; returns the C-ABI library."""
    if force or not is_current():
        nvcc = find_nvcc()
        OBJ_DIR.mkdir(parents=True, exist_ok=True)
        flags = ARCH_FLAGS + COMMON_FLAGS + (["-Xptxas", "-v"] if ptxas_info else [])

        def compile_one(unit):
            src, obj, extra = unit
            return _run([nvcc, *flags, *extra, "-c", str(src), "-o", str(obj)], verbose)

        units = _sources()
        with ThreadPoolExecutor(max_workers=min(len(units), os.cpu_count() or 2)) as ex:
            logs = list(ex.map(compile_one, units))
        if ptxas_info:
            print("\n".join(logs))
        objs = [str(obj) for _, obj, _ in units]
        _run([nvcc, *ARCH_FLAGS, "-shared", "-o", str(LIB_PATH), *objs, "-ldl"], verbose)
    build_torch_lib(force, verbose)
    return LIB_PATH


if __name__ == "__main__":
    path = build(force="--force" in sys.argv, verbose=True, ptxas_info="--ptxas-info" in sys.argv)
    print(path)
