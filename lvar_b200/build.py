"""In-tree build of ``liblvar_b200.so`` (sm_100a only) with plain nvcc.

``python -m lvar_b200.build`` compiles every ``csrc/*.cu`` to an object file and links them into
``lvar_b200/liblvar_b200.so``, and ``csrc/paged_host.cpp`` (the Python entry of the paged-cache calls, over the same
library and torch's headers) into ``lvar_b200/_paged_host.so``.  Objects are rebuilt only when a source or header is
newer, the module also for another torch or Python.  nvcc cross-compiles for sm_100a, so this also runs on a machine
without a GPU.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
CSRC = PKG_DIR / "csrc"
INCLUDE = PKG_DIR.parent / "include"
BUILD_DIR = PKG_DIR / "build"
LIB_PATH = PKG_DIR / "liblvar_b200.so"
HOST_PATH = PKG_DIR / "_paged_host.so"

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "-Xptxas", "-v",
]


def _nvcc() -> str:
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(exe):
        raise RuntimeError("nvcc not found: the sm_100a kernels cannot be built")
    return exe


def _stale(target: Path, deps: list[Path]) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(d.stat().st_mtime > t for d in deps)


def host_key() -> str:
    """What the compiled entry of the paged-cache calls is made for: it uses torch's C++ classes and CPython's."""
    import torch
    return f"torch {torch.__version__}, {sysconfig.get_config_var('SOABI')}, abi {int(torch._C._GLIBCXX_USE_CXX11_ABI)}"


def _build_host(force: bool) -> None:
    """The C++ entry of the paged-cache calls: a CPython module that links the library beside it and torch.  Built again when
    a source is newer or when torch or Python is another one than it was made for."""
    src, made_for, key = CSRC / "paged_host.cpp", BUILD_DIR / "paged_host.key", host_key()
    if not force and made_for.exists() and made_for.read_text() == key and not _stale(HOST_PATH, [src, INCLUDE / "lvar_b200.h"]):
        return
    import torch
    root = Path(torch.__file__).resolve().parent
    cuda = Path(os.environ.get("CUDA_HOME", Path(_nvcc()).resolve().parent.parent))
    cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-shared", "-fPIC",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f'-DLVAR_BUILT_FOR="{key}"',
           "-isystem", str(root / "include"), "-isystem", str(root / "include" / "torch" / "csrc" / "api" / "include"),
           "-isystem", str(cuda / "include"), "-isystem", sysconfig.get_paths()["include"], str(src), "-o", str(HOST_PATH),
           "-L", str(PKG_DIR), "-l:liblvar_b200.so", "-Wl,-rpath,$ORIGIN",
           "-L", str(root / "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed on {src.name}:\n{res.stdout}\n{res.stderr}")
    made_for.write_text(key)


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile and link the library; returns its path.  Raises on any compiler error."""
    BUILD_DIR.mkdir(exist_ok=True)
    sources = sorted(CSRC.glob("*.cu"))
    headers = sorted(CSRC.glob("*.cuh")) + sorted(INCLUDE.glob("*.h"))
    nvcc = _nvcc()
    logs = []

    def compile_one(src: Path) -> Path:
        obj = BUILD_DIR / (src.stem + ".o")
        if force or _stale(obj, [src] + headers):
            cmd = [nvcc, *NVCC_FLAGS, "-I", str(INCLUDE), "-c", str(src), "-o", str(obj)]
            res = subprocess.run(cmd, capture_output=True, text=True)
            logs.append((src.name, res.stderr))
            if res.returncode != 0:
                raise RuntimeError(f"nvcc failed on {src.name}:\n{res.stdout}\n{res.stderr}")
        return obj

    with ThreadPoolExecutor(max_workers=min(8, max(1, len(sources)))) as ex:
        objs = list(ex.map(compile_one, sources))

    if force or _stale(LIB_PATH, objs):
        cmd = [nvcc, "-shared", "-o", str(LIB_PATH), *map(str, objs)]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    _build_host(force)
    if verbose:
        for name, log in logs:
            keep = [ln for ln in log.splitlines() if "registers" in ln or "spill" in ln or "warning" in ln]
            print(f"== {name}\n" + "\n".join(keep))
    (BUILD_DIR / "ptxas.log").write_text("\n".join(f"== {n}\n{l}" for n, l in logs))
    return LIB_PATH


if __name__ == "__main__":
    path = build(force="--force" in sys.argv, verbose=True)
    print(path)
