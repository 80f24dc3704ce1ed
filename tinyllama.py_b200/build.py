"""Build libtinyllama_b200.so, the C-ABI library of the sm_100a decode kernels.

Every ``csrc/*.cu`` file is compiled with nvcc for ``sm_100a`` only
(``-gencode arch=compute_100a,code=sm_100a``) as relocatable device code, then
linked into one shared library next to the ``cscr`` package, where the op
modules load it. The library lives in-tree, so a copy of the repository
carries it as built.

``csrc/fast_calls.cpp`` (host code on torch's C++ headers) becomes the module
``cscr._fast`` beside it.

Usage: ``python tinyllama.py_b200/build.py [--force] [--verbose]``.
"""

from __future__ import annotations

import argparse
import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG_ROOT = Path(__file__).resolve().parent
CSRC = PKG_ROOT / "csrc"
INCLUDE = PKG_ROOT.parent / "include"
BUILD_DIR = PKG_ROOT.parent / "_build"
LIB_PATH = PKG_ROOT / "cscr" / "libtinyllama_b200.so"
FAST_SRC = CSRC / "fast_calls.cpp"
FAST_PATH = PKG_ROOT / "cscr" / f"_fast{sysconfig.get_config_var('EXT_SUFFIX')}"

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = [
    "-O3",
    "-lineinfo",
    "--use_fast_math",
    "-std=c++17",
    "-rdc=true",
    "-Xcompiler",
    "-fPIC,-O3,-fvisibility=hidden",
    "--expt-relaxed-constexpr",
]


def nvcc() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists():
        raise RuntimeError("nvcc not found: the CUDA toolkit is required to build")
    return cand


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def _deps() -> list[Path]:
    return sources() + sorted(CSRC.glob("*.h")) + sorted(CSRC.glob("*.cuh")) + sorted(
        INCLUDE.glob("*.h")
    )


def up_to_date() -> bool:
    return _lib_up_to_date() and _fast_up_to_date()


def _lib_up_to_date() -> bool:
    if not LIB_PATH.exists():
        return False
    built = LIB_PATH.stat().st_mtime
    return all(p.stat().st_mtime <= built for p in _deps())


def _torch_version() -> str:
    import torch

    return str(torch.__version__)


def _fast_up_to_date() -> bool:
    deps = [FAST_SRC, *INCLUDE.glob("*.h")]
    if not FAST_PATH.exists() or any(
            p.stat().st_mtime > FAST_PATH.stat().st_mtime for p in deps):
        return False
    # the module names the torch it was compiled against (its torch_version)
    return _torch_version().encode() + b"\0" in FAST_PATH.read_bytes()


def _build_fast() -> None:
    """Compile cscr._fast against the running interpreter and its torch. The ops run
    without it: a failure is a warning, and leaves no older module behind."""
    try:
        _compile_fast()
    except Exception as exc:  # noqa: BLE001 - whatever kept it from being built
        FAST_PATH.unlink(missing_ok=True)
        print(f"warning: cscr._fast is not built, calls take longer on the host: {exc}",
              file=sys.stderr)


def _compile_fast() -> None:
    import torch
    from torch.utils import cpp_extension

    cuda = Path(nvcc()).resolve().parent.parent
    lib = Path(torch.__file__).resolve().parent / "lib"
    tmp = FAST_PATH.with_suffix(".tmp")
    cmd = [shutil.which("g++") or "c++", "-O2", "-std=c++17", "-shared", "-fPIC",
           "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           *(f"-isystem{p}" for p in cpp_extension.include_paths()),
           f"-isystem{sysconfig.get_paths()['include']}", f"-isystem{cuda / 'include'}",
           f"-I{INCLUDE}", f'-DTLB_TORCH_VERSION="{_torch_version()}"', str(FAST_SRC), "-o",
           str(tmp), f"-L{lib}", "-ltorch_python", "-ltorch", "-ltorch_cpu",
           "-ltorch_cuda", "-lc10", "-lc10_cuda"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"compiling {FAST_SRC.name} failed:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, FAST_PATH)


def _compile(src: Path, verbose: bool) -> Path:
    obj = BUILD_DIR / (src.stem + ".o")
    cmd = [nvcc(), *ARCH_FLAGS, *NVCC_FLAGS, "-I", str(INCLUDE), "-dc", str(src), "-o", str(obj)]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src.name}:\n{res.stdout}\n{res.stderr}")
    if verbose and (res.stdout or res.stderr):
        print(res.stdout + res.stderr, file=sys.stderr)
    return obj


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile the kernels and link the shared library; returns its path."""
    stale = force or not _lib_up_to_date()
    BUILD_DIR.mkdir(parents=True, exist_ok=True)
    srcs = sources() if stale else []
    workers = min(len(srcs) + 1, os.cpu_count() or 4)
    with cf.ThreadPoolExecutor(max_workers=workers) as ex:
        fast = ex.submit(_build_fast) if force or not _fast_up_to_date() else None
        objs = list(ex.map(lambda s: _compile(s, verbose), srcs))
        if fast is not None:
            fast.result()
    if not stale:
        return LIB_PATH
    tmp = LIB_PATH.with_suffix(".so.tmp")
    cmd = [nvcc(), *ARCH_FLAGS, "-shared", "-o", str(tmp), *map(str, objs), "-cudart", "static"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true", help="print ptxas resource usage")
    args = ap.parse_args()
    print(build(force=args.force, verbose=args.verbose))


if __name__ == "__main__":
    main()
