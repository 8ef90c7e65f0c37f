"""Build liblara_b200.so in-tree with nvcc for sm_100a, and its Python binding.

``python -m lara_b200.build [--verbose]`` compiles every ``csrc/*.cu`` to an
object with ``-gencode arch=compute_100a,code=sm_100a -lineinfo -O3`` and
links them into ``lara_b200/liblara_b200.so`` (cudart linked statically, so
the library does not depend on which ``libcudart`` a host process has
loaded).  Objects go to ``lara_b200/_build``; a source newer than the library
triggers a rebuild.  After it ``csrc/binding.cpp``, the binding of the calls made
once per layer and token, is compiled with g++ against the installed torch into
``lara_b200/_binding.<Python's tag>.so``, again whenever torch is another one;
without what it needs (a torch with CUDA, g++, Python's headers) it is left out,
and the library alone is built.
"""

from __future__ import annotations

import argparse
import concurrent.futures as cf
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
INCLUDE = PKG.parent / "include"
BUILD = PKG / "_build"
LIB = PKG / "liblara_b200.so"
BINDING = PKG / ("_binding" + sysconfig.get_config_var("EXT_SUFFIX"))  # one Python's: another does not find it

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMMON_FLAGS = ["-O3", "-lineinfo", "-std=c++17", "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC",
                "-Xcompiler", "-fvisibility=hidden", "-I", str(INCLUDE), "-I", str(CSRC)]


def nvcc() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists():
        raise RuntimeError("nvcc not found: the CUDA toolkit is required to build liblara_b200.so")
    return cand


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def headers() -> list[Path]:
    return sorted(list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h")) + list(CSRC.glob("*.inc")) +
                  list(INCLUDE.glob("*.h")))


def needs_build() -> bool:
    if not LIB.exists():
        return True
    t = LIB.stat().st_mtime
    return any(p.stat().st_mtime > t for p in sources() + headers() + [Path(__file__)])


def _torch_include() -> Path | None:
    spec = importlib.util.find_spec("torch")
    return Path(spec.origin).parent / "include" if spec and spec.origin else None


def binding_lacks() -> str | None:
    """What the Python binding needs and this machine has not, or None."""
    inc = _torch_include()
    if inc is None:
        return "torch is not installed"
    if not (inc.parent / "lib" / "libc10_cuda.so").exists():
        return "the installed torch has no CUDA"
    if shutil.which("g++") is None:
        return "g++ was not found"
    if not (Path(sysconfig.get_paths()["include"]) / "Python.h").exists():
        return "Python's headers are not installed"
    return None


def build_binding(force: bool = False) -> Path | None:
    """Compile the Python binding; returns its path, or None where something for it is lacking."""
    lacks = binding_lacks()
    if lacks:
        sys.stderr.write(f"lara_b200: {BINDING.name} is left out: {lacks}\n")
        return None
    src, inc = CSRC / "binding.cpp", _torch_include()
    newest = max(p.stat().st_mtime for p in (src, INCLUDE / "lara_b200.h", Path(__file__)))
    stamp, torch_is = BUILD / "binding.torch", (inc.parent / "version.py").read_text()
    same_torch = stamp.exists() and stamp.read_text() == torch_is
    if not force and BINDING.exists() and BINDING.stat().st_mtime > newest and same_torch:
        return BINDING
    cuda = Path(nvcc()).resolve().parents[1] / "include"
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-shared", "-I", str(inc), "-I",
           str(inc / "torch" / "csrc" / "api" / "include"), "-I", sysconfig.get_paths()["include"], "-I", str(cuda)]
    tmp = BINDING.with_name(BINDING.name + ".tmp")
    libs = ["-L", str(inc.parent / "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    res = subprocess.run([*cmd, str(src), "-o", str(tmp), *libs], capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed on {src.name}:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, BINDING)
    BUILD.mkdir(exist_ok=True)
    stamp.write_text(torch_is)
    return BINDING


def _compile(src: Path, verbose: bool) -> Path:
    obj = BUILD / (src.stem + ".o")
    cmd = [nvcc(), *ARCH_FLAGS, *COMMON_FLAGS, "-c", str(src), "-o", str(obj)]
    if verbose:
        cmd += ["-Xptxas", "-v"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src.name}:\n{res.stdout}\n{res.stderr}")
    if verbose and res.stderr:
        sys.stderr.write(res.stderr)
    return obj


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile and link the library and its Python binding; returns the library's path."""
    build_library(force, verbose)
    build_binding(force)
    return LIB


def build_library(force: bool = False, verbose: bool = False) -> Path:
    """Compile and link the library; returns its path."""
    if not force and not needs_build():
        return LIB
    BUILD.mkdir(exist_ok=True)
    srcs = sources()
    with cf.ThreadPoolExecutor(max_workers=min(len(srcs), os.cpu_count() or 4)) as ex:
        objs = list(ex.map(lambda s: _compile(s, verbose), srcs))
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [nvcc(), *ARCH_FLAGS, "-shared", "-cudart", "static", "-o", str(tmp), *map(str, objs)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, LIB)
    return LIB


def main() -> int:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true", help="print ptxas register/smem usage")
    args = ap.parse_args()
    print(build(force=args.force, verbose=args.verbose))
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
