"""Build ``libfqkv_b200.so`` in-tree with nvcc for sm_100a.

    python "fused-quantized-kv-decode-attention_b200/build.py" [--force] [--verbose]

Each ``csrc/*.cu`` is compiled to an object in ``_build/`` (in parallel), then
linked into ``libfqkv_b200.so`` next to this file with the CUDA runtime linked
statically, so the library depends only on the NVIDIA driver.  ``-Xptxas -v``
register / spill / shared-memory reports are written to
``_build/ptxas_<name>.log``.  ``csrc/torch_binding.cpp`` becomes the extension
module ``_torch_binding.so`` (g++, the installed torch's headers); without
torch it is left out, and the library alone is built for users of the C entry
points.  Rebuilds only what a source or header is newer than (or all, with
``--force``).
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import os
import pathlib
import shutil
import subprocess
import sys
import sysconfig

HERE = pathlib.Path(__file__).resolve().parent
CSRC = HERE / "csrc"
INCLUDE = HERE.parent / "include"
BUILD = HERE / "_build"
LIB = HERE / "libfqkv_b200.so"
BINDING = HERE / "_torch_binding.so"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ARCH + [
    "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-O3",
    "--expt-relaxed-constexpr", "-Xptxas", "-v", f"-I{INCLUDE}", f"-I{CSRC}",
]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and pathlib.Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found; set NVCC or put the CUDA toolkit on PATH")


def sources() -> list[pathlib.Path]:
    return sorted(CSRC.glob("*.cu"))


def _stale(target: pathlib.Path, deps: list[pathlib.Path]) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(p.stat().st_mtime > t for p in [*deps, *INCLUDE.glob("*.h"), pathlib.Path(__file__)])


def _compile(src: pathlib.Path, verbose: bool) -> pathlib.Path:
    obj = BUILD / (src.stem + ".o")
    cmd = [nvcc(), *NVCC_FLAGS, "-c", str(src), "-o", str(obj)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    (BUILD / f"ptxas_{src.stem}.log").write_text(r.stdout + r.stderr)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src.name}:\n{r.stderr[-6000:]}")
    if verbose:
        print(f"compiled {src.name}")
    return obj


def _build_binding(verbose: bool) -> None:
    """The Python layer of the paged-cache operators, against the torch of this interpreter (if there is one)."""
    try:
        import torch
    except ImportError as exc:
        print(f"not built: {BINDING.name}, the Python calls of the paged cache ({exc})", file=sys.stderr)
        return

    root = pathlib.Path(torch.__file__).resolve().parent
    cuda = pathlib.Path(nvcc()).resolve().parents[1] / "include"
    tmp = BINDING.with_suffix(".so.tmp")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f'-DBUILT_FOR_TORCH="{torch.__version__}"', f"-I{INCLUDE}",
           "-isystem", sysconfig.get_paths()["include"], "-isystem", str(root / "include"),
           "-isystem", str(root / "include" / "torch" / "csrc" / "api" / "include"), "-isystem", str(cuda),
           str(CSRC / "torch_binding.cpp"), "-o", str(tmp),
           f"-L{root / 'lib'}", "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed for torch_binding.cpp:\n{r.stderr[-6000:]}")
    os.replace(tmp, BINDING)
    if verbose:
        print(f"built {BINDING}")


def _build_lib(ex: cf.Executor, verbose: bool) -> None:
    objs = list(ex.map(lambda s: _compile(s, verbose), sources()))
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [nvcc(), *ARCH, "-shared", "-cudart", "static", "-o", str(tmp), *map(str, objs)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stderr[-4000:]}")
    os.replace(tmp, LIB)
    if verbose:
        print(f"built {LIB}")


def build(force: bool = False, verbose: bool = False) -> pathlib.Path:
    lib = force or _stale(LIB, [*sources(), *CSRC.glob("*.h"), *CSRC.glob("*.cuh")])
    binding = force or _stale(BINDING, [CSRC / "torch_binding.cpp"])
    BUILD.mkdir(exist_ok=True)
    with cf.ThreadPoolExecutor(max_workers=min(len(sources()) + 1, os.cpu_count() or 4)) as ex:
        other = ex.submit(_build_binding, verbose) if binding else None
        if lib:
            _build_lib(ex, verbose)
        if other:
            other.result()  # its errors come behind a library that is whole
    return LIB


def main() -> int:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    args = ap.parse_args()
    build(force=args.force, verbose=args.verbose)
    return 0


if __name__ == "__main__":
    sys.exit(main())
