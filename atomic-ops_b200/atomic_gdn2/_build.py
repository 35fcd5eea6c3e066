"""Build the sm_100a shared library (plain nvcc, no torch extension machinery).

The library is written in-tree to ``atomic_gdn2/_lib/libgdn2_b200.so`` so that it
travels with the source tree, the serving operators' binding to torch tensors
(``csrc/gdn2_torch.cpp``, host code) to ``atomic_gdn2/_lib/gdn2_torch-<torch>-<python>.so``: it fits
the torch that it was built against and no other, so its name says which.  Each ``csrc/*.cu`` is
compiled to an object in parallel, then linked with ``-shared``.
"""
from __future__ import annotations

import concurrent.futures as cf
import os
import pathlib
import shutil
import subprocess
import sys

PKG_DIR = pathlib.Path(__file__).resolve().parent
ROOT = PKG_DIR.parent                      # atomic-ops_b200/
CSRC = ROOT / "csrc"
INCLUDE = ROOT.parent / "include"
LIB_DIR = PKG_DIR / "_lib"
LIB_NAME = "libgdn2_b200.so"
LIB_PATH = LIB_DIR / LIB_NAME
EXT_SRC = CSRC / "gdn2_torch.cpp"          # the serving operators' binding to torch tensors

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC",
              "-Xptxas", "-v", f"-I{INCLUDE}"]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and pathlib.Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found: the GDN-2 B200 library cannot be built")


def ext_path() -> pathlib.Path:
    """The torch binding for the running torch and Python."""
    import torch
    return LIB_DIR / f"gdn2_torch-{torch.__version__}-cp{sys.version_info[0]}{sys.version_info[1]}.so"


def sources() -> list[pathlib.Path]:
    return sorted(CSRC.glob("*.cu"))


def _stale() -> bool:
    ext = ext_path()
    if not LIB_PATH.exists() or not ext.exists():
        return True
    t = min(LIB_PATH.stat().st_mtime, ext.stat().st_mtime)
    deps = [EXT_SRC] + list(CSRC.glob("*.cu")) + list(CSRC.glob("*.cuh")) + list(INCLUDE.glob("*.h"))
    return any(p.stat().st_mtime > t for p in deps)


def _ext_object(obj_dir: pathlib.Path) -> pathlib.Path:
    """Compile the torch binding (host code only)."""
    import sysconfig
    import torch
    from torch.utils.cpp_extension import include_paths
    obj = obj_dir / (EXT_SRC.stem + ".o")
    nvcc_include = pathlib.Path(_nvcc()).resolve().parents[1] / "include"
    cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-c", str(EXT_SRC), "-o", str(obj),
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{INCLUDE}", f"-I{nvcc_include}",
           "-isystem", sysconfig.get_paths()["include"], *[x for p in include_paths() for x in ("-isystem", p)]]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for {EXT_SRC.name}:\n{r.stdout}\n{r.stderr}")
    return obj


def _link_ext(obj: pathlib.Path) -> None:
    import torch
    lib = pathlib.Path(torch.__file__).resolve().parent / "lib"
    path = ext_path()
    tmp = path.with_name(path.name + ".tmp")
    cmd = [shutil.which("g++") or "g++", "-shared", "-o", str(tmp), str(obj), f"-L{LIB_DIR}", f"-l:{LIB_NAME}",
           f"-L{lib}", "-ltorch_python", "-ltorch_cuda", "-ltorch_cpu", "-ltorch", "-lc10_cuda", "-lc10",
           "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, path)


def build_library(force: bool = False, verbose: bool = False) -> pathlib.Path:
    """Compile every csrc/*.cu for sm_100a and link libgdn2_b200.so, then the torch binding beside it;
    returns the library's path."""
    if not force and not _stale():
        return LIB_PATH
    nvcc = _nvcc()
    obj_dir = ROOT / "_build"
    obj_dir.mkdir(exist_ok=True)
    LIB_DIR.mkdir(exist_ok=True)

    def compile_one(src: pathlib.Path) -> tuple[pathlib.Path, str]:
        obj = obj_dir / (src.stem + ".o")
        cmd = [nvcc, *ARCH_FLAGS, *NVCC_FLAGS, "-c", str(src), "-o", str(obj)]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed for {src.name}:\n{r.stdout}\n{r.stderr}")
        return obj, r.stdout + r.stderr

    with cf.ThreadPoolExecutor(max_workers=min(9, (os.cpu_count() or 1) + 1)) as ex:
        ext = ex.submit(_ext_object, obj_dir)
        results = list(ex.map(compile_one, sources()))
    if verbose:
        for _, log in results:
            print(log)
    tmp = LIB_PATH.with_suffix(".so.tmp")
    cmd = [nvcc, *ARCH_FLAGS, "-shared", "-o", str(tmp), *[str(o) for o, _ in results], "-lcudart"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB_PATH)
    _link_ext(ext.result())
    return LIB_PATH


if __name__ == "__main__":
    print(build_library(force="--force" in sys.argv, verbose="-v" in sys.argv))
