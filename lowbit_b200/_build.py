"""Build of the CUDA library liblowbit_b200.so (sm_100a) from lowbit_b200/csrc.

The library is compiled in-tree with nvcc (one object per .cu, compiled in
parallel, linked with the static CUDA runtime) and loaded with ctypes. The
build output name does not change; a stamp file holding a hash of the sources
and flags decides whether a rebuild is needed. build_torch() compiles the
torch side of the KV-cache calls (csrc/kv8_torch.cpp, a CPython module on
torch's C++ headers) the same way.

Environment:
  NVCC                    nvcc binary (default: $CUDA_HOME/bin/nvcc or nvcc on PATH)
  LOWBIT_B200_LIB         path to a prebuilt liblowbit_b200.so (skips the build)
  LOWBIT_B200_TORCH_LIB   path to a prebuilt _kv8_torch.so (skips its build)
"""
from __future__ import annotations

import hashlib
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
INCLUDE = PKG.parent / "include"
LIB = PKG / "liblowbit_b200.so"
STAMP = PKG / ".liblowbit_b200.stamp"
TORCH_SRC = CSRC / "kv8_torch.cpp"
TORCH_LIB = PKG / "_kv8_torch.so"
TORCH_STAMP = PKG / "_build" / "kv8_torch.stamp"
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
# no fast-math: the activation quantizer relies on IEEE division and rint
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-Wall",
         "--expt-relaxed-constexpr", "-diag-suppress", "177"]


def nvcc() -> str:
    env = os.environ.get("NVCC")
    if env:
        return env
    home = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    cand = Path(home) / "bin" / "nvcc"
    if cand.exists():
        return str(cand)
    found = shutil.which("nvcc")
    if not found:
        raise RuntimeError("nvcc not found; set NVCC or CUDA_HOME")
    return found


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def _digest() -> str:
    h = hashlib.sha256()
    for p in sorted(list(CSRC.iterdir()) + list(INCLUDE.glob("*.h"))):
        if p.is_file() and p.suffix in (".cu", ".cuh", ".h"):
            h.update(p.name.encode())
            h.update(p.read_bytes())
    h.update(repr((ARCH, FLAGS)).encode())
    return h.hexdigest()[:16]


def up_to_date() -> bool:
    return LIB.exists() and STAMP.exists() and STAMP.read_text().strip() == _digest()


def build(verbose: bool = False, force: bool = False) -> Path:
    """Compile (if needed) and return the path of liblowbit_b200.so."""
    if os.environ.get("LOWBIT_B200_LIB"):
        return Path(os.environ["LOWBIT_B200_LIB"])
    if not force and up_to_date():
        return LIB
    cc = nvcc()
    objdir = PKG / "_build"
    objdir.mkdir(exist_ok=True)

    def compile_one(src: Path) -> Path:
        obj = objdir / (src.stem + ".o")
        cmd = [cc, *ARCH, *FLAGS, "-I", str(INCLUDE), "-c", str(src), "-o", str(obj)]
        if verbose:
            print(" ".join(cmd), flush=True)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src.name}:\n{r.stdout}\n{r.stderr}")
        return obj

    with ThreadPoolExecutor(max_workers=max(1, min(8, os.cpu_count() or 1))) as ex:
        objs = list(ex.map(compile_one, sources()))
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [cc, *ARCH, "-shared", "-cudart", "static", *map(str, objs), "-o", str(tmp)]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB)  # atomic for concurrent importers
    STAMP.write_text(_digest())
    return LIB


def cuda_include() -> Path:
    """Directory of the CUDA runtime headers; needs no compiler."""
    dirs = [Path(os.environ.get("CUDA_HOME", "/usr/local/cuda")) / "include"]
    dirs += [Path(p) / "nvidia" / "cuda_runtime" / "include" for p in sys.path]
    for d in dirs:
        if (d / "cuda_runtime_api.h").exists():
            return d
    try:
        return Path(nvcc()).resolve().parents[1] / "include"
    except RuntimeError:
        raise RuntimeError("CUDA headers not found; set CUDA_HOME, or LOWBIT_B200_TORCH_LIB to a prebuilt module") from None


def build_torch(force: bool = False) -> Path:
    """Compile (if needed) and return the path of the _kv8_torch module."""
    if os.environ.get("LOWBIT_B200_TORCH_LIB"):
        return Path(os.environ["LOWBIT_B200_TORCH_LIB"])
    import sysconfig

    import torch
    h = hashlib.sha256()
    for p in (TORCH_SRC, INCLUDE / "lowbit_b200.h"):
        h.update(p.read_bytes())
    h.update(f"{torch.__version__} {sys.version}".encode())
    digest = h.hexdigest()[:16]
    if not force and TORCH_LIB.exists() and TORCH_STAMP.exists() and TORCH_STAMP.read_text().strip() == digest:
        return TORCH_LIB
    root = Path(torch.__file__).parent
    inc = [root / "include", root / "include" / "torch" / "csrc" / "api" / "include", cuda_include(),
           sysconfig.get_paths()["include"]]
    TORCH_STAMP.parent.mkdir(exist_ok=True)
    tmp = TORCH_LIB.with_suffix(f".so.tmp{os.getpid()}")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *(a for p in inc for a in ("-isystem", str(p))),
           str(TORCH_SRC),
           "-o", str(tmp), f"-L{root / 'lib'}", "-ltorch_python", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-lc10",
           "-lc10_cuda"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{TORCH_SRC.name}: build failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, TORCH_LIB)
    TORCH_STAMP.write_text(digest)
    return TORCH_LIB


if __name__ == "__main__":
    from importlib.util import find_spec
    print(build(verbose=True, force="--force" in sys.argv))
    if find_spec("torch"):  # only the KV-cache calls need it
        build_torch(force="--force" in sys.argv)
