"""Build the CUDA library libnabla_g1.so for sm_100a and its torch host module nb_torch.so, in-tree
(nablaengine_b200/lib/).

nvcc cross-compiles without a GPU, so this runs anywhere the CUDA toolkit is installed; the built .so travels with
the repository to the GPU machines. `python -m nablaengine_b200.build` rebuilds when a source is newer than the
library or the library was built with other nvcc flags (recorded in a stamp file beside it).
"""
import hashlib
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
LIBDIR = PKG / "lib"
LIB = LIBDIR / "libnabla_g1.so"
SOURCES = [CSRC / n for n in ("nb_g1.cu", "nb_train.cu", "nb_layer_norm_f32.cu", "nb_layer_norm_bf16.cu",
                              "nb_layer_norm_f16.cu")]
# What the library exports: its C entries alone. Its kernels' host functions and what it remembers per kernel and device
# would otherwise be shared with another copy in the process (the profile build's, or a program's that compiles them in).
EXPORTS = CSRC / "nabla_g1.map"
DEPS = (SOURCES + sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h"))
        + [EXPORTS, PKG.parent / "include" / "nabla_g1.h"])
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-shared", "--cudart", "shared"]


def nvcc():
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found: the CUDA toolkit is needed to build libnabla_g1.so")


def _stamp(lib):
    return lib.with_name(lib.name + ".flags")


def _flags_text(extra):
    return " ".join([*ARCH, *FLAGS, *extra])


def stale(lib=LIB, extra=()):
    """True when `lib` is missing, older than a source, or was built with other nvcc flags (the stamp file beside it
    records them)."""
    if not lib.exists():
        return True
    t = lib.stat().st_mtime
    if any(p.stat().st_mtime > t for p in DEPS):
        return True
    stamp = _stamp(lib)
    return not stamp.exists() or stamp.read_text() != _flags_text(extra)


TORCH_LIB = LIBDIR / "nb_torch.so"
TORCH_DEPS = [CSRC / "nb_torch.cpp", PKG.parent / "include" / "nabla_g1.h"]


def _torch_key():
    """What nb_torch.so was built from and for: torch (whose inline C++ types it holds), Python and the sources. No path:
    a built tree may be moved."""
    import torch
    sources = hashlib.sha256(b"".join(p.read_bytes() for p in TORCH_DEPS)).hexdigest()
    return (f"torch {torch.__version__} abi {int(torch._C._GLIBCXX_USE_CXX11_ABI)} "
            f"python {sysconfig.get_config_var('SOABI')} sources {sources}")


def torch_stale():
    """True when nb_torch.so is missing, or was built from other sources or for another torch or Python."""
    stamp = _stamp(TORCH_LIB)
    return not TORCH_LIB.exists() or not stamp.exists() or stamp.read_text() != _torch_key()


def _torch_command(out):
    """The host compiler's command for nb_torch.so (torch's and Python's headers, libnabla_g1.so beside it)."""
    import torch
    root = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc()).resolve().parents[1] / "include"
    include = [root / "include", root / "include" / "torch" / "csrc" / "api" / "include",
               sysconfig.get_paths()["include"], cuda]
    return [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *[f"-I{d}" for d in include],
            str(TORCH_DEPS[0]), "-o", str(out), f"-L{root / 'lib'}", "-lc10", "-lc10_cuda", "-ltorch_cpu",
            "-ltorch_cuda", "-ltorch_python", f"-L{LIBDIR}", "-lnabla_g1", "-Wl,-rpath,$ORIGIN",
            f"-Wl,-rpath,{root / 'lib'}"]


def build_torch(force=False):
    """Compile nb_torch.so (the host side of the training operators) when it is stale; returns its path. libnabla_g1.so
    has to be there."""
    if not force and not torch_stale():
        return TORCH_LIB
    tmp = TORCH_LIB.with_suffix(f".tmp{os.getpid()}.so")
    cmd = _torch_command(tmp)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode:
        raise RuntimeError(f"{cmd[0]} failed ({r.returncode}):\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, TORCH_LIB)
    _stamp(TORCH_LIB).write_text(_torch_key())
    return TORCH_LIB


PROFILE_LIB = LIBDIR / "libnabla_g1_prof.so"


def build(force=False, verbose=False, extra=(), out=None):
    """Compile the library when it is missing, older than its sources or built with other flags; returns its path.
    `out` and `extra`: another output path and extra nvcc flags (the phase-profile build: -DNB_PROFILE into
    PROFILE_LIB)."""
    lib = Path(out) if out else LIB
    if not force and not stale(lib, extra):
        return lib
    LIBDIR.mkdir(exist_ok=True)
    tmp = lib.with_suffix(f".tmp{os.getpid()}.so")
    cmd = [nvcc(), *ARCH, *FLAGS, *extra, "-Xlinker", f"--version-script={EXPORTS}", "--threads", "0", "-o", str(tmp),
           *map(str, SOURCES)]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode:
        raise RuntimeError(f"nvcc failed ({r.returncode}):\n{r.stdout}\n{r.stderr}")
    if verbose:
        print(r.stderr, flush=True)
    os.replace(tmp, lib)
    _stamp(lib).write_text(_flags_text(extra))
    return lib


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
    print(build_torch(force="--force" in sys.argv))
