"""Build recipe for the in-tree CUDA library `libdraco_moe_b200.so` (sm_100a only).

    python -m dracomancer_llmengine_b200.build        # or build() from Python

Objects go to <repo>/_build/ (not committed); the shared library is written next to this file
so that it travels with the repository snapshot and is what `dracomancer_llmengine_b200`
loads, and beside it `_decoder`, the Python extension of `decoder` for torch tensors, where torch has CUDA.
Rebuilds only what changed (sources or headers newer than the object; the extension also for another torch, and
its name has the interpreter's tag, so that another Python does not load it).
"""
from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
BUILD = os.path.join(ROOT, "_build")
LIB = os.path.join(PKG, "libdraco_moe_b200.so")
EXT = os.path.join(PKG, "_decoder" + (sysconfig.get_config_var("EXT_SUFFIX") or ".so"))
EXT_FOR = os.path.join(BUILD, "decoder_py.torch")       # the torch that it was built for

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ARCH + ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-O2",
                     "--expt-relaxed-constexpr", "-I" + os.path.join(ROOT, "include")]


def nvcc() -> str:
    for c in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if c and os.path.exists(c):
            return c
    raise FileNotFoundError("nvcc not found")


def _headers():
    return [h for d, p in ((CSRC, "*.cuh"), (CSRC, "*.h"), (os.path.join(ROOT, "include"), "*.h"))
            for h in glob.glob(os.path.join(d, p))]


def build(verbose: bool = False, extra_flags=()) -> str:
    os.makedirs(BUILD, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    newest_hdr = max((os.path.getmtime(h) for h in _headers()), default=0.0)
    objs = []
    for s in srcs:
        o = os.path.join(BUILD, os.path.basename(s)[:-3] + ".o")
        objs.append(o)
        if os.path.exists(o) and os.path.getmtime(o) >= max(os.path.getmtime(s), newest_hdr):
            continue
        cmd = [nvcc()] + NVCC_FLAGS + list(extra_flags) + ["-c", s, "-o", o]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
    if not os.path.exists(LIB) or os.path.getmtime(LIB) < max(os.path.getmtime(o) for o in objs):
        tmp = LIB + ".tmp"
        cmd = [nvcc()] + ARCH + ["-shared", "-o", tmp] + objs + ["-lcudart", "-ldl"]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
        os.replace(tmp, LIB)
    build_decoder(verbose)
    return LIB


def build_decoder(verbose: bool = False) -> str | None:
    """The Python extension of `decoder` (argument checks and calls for torch tensors).  None where it cannot be of use or be
    built: no torch, a torch without CUDA, no headers of Python (the library does not need it)."""
    try:
        import torch
    except ImportError:
        return None
    at = os.path.dirname(torch.__file__)
    if torch.version.cuda is None:
        why = f"torch {torch.__version__} has no CUDA"
    elif not os.path.exists(os.path.join(sysconfig.get_paths()["include"], "Python.h")):
        why = "Python's headers are not installed"
    elif not os.path.exists(os.path.join(at, "include", "c10", "cuda", "CUDAStream.h")):
        why = "torch's headers are not installed"
    else:
        why = ""
    if why:
        print(f"_decoder is not built: {why}", file=sys.stderr)
        return None
    src, newest = os.path.join(CSRC, "decoder_py.cpp"), max(os.path.getmtime(h) for h in _headers())
    built_for = open(EXT_FOR).read() if os.path.exists(EXT_FOR) else ""
    if os.path.exists(EXT) and os.path.getmtime(EXT) >= max(os.path.getmtime(src), newest) and built_for == torch.__version__:
        return EXT
    cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f'-DDRACO_TORCH_VERSION="{torch.__version__}"', src, "-o", EXT + ".tmp"]
    cmd += ["-I" + d for d in (os.path.join(at, "include"), os.path.join(os.path.dirname(os.path.dirname(nvcc())), "include"),
                               sysconfig.get_paths()["include"])]
    cmd += ["-L" + os.path.join(at, "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(EXT + ".tmp", EXT)
    untagged = os.path.join(PKG, "_decoder.so")
    if EXT != untagged and os.path.exists(untagged):      # an earlier build's, for any Python
        os.remove(untagged)
    os.makedirs(BUILD, exist_ok=True)
    with open(EXT_FOR, "w") as f:
        f.write(torch.__version__)
    return EXT


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
