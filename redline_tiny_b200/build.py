"""Build libredline_b200.so in-tree with nvcc for sm_100a (no GPU needed: nvcc cross-compiles), and the Python extension
_rl_torch.so (the hot calls of ops.py in C++) beside it. The library needs nvcc alone; where torch, Python's headers or a C++
compiler are missing the extension is left out with a notice, and ops.py makes its calls through ctypes.

    python -m redline_tiny_b200.build [--verbose]
"""

import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
SRC = os.path.join(HERE, "csrc", "redline_b200.cu")
OUT = os.path.join(HERE, "libredline_b200.so")
NVCC_FLAGS = ["-O3", "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo",
              "-Xcompiler", "-fPIC", "-shared", "-I", os.path.join(ROOT, "include")]


EXT_SRC = os.path.join(HERE, "csrc", "rl_torch.cpp")
EXT = os.path.join(HERE, "_rl_torch.so")
EXT_FOR = EXT + ".txt"   # the Python and torch that it was built for
HEADER = os.path.join(ROOT, "include", "redline_b200.h")


def sources():
    d = os.path.join(HERE, "csrc")
    return [os.path.join(d, f) for f in sorted(os.listdir(d)) if f != "rl_torch.cpp"] + [HEADER]


def up_to_date(out=OUT, srcs=None):
    if not os.path.exists(out):
        return False
    t = os.path.getmtime(out)
    return all(os.path.getmtime(s) <= t for s in srcs or sources())


def build_extension(verbose=False, force=False):
    """The extension's path, or None where something that it needs is missing (an older one is then removed)."""
    cxx, include = os.environ.get("CXX", "g++"), sysconfig.get_paths()["include"]
    try:
        import torch
        missing = None if shutil.which(cxx) else f"the compiler {cxx}"
    except ImportError:
        missing = "torch"
    if not missing and not os.path.exists(os.path.join(include, "Python.h")):
        missing = "Python.h"
    if missing:
        sys.stderr.write(f"_rl_torch.so left out: {missing} is missing (ops.py calls the library through ctypes)\n")
        for f in (EXT, EXT_FOR):
            if os.path.exists(f):
                os.remove(f)
        return None
    built_for = f"python {sys.version_info[0]}.{sys.version_info[1]}, torch {torch.__version__}"
    if not force and up_to_date(EXT, [EXT_SRC, HEADER]) and os.path.exists(EXT_FOR):
        with open(EXT_FOR) as f:
            if f.read().strip() == built_for:
                return EXT
    t = os.path.dirname(torch.__file__)
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    _run([cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-o", EXT + ".tmp", EXT_SRC,
          f'-DRL_TORCH_VERSION="{torch.__version__}"', "-I", include, "-isystem", f"{t}/include", "-isystem",
          f"{t}/include/torch/csrc/api/include", "-isystem", f"{cuda}/include",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-L", HERE, "-l:libredline_b200.so", "-L",
          f"{t}/lib", "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda", "-Wl,-rpath,$ORIGIN"], verbose)
    os.replace(EXT + ".tmp", EXT)
    with open(EXT_FOR, "w") as f:
        f.write(built_for + "\n")
    return EXT


def _run(cmd, verbose):
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError(f"{cmd[0]} failed ({r.returncode}): {' '.join(cmd)}")
    if verbose:
        sys.stderr.write(r.stdout + r.stderr)


def build(verbose=False, force=False, need_extension=False):
    if force or not up_to_date():
        nvcc = os.environ.get("NVCC", "nvcc")
        _run([nvcc, *NVCC_FLAGS, *(["-Xptxas", "-v"] if verbose else []), "-o", OUT + ".tmp", SRC], verbose)
        os.replace(OUT + ".tmp", OUT)
    if build_extension(verbose, force) is None and need_extension:
        raise RuntimeError("the extension could not be built")
    return OUT


if __name__ == "__main__":
    print(build(verbose="--verbose" in sys.argv, force=True))
