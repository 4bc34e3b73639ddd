"""Builds libbmlattn.so (the CUDA library behind include/bml_attn.h) in-tree
for sm_100a with nvcc, and the Python binding of its paged calls with g++.  No
JIT cache is involved: the .so files sit next to this file and travel with the
source tree."""
from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libbmlattn.so")
CALLS = os.path.join(HERE, "_torch_calls.so")
CALLS_SRC = os.path.join(CSRC, "torch_calls.cpp")
CALLS_FOR = os.path.join(HERE, "_torch_calls.torch")  # the torch version that CALLS was built with
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def sources() -> list[str]:
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


BUILD_DIR = os.path.join(HERE, "_build")
FLAGS = ["-std=c++17", "-O3", *ARCH, "-lineinfo", "-Xcompiler", "-fPIC,-fvisibility=hidden"]


def headers() -> list[str]:
    return glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(HERE, "..", "include", "*.h"))


def needs_build() -> bool:
    return _older(LIB, sources() + headers()) or _calls_stale()


def _torch_version() -> str | None:
    """None without torch or a C++ compiler: then only the C library is built."""
    try:
        import torch
    except ImportError:
        return None
    return torch.__version__ if shutil.which(_cxx()) else None


def _cxx() -> str:
    return os.environ.get("CXX", "g++")


def _calls_stale() -> bool:
    """Whether the binding is to be built: it is older than its sources, or for
    another torch, whose C++ classes it takes apart."""
    want = _torch_version()
    if want is None:
        return False
    if _older(CALLS, [CALLS_SRC, *headers()]) or not os.path.exists(CALLS_FOR):
        return True
    with open(CALLS_FOR) as f:
        return f.read() != want


def _older(target: str, deps: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _build_calls(verbose: bool) -> None:
    """The Python binding of the paged calls (csrc/torch_calls.cpp): host code
    against the installed torch."""
    import sysconfig

    import torch
    root = os.path.join(os.path.dirname(torch.__file__))
    cuda = os.path.dirname(os.path.dirname(nvcc_path()))
    inc = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
           sysconfig.get_paths()["include"], os.path.join(cuda, "include")]
    cmd = [_cxx(), "-O2", f'-DBML_TORCH_VERSION="{torch.__version__}"', "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", *(f"-I{d}" for d in inc),
           "-o", CALLS + ".tmp", CALLS_SRC, "-L" + os.path.join(root, "lib"),
           *(f"-l{x}" for x in ("c10", "c10_cuda", "torch_cpu", "torch_cuda", "torch", "torch_python"))]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    subprocess.run(cmd, check=True)
    os.replace(CALLS + ".tmp", CALLS)
    with open(CALLS_FOR, "w") as f:
        f.write(torch.__version__)


def _object(src: str, newest_header: float, force: bool, verbose: bool) -> str:
    obj = os.path.join(BUILD_DIR, os.path.basename(src)[:-3] + ".o")
    if force or not os.path.exists(obj) or os.path.getmtime(obj) < max(os.path.getmtime(src), newest_header):
        cmd = [nvcc_path(), *FLAGS, "-c", "-o", obj + ".tmp", src]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
            print(" ".join(cmd), file=sys.stderr)
        subprocess.run(cmd, check=True)
        os.replace(obj + ".tmp", obj)
    return obj


def build(force: bool = False, verbose: bool = False) -> str:
    """Compiles every csrc/*.cu to an object (in parallel, each only when it
    or a header changed) and links libbmlattn.so; and _torch_calls.so, unless
    torch or the C++ compiler is missing (the C library needs neither)."""
    if not force and not needs_build():
        return LIB
    from concurrent.futures import ThreadPoolExecutor
    os.makedirs(BUILD_DIR, exist_ok=True)
    newest = max((os.path.getmtime(h) for h in headers()), default=0.0)
    srcs = sources()
    with ThreadPoolExecutor(max_workers=min(len(srcs), os.cpu_count() or 4) + 1) as ex:
        calls = ex.submit(_build_calls, verbose) if _torch_version() and (force or _calls_stale()) else None
        if force or _older(LIB, srcs + headers()):
            objs = list(ex.map(lambda f: _object(f, newest, force, verbose), srcs))
            subprocess.run([nvcc_path(), *ARCH, "-shared", "-o", LIB + ".tmp", *objs], check=True)
            os.replace(LIB + ".tmp", LIB)
        if calls is not None:
            calls.result()
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(LIB)
