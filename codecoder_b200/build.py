"""Build libbpc.so (the C-ABI library with every CUDA kernel) in-tree for sm_100a, and _torch_ops.so beside it.

    python -m codecoder_b200.build            # or __graft_entry__.build()

Each csrc/*.cu is compiled by nvcc with -gencode arch=compute_100a,code=sm_100a into _build/, then linked into
codecoder_b200/libbpc.so with the static CUDA runtime, so the library loads on a machine without a GPU (the driver is
only opened on first use).  csrc/torch_ops.cpp, the host side of the embedding, gradient-norm, group-norm and
linear-attention operators on torch tensors, is compiled by g++ against the installed torch into codecoder_b200/_torch_ops.so."""
from __future__ import annotations

import concurrent.futures as cf
import os
import shutil
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
OUT = os.path.join(PKG, "libbpc.so")
TORCH_SRC = os.path.join(CSRC, "torch_ops.cpp")
TORCH_OUT = os.path.join(PKG, "_torch_ops.so")
BUILD = os.path.join(REPO, "_build")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
         "--expt-relaxed-constexpr", "-I", os.path.join(REPO, "include")]


def nvcc() -> str:
    for c in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if c and os.path.exists(c):
            return c
    raise RuntimeError("nvcc not found")


def sources() -> list[str]:
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def _header() -> str:
    return os.path.join(REPO, "include", "bpc.h")


def _older(out: str, deps: list[str]) -> bool:
    return not os.path.exists(out) or any(os.path.getmtime(d) > os.path.getmtime(out) for d in deps if os.path.exists(d))


def _needs_build() -> bool:
    return _older(OUT, [os.path.join(CSRC, f) for f in os.listdir(CSRC) if not f.endswith(".cpp")] + [_header()])


def _run(cmd: list[str], what: str) -> str:
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{what} failed:\n{r.stdout}\n{r.stderr}")
    return r.stderr


def torch_ops_lack() -> str | None:
    """What this machine lacks to compile csrc/torch_ops.cpp, or None."""
    import sysconfig
    try:
        import torch
    except ImportError:
        return "torch cannot be imported"
    root = os.path.dirname(os.path.abspath(torch.__file__))
    for path in (os.path.join(root, "include", "c10", "cuda", "CUDAGuard.h"), os.path.join(root, "lib", "libc10_cuda.so"),
                 os.path.join(sysconfig.get_paths()["include"], "Python.h")):
        if not os.path.exists(path):
            return f"{path} is missing"
    return None


STAMP = b"torch_ops built for ["


def torch_stamp() -> str:
    """What a build of csrc/torch_ops.cpp depends on besides its sources: torch's C++ layout and Python's ABI."""
    import sysconfig

    import torch
    return (f"torch {torch.__version__}, CUDA {torch.version.cuda}, C++11 ABI {int(torch._C._GLIBCXX_USE_CXX11_ABI)}, "
            f"Python {sysconfig.get_config_var('SOABI')}")


def stamp_of(path: str) -> str | None:
    """The stamp that the built module carries, or None."""
    with open(path, "rb") as f:
        data = f.read()
    at = data.find(STAMP)
    return None if at < 0 else data[at + len(STAMP):data.index(b"]", at)].decode()


def build_torch_ops() -> str:
    """Compile csrc/torch_ops.cpp against the headers and libraries of the installed torch: with g++, the compiler nvcc
    uses, whatever $CXX says (another one may bring its own C++ runtime into the process)."""
    import sysconfig

    import torch
    root = os.path.dirname(os.path.abspath(torch.__file__))
    inc = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
           sysconfig.get_paths()["include"], os.path.join(os.path.dirname(os.path.dirname(nvcc())), "include"),
           os.path.join(REPO, "include")]
    tmp = TORCH_OUT + ".tmp"
    _run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
          "-DTORCH_EXTENSION_NAME=_torch_ops", f'-DBUILT_FOR="{torch_stamp()}"',
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
          *[f"-isystem{d}" for d in inc], TORCH_SRC, "-o", tmp, "-L", os.path.join(root, "lib"), "-lc10", "-lc10_cuda",
          "-ltorch_cpu", "-ltorch_python"], f"g++ on {TORCH_SRC}")
    os.replace(tmp, TORCH_OUT)
    return TORCH_OUT


def build_lib(verbose: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    cc = nvcc()

    def one(src):
        obj = os.path.join(BUILD, os.path.basename(src)[:-3] + ".o")
        cmd = [cc, *ARCH, *FLAGS, "-c", src, "-o", obj]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
        err = _run(cmd, f"nvcc on {src}")
        if verbose:
            sys.stderr.write(err)
        return obj

    with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        objs = list(ex.map(one, sources()))
    tmp = OUT + ".tmp"
    _run([cc, *ARCH, "-shared", "-cudart", "static", "-o", tmp, *objs, "-lrt", "-ldl", "-lpthread"], "link")
    os.replace(tmp, OUT)
    return OUT


def build(force: bool = False, verbose: bool = False) -> str:
    """Both libraries, where they are older than their sources; libbpc.so alone where there is no torch to compile against
    (a C caller's machine: _lib.torch_ops() says then what is missing)."""
    lack = torch_ops_lack()
    wanted = force or _older(TORCH_OUT, [TORCH_SRC, _header()]) or not lack and stamp_of(TORCH_OUT) != torch_stamp()
    if wanted and lack:
        sys.stderr.write(f"{os.path.basename(TORCH_OUT)} is not built: {lack}\n")
    with cf.ThreadPoolExecutor(max_workers=1) as ex:
        host = ex.submit(build_torch_ops) if wanted and not lack else None
        if force or _needs_build():
            build_lib(verbose)
        if host is not None:
            host.result()
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
