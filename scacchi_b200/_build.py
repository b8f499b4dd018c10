"""Build the CUDA library in-tree (sm_100a only)."""

from __future__ import annotations

import os
import subprocess
import sys
import threading
import warnings

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libscacchi_b200.so")
# (source, extra flags).  The search kernels are bit-reproducible against
# the oracle: no implicit multiply-add contraction (they call fmaf()
# explicitly where they want one), and the AdamW step's 8-bit codes against
# their definition.  The network kernels are checked to a
# tolerance and keep contraction.
UNITS = [(os.path.join(CSRC, "search.cu"), ["-fmad=false"]), (os.path.join(CSRC, "tower.cu"), []),
         (os.path.join(CSRC, "hex.cu"), ["-fmad=false"]), (os.path.join(CSRC, "targets.cu"), ["-fmad=false"]),
         (os.path.join(CSRC, "policy_loss.cu"), []), (os.path.join(CSRC, "muon.cu"), []),
         (os.path.join(CSRC, "adamw.cu"), ["-fmad=false"]), (os.path.join(CSRC, "log_probs.cu"), [])]
SOURCES = [u[0] for u in UNITS]
HEADERS = [os.path.join(CSRC, h) for h in ("smath.h", "threefry.h", "synthetic_env.h", "lane_cta.cuh", "tc05.cuh",
                                            "row_log.cuh")] + [
    os.path.join(ROOT, "include", "scacchi_b200.h")]

NVCC_FLAGS = ["-O3", "-std=c++17", "-Xcompiler", "-fPIC", "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo"]


def nvcc() -> str:
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    path = os.path.join(cuda, "bin", "nvcc")
    return path if os.path.exists(path) else "nvcc"


def stale() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    return any(os.path.getmtime(p) > t for p in SOURCES + HEADERS)


def build(force: bool = False, verbose: bool = False, out: str | None = None, defines: tuple = ()) -> str:
    """The library by nvcc alone, then the extension module, which needs
    torch's and Python's headers: without them its calls go through Python."""
    out = out or LIB
    if out != LIB or force or stale():
        _build_library(out, verbose, defines)
    if out == LIB:
        try:
            build_host(force)
        except Exception as e:  # (no torch, no headers, no compiler)
            warnings.warn(f"the extension module was not built: {e!r}", RuntimeWarning, stacklevel=2)
    return out


def _build_library(out: str, verbose: bool, defines: tuple) -> None:
    objs = []
    build_dir = os.path.join(HERE, "_build")
    os.makedirs(build_dir, exist_ok=True)
    procs = []
    for src, extra in UNITS:
        obj = os.path.join(build_dir, os.path.basename(src) + ".o")
        cmd = [nvcc(), *NVCC_FLAGS, *extra, *defines, "-I", os.path.join(ROOT, "include"), "-c", src, "-o", obj]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
        procs.append(subprocess.Popen(cmd))
        objs.append(obj)
    for p in procs:
        if p.wait() != 0:
            raise RuntimeError("nvcc failed")
    subprocess.run([nvcc(), "-shared", "-gencode", "arch=compute_100a,code=sm_100a", "-o", out, *objs], check=True)


def host_path() -> str:
    """The extension module (csrc/host.cpp: Python's calls of some operators).
    It holds to the C++ of the torch and the Python that it was built against,
    so its name tells them: another torch finds none and builds its own."""
    import torch

    version, abi = torch.__version__.replace("+", "."), int(torch._C._GLIBCXX_USE_CXX11_ABI)
    return os.path.join(HERE, f"_host.{sys.implementation.cache_tag}-torch{version}-abi{abi}.so")


def build_host(force: bool = False) -> str:
    """The extension module, by the host's compiler against torch's headers."""
    src, header = os.path.join(CSRC, "host.cpp"), os.path.join(ROOT, "include", "scacchi_b200.h")
    path = host_path()
    if not force and os.path.exists(path) and all(os.path.getmtime(p) <= os.path.getmtime(path) for p in (src, header)):
        return path
    import sysconfig

    import torch

    base = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(nvcc())) or "/usr/local/cuda"
    part = f"{path}.{os.getpid()}.{threading.get_ident()}"  # renamed when whole: several may build at once
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC",
                    f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{base}/include",
                    f"-I{base}/include/torch/csrc/api/include", f"-I{sysconfig.get_paths()['include']}",
                    f"-I{cuda}/include", src, "-o", part, f"-L{base}/lib", "-ltorch_python", "-ltorch", "-ltorch_cpu",
                    "-lc10", "-lc10_cuda", f"-Wl,-rpath,{base}/lib"], check=True)
    os.replace(part, path)
    return path


if __name__ == "__main__":
    print(build(force=True, verbose=True))
