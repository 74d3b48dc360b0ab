"""Build the ferrum-gpu B200 libraries in-tree.

Outputs (next to the Python package so they travel with the source tree):
  ferrum_gpu/libferrum_fft.so                    C ABI (include/ferrum_fft.h, ferrum_seq.h) + sm_100a kernels
  ferrum_gpu/_native.<python-ext-suffix>         pybind11 module over the C ABI
  ferrum_gpu/_sequence.<python-ext-suffix>       the sequence operators on torch tensors (where
                                                 torch is installed, against that version)

Every .cu is compiled with
  nvcc -gencode arch=compute_100a,code=sm_100a -lineinfo -O3
and the CUDA runtime is linked statically. Objects go to _build/. A target
is rebuilt only when a source or header is newer than it.

Usage: python ferrum-gpu_b200/build.py [-j JOBS] [--force]
"""

from __future__ import annotations

import argparse
import concurrent.futures as cf
import glob
import os
import shutil
import subprocess
import sys
import sysconfig
from importlib import metadata

HERE = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
PKG = os.path.join(HERE, "ferrum_gpu")
BUILD = os.path.join(HERE, "_build")
INCLUDE = os.path.join(REPO, "include")

CUDA_HOME = os.environ.get("CUDA_HOME", "/usr/local/cuda")
NVCC = shutil.which("nvcc") or os.path.join(CUDA_HOME, "bin", "nvcc")
# The system g++ builds the pybind11 module: it must match the libstdc++ the
# interpreter loads at run time.
CXX = "/usr/bin/g++" if os.path.exists("/usr/bin/g++") else (shutil.which("g++") or "g++")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-std=c++17", "-O3", "-lineinfo", "-Xcompiler", "-fPIC", "-Xcompiler", "-Wall",
              "--expt-relaxed-constexpr", f"-I{INCLUDE}"] + ARCH

CU_SOURCES = ["launch_rows.cu", "launch_pass.cu", "launch_misc.cu", "launch_tile.cu", "capi.cu", "host_path.cu", "dist.cu",
              "no_alloc.cu", "substrate.cu"]
# Sequence operators (include/ferrum_seq.h).
SEQ_SOURCES = ["seq_common.cu", "conv1d.cu", "scan_fwd.cu", "scan_bwd.cu", "norm.cu",
               "long_conv.cu", "recurrence.cu", "dropout.cu", "cross_entropy.cu",
               "cross_entropy_f32.cu", "cross_entropy_tc.cu"]
LIB = os.path.join(PKG, "libferrum_fft.so")
EXT = os.path.join(PKG, "_native" + sysconfig.get_config_var("EXT_SUFFIX"))
SEQ_EXT = os.path.join(PKG, "_sequence" + sysconfig.get_config_var("EXT_SUFFIX"))


def _headers(seq: bool = False) -> list[str]:
    fft = (glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.cuh"))
           + [os.path.join(INCLUDE, "ferrum_fft.h")])
    if not seq:
        return fft
    return fft + glob.glob(os.path.join(CSRC, "seq", "*.cuh")) + [os.path.join(INCLUDE, "ferrum_seq.h")]


def _stale(target: str, deps: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _run(cmd: list[str]) -> None:
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(" ".join(cmd) + "\n" + r.stdout + r.stderr)
        raise RuntimeError(f"command failed ({r.returncode}): {cmd[0]} ... {cmd[-1]}")


def _compile_cu(src: str, force: bool) -> str:
    obj = os.path.join(BUILD, os.path.basename(src).replace(".cu", ".o"))
    if force or _stale(obj, [src] + _headers(os.path.dirname(src) != CSRC)):
        _run([NVCC] + NVCC_FLAGS + ["-c", src, "-o", obj])
    return obj


def build(jobs: int = 4, force: bool = False) -> None:
    os.makedirs(BUILD, exist_ok=True)
    srcs = ([os.path.join(CSRC, s) for s in CU_SOURCES]
            + [os.path.join(CSRC, "seq", s) for s in SEQ_SOURCES])
    with cf.ThreadPoolExecutor(max_workers=jobs) as ex:
        objs = list(ex.map(lambda s: _compile_cu(s, force), srcs))
    if force or _stale(LIB, objs):
        _run([NVCC] + ARCH + ["-shared", "-cudart", "static", "-o", LIB] + objs
             + ["-ldl", "-lpthread", "-lrt"])
    native_src = os.path.join(CSRC, "native_py.cpp")
    if force or _stale(EXT, [native_src, LIB] + _headers()):
        import pybind11

        py_inc = sysconfig.get_paths()["include"]
        _run([CXX, "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
              f"-I{pybind11.get_include()}", f"-I{py_inc}", f"-I{INCLUDE}", native_src,
              "-o", EXT, f"-L{PKG}", "-lferrum_fft", "-Wl,-rpath,$ORIGIN"])
    if not build_sequence(force):
        print("torch is not installed: ferrum_gpu.sequence is left out", file=sys.stderr)


def _torch_version() -> str | None:
    try:
        return metadata.version("torch")
    except metadata.PackageNotFoundError:
        return None


def build_sequence(force: bool = False) -> bool:
    """The module on torch tensors; False where torch is not installed. It is
    rebuilt for another torch, whose C++ interface it is compiled against."""
    version = _torch_version()
    if version is None:
        return False
    src = os.path.join(CSRC, "seq", "torch_binding.cpp")
    stamp = os.path.join(BUILD, "torch_version")
    built = ""
    if os.path.exists(stamp):
        with open(stamp) as f:
            built = f.read()
    if force or built != version or _stale(SEQ_EXT, [src, LIB] + _headers(seq=True)):
        import torch

        torch_dir = os.path.dirname(torch.__file__)
        py_inc = sysconfig.get_paths()["include"]
        _run([CXX, "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
              f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
              f"-I{torch_dir}/include", f"-I{torch_dir}/include/torch/csrc/api/include",
              f"-I{CUDA_HOME}/include", f"-I{py_inc}", f"-I{INCLUDE}", src, "-o", SEQ_EXT,
              f"-L{torch_dir}/lib", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python",
              f"-L{PKG}", "-lferrum_fft", "-Wl,-rpath,$ORIGIN"])
        with open(stamp, "w") as f:
            f.write(version)
    return True


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("-j", "--jobs", type=int, default=4)
    ap.add_argument("--force", action="store_true")
    a = ap.parse_args()
    build(a.jobs, a.force)
    print(LIB)
    print(EXT)
    if _torch_version() is not None:
        print(SEQ_EXT)


if __name__ == "__main__":
    main()
