"""In-tree build of the CUDA library (``lib/libb200attn.so``) with nvcc for sm_100a, and of the extension module that puts its
training-step operators into torch (``lib/_train_binding.*.so``, its name with the torch and the Python it is for) with the host compiler."""
from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sysconfig

import torch

_PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(_PKG, "csrc")
LIB_DIR = os.path.join(_PKG, "lib")
LIB_PATH = os.path.join(LIB_DIR, "libb200attn.so")
HEADERS = [os.path.join(os.path.dirname(_PKG), "include", h) for h in ("b200attn.h", "b200moe.h", "b200train.h")]
UNITS = ("b200attn_api.cu", "b200moe_api.cu", "b200train_api.cu")   # one translation unit per header

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-shared", "-Xcompiler", "-fPIC",
]


def _sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh")) + HEADERS)


def _older(path: str, sources) -> bool:
    return not os.path.exists(path) or any(os.path.getmtime(s) > os.path.getmtime(path) for s in sources)


def binding_path() -> str:
    """The extension module: torch's C++ interface changes between versions, so a module built for another one is another file."""
    return os.path.join(LIB_DIR, f"_train_binding.torch-{torch.__version__}{sysconfig.get_config_var('EXT_SUFFIX')}")


def _binding_sources():
    return [os.path.join(CSRC, "train_binding.cpp"), *HEADERS]


def is_stale() -> bool:
    return _older(LIB_PATH, _sources()) or _older(binding_path(), _binding_sources())


def find_nvcc() -> str | None:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    return None


def _binding_command(nvcc: str) -> list:
    root = os.path.dirname(torch.__file__)
    lib = os.path.join(root, "lib")
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(nvcc)))
    # (the system's compiler, whatever CXX says: the module has to share torch's libstdc++, and a toolchain that brings its own
    # library links it in a second time, where streams and exceptions of the two meet and crash)
    return [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-shared", "-fPIC", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            "-I" + os.path.join(root, "include"), "-I" + os.path.join(root, "include", "torch", "csrc", "api", "include"),
            "-I" + os.path.join(cuda, "include"), "-I" + sysconfig.get_paths()["include"], "-o", binding_path(),
            os.path.join(CSRC, "train_binding.cpp"), "-L" + lib, "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python"]


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile the translation units of ``csrc/`` (each includes its kernels) into ``lib/libb200attn.so``, and the extension module."""
    if not force and not is_stale():
        return LIB_PATH
    nvcc = find_nvcc()
    if nvcc is None:
        raise RuntimeError("nvcc not found: cannot build libb200attn.so")
    os.makedirs(LIB_DIR, exist_ok=True)
    commands = []
    if force or _older(LIB_PATH, _sources()):
        commands.append([nvcc, *NVCC_FLAGS, *(["-Xptxas=-v"] if verbose else []), "-o", LIB_PATH, *[os.path.join(CSRC, u) for u in UNITS]])
    if force or _older(binding_path(), _binding_sources()):
        commands.append(_binding_command(nvcc))
    running = [subprocess.Popen(cmd) for cmd in commands]
    codes = [p.wait() for p in running]
    for cmd, code in zip(commands, codes):
        if code != 0:
            raise subprocess.CalledProcessError(code, cmd)
    return LIB_PATH


if __name__ == "__main__":
    print(build(force=True, verbose=True))
