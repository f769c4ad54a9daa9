"""Builds libxnor_b200.so (the CUDA kernels and their C ABI) in-tree with nvcc for sm_100a, and _fourbit.so (the host side of
darknet_b200.fourbit's calls into it) with the host compiler.

Usage: ``python -m darknet_b200.build [--force] [--verbose]``.  nvcc cross-compiles, so no GPU is
needed.  Each is rebuilt when any source or header of it is newer than the existing one, _fourbit.so also when torch is another version.
libxnor_b200.so needs no torch to build.
"""
from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sys

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
REPO_DIR = os.path.dirname(PKG_DIR)
CSRC = os.path.join(PKG_DIR, "csrc")
INCLUDE = os.path.join(REPO_DIR, "include")
LIB_PATH = os.path.join(PKG_DIR, "libxnor_b200.so")
BINDINGS = os.path.join(PKG_DIR, "bindings")
BINDING_PATH = os.path.join(PKG_DIR, "_fourbit.so")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "--shared", "-Xcompiler", "-fPIC,-fvisibility=hidden",
    "-Xptxas", "-v",
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found; the xnor_b200 library cannot be built")


def sources() -> list[str]:
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cpp")))


def _older(path: str, deps: list[str]) -> bool:
    return not os.path.exists(path) or any(os.path.getmtime(d) > os.path.getmtime(path) for d in deps)


def _stale() -> bool:
    return _older(LIB_PATH, sources() + glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.hpp")) + glob.glob(os.path.join(INCLUDE, "*.h")))


def _torch():
    """torch, whose tensors _fourbit.so is handed; None where there is none, or no headers to build a Python extension with: the library
    itself needs neither."""
    import sysconfig

    try:
        import torch
    except ImportError:
        return None
    return torch if os.path.exists(os.path.join(sysconfig.get_paths()["include"], "Python.h")) else None


def _built_for(torch) -> str:
    """What _fourbit.so says it was built for: torch's C++ interface changes from one version to the next."""
    return torch.__version__


def _binding_stale(torch) -> bool:
    if _older(BINDING_PATH, glob.glob(os.path.join(BINDINGS, "*.cpp")) + glob.glob(os.path.join(INCLUDE, "*.h"))):
        return True
    with open(BINDING_PATH, "rb") as fh:
        return f"built for torch {_built_for(torch)};".encode() not in fh.read()


def _binding(torch, obj: str) -> tuple[list[str], list[str]]:
    """The commands that compile and link _fourbit.so: torch's headers for the tensors it is handed, the C ABI for everything else."""
    import sysconfig

    root = os.path.dirname(torch.__file__)
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(_nvcc()))), "include")
    compile_ = ["g++", "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
                f'-DBUILT_FOR_TORCH="{_built_for(torch)}"',
                "-I", INCLUDE, "-isystem", os.path.join(root, "include"), "-isystem", os.path.join(root, "include", "torch", "csrc", "api", "include"),
                "-isystem", cuda, "-I", sysconfig.get_paths()["include"], "-c", os.path.join(BINDINGS, "fourbit_calls.cpp"), "-o", obj]
    link = ["g++", "-shared", "-o", BINDING_PATH, obj, "-L", os.path.join(root, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python",
            "-L", os.path.dirname(LIB_PATH), "-lxnor_b200", "-Wl,-rpath,$ORIGIN"]
    return compile_, link


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile every CUDA source into libxnor_b200.so, and the binding beside it where there is a torch to build it for; returns the
    library's path."""
    torch = _torch()
    library, binding = force or _stale(), torch is not None and (force or _binding_stale(torch))
    if torch is None:
        sys.stderr.write("no torch, or no headers of this Python: _fourbit.so, which darknet_b200.fourbit calls through, is not built\n")
    if not library and not binding:
        return LIB_PATH
    objs = []
    obj_dir = os.path.join(PKG_DIR, "build")
    os.makedirs(obj_dir, exist_ok=True)
    nvcc = _nvcc()
    procs = []
    if binding:
        binding_compile, binding_link = _binding(torch, os.path.join(obj_dir, "fourbit_calls.o"))
        binding_proc = subprocess.Popen(binding_compile, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    for src in sources() if library else []:
        obj = os.path.join(obj_dir, os.path.basename(src) + ".o")
        objs.append(obj)
        cmd = [nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
               "-Xcompiler", "-fPIC,-fvisibility=hidden", "-Xptxas", "-v", "-DXNOR_B200_BUILD",
               "-I", INCLUDE, "-I", CSRC, "-c", src, "-o", obj]
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    log = []
    failed = False
    for src, proc in procs:
        out, _ = proc.communicate()
        log.append(f"== {os.path.basename(src)}\n{out}")
        failed |= proc.returncode != 0
    binding_out = binding_proc.communicate()[0] if binding else ""
    if library:
        with open(os.path.join(obj_dir, "ptxas.log"), "w") as fh:
            fh.write("\n".join(log))
    if failed or verbose:
        sys.stderr.write("\n".join(log))
    if failed:
        raise RuntimeError("nvcc failed; see messages above")
    if library:
        subprocess.check_call([nvcc, "--shared", "-o", LIB_PATH] + objs)
    if binding:
        if binding_proc.returncode != 0:
            sys.stderr.write(binding_out)
            raise RuntimeError(f"{LIB_PATH} is built; its binding for torch {_built_for(torch)} is not, see messages above")
        subprocess.check_call(binding_link)
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
