"""Build libnv4.so, the sm_100a kernel library, and its torch binding in-tree.

    python nano-vllm-int4_b200/build_native.py [--force] [--ptxas-verbose] [--no-binding]

nvcc cross-compiles for sm_100a without a GPU.  All kernel sources are
compiled as one translation unit (csrc/nv4_unity.cu) so the device-side error
word is a single symbol without relocatable device code.  The CUDA runtime is
linked statically and the driver's tensor-map encoder is resolved at run time,
so the library depends on nothing but the driver.

_nv4_serving.so (csrc/serving_binding.cpp, a host compiler only) is a Python
module for the short calls of the serving operators: it checks and allocates
torch tensors and calls libnv4.so beside it.  It holds to the torch and Python
that it was compiled against, so these belong to its stamp; a user of the C ABI
alone, without torch, leaves it out with --no-binding.
"""
from __future__ import annotations

import argparse
import hashlib
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
OUT_DIR = os.path.join(HERE, "nanovllm", "_lib")
OUT = os.path.join(OUT_DIR, "libnv4.so")
BINDING = os.path.join(OUT_DIR, "_nv4_serving.so")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def _digest(names: list[tuple[str, str]], rest: str) -> str:
    h = hashlib.sha256()
    for d, name in names:
        with open(os.path.join(d, name), "rb") as f:
            h.update(name.encode() + b"\0" + f.read())
    h.update(rest.encode())
    return h.hexdigest()


def source_hash() -> str:
    """Of what libnv4.so is built from."""
    return _digest([(d, n) for d in (CSRC, INCLUDE) for n in sorted(os.listdir(d)) if n.endswith((".cu", ".cuh", ".h"))],
                   " ".join(ARCH))


def binding_hash() -> str:
    """Of what _nv4_serving.so is built from and against: a module of another torch
    or Python may load and then misread their objects."""
    import sysconfig

    import torch
    return _digest([(CSRC, "serving_binding.cpp"), (INCLUDE, "nv4.h")],
                   " ".join((torch.__version__, str(torch.compiled_with_cxx11_abi()),
                             sysconfig.get_config_var("EXT_SUFFIX") or sys.version)))


def _fresh(built: str, digest: str) -> bool:
    stamp = built + ".srchash"
    if not os.path.exists(built) or not os.path.exists(stamp):
        return False
    with open(stamp) as f:
        return f.read().strip() == digest


def _replace(built: str, cmd: list[str], digest: str, failure: str) -> str:
    """Runs cmd, which writes built + ".tmp", and puts that and its stamp in place."""
    stamp = built + ".srchash"
    if os.path.exists(stamp):
        os.remove(stamp)
    log = _run(cmd, failure)
    os.replace(built + ".tmp", built)
    with open(stamp, "w") as f:
        f.write(digest + "\n")
    return log


def _run(cmd: list[str], failure: str) -> str:
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        sys.stderr.write(proc.stdout + proc.stderr)
        raise RuntimeError(failure)
    return proc.stderr


def _binding_command() -> list[str]:
    import sysconfig

    import torch
    base = os.path.join(os.path.dirname(torch.__file__))
    lib = os.path.join(base, "lib")
    cuda = os.path.dirname(os.path.dirname(NVCC))
    return [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
            "-isystem", os.path.join(base, "include"),
            "-isystem", os.path.join(base, "include", "torch", "csrc", "api", "include"),
            "-isystem", sysconfig.get_paths()["include"], "-isystem", os.path.join(cuda, "include"),
            "-o", BINDING + ".tmp", os.path.join(CSRC, "serving_binding.cpp"), "-L", OUT_DIR, "-lnv4", "-L", lib,
            "-ltorch", "-ltorch_cpu", "-ltorch_python", "-lc10", "-lc10_cuda", "-Wl,-rpath,$ORIGIN"]


def build(force: bool = False, verbose_ptxas: bool = False, binding: bool = True) -> str:
    """Builds what is not current; `binding` false leaves _nv4_serving.so (and torch) aside."""
    os.makedirs(OUT_DIR, exist_ok=True)
    digest = source_hash()
    if force or not _fresh(OUT, digest):
        cmd = [NVCC, *ARCH, "-O3", "-lineinfo", "-std=c++17", "-shared", "-Xcompiler", "-fPIC",
               "-Xcompiler", "-fvisibility=hidden", "--cudart", "static", "-I", INCLUDE,
               "-o", OUT + ".tmp", os.path.join(CSRC, "nv4_unity.cu")]
        if verbose_ptxas:
            cmd[1:1] = ["-Xptxas", "-v"]
        log = _replace(OUT, cmd, digest, "nvcc failed building libnv4.so")
        if verbose_ptxas:
            sys.stderr.write(log)
    if binding:
        digest = binding_hash()
        if force or not _fresh(BINDING, digest):
            _replace(BINDING, _binding_command(), digest, "the host compiler failed building _nv4_serving.so")
    return OUT


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--ptxas-verbose", action="store_true")
    ap.add_argument("--no-binding", action="store_true")
    args = ap.parse_args()
    print(build(args.force, args.ptxas_verbose, not args.no_binding))
