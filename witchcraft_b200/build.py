"""Builds the native library `witchcraft_b200/libwc_t5cuda.so` in-tree.

Every CUDA translation unit is compiled for sm_100a only
(`-gencode arch=compute_100a,code=sm_100a`); the host C++ parts with g++.
The library links the CUDA runtime statically and reaches the driver's
cuTensorMapEncodeTiled through cudaGetDriverEntryPointByVersion, so it needs
no libcuda at link time and no torch at all.  The torch binding of the 8-bit
operators is a second, small library, `witchcraft_b200/_fp8_torch.so`, built
where torch with CUDA is installed and again for another version of it.

Usage: python -m witchcraft_b200.build   (or witchcraft_b200.build.build())
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libwc_t5cuda.so")
TORCH_BINDING = os.path.join(HERE, "_fp8_torch.so")
BUILD_DIR = os.path.join(HERE, "_build")

CUDA_SOURCES = ["gemm_q4k.cu", "gemm2_q4k.cu", "gemv_q4k.cu", "attention_tc.cu", "attention_small.cu", "elementwise.cu",
                "runtime.cu", "codec.cu", "index.cu", "query.cu", "fp8_rows.cu", "fp8_gemm.cu"]
CXX_SOURCES = ["t5_host.cpp", "fp8.cpp"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def _run(cmd):
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("build step failed:\n" + " ".join(cmd) + "\n" + r.stdout + r.stderr)
    return r.stdout + r.stderr


def _stale(target: str, deps: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build(verbose: bool = False, force: bool = False) -> str:
    nvcc = _nvcc()
    os.makedirs(BUILD_DIR, exist_ok=True)
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".h", ".cuh"))]
    inc = os.path.join(os.path.dirname(HERE), "include")
    headers += [os.path.join(inc, f) for f in os.listdir(inc) if f.endswith(".h")]
    objs = []
    for src in CUDA_SOURCES:
        s = os.path.join(CSRC, src)
        o = os.path.join(BUILD_DIR, src + ".o")
        objs.append(o)
        if force or _stale(o, [s] + headers):
            extra = os.environ.get("WC_EXTRA_NVCC_FLAGS", "").split()
            out = _run([nvcc, *ARCH, *extra, "-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-Xptxas", "-v",
                        "--expt-relaxed-constexpr", "-c", s, "-o", o])
            if verbose:
                print(out)
    for src in CXX_SOURCES:
        s = os.path.join(CSRC, src)
        o = os.path.join(BUILD_DIR, src + ".o")
        objs.append(o)
        if force or _stale(o, [s] + headers):
            _run(["g++", "-O2", "-std=c++17", "-fPIC", "-I/usr/local/cuda/include", "-c", s, "-o", o])
    if force or _stale(LIB, objs):
        _run([nvcc, *ARCH, "-shared", "-Xcompiler", "-fPIC", "-cudart", "static", "-o", LIB, *objs])
    build_torch_binding(force)
    return LIB


def build_torch_binding(force: bool = False) -> str | None:
    """The torch binding of the 8-bit operators (witchcraft_b200/fp8.py), or
    None without torch or with one built without CUDA: the library itself needs
    neither."""
    try:
        import torch
    except ImportError:
        return None
    if torch.version.cuda is None:
        return None
    import sysconfig
    src = os.path.join(CSRC, "fp8_torch.cpp")
    header = os.path.join(os.path.dirname(HERE), "include", "wc_fp8.h")
    stamp = os.path.join(BUILD_DIR, "fp8_torch.version")  # what the binding was built for
    version = f"torch {torch.__version__}, python {sysconfig.get_config_var('SOABI')}"
    built_for = open(stamp).read() if os.path.exists(stamp) else ""
    if force or built_for != version or _stale(TORCH_BINDING, [src, header]):
        from torch.utils.cpp_extension import include_paths, library_paths
        inc = [f"-I{d}" for d in include_paths()] + [f"-I{sysconfig.get_paths()['include']}", "-I/usr/local/cuda/include"]
        abi = int(torch.compiled_with_cxx11_abi())
        _run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={abi}", *inc, src, "-o",
              TORCH_BINDING, *[f"-L{d}" for d in library_paths()], "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch",
              "-ltorch_python"])
        with open(stamp, "w") as f:
            f.write(version)
    return TORCH_BINDING


def build_oracle() -> str:
    """Builds the CPU oracle (test infrastructure) with its Makefile."""
    d = os.path.join(os.path.dirname(HERE), "oracle")
    _run(["make", "-C", d, "CC=gcc"])
    return os.path.join(d, "liboracle.so")


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv, force="-f" in sys.argv))
