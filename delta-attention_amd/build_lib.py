"""Build libdelta_attn.so (the C-ABI library) for gfx950 with hipcc, and the
extension module of the 8-bit cache's Python calls with a host compiler.

Run as a script or call ``build()``. Both land next to the Python package
(delta_attention/libdelta_attn.so, _kv8_ext.so) so that they travel with the
tree.
"""

from __future__ import annotations

import os
import shlex
import shutil
import subprocess
import sys
import sysconfig
import tempfile
import warnings
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(REPO, "include")
OUT = os.path.join(HERE, "delta_attention", "libdelta_attn.so")
SOURCES = ["attn_kernels.hip", "attn_bwd.hip", "delta_add.hip", "rope.hip", "norm.hip",
           "anchor_cos.hip", "adapt_loop.hip", "kv8.hip"]
ARCH = "gfx950"
EXT_SOURCE = "kv8_bind.cpp"
EXT_OUT = os.path.join(HERE, "delta_attention", "_kv8_ext.so")

# Packed fp32 VALU ops are disabled: they are not used by hand and must not be
# formed by the compiler either.
HIPCC_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-shared",
    "-Wall",
    "-Wno-unused-function",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    # MFMAs the compiler emits keep their accumulators in VGPRs also in the
    # one-wave-per-SIMD kernels (their default there is the AGPR form, whose
    # score tiles the softmax would have to copy out); the accumulators meant
    # for AGPRs are placed there by inline asm
    "-mllvm", "-amdgpu-mfma-vgpr-form",
]


def hipcc() -> str:
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    path = os.path.join(rocm, "bin", "hipcc")
    return path if os.path.exists(path) else "hipcc"


def host_cxx() -> list:
    """The C++ compiler of host code: $CXX, or the first of g++, c++ and ROCm's
    clang++ that is there."""
    if os.environ.get("CXX"):
        return shlex.split(os.environ["CXX"])
    rocm = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "bin", "amdclang++")
    return [next((c for c in ("g++", "c++", rocm) if shutil.which(c)), "g++")]


def _run(cmd, verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    # the host pass warns that it does not know the packed-fp32 feature
    warn = "\n".join(l for l in res.stderr.splitlines()
                     if "packed-fp32-ops" not in l and l.strip())
    if res.returncode != 0:
        raise RuntimeError(f"{os.path.basename(cmd[0])} failed ({res.returncode}):\n{warn}")
    if warn and verbose:
        print(warn, file=sys.stderr)


def _compile_ext(verbose: bool, out: str) -> None:
    import torch          # (the extension is built against it)
    t = os.path.dirname(torch.__file__)
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    _run([*host_cxx(), "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
          f"-I{INCLUDE}", f"-I{sysconfig.get_paths()['include']}", "-isystem", os.path.join(t, "include"),
          "-isystem", os.path.join(t, "include", "torch", "csrc", "api", "include"),
          "-isystem", os.path.join(rocm, "include"), os.path.join(CSRC, EXT_SOURCE), "-o", out,
          f"-L{t}/lib", "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_hip",
          "-L" + os.path.join(rocm, "lib"), "-lamdhip64", f"-Wl,-rpath,{t}/lib"], verbose)


def build_ext(verbose: bool = False, out: str = EXT_OUT) -> str:
    """The extension module of the 8-bit cache's calls (host code, against the
    installed torch)."""
    _compile_ext(verbose, out + ".tmp")
    os.replace(out + ".tmp", out)
    return out


def build(verbose: bool = False, out: str = OUT) -> str:
    """Every source at once (each an object of its own), then the library; the
    extension beside it when the library is the package's. hipcc is all that the
    library needs: without a host compiler, Python's headers or torch only the
    extension is left out, with a warning, and the calls that need it say so."""
    compile_flags = [f for f in HIPCC_FLAGS if f != "-shared"]
    with tempfile.TemporaryDirectory() as tmp, ThreadPoolExecutor(len(SOURCES) + 1) as pool:
        objs = [os.path.join(tmp, s + ".o") for s in SOURCES]
        jobs = [pool.submit(_run, [hipcc(), *compile_flags, f"-I{INCLUDE}", f"-I{CSRC}", "-c",
                                   os.path.join(CSRC, s), "-o", o], verbose)
                for s, o in zip(SOURCES, objs)]
        ext = pool.submit(_compile_ext, verbose, EXT_OUT + ".tmp") if out == OUT else None
        for j in jobs:
            j.result()
        _run([hipcc(), f"--offload-arch={ARCH}", "-fPIC", "-shared", *objs, "-o", out + ".tmp"], verbose)
    os.replace(out + ".tmp", out)
    if ext is not None:
        if ext.exception() is None:
            os.replace(EXT_OUT + ".tmp", EXT_OUT)
        else:
            if os.path.exists(EXT_OUT):      # (an older one's structs need not be this library's)
                os.remove(EXT_OUT)
            warnings.warn(f"the 8-bit cache's calls are not built: {ext.exception()}")
    return out


if __name__ == "__main__":
    print(build(verbose=True))
