"""Build libpsquant.so (gfx950 HIP kernels + C ABI) in-tree with hipcc.

    python comfyui-powershard_amd/powershard_amd/build_lib.py [-j N]

Each ``csrc/*.hip`` compiles to an object under ``_build/``; the objects link into
``lib/libpsquant.so``.  Flags:

* ``--offload-arch=gfx950`` only: no other target, no CUDA path.
* ``-ffp-contract=off``: no silent FMA fusion (the kernels call fmaf where the convention
  fuses), so the quantization and epilogue arithmetic matches the CPU oracle bit for bit.
* ``-fhip-fp32-correctly-rounded-divide-sqrt``: IEEE division for the per-row 127/absmax.
* ``-fno-gpu-flush-denormals-to-zero``: fp32 denormals are kept, as on the CPU.
* ``-Xclang -target-feature -Xclang -packed-fp32-ops``: no packed fp32 VALU instructions.

``csrc/direct.cpp`` (host code only) is built beside it with the host compiler against the installed
torch's headers: ``lib/psq_direct.so``.  The library works without it (the decoder operators' calls take longer), so
where that fails (no host compiler, no torch headers) the build says so and goes on.
"""
import argparse
import concurrent.futures
import os
import subprocess
import sys
import warnings
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
BUILD = PKG / "_build"
LIB = PKG / "lib" / "libpsquant.so"
DIRECT = PKG / "lib" / "psq_direct.so"
INCLUDE = PKG.parent.parent / "include"

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ARCH = "gfx950"
CFLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-fPIC", "-std=c++20",
    "-ffp-contract=off", "-fhip-fp32-correctly-rounded-divide-sqrt", "-fno-gpu-flush-denormals-to-zero",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-fvisibility=hidden", "-Wall", "-Wno-unused-function", f"-I{INCLUDE}",
]


def sources():
    return sorted(CSRC.glob("*.hip"))


def _compile(src):
    obj = BUILD / (src.stem + ".o")
    cmd = [HIPCC, *CFLAGS, "-c", str(src), "-o", str(obj)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src.name}:\n{r.stdout}\n{r.stderr}")
    # surface warnings other than the known host-pass note about the packed-fp32 feature
    for line in r.stderr.splitlines():
        if "warning" in line and "packed-fp32-ops" not in line:
            print(line, file=sys.stderr)
    return obj


def _build_direct():
    """lib/psq_direct.so, or a warning and no such file: one of another build would not fit the library."""
    try:
        _compile_direct()
    except Exception as error:   # whatever the compiler or torch's build helpers run into
        DIRECT.unlink(missing_ok=True)
        warnings.warn(f"psquant: {DIRECT.name} was not built: {error}")


def _compile_direct():
    """lib/psq_direct.so, the CPython module of the decoder operators' direct calls."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension
    tmp = DIRECT.with_suffix(".so.tmp")
    headers = [*cpp_extension.include_paths(), sysconfig.get_paths()["include"]]
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-Wall",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", f"-I{INCLUDE}",
           *(flag for path in headers for flag in ("-isystem", path)), str(CSRC / "direct.cpp"), "-o", str(tmp),
           f"-L{cpp_extension.TORCH_LIB_PATH}", "-ltorch_python", "-ltorch_cpu", "-lc10"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed for direct.cpp:\n{r.stdout}\n{r.stderr}")
    if r.stderr:
        print(r.stderr, file=sys.stderr)
    os.replace(tmp, DIRECT)


def _check_stubs(lib):
    """Fail on an undefined symbol of the library's own namespace.  When the host pass of a .hip
    file rejects a kernel body (a target builtin it cannot check there), clang drops the kernel's
    launch stub without an error, and the library then fails to load on the GPU host."""
    r = subprocess.run(["nm", "-D", "--undefined-only", str(lib)], capture_output=True, text=True)
    if r.returncode != 0:
        return   # no binutils: the ABI test's load of the library still catches it
    missing = [line.split()[-1] for line in r.stdout.splitlines() if "_ZN3psq" in line]
    if missing:
        raise RuntimeError("kernel launch stubs missing (host pass dropped them): " + ", ".join(missing[:4]))


def build(jobs=None, verbose=False):
    """Compile every csrc/*.hip for gfx950 and link lib/libpsquant.so, and lib/psq_direct.so beside it.
    Returns the library's path."""
    BUILD.mkdir(exist_ok=True)
    LIB.parent.mkdir(exist_ok=True)
    srcs = sources()
    jobs = jobs or min(len(srcs), os.cpu_count() or 1, 8)
    with concurrent.futures.ThreadPoolExecutor(jobs) as ex:
        direct = ex.submit(_build_direct)
        objs = list(ex.map(_compile, srcs))
        direct.result()
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", str(tmp), *map(str, objs)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    _check_stubs(tmp)
    os.replace(tmp, LIB)
    if verbose:
        print(f"built {LIB}")
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("-j", type=int, default=None)
    build(ap.parse_args().j, verbose=True)
