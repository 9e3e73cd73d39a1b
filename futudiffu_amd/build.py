"""Build recipe for libsage_mi355x.so (gfx950 only).

Compiles the HIP sources under ``csrc/`` with ``hipcc`` into one in-tree
shared library, and the host side of the block operators (``block_ops.cpp``) into a
Python extension beside it.  Packed fp32 VALU instructions are disabled
(``-packed-fp32-ops``); no fast-math flags are used, so fp32 division stays
correctly rounded, which the quantization codes depend on.
"""

from __future__ import annotations

import concurrent.futures
import os
import shutil
import subprocess
import sys
import sysconfig
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB_NAME = "libsage_mi355x.so"
LIB_PATH = os.path.join(HERE, LIB_NAME)
# the measurement build: the same library with per-phase s_memtime timing of
# the attention kernel's pipelined loop (sage_phase_read), for bench.py
# --phase-timing; never loaded by the product path
PHASE_LIB_PATH = os.path.join(HERE, "libsage_mi355x_phase.so")
SOURCES = ["sage_quant.hip", "sage_attn.hip", "sage_mask.hip", "sage_bwd.hip", "sage_capi.hip",
           "sage_norm.hip", "sage_linear.hip"]
# the host side of the block operators: a Python extension over torch's C++ API, which takes
# the library's entry points from the loaded library
EXT_SOURCE = "block_ops.cpp"
EXT_PATH = os.path.join(HERE, "_block_ops.so")
ARCH = "gfx950"


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found (set HIPCC or install ROCm under /opt/rocm)")


def flags() -> list[str]:
    return [
        f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC",
        "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
        "-Wno-unused-command-line-argument",
    ]


def _link(cc: str, objs: list[str], tmp: str, path: str) -> None:
    tmp_lib = os.path.join(tmp, os.path.basename(path))
    cmd = [cc, f"--offload-arch={ARCH}", "-shared", "-fPIC", *objs, "-o", tmp_lib]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stderr}")
    shutil.copyfile(tmp_lib, path + ".tmp")
    os.replace(path + ".tmp", path)


def ext_command(out: str) -> list[str]:
    import torch

    root = os.path.dirname(torch.__file__)
    cxx = os.environ.get("CXX") or shutil.which("g++") or "c++"
    return [cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
            "-DTORCH_EXTENSION_NAME=_block_ops", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            f"-I{root}/include", f"-I{root}/include/torch/csrc/api/include", "-I/opt/rocm/include",
            f"-I{sysconfig.get_paths()['include']}", os.path.join(CSRC, EXT_SOURCE), f"-L{root}/lib", "-lc10",
            "-lc10_hip", "-ltorch_cpu", "-ltorch", "-ltorch_python", "-o", out]


def build(verbose: bool = False, phase_timing: bool = False) -> str:
    """Compile every source and link LIB_PATH atomically; returns LIB_PATH.
    With phase_timing, builds PHASE_LIB_PATH (-DSAGE_PHASE_TIMING) instead."""
    cc = hipcc()
    extra = ["-DSAGE_PHASE_TIMING"] if phase_timing else []
    out_path = PHASE_LIB_PATH if phase_timing else LIB_PATH
    with tempfile.TemporaryDirectory(prefix="sage_build_") as tmp:
        srcs = SOURCES
        objs = [os.path.join(tmp, src + ".o") for src in srcs]

        def compile_one(i: int) -> None:
            cmd = [cc, *flags(), *extra, "-c", os.path.join(CSRC, srcs[i]), "-o", objs[i]]
            if verbose:
                print(" ".join(cmd), flush=True)
            res = subprocess.run(cmd, capture_output=True, text=True)
            if res.returncode != 0:
                raise RuntimeError(f"hipcc failed on {srcs[i]}:\n{res.stderr}")

        ext = os.path.join(tmp, os.path.basename(EXT_PATH))

        def compile_ext() -> None:
            cmd = ext_command(ext)
            if verbose:
                print(" ".join(cmd), flush=True)
            res = subprocess.run(cmd, capture_output=True, text=True)
            if res.returncode != 0:
                raise RuntimeError(f"the compiler failed on {EXT_SOURCE}:\n{res.stderr}")

        # one compiler process per source file, at most four at a time
        with concurrent.futures.ThreadPoolExecutor(max_workers=min(4, len(srcs))) as pool:
            jobs = [pool.submit(compile_one, i) for i in range(len(srcs))]
            if not phase_timing:
                jobs.append(pool.submit(compile_ext))
            for f in jobs:
                f.result()
        _link(cc, objs, tmp, out_path)
        if not phase_timing:
            shutil.copyfile(ext, EXT_PATH + ".tmp")
            os.replace(EXT_PATH + ".tmp", EXT_PATH)
    return out_path


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv, phase_timing="--phase-timing" in sys.argv))
