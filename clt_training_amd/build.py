"""Build libcltmi355.so in-tree with hipcc for gfx950 (cross-compiles without a GPU)."""
from __future__ import annotations

import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
LIB = HERE / "libcltmi355.so"
SOURCES = ["common.hip", "decode.hip", "segments.hip", "decode_rows.hip", "topk.hip", "encoder_gemm.hip", "encoder_gemm_fast.hip", "encoder_gemm_fast16.hip", "encoder_gemm_w8.hip", "fvu.hip", "adam.hip", "adamw.hip", "mxfp4.hip"]
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
# (no packed fp32 arithmetic: some forms of v_pk_{add,mul,fma}_f32 have given wrong results on gfx950 now and then; hipcc's
# host pass does not know the feature and says so, which is harmless)
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Wno-unused-result",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


# The compiled host side (csrc/host.cpp): a Python module against this process's torch, built by the host compiler.
HOST_LIB = HERE / "_clthost.so"


def _host_command(out: Path) -> list:
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths

    lib = Path(torch.__file__).resolve().parent / "lib"
    includes = [*include_paths(), "/opt/rocm/include", sysconfig.get_paths()["include"]]
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            *(a for p in includes for a in ("-isystem", str(p))), str(CSRC / "host.cpp"), "-o", str(out), f"-L{lib}",
            "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch_hip", "-ltorch", "-ltorch_python"]


def _stale(out: Path, deps) -> bool:
    if not out.exists():
        return True
    t = out.stat().st_mtime
    return any(Path(d).stat().st_mtime > t for d in deps)


def build(force: bool = False, verbose: bool = True, tuning: bool = False) -> Path:
    """tuning=True: -DCLT_TUNING (the kernels' timing / A-B switches read the environment) into libcltmi355_tuning.so,
    for tools/ only (select it with CLT_LIB=...); the shipped library never reads the environment."""
    objdir = HERE / ("build_tuning" if tuning else "build")
    objdir.mkdir(exist_ok=True)
    flags = FLAGS + (["-DCLT_TUNING"] if tuning else [])
    lib = HERE / "libcltmi355_tuning.so" if tuning else LIB
    headers = [*CSRC.glob("*.h"), HERE.parent / "include" / "clt_mi355.h"]

    def compile_one(src):
        obj = objdir / (Path(src).stem + ".o")
        if force or _stale(obj, [CSRC / src, *headers]):
            cmd = [HIPCC, *flags, "-c", str(CSRC / src), "-o", str(obj)]
            if verbose:
                print(" ".join(cmd), flush=True)
            subprocess.run(cmd, check=True)
        return obj

    def compile_host():
        if force or _stale(HOST_LIB, [CSRC / "host.cpp", HERE.parent / "include" / "clt_mi355.h"]):
            cmd = _host_command(HOST_LIB)
            if verbose:
                print(" ".join(cmd), flush=True)
            subprocess.run(cmd, check=True)

    with ThreadPoolExecutor(max_workers=min(8, len(SOURCES) + 1)) as ex:
        host = ex.submit(compile_host)
        objs = list(ex.map(compile_one, SOURCES))
        host.result()
    if force or _stale(lib, objs):
        cmd = [HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", str(lib), *map(str, objs)]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
    return lib


if __name__ == "__main__":
    build(force="--force" in sys.argv, tuning="--tuning" in sys.argv)
