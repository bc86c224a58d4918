"""Build the native parts of gpuos_b200 in-tree for sm_100a.

    python -m gpuos_b200._build          # incremental
    python -m gpuos_b200._build --force  # rebuild everything

Outputs (next to this file, git-ignored, shipped with the tree):
    libgpuos_b200.so   the executor (CUDA kernels + C++ runtime + C ABI, with
                       the multi-process IPC server and client) and the row
                       operators, cudart linked statically
    gpuos_ext*.so      the Python module with the reference's API

No GPU is needed to build: nvcc cross-compiles for sm_100a.
"""
from __future__ import annotations

import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
ROOT = HERE.parent
BUILD = ROOT / "_build"
CUDA_HOME = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda"))
NVCC = str(CUDA_HOME / "bin" / "nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]

LIB = HERE / "libgpuos_b200.so"
EXT = HERE / ("gpuos_ext" + sysconfig.get_config_var("EXT_SUFFIX"))

DEV_HEADERS = [CSRC / "gpuos_abi.h", CSRC / "ops.cuh", CSRC / "executor.cuh", CSRC / "batch.cuh",
               CSRC / "lean.cuh"]
# gpuos_rotary, gpuos_cache_*, gpuos_attend, gpuos_route*, gpuos_order / dispatch / combine*, gpuos_logprobs*, gpuos_verify
ROWOPS = ["rotary", "cache", "attend", "attend_int8", "attend_e4m3", "route", "experts", "logprobs", "verify"]
HOST_HEADERS = [CSRC / "gpuos_abi.h", CSRC / "runtime.h", CSRC / "jit.h", ROOT / "include" / "gpuos_b200.h"]


def _stale(out: Path, deps) -> bool:
    if not out.exists():
        return True
    t = out.stat().st_mtime
    return any(Path(d).stat().st_mtime > t for d in deps)


def _run(cmd, verbose):
    if verbose:
        print(" ".join(str(c) for c in cmd), flush=True)
    r = subprocess.run([str(c) for c in cmd], capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError(f"build step failed: {cmd[0]} ... -> exit {r.returncode}")
    return r


def build_lib(force=False, verbose=False) -> Path:
    BUILD.mkdir(exist_ok=True)
    abi = ROOT / "include" / "gpuos_b200.h"
    nvcc = [NVCC, *ARCH, "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC"]
    gxx = ["g++", "-std=c++17", "-O2", "-fPIC", "-Wall", "-Wno-unused-parameter", f"-I{CUDA_HOME / 'include'}"]
    # (object, its command up to -o, what it depends on)
    steps = [(BUILD / "kernels.o", [*nvcc, "-c", CSRC / "kernels.cu"], [CSRC / "kernels.cu", *DEV_HEADERS]),
             (BUILD / "noalloc.o", [*nvcc, "-c", CSRC / "noalloc.cu"], [CSRC / "noalloc.cu", abi, *DEV_HEADERS]),
             (BUILD / "rowops.o", [*gxx, "-c", CSRC / "rowops.cpp"], [CSRC / "rowops.cpp"]),
             (BUILD / "jit.o", [*gxx, "-c", CSRC / "jit.cpp"], [CSRC / "jit.cpp", CSRC / "jit.h", *HOST_HEADERS]),
             (BUILD / "runtime.o", [*gxx, "-c", CSRC / "runtime.cpp"], [CSRC / "runtime.cpp", *HOST_HEADERS]),
             (BUILD / "ipc.o", [*gxx, "-c", CSRC / "ipc.cpp"], [CSRC / "ipc.cpp", *HOST_HEADERS])]
    for name in ROWOPS:
        src = CSRC / f"{name}.cu"
        deps = [src, CSRC / "rowops.cuh", CSRC / "rowops.h", abi]
        if name.startswith("attend"):
            deps += [CSRC / "attend.h", CSRC / "attend.cuh", CSRC / "attend_wide.cuh"]
        steps.append((BUILD / f"{name}.o", [*nvcc, "-c", src], deps))
    jcubin = BUILD / "jit_kernel.cubin"
    jblob = BUILD / "jit_blob.cpp"
    jbobj = BUILD / "jit_blob.o"

    def embed():
        # the relocatable batch kernel for custom expressions, embedded as bytes
        if force or _stale(jcubin, [CSRC / "jit_kernel.cu", *DEV_HEADERS]):
            _run([NVCC, *ARCH, "-O3", "-std=c++17", "-rdc=true", "-cubin",
                  CSRC / "jit_kernel.cu", "-o", jcubin], verbose)
        if force or _stale(jbobj, [jcubin]):
            data = jcubin.read_bytes()
            lines = ["// generated by _build.py from jit_kernel.cu: the relocatable batch kernel",
                     'extern "C" const unsigned long long gpuos_jit_cubin_size = %d;' % len(data),
                     'extern "C" alignas(64) const unsigned char gpuos_jit_cubin[] = {']
            for k in range(0, len(data), 24):
                lines.append(",".join(str(b) for b in data[k:k + 24]) + ",")
            lines.append("};")
            jblob.write_text("\n".join(lines) + "\n")
            _run(["g++", "-O0", "-fPIC", "-c", jblob, "-o", jbobj], verbose)

    def compile_one(step):
        out, cmd, deps = step
        if force or _stale(out, deps):
            _run([*cmd, "-o", out], verbose)

    with ThreadPoolExecutor(max_workers=os.cpu_count() or 1) as pool:
        for f in [pool.submit(embed), *(pool.submit(compile_one, s) for s in steps)]:
            f.result()
    objs = [out for out, _, _ in steps] + [jbobj]
    if force or _stale(LIB, objs):
        _run([NVCC, *ARCH, "-shared", "-cudart", "static", "-o", LIB, *objs,
              "-Xlinker", "--no-undefined", "-lpthread", "-ldl", "-lrt"], verbose)
    return LIB


def build_ext(force=False, verbose=False) -> Path:
    import torch
    from torch.utils import cpp_extension

    lib = build_lib(force, verbose)
    if not (force or _stale(EXT, [CSRC / "ext.cpp", CSRC / "rowops_ext.cpp", lib, *HOST_HEADERS])):
        return EXT
    inc = [f"-I{p}" for p in cpp_extension.include_paths()]
    inc += [f"-I{sysconfig.get_paths()['include']}", f"-I{CUDA_HOME / 'include'}"]
    tlib = cpp_extension.library_paths()[0]
    abi = int(torch._C._GLIBCXX_USE_CXX11_ABI)
    _run(["g++", "-std=c++17", "-O2", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={abi}",
          "-DTORCH_EXTENSION_NAME=gpuos_ext", *inc, CSRC / "ext.cpp", CSRC / "rowops_ext.cpp",
          "-o", EXT,
          f"-L{HERE}", "-lgpuos_b200", f"-L{tlib}", "-ltorch_python", "-ltorch", "-ltorch_cpu",
          "-ltorch_cuda", "-lc10", "-lc10_cuda", "-Wl,-rpath,$ORIGIN", f"-Wl,-rpath,{tlib}"], verbose)
    return EXT


def build(force=False, verbose=False):
    build_ext(force, verbose)


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(LIB)
    print(EXT)
