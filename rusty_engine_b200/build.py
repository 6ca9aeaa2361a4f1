"""Build librmoe.so in-tree: every .cu under csrc/ compiled for sm_100a by nvcc, linked shared.

Run as ``python -m rusty_engine_b200.build`` (or through ``__graft_entry__.build()``).  The
output lands next to this file so it travels with the repository snapshot.
"""
from __future__ import annotations

import concurrent.futures as cf
import glob
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "librmoe.so")
OBJ = os.path.join(HERE, "_build")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ARCH + [
    "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
    "--expt-relaxed-constexpr", "-Xptxas", "-v", "-DRMOE_BUILD",
]


def _nvcc() -> str:
    for c in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if c and os.path.exists(c):
            return c
    raise RuntimeError("nvcc not found")


def _nccl_flags():
    """NCCL headers/lib: prefer the copy torch loads (same soname, one NCCL per process)."""
    try:
        import nvidia.nccl  # type: ignore

        base = os.path.dirname(nvidia.nccl.__file__) if nvidia.nccl.__file__ else list(nvidia.nccl.__path__)[0]
        inc, lib = os.path.join(base, "include"), os.path.join(base, "lib")
        if os.path.exists(os.path.join(inc, "nccl.h")):
            return ["-I" + inc], ["-L" + lib, "-Xlinker", "-rpath=" + lib, "-l:libnccl.so.2"]
    except Exception:
        pass
    return [], ["-lnccl"]


BINDING_SRC = os.path.join(HERE, "binding", "kv_ops.cpp")
BINDING = os.path.join(HERE, "_kv_ops.so")


def build_binding():
    """The torch-tensor entry of kv.py (binding/kv_ops.cpp), linked against librmoe.so and torch; its
    path, or None where what it needs is missing (torch with CUDA, g++, Python's headers): librmoe.so
    needs none of these, and kv.py says so when it is used."""
    deps = [BINDING_SRC, os.path.join(HERE, "..", "include", "rmoe.h")]
    if os.path.exists(BINDING) and os.path.getmtime(BINDING) >= max(os.path.getmtime(d) for d in deps):
        return BINDING
    import sysconfig

    try:
        import torch
        from torch.utils.cpp_extension import include_paths
    except (ImportError, OSError) as e:
        return _no_binding(str(e))
    needs = [(os.path.join(os.path.dirname(torch.__file__), "lib", "libc10_cuda.so"), "torch without CUDA"),
             (shutil.which("g++") or "", "no g++"),
             (os.path.join(sysconfig.get_paths()["include"], "Python.h"), "no Python.h")]
    for path, why in needs:
        if not os.path.exists(path):
            return _no_binding(why)

    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    cuda_inc = os.path.join(os.path.dirname(os.path.dirname(_nvcc())), "include")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-I" + sysconfig.get_paths()["include"], "-I" + cuda_inc] + ["-I" + p for p in include_paths()] + [
        BINDING_SRC, "-o", BINDING, "-L" + lib, "-ltorch_python", "-ltorch_cpu", "-ltorch", "-lc10", "-lc10_cuda",
        OUT, "-Wl,-rpath," + lib, "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for {BINDING_SRC}:\n{r.stderr}")
    return BINDING


def _no_binding(why: str):
    print(f"{os.path.basename(BINDING)} not built ({why}): rusty_engine_b200.kv needs it, the C library does not", file=sys.stderr)
    return None


def build(verbose: bool = False, jobs: int = 8) -> str:
    nvcc = _nvcc()
    os.makedirs(OBJ, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    headers = glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(
        os.path.join(HERE, "..", "include", "*.h"))
    newest_h = max(os.path.getmtime(h) for h in headers)
    inc_nccl, link_nccl = _nccl_flags()

    def compile_one(src):
        obj = os.path.join(OBJ, os.path.basename(src) + ".o")
        if os.path.exists(obj) and os.path.getmtime(obj) >= max(os.path.getmtime(src), newest_h):
            return obj, ""
        cmd = [nvcc] + NVCC_FLAGS + inc_nccl + ["-c", src, "-o", obj]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed for {src}:\n{r.stderr}")
        return obj, r.stderr

    with cf.ThreadPoolExecutor(jobs) as ex:
        results = list(ex.map(compile_one, srcs))
    if verbose:
        for obj, log in results:
            if log:
                print(log, file=sys.stderr)
    objs = [o for o, _ in results]
    if not os.path.exists(OUT) or os.path.getmtime(OUT) < max(os.path.getmtime(o) for o in objs):
        cmd = [nvcc] + ARCH + ["-shared", "-Xlinker", "-soname=librmoe.so", "-o", OUT] + objs + link_nccl
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stderr}")
    build_binding()
    return OUT


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
