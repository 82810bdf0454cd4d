"""Build libtrb_kv.so (the C-ABI CUDA library) in-tree for sm_100a with nvcc.

    python -m tokenrush_b200.build [--force] [--verbose] [--timeline]

--timeline builds a second, diagnostic library (libtrb_kv_timeline.so) whose decode kernel records
per-CTA time stamps; `bench.py --workload timeline` loads it.

The library has no dependency on torch or Python; the host package loads it with ctypes.  The argument
checks of the batched calls are native too (csrc/binding.cpp, built with the host compiler against torch).
"""
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libtrb_kv.so")
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
              "-shared", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr", "-Xcudafe", "--diag_suppress=177"]


def sources():
    out = [os.path.join(HERE, "..", "include", "trb_kv.h")]
    for f in sorted(os.listdir(CSRC)):
        if f.endswith((".cu", ".cuh", ".h")):
            out.append(os.path.join(CSRC, f))
    return out


def up_to_date(lib: str = LIB) -> bool:
    if not os.path.exists(lib):
        return False
    t = os.path.getmtime(lib)
    return all(os.path.getmtime(s) <= t for s in sources())


LIB_TIMELINE = os.path.join(HERE, "libtrb_kv_timeline.so")


BINDING = os.path.join(HERE, "_binding.so")


def binding_sources():
    import torch
    # (the binding is built against one torch: another one, installed later, makes it out of date)
    return [os.path.join(CSRC, "binding.cpp"), os.path.join(HERE, "..", "include", "trb_kv.h"), os.path.join(os.path.dirname(torch.__file__), "version.py")]


def build_binding(force: bool = False) -> str:
    src = os.path.join(CSRC, "binding.cpp")
    if not force and os.path.exists(BINDING) and all(os.path.getmtime(d) <= os.path.getmtime(BINDING) for d in binding_sources()):
        return BINDING
    import sysconfig
    import torch
    from torch.utils.cpp_extension import include_paths, library_paths
    cuda = os.path.join(os.path.dirname(os.path.dirname(shutil.which(os.environ.get("NVCC", "nvcc")) or "/usr/local/cuda/bin/nvcc")), "include")
    includes = include_paths() + [sysconfig.get_path("include"), cuda]
    libs = [f for p in library_paths() for f in ("-L" + p, "-Wl,-rpath," + p)] + ["-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", "-w",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"] + ["-I" + p for p in includes] + ["-o", BINDING, src] + libs
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError("the host compiler failed building _binding.so")
    return BINDING


def build(force: bool = False, verbose: bool = False, timeline: bool = False) -> str:
    lib = LIB_TIMELINE if timeline else LIB
    build_binding(force)
    if not force and up_to_date(lib):
        return lib
    nvcc = os.environ.get("NVCC", "nvcc")
    cmd = [nvcc] + NVCC_FLAGS + (["-DTRB_TIMELINE"] if timeline else []) + (["-Xptxas", "-v"] if verbose else []) + ["-o", lib, os.path.join(CSRC, "trb_kv.cu")]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError("nvcc failed building libtrb_kv.so")
    if verbose:
        sys.stderr.write(r.stderr)
    return lib


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv, timeline="--timeline" in sys.argv))
