"""Build in-tree: the b200q C-ABI library ``_lib/libb200q.so`` (sm_100a) and, on
top of it, ``_lib/b200q_bindings.so``, the CPython bindings of the low-bit decode
operators (``bindings.cpp``, against torch's headers).  The library needs nvcc alone;
where a C++ compiler, Python.h or torch's headers are missing the bindings are left
out with a message, and the low-bit operators raise.

Usage: ``python csrc/build.py [--verbose]``.  Rebuilds only when a source is
newer than the library.  nvcc cross-compiles, so no GPU is needed.  The
translation units are compiled without --use_fast_math: the INT8 epilogue and the
quantizers rely on IEEE round-to-nearest fp32 arithmetic.
"""
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
PACK = os.path.dirname(HERE)
ROOT = os.path.dirname(PACK)
OUT = os.path.join(PACK, "_lib", "libb200q.so")
HEADER = os.path.join(ROOT, "include", "b200q.h")
# translation unit -> the headers it includes (each is compiled on its own, in
# parallel, and only when one of its sources is newer than its object)
UNITS = {
    "capi.cu": ["host.h", "gemm8.cuh", "prologue.cuh", "qkv_rope.cuh", "quant.cuh", "w8a16.cuh",
                "w8a16_planes.cuh", "numerics.cuh", "ptx.cuh"],
    "lowbit.cu": ["host.h", "digits.cuh", "w4a16.cuh", "w4_tile.cuh", "block_norm.cuh", "kv8.cuh",
                  "kv8_prefill.cuh", "numerics.cuh", "ptx.cuh"],
}
SOURCES = sorted({f for unit, deps in UNITS.items() for f in (unit, *deps)})
FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-lineinfo", "-std=c++17",
         "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden"]


def nvcc_cmd(unit, out, extra=()):
    nvcc = os.environ.get("NVCC", "nvcc")
    return [nvcc, *FLAGS, "-c", "-o", out, os.path.join(HERE, unit), *extra]


def link_cmd(objects, out=OUT):
    nvcc = os.environ.get("NVCC", "nvcc")
    return [nvcc, *FLAGS, "-shared", "-Xlinker", "-soname=libb200q.so", "-o", out, *objects]


BINDINGS = os.path.join(PACK, "_lib", "b200q_bindings.so")
BINDINGS_SOURCES = [os.path.join(HERE, "bindings.cpp"), HEADER]


def cxx_runtime():
    """The libstdc++.so.6 that torch has loaded into this process.  The bindings share
    exceptions with torch, so they must not bring a runtime of their own, and a
    compiler may have only the static one beside it."""
    with open("/proc/self/maps") as f:
        for line in f:
            path = line.split(maxsplit=5)[-1].strip()
            if os.path.basename(path).startswith("libstdc++.so.6"):
                return path
    return "-lstdc++"


def bindings_lack():
    """What the bindings need and this machine has not, or None."""
    import sysconfig
    try:
        import torch
    except ImportError:
        return "torch"
    cxx = os.environ.get("CXX", "g++")
    if not shutil.which(cxx):
        return f"a C++ compiler ({cxx})"
    for header in (os.path.join(sysconfig.get_paths()["include"], "Python.h"),
                   os.path.join(os.path.dirname(torch.__file__), "include", "ATen", "ATen.h")):
        if not os.path.exists(header):
            return header
    return None


def bindings_cmd(out=BINDINGS):
    import sysconfig
    import torch
    base = os.path.dirname(torch.__file__)
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    inc = [os.path.join(base, "include"), os.path.join(base, "include", "torch", "csrc", "api", "include"),
           os.path.join(cuda, "include"), sysconfig.get_paths()["include"]]
    return [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-shared",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            *[a for d in inc for a in ("-isystem", d)], "-o", out, os.path.join(HERE, "bindings.cpp"),
            OUT, "-L" + os.path.join(base, "lib"), "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10",
            "-lc10_cuda", "-nostdlib++", cxx_runtime(), "-Wl,-rpath,$ORIGIN"]


def object_of(unit):
    return os.path.join(PACK, "_lib", unit.replace(".cu", ".o"))


def newer(target, sources):
    """True when `target` exists and no source is newer."""
    if not os.path.exists(target):
        return False
    t = os.path.getmtime(target)
    return all(os.path.getmtime(s) <= t for s in sources if os.path.exists(s))


def unit_sources(unit):
    return [os.path.join(HERE, f) for f in (unit, *UNITS[unit])] + [HEADER]


def up_to_date():
    return (newer(OUT, [s for unit in UNITS for s in unit_sources(unit)])
            and newer(BINDINGS, BINDINGS_SOURCES))


def build(force=False, verbose=False):
    if not force and up_to_date():
        return OUT
    os.makedirs(os.path.dirname(OUT), exist_ok=True)
    jobs = []
    for unit in UNITS:
        obj = object_of(unit)
        if not force and newer(obj, unit_sources(unit)):
            continue
        cmd = nvcc_cmd(unit, obj, ["-Xptxas", "-v"] if verbose == "ptxas" else ())
        if verbose:
            print(" ".join(cmd))
        jobs.append((obj, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT,
                                           text=True)))
    failed = []
    for obj, job in jobs:
        text = job.communicate()[0]
        msg = "\n".join(l for l in text.splitlines() if "compute_" not in l or "Warning" not in l)
        if job.returncode != 0:
            failed.append(f"nvcc failed ({job.returncode}):\n{msg}")
            if os.path.exists(obj):
                os.remove(obj)
        elif verbose and msg.strip():
            print(msg)
    if failed:
        raise RuntimeError("\n".join(failed))
    run(link_cmd([object_of(u) for u in UNITS]), verbose)
    if force or not newer(BINDINGS, BINDINGS_SOURCES):
        lack = bindings_lack()
        if lack:
            print(f"[b200q] {BINDINGS} not built: {lack} is missing; the low-bit operators will raise")
            if os.path.exists(BINDINGS):
                os.remove(BINDINGS)  # one of another source
        else:
            run(bindings_cmd(), verbose)
    return OUT


def run(cmd, verbose):
    if verbose:
        print(" ".join(cmd))
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{os.path.basename(cmd[0])} failed ({r.returncode}):\n{r.stdout}{r.stderr}")


if __name__ == "__main__":
    v = "ptxas" if "--ptxas" in sys.argv else "--verbose" in sys.argv
    print(build(force="--force" in sys.argv, verbose=v))
