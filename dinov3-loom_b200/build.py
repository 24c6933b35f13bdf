"""Build libdinov3.so (CUDA kernels for sm_100a + the C++ host library + the C ABI) in-tree.

    python dinov3-loom_b200/build.py [--force] [--verbose]

Every source in csrc/ is compiled by nvcc with `-gencode arch=compute_100a,code=sm_100a`
(`-Xptxas -v` output lands in _build/ptxas.log) and linked with the static CUDA runtime into
dinov3_b200/libdinov3.so. The library does not link libcuda (driver entry points are looked up
at run time), so it loads on a machine without a GPU. Objects are rebuilt when a source or
header is newer than them. Where a torch with CUDA is installed, binding/sequence.cpp is compiled
into dinov3_b200/_sequence.so (the tensor arguments of dinov3_b200/sequence.py), anew when torch or Python
change; nothing else needs it, and the library is built whether or not that succeeds.
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import glob
import importlib.util
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "dinov3_b200", "libdinov3.so")
BINDING = os.path.join(HERE, "binding", "sequence.cpp")
BINDING_LIB = os.path.join(HERE, "dinov3_b200", "_sequence.so")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMMON = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC,-fvisibility=hidden",
          "-I" + CSRC, "-I" + os.path.join(ROOT, "include")]


def _sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cpp")))


def _headers():
    return glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.cuh")) + \
        glob.glob(os.path.join(ROOT, "include", "*.h"))


def _compile(src: str, force: bool):
    obj = os.path.join(BUILD, os.path.basename(src) + ".o")
    newest = max([os.path.getmtime(src)] + [os.path.getmtime(h) for h in _headers()])
    if not force and os.path.exists(obj) and os.path.getmtime(obj) >= newest:
        return obj, ""
    cmd = [NVCC, *ARCH, *COMMON, "-c", src, "-o", obj]
    if src.endswith(".cu"):
        cmd += ["-Xptxas", "-v"]
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {os.path.basename(src)}:\n{r.stdout}")
    return obj, r.stdout


def _build_binding(force: bool) -> str:
    """Build the tensor binding where torch is installed; returns why it could not be, or ""."""
    found = importlib.util.find_spec("torch")
    if found is None:
        return ""
    torch = found.submodule_search_locations[0]
    if not os.path.exists(os.path.join(torch, "lib", "libtorch_cuda.so")):
        return "the torch that is installed has no CUDA libraries"
    include = [os.path.join(ROOT, "include"), os.path.join(torch, "include"),
               os.path.join(torch, "include", "torch", "csrc", "api", "include"),
               sysconfig.get_paths()["include"]]
    cmd = [NVCC, "-O2", "-std=c++17", "-shared", "-cudart", "none", "-Xcompiler", "-fPIC,-fvisibility=hidden",
           *("-I" + d for d in include), BINDING, "-o", BINDING_LIB, "-L" + os.path.join(torch, "lib"),
           "-ltorch_python", "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda"]
    # what it is built against: it must not be loaded under another torch or Python
    with open(os.path.join(torch, "version.py")) as f:
        key = "\n".join([*cmd, str(sysconfig.get_config_var("SOABI")), f.read()]).replace(ROOT, ".")
    stamp = os.path.join(BUILD, "sequence.stamp")
    newest = max(os.path.getmtime(f) for f in [BINDING, *glob.glob(os.path.join(ROOT, "include", "*.h"))])
    if not force and os.path.exists(BINDING_LIB) and os.path.getmtime(BINDING_LIB) >= newest and os.path.exists(stamp):
        with open(stamp) as f:
            if f.read() == key:
                return ""
    if os.path.exists(BINDING_LIB):
        os.unlink(BINDING_LIB)
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if r.returncode != 0:
        return r.stdout
    with open(stamp, "w") as f:
        f.write(key)
    return ""


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    srcs = _sources()
    with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 4)) as ex:
        binding = ex.submit(_build_binding, force)
        results = list(ex.map(lambda s: _compile(s, force), srcs))
    objs = [o for o, _ in results]
    log = "".join(out for _, out in results)
    if log:
        with open(os.path.join(BUILD, "ptxas.log"), "w") as f:
            f.write(log)
        if verbose:
            print(log)
    if force or not os.path.exists(LIB) or any(os.path.getmtime(o) > os.path.getmtime(LIB) for o in objs):
        cmd = [NVCC, *ARCH, "-shared", "-cudart", "static", "-o", LIB, *objs, "-lpthread", "-ldl", "-lrt"]
        r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}")
    # nothing but the sequence operators' Python face needs the binding, and that says so when it is missing
    if why := binding.result():
        print(f"the tensor binding _sequence.so is not built: {why}", file=sys.stderr)
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args()
    try:
        print(build(a.force, a.verbose))
    except RuntimeError as e:
        print(e, file=sys.stderr)
        sys.exit(1)
