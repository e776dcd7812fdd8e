"""Build libclusterfusion_b200.so in-tree with nvcc for sm_100a.

    python clusterfusionplus_b200/build.py [--force] [--verbose]

Nine translation units, compiled separately (objects cached under lib/obj/) and linked into one
shared library: the decode kernel with the C ABI, the batched Llama decode blocks (hand-written
tcgen05 skinny GEMMs + paged attention), the elementwise kernels of the prompt pass, the plan of a step over a
paged cache, the cache held in 4 bits (append and read; attention of few query rows; of many), the log probabilities of
tokens, and the tensor-core prefill GEMM, which is built from the CUTLASS / CuTe headers found in the Python
environment (the `flashinfer` wheel vendors them; set CUTLASS_INCLUDE to use another copy).  The library has no torch dependency;
it links the CUDA runtime statically and finds the driver's tensor-map encoder at run time.  Beside it, lib/_serving.so binds
the serving calls to Python (g++, torch's C++ headers).
"""
from __future__ import annotations

import importlib.util
import os
import re
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
HEADER = os.path.join(os.path.dirname(HERE), "include", "clusterfusion_b200.h")
OUT = os.path.join(HERE, "lib", "libclusterfusion_b200.so")
OBJ = os.path.join(HERE, "lib", "obj")

# source -> (dependencies besides itself, needs the CUTLASS headers)
UNITS = {
    "capi.cu": (["decode_kernel.cuh", "pipeline.cuh", "dsm.cuh", "prefill_gemm.h", "host_common.h", HEADER], False),
    "llama_batch.cu": (["llama_batch_kernel.cuh", "pipeline.cuh", "host_common.h", HEADER], False),
    "prefill_gemm.cu": (["prefill_gemm.h"], True),
    "prefill_ops.cu": (["host_common.h", HEADER], False),
    "serve_plan.cu": (["host_common.h", HEADER], False),
    "kv4_cache.cu": (["f32x2.cuh", "kv4_layout.cuh", "kv4_attention.h", "host_common.h", HEADER], False),
    "kv4_decode.cu": (["kv4_layout.cuh", "kv4_attention.h", "mma.cuh"], False),
    "kv4_prompt.cu": (["f32x2.cuh", "kv4_layout.cuh", "kv4_attention.h", "mma.cuh", "pipeline.cuh"], False),
    "logprobs.cu": (["f32x2.cuh", "mma.cuh", "host_common.h", HEADER], False),
}
BINDING = os.path.join(CSRC, "serving_binding.cpp")
BINDING_OUT = os.path.join(HERE, "lib", "_serving.so")
BINDING_TORCH = os.path.join(HERE, "lib", "_serving.torch")  # the torch version that it was built for
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def cutlass_includes() -> list:
    """Include directories of a CUTLASS tree that has the sm_100 collectives."""
    roots = []
    if os.environ.get("CUTLASS_INCLUDE"):
        roots.append(os.path.dirname(os.environ["CUTLASS_INCLUDE"].rstrip("/")))
    spec = importlib.util.find_spec("flashinfer")
    if spec and spec.submodule_search_locations:
        roots.append(os.path.join(list(spec.submodule_search_locations)[0], "data", "cutlass"))
    for root in roots:
        inc = os.path.join(root, "include")
        if os.path.exists(os.path.join(inc, "cutlass", "gemm", "collective", "collective_builder.hpp")):
            dirs = [inc]
            util = os.path.join(root, "tools", "util", "include")
            if os.path.isdir(util):
                dirs.append(util)
            return dirs
    raise RuntimeError("CUTLASS headers not found: set CUTLASS_INCLUDE to <cutlass>/include")


def _deps(src: str) -> list:
    extra, _ = UNITS[src]
    return [os.path.join(CSRC, src)] + [d if os.path.isabs(d) else os.path.join(CSRC, d) for d in extra]


def _stale(target: str, deps: list) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _compile(src: str, verbose: bool) -> str:
    obj = os.path.join(OBJ, src.replace(".cu", ".o"))
    cmd = [nvcc_path(), *ARCH, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-c", "-o", obj,
           os.path.join(CSRC, src)]
    if UNITS[src][1]:
        cmd += ["--expt-relaxed-constexpr"] + [f"-I{d}" for d in cutlass_includes()]
    if verbose:
        cmd[1:1] = ["-Xptxas", "-v"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if verbose or r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src}")
    return obj


def torch_version() -> str:
    """torch.__version__, without the import."""
    path = os.path.join(os.path.dirname(importlib.util.find_spec("torch").origin), "version.py")
    with open(path) as f:
        return re.search(r"^__version__\s*=\s*['\"]([^'\"]+)['\"]", f.read(), re.M).group(1)


def _binding_stale() -> bool:
    if _stale(BINDING_OUT, [BINDING, HEADER]) or not os.path.exists(BINDING_TORCH):
        return True
    with open(BINDING_TORCH) as f:
        return f.read() != torch_version()


def _bind(verbose: bool) -> None:
    torch = os.path.dirname(importlib.util.find_spec("torch").origin)
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(nvcc_path())))
    dirs = [os.path.join(torch, "include"), os.path.join(torch, "include", "torch", "csrc", "api", "include"), sysconfig.get_paths()["include"], os.path.join(cuda, "include")]
    # the compiler that nvcc takes too: one that links libstdc++ statically would put a second copy next to torch's
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", *(x for d in dirs for x in ("-isystem", d)), "-o", BINDING_OUT, BINDING,
           "-L" + os.path.join(torch, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if verbose or r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
    if r.returncode != 0:
        raise RuntimeError("g++ failed on serving_binding.cpp")
    with open(BINDING_TORCH, "w") as f:
        f.write(torch_version())


def up_to_date() -> bool:
    return not _stale(OUT, [d for s in UNITS for d in _deps(s)]) and not _binding_stale()


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and up_to_date():
        return OUT
    os.makedirs(OBJ, exist_ok=True)
    todo = [s for s in UNITS if force or _stale(os.path.join(OBJ, s.replace(".cu", ".o")), _deps(s))]
    with ThreadPoolExecutor(max_workers=len(UNITS) + 1) as ex:
        binding = ex.submit(_bind, verbose) if force or _binding_stale() else None
        list(ex.map(lambda s: _compile(s, verbose), todo))
        if binding:
            binding.result()
    objs = [os.path.join(OBJ, s.replace(".cu", ".o")) for s in UNITS]
    r = subprocess.run([nvcc_path(), *ARCH, "-shared", "-o", OUT, *objs], capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError("linking libclusterfusion_b200.so failed")
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
