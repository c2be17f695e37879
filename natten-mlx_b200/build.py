"""Build ``libnatten_b200.so`` in-tree with nvcc for sm_100a.

    python natten-mlx_b200/build.py [--force] [--verbose]

Each ``csrc/*.cu`` is compiled to an object (in parallel, skipped when the
object is newer than every source and header) and linked into
``natten_mlx_b200/libnatten_b200.so``.  ``csrc/torch_binding.cpp`` becomes the extension module
``natten_mlx_b200/_torch_binding.*.so``, against the headers of the torch that runs the build.  No GPU is needed to build.
"""

from __future__ import annotations

import concurrent.futures
import glob
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "build")
OUT = os.path.join(HERE, "natten_mlx_b200", "libnatten_b200.so")
BINDING = os.path.join(HERE, "natten_mlx_b200", "_torch_binding" + sysconfig.get_config_var("EXT_SUFFIX"))
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
         "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr"] + os.environ.get("NATTEN_B200_NVCC_FLAGS", "").split()


def _newest(paths):
    return max(os.path.getmtime(p) for p in paths)


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(OBJ, exist_ok=True)
    sources = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    headers = (glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.inc")) +
               glob.glob(os.path.join(HERE, "..", "include", "*.h")))
    dep_time = _newest(headers) if headers else 0.0

    def compile_one(src):
        obj = os.path.join(OBJ, os.path.basename(src)[:-3] + ".o")
        if not force and os.path.exists(obj) and os.path.getmtime(obj) > max(os.path.getmtime(src), dep_time):
            return obj, ""
        cmd = [NVCC] + FLAGS + (["-Xptxas", "-v"] if verbose else []) + ["-c", src, "-o", obj]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src}:\n{r.stdout}\n{r.stderr}")
        return obj, r.stderr

    with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, len(sources))) as pool:
        results = list(pool.map(compile_one, sources))
    objs = [o for o, _ in results]
    if verbose:
        for _, log in results:
            sys.stderr.write(log)
    if force or not os.path.exists(OUT) or os.path.getmtime(OUT) < _newest(objs):
        cmd = [NVCC, "-shared", "-o", OUT] + objs + ["-gencode", "arch=compute_100a,code=sm_100a"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    build_binding(force)
    return OUT


def build_binding(force: bool = False) -> str:
    """The torch side of the operators that have one; rebuilt when its source, the C header or torch changed."""
    import torch
    from torch.utils.cpp_extension import include_paths

    src = os.path.join(CSRC, "torch_binding.cpp")
    stamp = os.path.join(OBJ, "torch_binding.version")
    version = torch.__version__ + "\n" + sys.version
    newest = _newest([src] + glob.glob(os.path.join(HERE, "..", "include", "*.h")))
    old = open(stamp).read() if os.path.exists(stamp) else ""
    if not force and old == version and os.path.exists(BINDING) and os.path.getmtime(BINDING) > newest:
        return BINDING
    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    includes = include_paths() + [sysconfig.get_paths()["include"], os.path.join(os.path.dirname(NVCC), "..", "include")]
    # the host compiler that nvcc takes, and so the system's C++ runtime, which torch shares: one that links its own
    # copy in (a CXX of another toolchain may) breaks the first stream of a number
    cmd = (["g++", "-shared", "-fPIC", "-O2", "-std=c++17", "-fvisibility=hidden",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
           + [a for p in includes for a in ("-isystem", p)] + [src, "-o", BINDING]
           + [f"-L{lib}", "-ltorch", "-ltorch_cpu", "-ltorch_python", "-lc10", "-lc10_cuda", "-ldl"])
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed on {src}:\n{r.stdout}\n{r.stderr}")
    with open(stamp, "w") as fh:
        fh.write(version)
    return BINDING


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
