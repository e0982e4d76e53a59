"""Build the native library ``libkvs_b200.so`` in-tree.

Every ``.cu`` file under ``csrc/`` is compiled by nvcc for sm_100a only
(``-gencode arch=compute_100a,code=sm_100a``), every ``.cpp`` by g++, and the
objects are linked by nvcc with a static CUDA runtime.  The library has no
link-time dependency on ``libcuda``: driver entry points (tensor-map
encoding) are fetched at run time with ``cudaGetDriverEntryPoint``, so the
library also loads on machines without a GPU driver (its CPU codec then
works and its device entry points return errors).

``csrc/torch/*.cpp`` (host code that takes torch tensors) is compiled against
this interpreter's torch into a second module, ``_paged_ops`` with the
interpreter's suffix, linked to the library next to it.  Without a torch for
CUDA it is left out, with a warning: the library does not need one.

Usage: ``python -m kvserve_hpdps_b200.ops.build [-v] [--force]``.
Objects go to ``ops/_build/``; rebuilding is incremental on file mtimes.
"""

from __future__ import annotations

import argparse
import concurrent.futures as cf
import glob
import os
import shutil
import subprocess
import sys
import sysconfig
import warnings

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
LIB_NAME = "libkvs_b200.so"
LIB_PATH = os.path.join(HERE, LIB_NAME)
BIND_NAME = "_paged_ops"
BIND_PATH = os.path.join(HERE, BIND_NAME + sysconfig.get_config_var("EXT_SUFFIX"))

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def _cuda_home() -> str:
    for cand in (os.environ.get("CUDA_HOME"), "/usr/local/cuda"):
        if cand and os.path.exists(os.path.join(cand, "bin", "nvcc")):
            return cand
    nvcc = shutil.which("nvcc")
    if nvcc:
        return os.path.dirname(os.path.dirname(nvcc))
    raise RuntimeError("nvcc not found (set CUDA_HOME)")


def _headers() -> list[str]:
    return sorted(glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.h")))


def _stale(obj: str, src: str, deps: list[str]) -> bool:
    if not os.path.exists(obj):
        return True
    t = os.path.getmtime(obj)
    return any(os.path.getmtime(p) > t for p in [src] + deps)


def _compile(src: str, obj: str, cuda: str, verbose: bool) -> tuple[str, str]:
    if src.endswith(".cu"):
        cmd = [os.path.join(cuda, "bin", "nvcc"), *ARCH_FLAGS, "-O3", "-lineinfo", "-std=c++17",
               "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr", "-I", CSRC, "-c", src, "-o", obj]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
    else:
        cmd = ["g++", "-O3", "-fPIC", "-std=c++17", "-pthread", "-I", CSRC,
               "-I", os.path.join(cuda, "include"), "-c", src, "-o", obj]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"compile failed: {' '.join(cmd)}\n{res.stdout}\n{res.stderr}")
    return src, (res.stdout + res.stderr)


def _no_bindings() -> str | None:
    """Why the torch module cannot be built here; None if it can."""
    try:
        import torch
    except ImportError as e:
        return f"torch cannot be imported ({e})"
    if torch.version.cuda is None:
        return f"torch {torch.__version__} is not built for CUDA"
    return None


def _build_bindings(jobs: int, force: bool) -> str:
    """Compile csrc/torch/*.cpp against torch and link it to the library."""
    import torch
    from torch.utils import cpp_extension
    srcs = sorted(glob.glob(os.path.join(CSRC, "torch", "*.cpp")))
    deps = _headers()
    objs, todo = [], []
    flags = [f"-DTORCH_EXTENSION_NAME={BIND_NAME}", "-DTORCH_API_INCLUDE_EXTENSION_H",
             f'-DKVS_TORCH_VERSION="{torch.__version__}"',
             f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
    incs = cpp_extension.include_paths("cuda") + [sysconfig.get_paths()["include"]]
    made_for = f"{torch.__version__}_{sysconfig.get_config_var('SOABI')}"
    for src in srcs:
        obj = os.path.join(BUILD, f"torch_{made_for}_{os.path.basename(src)}.o")
        objs.append(obj)
        if force or _stale(obj, src, deps):
            todo.append(["g++", "-O2", "-fPIC", "-std=c++17", "-fvisibility=hidden", *flags,
                         *[x for i in incs for x in ("-isystem", i)], "-c", src, "-o", obj])

    def run(cmd):
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"failed: {' '.join(cmd)}\n{res.stdout}\n{res.stderr}")
    with cf.ThreadPoolExecutor(max_workers=jobs) as ex:
        list(ex.map(run, todo))
    # What the module was linked for: an older object of another torch is no newer than it.
    stamp = os.path.join(BUILD, BIND_NAME + ".made_for")
    if os.path.exists(stamp):
        with open(stamp) as f:
            last = f.read()
    else:
        last = None
    if todo or last != made_for or not os.path.exists(BIND_PATH) or any(
            os.path.getmtime(o) > os.path.getmtime(BIND_PATH) for o in objs):
        libdir = cpp_extension.library_paths("cuda")[0]
        tmp = BIND_PATH + ".tmp"
        run(["g++", "-shared", "-o", tmp, *objs, f"-L{HERE}", f"-l:{LIB_NAME}",
             "-Wl,-rpath,$ORIGIN", f"-L{libdir}", "-lc10", "-lc10_cuda", "-ltorch_cpu",
             "-ltorch_cuda", "-ltorch", "-ltorch_python"])
        os.replace(tmp, BIND_PATH)
        with open(stamp, "w") as f:
            f.write(made_for)
    return BIND_PATH


def _build_library(verbose: bool, force: bool, jobs: int | None) -> None:
    cuda = _cuda_home()
    os.makedirs(BUILD, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cpp")))
    deps = _headers()
    todo = []
    objs = []
    for s in srcs:
        o = os.path.join(BUILD, os.path.basename(s) + ".o")
        objs.append(o)
        if force or _stale(o, s, deps):
            todo.append((s, o))
    if todo:
        with cf.ThreadPoolExecutor(max_workers=jobs or min(8, os.cpu_count() or 4)) as ex:
            futs = [ex.submit(_compile, s, o, cuda, verbose) for s, o in todo]
            for f in cf.as_completed(futs):
                src, log = f.result()
                if verbose and log.strip():
                    print(f"--- {os.path.basename(src)}\n{log}")
    if todo or force or not os.path.exists(LIB_PATH) or any(
            os.path.getmtime(o) > os.path.getmtime(LIB_PATH) for o in objs):
        tmp = LIB_PATH + ".tmp"
        cmd = [os.path.join(cuda, "bin", "nvcc"), *ARCH_FLAGS, "-shared", "-o", tmp, *objs,
               "-cudart", "static", "-lpthread"]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"link failed: {' '.join(cmd)}\n{res.stdout}\n{res.stderr}")
        os.replace(tmp, LIB_PATH)


def build(verbose: bool = False, force: bool = False, jobs: int | None = None) -> str:
    """Compile and link; returns the library path."""
    _build_library(verbose, force, jobs)
    why = _no_bindings()
    if why is None:
        _build_bindings(jobs or min(8, os.cpu_count() or 4), force)
    else:
        warnings.warn(f"built without the paged-cache operators: {why}", stacklevel=2)
    return LIB_PATH


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("-v", "--verbose", action="store_true", help="ptxas -v and compiler output")
    ap.add_argument("--force", action="store_true")
    args = ap.parse_args(argv)
    path = build(verbose=args.verbose, force=args.force)
    print(path)
    return 0


if __name__ == "__main__":
    sys.exit(main())
