"""Builds libtbe_b200.so (the C-ABI library declared in include/tbe_b200.h) with nvcc for sm_100a.

Run as ``python -m sparse_ads_baselines_b200.build`` or call :func:`build`.  Each ``csrc/*.cu`` is
compiled to an object file (in parallel, skipped when up to date) and linked into
``sparse_ads_baselines_b200/libtbe_b200.so``; the CUDA runtime is linked statically so the library
depends on nothing but the driver.  ``csrc/torch_glue.cpp`` -- the PyTorch side of expert routing and
gradient clipping -- becomes the extension module ``_torch_glue.so`` beside it, linked to that library and
to the PyTorch that builds it; without PyTorch it is left out.
"""
import concurrent.futures
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "build")
LIB = os.path.join(HERE, "libtbe_b200.so")
GLUE = os.path.join(HERE, "_torch_glue.so")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "--expt-relaxed-constexpr",
    "-Xcompiler", "-fPIC",
    "-Xcompiler", "-fvisibility=hidden",
]


def _nvcc():
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(exe):
        raise RuntimeError("nvcc not found; libtbe_b200.so cannot be built")
    return exe


def _newer(target, deps):
    if not os.path.exists(target):
        return False
    t = os.path.getmtime(target)
    return all(os.path.getmtime(d) <= t for d in deps)


def _build_glue(force):
    try:
        import torch
    except ImportError as e:  # a host without PyTorch binds the C library
        sys.stderr.write("PyTorch cannot be imported (%s): _torch_glue.so is not built\n" % e)
        return
    from torch.utils import cpp_extension
    src = os.path.join(CSRC, "torch_glue.cpp")
    header = os.path.join(HERE, "..", "include", "tbe_b200.h")
    if not force and _newer(GLUE, [src, header, os.path.abspath(__file__), torch.__file__]):
        return
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(_nvcc())))
    includes = cpp_extension.include_paths() + [os.path.join(cuda, "include"), sysconfig.get_paths()["include"]]
    cmd = (["g++", "-shared", "-fPIC", "-O2", "-std=c++17", "-fvisibility=hidden", "-w",
            "-D_GLIBCXX_USE_CXX11_ABI=%d" % torch._C._GLIBCXX_USE_CXX11_ABI, src, "-o", GLUE]
           + [f for p in includes for f in ("-isystem", p)]
           + [f for p in cpp_extension.library_paths() for f in ("-L" + p,)]
           + ["-L" + HERE, "-l:" + os.path.basename(LIB), "-Wl,-rpath,$ORIGIN",
              "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10_cuda", "-lc10"])
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("g++ failed for torch_glue.cpp:\n%s\n%s" % (r.stdout, r.stderr))


def build(verbose=False, force=False, ptxas_info=False):
    os.makedirs(OBJ, exist_ok=True)
    nvcc = _nvcc()
    sources = sorted(f for f in os.listdir(CSRC) if f.endswith(".cu"))
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cuh")]
    headers.append(os.path.join(HERE, "..", "include", "tbe_b200.h"))
    headers.append(os.path.abspath(__file__))

    def compile_one(src):
        obj = os.path.join(OBJ, src[:-3] + ".o")
        path = os.path.join(CSRC, src)
        if not force and _newer(obj, [path] + headers):
            return obj, ""
        cmd = [nvcc] + NVCC_FLAGS + (["-Xptxas", "-v"] if ptxas_info else []) + ["-c", path, "-o", obj]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("nvcc failed for %s:\n%s\n%s" % (src, r.stdout, r.stderr))
        return obj, r.stderr

    with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, len(sources))) as pool:
        results = list(pool.map(compile_one, sources))
    objs = [o for o, _ in results]
    if verbose or ptxas_info:
        for _, log in results:
            if log:
                sys.stderr.write(log)
    if force or not _newer(LIB, objs):
        cmd = [nvcc, "-shared", "-o", LIB] + objs + ["-gencode", "arch=compute_100a,code=sm_100a",
                                                     "-cudart", "static", "-Xcompiler", "-fPIC"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("link failed:\n%s\n%s" % (r.stdout, r.stderr))
    _build_glue(force)
    return LIB


if __name__ == "__main__":
    print(build(verbose=True, force="--force" in sys.argv, ptxas_info="--ptxas" in sys.argv))
