"""Build recipe for the sm_100a C-ABI library ``compressai_b200/lib/libvq2_b200.so``.

Every ``csrc/*.cu`` is compiled by nvcc for ``sm_100a`` only (no PTX for other targets) and
linked into one shared library with a static CUDA runtime; the library exports only the
``vq2_*`` symbols declared in ``include/vq2_b200.h``. Object files are cached under
``compressai_b200/_build`` and rebuilt when a source or header is newer.

``csrc/attention_host.cpp``, the host side of ``compressai_b200.attention``, is compiled by g++
against the installed torch into ``lib/_attention_host.so`` beside it.

Usage: python -m compressai_b200.build [--force] [--jobs N]
"""
import argparse
import concurrent.futures as cf
import glob
import os
import shutil
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(REPO, "include")
BUILD = os.path.join(PKG, "_build")
LIBDIR = os.path.join(PKG, "lib")
LIB = os.path.join(LIBDIR, "libvq2_b200.so")
HOST = os.path.join(LIBDIR, "_attention_host.so")
HOST_STAMP = os.path.join(BUILD, "attention_host.key")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC,-fvisibility=hidden",
              "--expt-relaxed-constexpr", "-Xptxas", "-v", "-DVQ2_BUILD"]


def nvcc():
    p = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(p):
        raise RuntimeError("nvcc not found; the CUDA toolkit is required to build compressai_b200")
    return p


def _headers():
    return glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(INCLUDE, "*.h"))


def _stale(obj, src):
    if not os.path.exists(obj):
        return True
    t = os.path.getmtime(obj)
    return any(os.path.getmtime(f) > t for f in [src] + _headers())


def _compile(src, force):
    obj = os.path.join(BUILD, os.path.basename(src) + ".o")
    log = obj + ".ptxas.txt"
    if not force and not _stale(obj, src):
        return obj, None
    cmd = [nvcc(), *ARCH, *NVCC_FLAGS, "-I", INCLUDE, "-I", CSRC, "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src}:\n{r.stdout}\n{r.stderr}")
    with open(log, "w") as f:
        f.write(r.stderr)
    return obj, log


def _host_key():
    """What the host module is compiled against, beside the sources: the interpreter's ABI and torch's."""
    import sysconfig

    import torch
    return f"{sysconfig.get_config_var('EXT_SUFFIX')} torch {torch.__version__}"


def _host_stale(src):
    try:
        with open(HOST_STAMP) as f:
            return f.read() != _host_key() or _stale(HOST, src)
    except FileNotFoundError:
        return True


def _build_host(force):
    """lib/_attention_host.so: a CPython module over torch's C++ headers; rebuilt when torch changes too."""
    import sysconfig

    import torch
    src = os.path.join(CSRC, "attention_host.cpp")
    if not force and not _host_stale(src):
        return HOST
    root = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(nvcc()))
    tmp = HOST + ".tmp"
    cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I", INCLUDE,
           "-I", sysconfig.get_paths()["include"], "-isystem", os.path.join(root, "include"),
           "-isystem", os.path.join(root, "include", "torch", "csrc", "api", "include"),
           "-isystem", os.path.join(cuda, "include"), src, "-o", tmp, "-L", os.path.join(root, "lib"),
           "-ltorch_python", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for {src}:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, HOST)
    with open(HOST_STAMP, "w") as f:
        f.write(_host_key())
    return HOST


def build(force=False, jobs=None):
    """Compile every csrc/*.cu for sm_100a and link lib/libvq2_b200.so (returned), and lib/_attention_host.so."""
    os.makedirs(BUILD, exist_ok=True)
    os.makedirs(LIBDIR, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    jobs = jobs or min(len(srcs), os.cpu_count() or 4)
    with cf.ThreadPoolExecutor(jobs + 1) as ex:
        host = ex.submit(_build_host, force)
        objs = [o for o, _ in ex.map(lambda s: _compile(s, force), srcs)]
        host.result()
    if force or not os.path.exists(LIB) or any(os.path.getmtime(o) > os.path.getmtime(LIB) for o in objs):
        tmp = LIB + ".tmp"
        cmd = [nvcc(), *ARCH, "-shared", "-cudart", "static", "-o", tmp, *objs]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
        os.replace(tmp, LIB)
    return LIB


def main(argv=None):
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--jobs", type=int, default=None)
    a = ap.parse_args(argv)
    print(build(force=a.force, jobs=a.jobs))


if __name__ == "__main__":
    sys.exit(main())
