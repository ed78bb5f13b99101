"""Build ``libhdcmamba_b200.so`` (all CUDA sources under csrc/) for sm_100a with nvcc, and with the
host compiler the Python module ``_host.so`` (csrc/host.cpp, against torch's headers) that calls it.

Both are built in-tree, next to this file, so that they travel with the source tree.  Usage: ``python -m hdcmamba_b200.build [--force] [-j N]``.
"""
import argparse
import concurrent.futures as cf
import os
import platform
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libhdcmamba_b200.so")
HOST = os.path.join(HERE, "_host.so")
HOST_SRC = os.path.join(CSRC, "host.cpp")
OBJ = os.path.join(HERE, "_build")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
         "-DHDC_BUILT_ARCH=100", "-Xptxas", "-warn-spills"]


def nvcc():
    for c in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if c and os.path.exists(c):
            return c
    raise RuntimeError("nvcc not found: the CUDA toolkit is required to build hdcmamba_b200")


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def _deps():
    files = sources() + [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    files.append(HOST_SRC)
    files.append(os.path.join(os.path.dirname(HERE), "include", "hdcmamba_b200.h"))
    files.append(os.path.abspath(__file__))
    return files


def up_to_date():
    if not os.path.exists(LIB) or not os.path.exists(HOST):
        return False
    t = min(os.path.getmtime(LIB), os.path.getmtime(HOST))
    return all(os.path.getmtime(f) <= t for f in _deps() if os.path.exists(f)) and host_matches()


def host_tag():
    """What the host module is compiled against, as it stands in the module."""
    import torch
    return (f"hdcmamba_b200._host for torch {torch.__version__}, C++ ABI {int(torch._C._GLIBCXX_USE_CXX11_ABI)}, "
            f"Python {'.'.join(platform.python_version().split('.')[:2])};")


def host_matches():
    """Whether ``_host.so`` was compiled against this torch and Python; read from the file, since loading another's
    may end in undefined symbols or in objects of another layout."""
    with open(HOST, "rb") as f:
        return host_tag().encode() in f.read()


def host_command(obj):
    """Compile host.cpp, with torch's own headers and C++ ABI."""
    import torch
    root = os.path.join(os.path.dirname(torch.__file__), "include")
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc()))), "include")
    dirs = (root, os.path.join(root, "torch", "csrc", "api", "include"), cuda, sysconfig.get_paths()["include"])
    return ["g++", "-O2", "-std=c++17", "-fPIC", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            f'-DHDC_HOST_TAG="{host_tag()}"', *[f"-I{d}" for d in dirs], "-c", HOST_SRC, "-o", obj], os.path.join(os.path.dirname(torch.__file__), "lib")


def build(force=False, jobs=None, verbose=False, extra=()):
    if not force and up_to_date():
        return LIB
    os.makedirs(OBJ, exist_ok=True)
    cc = nvcc()

    def compile_one(src):
        obj = os.path.join(OBJ, os.path.basename(src) + ".o")
        cmd = [cc, *ARCH, *FLAGS, *extra, "-c", src, "-o", obj]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src}:\n{r.stderr}")
        return obj, r.stderr

    host_obj = os.path.join(OBJ, "host.o")
    host_cmd, torch_lib = host_command(host_obj)

    def compile_host():
        r = subprocess.run(host_cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"g++ failed on {HOST_SRC}:\n{r.stderr}")

    with cf.ThreadPoolExecutor(max_workers=jobs or os.cpu_count() or 4) as ex:
        host = ex.submit(compile_host)
        results = list(ex.map(compile_one, sources()))
        host.result()
    for obj, err in results:
        if verbose and err.strip():
            print(err, file=sys.stderr)
    tmp = LIB + ".tmp"
    cmd = [cc, *ARCH, "-shared", "-o", tmp, *[o for o, _ in results], "-lcudart"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stderr}")
    os.replace(tmp, LIB)
    tmp = HOST + ".tmp"
    cmd = ["g++", "-shared", "-o", tmp, host_obj, f"-L{HERE}", "-l:libhdcmamba_b200.so", f"-L{torch_lib}", "-ltorch_python",
           "-ltorch", "-ltorch_cpu", "-lc10_cuda", "-lc10", "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link of the host module failed:\n{r.stderr}")
    os.replace(tmp, HOST)
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-j", type=int, default=None)
    ap.add_argument("-v", action="store_true", help="print ptxas output (registers / spills)")
    a = ap.parse_args()
    extra = ("-Xptxas", "-v") if a.v else ()
    print(build(force=a.force, jobs=a.j, verbose=a.v, extra=extra))
