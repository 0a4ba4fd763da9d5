"""Build the sm_100a shared library ``unblend_b200/_lib/libunblend_b200.so``.

Every ``csrc/*.cu`` file is compiled with ``nvcc -gencode
arch=compute_100a,code=sm_100a`` and linked into one C-ABI shared library that
the host code loads with ctypes. That needs nvcc alone; where torch, g++ and Python's
headers are installed, ``csrc/tensor_lists.cpp`` becomes a Python extension beside it.
Objects are rebuilt only when a source or header is newer. The FFT twiddle table
(``csrc/twiddle4096.inc``) is generated here in double precision, so the kernels hold
it as static module data.

Usage: ``python -m unblend_b200.build [-j N] [--force]``.
"""

from __future__ import annotations

import argparse
import glob
import math
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
ROOT = os.path.dirname(HERE)
INCLUDE = os.path.join(ROOT, "include")
LIBDIR = os.path.join(HERE, "_lib")
OBJDIR = os.path.join(HERE, "_build")
LIBNAME = "libunblend_b200.so"

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC",
              "-Xptxas", "-v", "--expt-relaxed-constexpr"]


def nvcc() -> str:
    """Path of the nvcc binary."""
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def write_twiddles(n: int = 4096) -> str:
    """Write ``exp(-2 pi i m / n)`` rounded from double to float, one pair per line."""
    path = os.path.join(CSRC, f"twiddle{n}.inc")
    lines = []
    for m in range(n):
        a = -2.0 * math.pi * m / n
        lines.append(f"{{{float.hex(float(_f32(math.cos(a))))}f, {float.hex(float(_f32(math.sin(a))))}f}},")
    text = "// generated by unblend_b200/build.py\n" + "\n".join(lines) + "\n"
    if not os.path.exists(path) or open(path).read() != text:
        with open(path, "w") as f:
            f.write(text)
    return path


def _f32(x: float) -> float:
    import struct

    return struct.unpack("f", struct.pack("f", x))[0]


def source_digest() -> str:
    """SHA-256 over the library's sources (kernels, generated tables, C header), in name order."""
    import hashlib

    files = []
    for pat in ("*.cu", "*.cuh", "*.inc", "*.cpp"):
        files += glob.glob(os.path.join(CSRC, pat))
    files += glob.glob(os.path.join(INCLUDE, "*.h"))
    h = hashlib.sha256()
    for f in sorted(files, key=os.path.basename):
        h.update(os.path.basename(f).encode())
        with open(f, "rb") as fh:
            h.update(fh.read())
    return h.hexdigest()


EXTENSION = "tensor_lists"
STAMP_SUFFIX = ".torch"


def extension_stamp() -> str:
    """What the extension is built for: another torch or Python needs another build."""
    import sysconfig

    import torch

    return f"torch {torch.__version__}, {sysconfig.get_config_var('SOABI')}"


def _extension(force: bool) -> str | None:
    """Build the Python extension against the headers of the installed torch; on a machine that lacks what this needs,
    return what that is (the library and its C interface need none of it)."""
    import sysconfig

    src, out = os.path.join(CSRC, EXTENSION + ".cpp"), os.path.join(LIBDIR, EXTENSION + ".so")
    stamp = out + STAMP_SUFFIX
    cxx = os.environ.get("CXX", "g++")
    try:
        from torch.utils.cpp_extension import include_paths, library_paths

        import torch
    except (ImportError, OSError) as e:  # OSError: a library of its own that does not load
        lacking: str | None = f"torch ({e})"
    else:
        lacking = cxx if shutil.which(cxx) is None else None
        if not os.path.exists(os.path.join(sysconfig.get_path("include"), "Python.h")):
            lacking = "Python.h"
    if lacking is None and not force and os.path.exists(out) and os.path.exists(stamp) and \
            open(stamp).read() == extension_stamp() and os.path.getmtime(out) >= max(os.path.getmtime(src), _deps()):
        return None
    for f in (out, stamp):  # from here on it does not belong to the library
        if os.path.exists(f):
            os.remove(f)
    if lacking is not None:
        return lacking
    cmd = [cxx, "-O2", "-std=c++17", "-shared", "-fPIC", "-Wall",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *(f for p in include_paths() for f in ("-isystem", p)), "-isystem", sysconfig.get_path("include"),
           src, "-o", out + ".tmp", *(f"-L{p}" for p in library_paths()), "-ltorch_python", "-ltorch_cpu", "-lc10"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{cxx} failed for {src}:\n{res.stderr}")
    os.replace(out + ".tmp", out)
    with open(stamp, "w") as f:
        f.write(extension_stamp())
    return None


DIGEST_NAME = "libunblend_b200.digest"


def _deps() -> float:
    files = glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.inc"))
    files += glob.glob(os.path.join(INCLUDE, "*.h"))
    return max((os.path.getmtime(f) for f in files), default=0.0)


def _compile(src: str, force: bool, log: list) -> str:
    obj = os.path.join(OBJDIR, os.path.basename(src).replace(".cu", ".o"))
    if not force and os.path.exists(obj) and os.path.getmtime(obj) >= max(os.path.getmtime(src), _deps()):
        return obj
    cmd = [nvcc(), *ARCH_FLAGS, *NVCC_FLAGS, "-I", INCLUDE, "-c", src, "-o", obj]
    res = subprocess.run(cmd, capture_output=True, text=True)
    log.append((src, res.stdout + res.stderr))
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src}:\n{res.stderr}")
    return obj


def build(force: bool = False, jobs: int = 8, verbose: bool = False) -> str:
    """Compile and link the library, and build the extension beside it where torch, its compiler and Python's headers
    are there; return the library's path."""
    os.makedirs(OBJDIR, exist_ok=True)
    os.makedirs(LIBDIR, exist_ok=True)
    write_twiddles()
    sources = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    log: list = []
    with ThreadPoolExecutor(max_workers=jobs) as ex:
        extension = ex.submit(_extension, force)
        objs = list(ex.map(lambda s: _compile(s, force, log), sources))
    lib = os.path.join(LIBDIR, LIBNAME)
    if force or not os.path.exists(lib) or os.path.getmtime(lib) < max(os.path.getmtime(o) for o in objs):
        cmd = [nvcc(), *ARCH_FLAGS, "-shared", "-Xcompiler", "-fPIC", *objs, "-o", lib + ".tmp", "-lcuda"]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"link failed:\n{res.stderr}")
        os.replace(lib + ".tmp", lib)
    # Stamp the library with the sources it was built from; the loader refuses a
    # library whose stamp differs from the sources next to it.
    with open(os.path.join(LIBDIR, DIGEST_NAME), "w") as f:
        f.write(source_digest() + "\n")
    lacking = extension.result()  # raises after the library is in place
    if lacking is not None:
        print(f"{EXTENSION} not built, {lacking} is missing: the library and its C interface work without it, the rotary "
              "operators, AdamW and the gradient norm of unblend_b200.training do not", file=sys.stderr)
    if verbose:
        for src, text in log:
            print(f"== {os.path.basename(src)}\n{text}")
    return lib


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("-j", type=int, default=os.cpu_count() or 4)
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-v", action="store_true")
    args = ap.parse_args()
    print(build(force=args.force, jobs=args.j, verbose=args.v))


if __name__ == "__main__":
    sys.exit(main())
