"""Builds the package's CUDA library (reworld_b200/_lib/libreworld_b200.so) for sm_100a.

Each .cu file under csrc/ is compiled with nvcc for `-gencode
arch=compute_100a,code=sm_100a` and the objects are linked into one shared
library that the package loads with ctypes.  csrc/paged_bind.cpp (argument checks
of paged.py on torch's C++ tensors, no device code) becomes a Python module beside
it, linked to that library.  Run `python reworld_b200/build.py`
(by path: importing the package requires the library to exist) or call build().
"""
import concurrent.futures
import importlib.util
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT_DIR = os.path.join(HERE, "_lib")
LIB_NAME = "libreworld_b200.so"
BIND_NAME = "paged_bind.so"
CXX = os.environ.get("CXX", "g++")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr"]


def _sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def _newest_input_mtime():
    files = [os.path.join(CSRC, f) for f in os.listdir(CSRC)]
    files.append(os.path.join(HERE, "..", "include", "reworld_b200.h"))
    files.append(os.path.abspath(__file__))
    return max(os.path.getmtime(f) for f in files if os.path.exists(f))


def lib_path():
    return os.path.join(OUT_DIR, LIB_NAME)


def bind_path():
    return os.path.join(OUT_DIR, BIND_NAME)


def bind_stamp_path():
    return bind_path() + ".for"


def _torch_dir():
    # found, not imported: a build needs torch's headers and libraries only
    return list(importlib.util.find_spec("torch").submodule_search_locations)[0]


def bind_stamp():
    """What paged_bind.so is made for: torch's C++ interface and Python's differ from one version to the next."""
    version = {}
    with open(os.path.join(_torch_dir(), "version.py")) as f:
        exec(f.read(), version)
    return f"torch {version['__version__']} {sysconfig.get_config_var('SOABI')}"


def bind_made_for():
    """The stamp beside paged_bind.so, or None."""
    try:
        with open(bind_stamp_path()) as f:
            return f.read()
    except OSError:
        return None


def _compile_bind(obj):
    """Compiles paged_bind.cpp to `obj` and returns the command that links it."""
    torch_dir = _torch_dir()
    inc = os.path.join(torch_dir, "include")
    lib = os.path.join(torch_dir, "lib")
    cuda = os.path.join(os.path.dirname(os.path.dirname(NVCC)), "include")
    cmd = [CXX, "-O2", "-std=c++20", "-fPIC", "-fvisibility=hidden", "-Wall", "-Wextra", "-c", os.path.join(CSRC, "paged_bind.cpp"),
           "-o", obj, "-isystem", inc, "-isystem", os.path.join(inc, "torch", "csrc", "api", "include"), "-isystem", cuda,
           "-isystem", sysconfig.get_paths()["include"]]
    _run(cmd)
    return [CXX, "-shared", "-o", bind_path() + ".tmp", obj, "-L" + lib, "-ltorch_python", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda",
           "-L" + OUT_DIR, "-lreworld_b200",
           # the C++ and CUDA runtimes that torch loads: a second, static C++ runtime (a compiler that comes with
           # libstdc++.a alone takes that) is mixed with torch's, and the first formatted message ends the process
           "-l:libstdc++.so.6", "-Wl,--copy-dt-needed-entries", "-Wl,-rpath," + lib, "-Wl,-rpath,$ORIGIN"]


def _run(cmd):
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{' '.join(cmd)} failed:\n{r.stdout}\n{r.stderr}")
    sys.stderr.write(r.stderr)                           # warnings


def build(force=False, verbose=False):
    """Compiles csrc/*.cu into _lib/libreworld_b200.so and csrc/paged_bind.cpp into
    _lib/paged_bind.so (skipped when up to date: newer than the sources, and the second
    one made for this torch and Python)."""
    os.makedirs(OUT_DIR, exist_ok=True)
    out = lib_path()
    newest = _newest_input_mtime()
    if (not force and all(os.path.exists(f) and os.path.getmtime(f) >= newest for f in (out, bind_path()))
            and bind_made_for() == bind_stamp()):
        return out
    objs = []

    def compile_one(src):
        obj = os.path.join(OUT_DIR, os.path.basename(src)[:-3] + ".o")
        cmd = [NVCC, *ARCH, *FLAGS, "-c", src, "-o", obj]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed for {src}:\n{r.stdout}\n{r.stderr}")
        if verbose:
            sys.stdout.write(r.stdout + r.stderr)
        return obj

    with concurrent.futures.ThreadPoolExecutor(max_workers=os.cpu_count() or 4) as ex:
        bind_obj = os.path.join(OUT_DIR, "paged_bind.o")
        bind = ex.submit(_compile_bind, bind_obj)
        objs = list(ex.map(compile_one, _sources()))
    tmp = out + ".tmp"
    cmd = [NVCC, *ARCH, "-shared", "-o", tmp, *objs, "-cudart=static"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, out)
    # (behind the library, which is there whatever becomes of this: it needs no C++ compiler and no torch with CUDA)
    _run(bind.result())
    if os.path.exists(bind_stamp_path()):
        os.remove(bind_stamp_path())
    os.replace(bind_path() + ".tmp", bind_path())
    with open(bind_stamp_path(), "w") as f:
        f.write(bind_stamp())
    for o in objs + [bind_obj]:
        os.remove(o)
    return out


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
