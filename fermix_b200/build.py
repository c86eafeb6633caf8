"""Build libfermix_b200.so in-tree for sm_100a (nvcc cross-compiles without a GPU).

Each csrc/*.cu is compiled to an object of its own, in parallel, then linked into one
shared library; csrc/torch_binding.cpp becomes the Python module that binds the operators on
tokens to torch (fermix_torch.so, against the installed torch):

    python -m fermix_b200.build [--force] [-j N]
"""

import concurrent.futures
import glob
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
OUT_DIR = os.path.join(HERE, "_lib")
OBJ_DIR = os.path.join(OUT_DIR, "obj")
OUT = os.path.join(OUT_DIR, "libfermix_b200.so")
BINDING = os.path.join(CSRC, "torch_binding.cpp")
BINDING_OBJ = os.path.join(OBJ_DIR, "torch_binding.o")
BINDING_OUT = os.path.join(OUT_DIR, "fermix_torch.so")
BINDING_FOR = BINDING_OUT + ".for"  # the torch and the Python that it was built for
INCLUDE = os.path.join(ROOT, "include")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", *ARCH, "-lineinfo", "-Xcompiler", "-fPIC"]


def _nvcc():
    for c in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if c and (os.path.sep not in c or os.path.exists(c)):
            return c
    return "nvcc"


def units():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def headers():
    return sorted(glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.inl")) +
                  glob.glob(os.path.join(INCLUDE, "*.h")))


def sources():
    return units() + headers()


def _obj(cu):
    return os.path.join(OBJ_DIR, os.path.basename(cu)[:-3] + ".o")


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _binding_deps():
    return [BINDING, os.path.abspath(__file__)] + glob.glob(os.path.join(INCLUDE, "*.h"))


def _installed():
    import torch

    return f"torch {torch.__version__}, C++11 ABI {int(torch.compiled_with_cxx11_abi())}, {sys.implementation.cache_tag}"


def _binding_for():
    try:
        with open(BINDING_FOR) as f:
            return f.read()
    except OSError:
        return None


def up_to_date():
    return (not _stale(OUT, sources() + [os.path.abspath(__file__)]) and not _stale(BINDING_OUT, _binding_deps()) and
            _binding_for() == _installed())


def _run(cmd, name, verbose):
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed on {name}:\n{r.stdout}\n{r.stderr}")
    if verbose and (r.stdout.strip() or r.stderr.strip()):
        print(r.stdout + r.stderr, flush=True)


def _compile_binding(verbose):
    import sysconfig

    import torch

    root = os.path.join(os.path.dirname(torch.__file__), "include")
    cuda = os.path.join(os.path.dirname(os.path.dirname(_nvcc())) if os.path.sep in _nvcc() else "/usr/local/cuda", "include")
    obj = BINDING_OBJ
    _run(["g++", "-O2", "-std=c++17", "-fPIC", "-c", "-DTORCH_EXTENSION_NAME=fermix_torch",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", "-I", INCLUDE, "-isystem", root, "-isystem",
          os.path.join(root, "torch", "csrc", "api", "include"), "-isystem", cuda, "-isystem",
          sysconfig.get_paths()["include"], "-o", obj + ".tmp", BINDING], os.path.basename(BINDING), verbose)
    os.replace(obj + ".tmp", obj)


def _link_binding(verbose):
    import torch

    _run(["g++", "-shared", "-o", BINDING_OUT + ".tmp", BINDING_OBJ,
          "-L", os.path.join(os.path.dirname(torch.__file__), "lib"), "-lc10", "-ltorch", "-ltorch_cpu", "-ltorch_python",
          "-lc10_cuda", "-ltorch_cuda", "-L", OUT_DIR, "-l:libfermix_b200.so", "-Wl,-rpath,$ORIGIN"],
         os.path.basename(BINDING_OUT), verbose)
    os.replace(BINDING_OUT + ".tmp", BINDING_OUT)


def _compile(cu, verbose):
    obj = _obj(cu)
    _run([_nvcc(), *NVCC_FLAGS, "-I", INCLUDE, "-c", "-o", obj + ".tmp", cu], os.path.basename(cu), verbose)
    os.replace(obj + ".tmp", obj)
    return obj


def build(force=False, verbose=False, jobs=None):
    if not force and up_to_date():
        return OUT
    os.makedirs(OBJ_DIR, exist_ok=True)
    hdr = headers() + [os.path.abspath(__file__)]
    todo = [cu for cu in units() if force or _stale(_obj(cu), [cu] + hdr)]
    other = _binding_for() != _installed()  # until a module of the installed torch is linked
    bind = force or other or _stale(BINDING_OBJ, _binding_deps())
    jobs = jobs or max(1, min(len(todo) + bind, os.cpu_count() or 1))
    with concurrent.futures.ThreadPoolExecutor(max_workers=jobs) as ex:
        work = [ex.submit(_compile_binding, verbose)] if bind else []
        work += [ex.submit(_compile, cu, verbose) for cu in todo]
        for f in work:
            f.result()
    # what a call that failed half way has left is linked by the next: by the objects' times, not by what this call compiled
    objs = [_obj(cu) for cu in units()]
    if force or _stale(OUT, objs + sources()):
        _run([_nvcc(), *ARCH, "-shared", "-Xcompiler", "-fPIC", "-o", OUT + ".tmp", *objs], os.path.basename(OUT), verbose)
        os.replace(OUT + ".tmp", OUT)
    if force or other or _stale(BINDING_OUT, [BINDING_OBJ] + _binding_deps()):
        _link_binding(verbose)
        with open(BINDING_FOR, "w") as f:
            f.write(_installed())
    return OUT


if __name__ == "__main__":
    j = None
    if "-j" in sys.argv:
        j = int(sys.argv[sys.argv.index("-j") + 1])
    print(build(force="--force" in sys.argv, verbose=True, jobs=j))
