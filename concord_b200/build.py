"""Build the in-tree CUDA library `concord_b200/_lib/libconcord_b200.so`.

    python -m concord_b200.build

Compiles every .cu file under concord_b200/csrc for sm_100a with nvcc and
links one shared library with a plain C ABI (include/concord_b200.h).  The
step kernels are built with -fmad=false: the reference's arithmetic rounds
every fp32 multiply and add separately, and bit-exact words depend on the
compiler not fusing them.  Also builds the host copy of the correctly
rounded log2/exp2 (libcrmath_check.so) that the CPU tests check, and
`_lib/_native.so`, the Python extension with the training operators' autograd
nodes (csrc/torch_ops.cpp, compiled by g++ against the installed torch and
again when another torch or Python is installed).  Users of the C ABI need
neither: `--library` (build(extension=False)) leaves the extension out.
"""
import glob
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIBDIR = os.path.join(HERE, "_lib")
OUT = os.path.join(LIBDIR, "libconcord_b200.so")
NATIVE = os.path.join(LIBDIR, "_native.so")
STAMP = os.path.join(LIBDIR, "_native.stamp")      # what NATIVE was built for
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVFLAGS = ARCH + ["-O3", "-lineinfo", "-std=c++17", "-fmad=false", "-Xcompiler", "-fPIC",
                  "-Xcompiler", "-ffp-contract=off", "--expt-relaxed-constexpr"]


def _cutlass_root():
    """CUTLASS/CuTe headers (a vendored header tree shipped inside flashinfer)."""
    env = os.environ.get("CUTLASS_DIR")
    if env:
        return env
    import importlib.util
    spec = importlib.util.find_spec("flashinfer")
    if spec is None or not spec.submodule_search_locations:
        raise RuntimeError("CUTLASS headers not found: set CUTLASS_DIR")
    return os.path.join(list(spec.submodule_search_locations)[0], "data", "cutlass")


def _flags_for(cu):
    if os.path.basename(cu) in ("gemm.cu", "convgemm.cu"):
        root = _cutlass_root()
        # tensor-core GEMMs: contraction order is the hardware's; no -fmad=false needed
        return ARCH + ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
                       "-I" + os.path.join(root, "include"),
                       "-I" + os.path.join(root, "tools", "util", "include"),
                       "-DNDEBUG", "-Xcompiler", "-Wno-psabi", "-diag-suppress", "20012"]
    if os.path.basename(cu) in ("norm.cu", "distill.cu", "attention.cu", "embed.cu", "qknorm.cu", "eight.cu",
                                "gemm8.cu"):
        # no reference arithmetic to reproduce: a multiply and an add may become one fma
        return ARCH + ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr"]
    return NVFLAGS


def _newer(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _native_command(src):
    """g++ command of the Python extension: torch's headers and libraries, and
    libconcord_b200 beside it."""
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths, library_paths
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-DTORCH_EXTENSION_NAME=_native",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
    cmd += ["-I" + p for p in include_paths("cuda") + [sysconfig.get_paths()["include"]]]
    cmd += ["-I" + os.path.join(os.path.dirname(os.path.dirname(NVCC)), "include"), src, "-o", NATIVE]
    cmd += ["-L" + LIBDIR, "-lconcord_b200", "-Wl,-rpath,$ORIGIN"] + ["-L" + p for p in library_paths("cuda")]
    return cmd + ["-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python"]


def built_for():
    """The torch and Python that an extension built now works with."""
    import torch
    return f"torch {torch.__version__}, {sys.implementation.cache_tag}"


def stamp():
    """What the extension that is there was built for (None: not known)."""
    try:
        with open(STAMP) as f:
            return f.read().strip()
    except OSError:
        return None


def build(verbose=False, force=False, extension=True):
    os.makedirs(LIBDIR, exist_ok=True)
    objdir = os.path.join(LIBDIR, "obj")
    os.makedirs(objdir, exist_ok=True)
    headers = glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.cuh")) + \
        [os.path.join(HERE, "..", "include", "concord_b200.h")]
    objs = []
    for cu in sorted(glob.glob(os.path.join(CSRC, "*.cu"))):
        obj = os.path.join(objdir, os.path.basename(cu) + ".o")
        objs.append(obj)
        if force or _newer(obj, [cu] + headers):
            cmd = [NVCC] + _flags_for(cu) + ["-c", cu, "-o", obj]
            if verbose:
                print(" ".join(cmd), flush=True)
            subprocess.check_call(cmd)
    if force or _newer(OUT, objs):
        subprocess.check_call([NVCC] + ARCH + ["-shared", "-o", OUT] + objs + ["-lcudart"])
    chk = os.path.join(LIBDIR, "libcrmath_check.so")
    src = os.path.join(CSRC, "crmath_check.cpp")
    if force or _newer(chk, [src, os.path.join(CSRC, "crmath.h")]):
        subprocess.check_call(["g++", "-O2", "-fPIC", "-ffp-contract=off", "-shared", "-o", chk, src])
    if not extension:
        return OUT
    src = os.path.join(CSRC, "torch_ops.cpp")
    if force or stamp() != built_for() or _newer(NATIVE, [src, os.path.join(HERE, "..", "include", "concord_b200.h")]):
        cmd = _native_command(src)
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.check_call(cmd)
        with open(STAMP, "w") as f:
            f.write(built_for() + "\n")
    return OUT


if __name__ == "__main__":
    print(build(verbose=True, force="--force" in sys.argv, extension="--library" not in sys.argv))
