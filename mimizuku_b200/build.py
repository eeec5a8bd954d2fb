"""Builds libmimizuku_b200.so in-tree: the sm_100a kernels (nvcc, -gencode arch=compute_100a,code=sm_100a), the C++
engine and CPU stages, linked against cuBLAS with a static CUDA runtime; and, where a torch with CUDA is installed, the
compiled calls over torch tensors (_serving.so).

    python mimizuku_b200/build.py [--force] [-j N]      (by path: importing the package needs the library)

Objects go to mimizuku_b200/_build/; a source is recompiled when it or a header changed.
"""
import argparse
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libmimizuku_b200.so")
CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")
NVCC = os.path.join(CUDA, "bin", "nvcc")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ARCH + ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-Xptxas", "-warn-spills",
                     "--expt-relaxed-constexpr"]
CXX_FLAGS = ["-O3", "-std=c++17", "-fPIC", "-Wall", "-Wno-unused-function", f"-I{CUDA}/include"]

CU = ["runtime.cu", "dec_attn.cu", "enc_attn.cu", "ln.cu", "misc.cu", "cross_noalloc.cu", "align.cu", "dec_linear.cu", "logmel.cu", "logits_argmax.cu", "gemm.cu", "gemv.cu", "kv8.cu", "attn8.cu",
      "logprobs.cu", "linear_logprobs.cu"]
CPP = ["host_cpu.cpp", "engine.cpp", "capi.cpp"]
HEADERS = ["common.cuh", "launch.h", "engine.h", "host_cpu.h", "ln_row.cuh", "gemv_row.cuh", "fp8_cache.cuh", "attn8.h",
           "logprobs.h", "logprobs.cuh"]
# kernels under the reference's own names, as an image its host loads by name (not linked into the library)
DROPIN_SRC = os.path.join(CSRC, "dropin.cu")
DROPIN = os.path.join(HERE, "dropin_sm100a.fatbin")
# the calls over torch tensors: a Python module that links the library (which itself knows nothing of torch or Python)
SERVING_SRC = os.path.join(CSRC, "serving.cpp")
SERVING = os.path.join(HERE, "_serving.so")


def _newest_header():
    paths = [os.path.join(CSRC, h) for h in HEADERS] + [os.path.join(HERE, "..", "include", "mimizuku_b200.h")]
    return max(os.path.getmtime(p) for p in paths if os.path.exists(p))


def _compile(src, force, hdr_time):
    path = os.path.join(CSRC, src)
    obj = os.path.join(BUILD, src + ".o")
    if not force and os.path.exists(obj) and os.path.getmtime(obj) >= max(os.path.getmtime(path), hdr_time):
        return obj, None
    if src.endswith(".cu"):
        cmd = [NVCC] + NVCC_FLAGS + ["-c", path, "-o", obj]
    else:
        cxx = os.environ.get("CXX", "g++")
        extra = ["-ffp-contract=off"] if src == "host_cpu.cpp" else []
        cmd = [cxx] + CXX_FLAGS + extra + ["-c", path, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        return obj, f"{' '.join(cmd)}\n{r.stdout}{r.stderr}"
    return obj, None


def _build_serving(force, hdr, verbose):
    """Compiles _serving.so for the Python and torch that run this. Without torch or a torch with CUDA there is nothing to
    call it with; where it does not compile, the library is whole all the same: a warning, and no module of another torch
    is left behind (importing the calls says what is missing)."""
    torch = importlib.util.find_spec("torch")
    at = torch.submodule_search_locations[0] if torch else None
    if not at or not os.path.exists(os.path.join(at, "lib", "libc10_cuda.so")):
        if verbose:
            print("no torch with CUDA: _serving.so is not built")
        return
    with open(os.path.join(at, "version.py")) as f:  # torch's C++ interface changes with its version
        made_for = f"{sys.version}\n{at}\n{f.read()}"
    stamp = os.path.join(BUILD, "serving.txt")
    if not force and os.path.exists(SERVING) and os.path.getmtime(SERVING) >= max(os.path.getmtime(SERVING_SRC), hdr):
        if os.path.exists(stamp) and open(stamp).read() == made_for:
            return
    cmd = [os.environ.get("CXX", "g++")] + CXX_FLAGS + [
        "-shared", SERVING_SRC, "-o", SERVING + ".tmp", "-I", os.path.join(HERE, "..", "include"),
        "-isystem", sysconfig.get_path("include"), "-isystem", os.path.join(at, "include"),
        "-isystem", os.path.join(at, "include", "torch", "csrc", "api", "include"), f"-L{HERE}",
        "-l:" + os.path.basename(LIB), "-L" + os.path.join(at, "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10_cuda",
        "-lc10", "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        for path in (SERVING, stamp):
            if os.path.exists(path):
                os.remove(path)
        print(f"warning: _serving.so (the calls over torch tensors) is not built:\n{' '.join(cmd)}\n{r.stdout}{r.stderr}",
              file=sys.stderr)
        return
    shutil.move(SERVING + ".tmp", SERVING)
    with open(stamp, "w") as f:
        f.write(made_for)
    if verbose:
        print(f"built {SERVING}")


def build(force=False, jobs=None, verbose=False):
    """Compiles every source and links the library; raises RuntimeError with the compiler output on failure."""
    if not os.path.exists(NVCC):
        raise RuntimeError(f"nvcc not found at {NVCC}")
    os.makedirs(BUILD, exist_ok=True)
    hdr = _newest_header()
    srcs = CU + CPP
    with ThreadPoolExecutor(max_workers=jobs or min(len(srcs), os.cpu_count() or 4)) as ex:
        results = list(ex.map(lambda s: _compile(s, force, hdr), srcs))
    errs = [e for _, e in results if e]
    if errs:
        raise RuntimeError("build failed:\n" + "\n".join(errs))
    objs = [o for o, _ in results]
    if force or not os.path.exists(DROPIN) or os.path.getmtime(DROPIN) < max(os.path.getmtime(DROPIN_SRC), hdr):
        cmd = [NVCC] + ARCH + ["-O3", "-std=c++17", "-lineinfo", "-fatbin", DROPIN_SRC, "-o", DROPIN]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"build failed:\n{' '.join(cmd)}\n{r.stdout}{r.stderr}")
    if force or not os.path.exists(LIB) or os.path.getmtime(LIB) < max(os.path.getmtime(o) for o in objs):
        tmp = LIB + ".tmp"
        cmd = [NVCC] + ARCH + ["-shared", "-o", tmp] + objs + [
            f"-L{CUDA}/lib64", "-lcublas", "-lcublasLt", "-Xlinker", f"-rpath,{CUDA}/lib64", "-cudart", "static"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{' '.join(cmd)}\n{r.stdout}{r.stderr}")
        shutil.move(tmp, LIB)
        if verbose:
            print(f"built {LIB}")
    _build_serving(force, hdr, verbose)
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-j", type=int, default=None)
    a = ap.parse_args()
    try:
        build(a.force, a.j, verbose=True)
    except RuntimeError as e:
        print(e, file=sys.stderr)
        sys.exit(1)
