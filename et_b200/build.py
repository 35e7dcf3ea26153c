"""Builds libet_b200.so (the C-ABI library: hand-written sm_100a kernels + host C++) in-tree with nvcc, and, where there is a torch, the extension _binding.*.so (Python's fast way
to some of its entry points) with g++."""
import importlib.util
import os
import re
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libet_b200.so")
SOURCES = ["error.cu", "layernorm.cu", "softmax.cu", "tile_gemm.cu", "attention.cu", "attention_tc.cu", "dense_gemm.cu", "resident_gemm.cu", "formats.cu",
           "encoder.cu", "api.cu", "rotary.cu", "adapter.cu", "adapter_tc.cu", "attention_rules.cu", "attention_rules_tc.cu", "attention_rules_token.cu",
           "rmsnorm.cu", "fp8_gemm.cu", "kv_cache.cu", "attention_tree.cu", "attention_tree_tc.cu"]
FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-lineinfo",
         "--expt-relaxed-constexpr", "-t", "0", "-Xcompiler", "-fPIC", "-Xcompiler", "-Wall", "-shared"]

DEPS = (os.path.join(HERE, "..", "include", "et_b200.h"), os.path.abspath(__file__))


def binding_path():
    """The extension for this Python and this torch, whose objects it reads as they lie in memory: its name says which. None where there is no torch, or not what it is compiled with."""
    spec = importlib.util.find_spec("torch")
    if spec is None or not spec.origin:
        return None
    with open(os.path.join(os.path.dirname(spec.origin), "version.py")) as f:
        version = re.search(r"__version__[^=\n]*= *['\"]([^'\"]+)", f.read())
    return os.path.join(HERE, f"_binding.{sys.implementation.cache_tag}.torch-{version.group(1)}.so") if version else None


def newer(path, deps):
    """Whether the file is there and newer than what it is made from."""
    return os.path.exists(path) and all(os.path.getmtime(d) <= os.path.getmtime(path) for d in deps)


def needs_library():
    return not newer(LIB, [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f != "binding.cpp"] + list(DEPS))


def needs_binding():
    path = binding_path()
    return path is not None and not newer(path, [os.path.join(CSRC, "binding.cpp")] + list(DEPS))


def needs_build():
    return needs_library() or needs_binding()


def build_binding():
    """Compiles the extension. The library does not need it and Python does the same checks without it, so what is missing here ends no build."""
    path = binding_path()
    torch = os.path.dirname(importlib.util.find_spec("torch").origin)
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    include = [sysconfig.get_paths()["include"], os.path.join(torch, "include"), os.path.join(torch, "include", "torch", "csrc", "api", "include"), os.path.join(cuda, "include")]
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall"] + ["-I" + i for i in include] + [os.path.join(CSRC, "binding.cpp"), "-o", path, "-L" + os.path.join(torch, "lib")] + \
        ["-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    for f in os.listdir(HERE):
        if f.startswith("_binding.") and f.endswith(".so"):
            os.remove(os.path.join(HERE, f))
    try:
        res = subprocess.run(cmd, capture_output=True, text=True)
        problem = None if res.returncode == 0 else res.stdout + res.stderr
    except OSError as e:
        problem = f"{e}\n"
    if problem is not None:
        sys.stderr.write(problem + f"{os.path.basename(path)} has not been built: the 8-bit operators' arguments are checked in Python\n")


def build(force=False, verbose=False):
    if force or needs_library():
        cmd = ["nvcc"] + FLAGS + (["-Xptxas", "-v"] if verbose else []) + \
            ["-o", LIB] + [os.path.join(CSRC, s) for s in SOURCES]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            sys.stderr.write(res.stdout + res.stderr)
            raise RuntimeError("nvcc failed building libet_b200.so")
        if verbose:
            print(res.stderr)
    if binding_path() is not None and (force or needs_binding()):
        build_binding()
    return LIB


if __name__ == "__main__":
    print(build(force=True, verbose="-v" in sys.argv))
