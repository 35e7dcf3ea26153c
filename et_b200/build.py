"""Builds libet_b200.so (the C-ABI library: hand-written sm_100a kernels + host C++) in-tree with nvcc, and _binding.so (Python's fast way to some of its entry points) with g++."""
import importlib.util
import os
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


BINDING = os.path.join(HERE, "_binding.so")


def needs_build():
    if not os.path.exists(LIB) or not os.path.exists(BINDING):
        return True
    t = min(os.path.getmtime(LIB), os.path.getmtime(BINDING))
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC)] + [
        os.path.join(HERE, "..", "include", "et_b200.h"), os.path.abspath(__file__)]
    return any(os.path.getmtime(d) > t for d in deps)


def build_binding():
    torch = os.path.dirname(importlib.util.find_spec("torch").origin)
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    include = [sysconfig.get_paths()["include"], os.path.join(torch, "include"), os.path.join(torch, "include", "torch", "csrc", "api", "include"), os.path.join(cuda, "include")]
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall"] + ["-I" + i for i in include] + [os.path.join(CSRC, "binding.cpp"), "-o", BINDING, "-L" + os.path.join(torch, "lib")] + \
        ["-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("g++ failed building _binding.so")


def build(force=False, verbose=False):
    if not force and not needs_build():
        return LIB
    cmd = ["nvcc"] + FLAGS + (["-Xptxas", "-v"] if verbose else []) + \
        ["-o", LIB] + [os.path.join(CSRC, s) for s in SOURCES]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("nvcc failed building libet_b200.so")
    if verbose:
        print(res.stderr)
    build_binding()
    return LIB


if __name__ == "__main__":
    print(build(force=True, verbose="-v" in sys.argv))
