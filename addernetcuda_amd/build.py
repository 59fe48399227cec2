"""Build libaddernet_hip.so for gfx950 with plain hipcc (no hipify), and beside it the host module _nodes.so.

The library has a C ABI (include/addernet_hip.h) and links only the HIP
runtime, so the Python side can load it with ctypes.  _nodes.so (csrc/nodes*.cpp) is host code on torch's C++ interface that calls the library
by the addresses it is given.
"""
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libaddernet_hip.so")
NODES = os.path.join(HERE, "_nodes.so")
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
SOURCES = ["api.hip", "fwd.hip", "fwd_nine.hip", "fwd_tap.hip", "fwd_tile.hip", "grad_x.hip", "grad_x_nine.hip", "grad_x_s2.hip", "grad_x_tap.hip", "grad_w.hip", "grad_w_mfma.hip", "grad_w_i8.hip", "conv1x1.hip", "col.hip", "bn_act.hip", "head.hip", "sgd.hip", "api_layers.hip", "layer_norm.hip", "linear.hip", "linear_stream.hip", "linear_staged.hip", "linear_rows.hip", "adamw.hip", "api_blocks.hip", "rms_norm.hip", "fp8.hip", "fp8_product.hip", "gated.hip", "distill.hip"]
NODE_SOURCES = ["nodes.cpp", "nodes_blocks.cpp"]
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-fvisibility=hidden",
    # keep hipcc from forming packed fp32 instructions out of scalar float code
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall", "-Wno-unused-function",
]


def _compile(src, verbose):
    obj = os.path.join(CSRC, src.replace(".hip", ".o"))
    cmd = [HIPCC, *FLAGS, "-c", os.path.join(CSRC, src), "-o", obj]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    out = "\n".join(l for l in r.stdout.splitlines() if "packed-fp32-ops" not in l)
    if r.returncode:
        raise RuntimeError(f"hipcc failed on {src}:\n{out}")
    if out.strip() and verbose:
        print(out)
    return obj


def _build_nodes(verbose):
    import sysconfig
    from torch.utils import cpp_extension
    includes = [*cpp_extension.include_paths(), os.path.join(ROCM, "include"), sysconfig.get_paths()["include"]]
    libs = cpp_extension.library_paths()
    cmd = ["g++", "-std=c++17", "-O2", "-fPIC", "-shared", "-fvisibility=hidden", "-Wall", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
           *[a for i in includes for a in ("-isystem", i)], *[os.path.join(CSRC, f) for f in NODE_SOURCES], "-o", NODES,
           *["-L" + d for d in libs], "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_hip"]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if r.returncode:
        raise RuntimeError(f"g++ failed on {', '.join(NODE_SOURCES)}:\n{r.stdout}")
    return NODES


def build(verbose=False, jobs=4):
    with ThreadPoolExecutor(max_workers=jobs) as ex:
        nodes = ex.submit(_build_nodes, verbose)
        objs = list(ex.map(lambda s: _compile(s, verbose), SOURCES))
    cmd = [HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB, *objs]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    nodes.result()   # (an error here leaves the library, which does without)
    return LIB


if __name__ == "__main__":
    build(verbose="-q" not in sys.argv)
    print("built", LIB)
