"""Build the HIP engine (gfx950) in-tree: fable5_llm_amd/libfable5_w4a8.so.

    python -m fable5_llm_amd.build

The library is a plain C-ABI shared object (include/fable5_w4a8.h) linked
against the HIP runtime only; Python reaches it through ctypes.
"""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libfable5_w4a8.so")
SOURCES = ["w4a8_kernels.hip", "w4a8_stream.hip", "w4a8_mfma.hip", "w4a8_topk.hip",
           "w4a8_kv.hip", "w4a8_attend.hip", "w4a8_chunk.hip", "w4a8_rotary.hip",
           "w4a8_logprobs.hip", "w4a8_delta.hip", "w4a8_abi.hip"]
ARCH = os.environ.get("FABLE5_OFFLOAD_ARCH", "gfx950")


def hipcc():
    for c in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", "hipcc"):
        if c and (os.path.sep not in c or os.path.exists(c)):
            return c
    return "hipcc"


def flags():
    return [f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC",
            "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
            "-Wall", "-Wno-unused-result", f"-I{os.path.join(ROOT, 'include')}"]


def build(verbose=False):
    """Compile every source to an object, then link the shared library."""
    objdir = os.path.join(ROOT, "_build", "hip")
    os.makedirs(objdir, exist_ok=True)
    objs = []
    for s in SOURCES:
        src = os.path.join(CSRC, s)
        obj = os.path.join(objdir, s + ".o")
        cmd = [hipcc()] + flags() + ["-c", src, "-o", obj]
        _run(cmd, verbose)
        objs.append(obj)
    tmp = LIB + ".tmp"
    _run([hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", tmp] + objs,
         verbose)
    os.replace(tmp, LIB)
    return LIB


def _run(cmd, verbose):
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT,
                       text=True)
    out = "\n".join(l for l in r.stdout.splitlines()
                    if "packed-fp32-ops" not in l)
    if r.returncode != 0:
        raise RuntimeError(f"build failed: {' '.join(cmd)}\n{out}")
    if verbose and out.strip():
        print(out)


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
