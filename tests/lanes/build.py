"""The attention sources of the library (trace_amd/csrc) compiled for this machine's CPU against hip/hip_runtime.h beside this
file: liblanes.so has the same C entries, on host memory.  Shared memory becomes plain memory in copies of the sources."""
import os
import shutil
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(os.path.dirname(HERE))
CSRC = os.path.join(ROOT, "trace_amd", "csrc")
SOURCES = ["attention.hip", "attn_f32.hip", "attn_bf16.hip", "attn_f16.hip"]
HEADERS = ["common.h", "layer_types.h", "attn_kernels.h", "attn_launch.h"]


def _compiler():
    for c in ("/opt/rocm/llvm/bin/clang++", shutil.which("clang++")):
        if c and os.path.exists(c):
            return c
    raise RuntimeError("clang++ not found (the sources use its vector types)")


def build(to):
    """Compiles into the folder `to`; returns the library's path."""
    csrc = os.path.join(to, "csrc")
    os.makedirs(csrc, exist_ok=True)
    for f in SOURCES + HEADERS:
        text = open(os.path.join(CSRC, f)).read()
        text = text.replace("extern __shared__", "extern").replace("__shared__", "static")
        open(os.path.join(csrc, f), "w").write(text)
    flags = ["-x", "c++", "-std=c++17", "-O1", "-fPIC", "-w", "-mf16c", "-mfma", "-I", HERE, "-I", os.path.join(ROOT, "include"), "-I", csrc]
    jobs, objs = [], []
    for f in [os.path.join(csrc, s) for s in SOURCES] + [os.path.join(HERE, "lanes.cpp")]:
        objs.append(os.path.join(to, os.path.basename(f) + ".o"))
        jobs.append(subprocess.Popen([_compiler()] + flags + ["-c", f, "-o", objs[-1]]))
    if any([p.wait() for p in jobs]):
        raise RuntimeError("the attention sources do not compile for the CPU")
    lib = os.path.join(to, "liblanes.so")
    subprocess.run([_compiler(), "-shared", "-o", lib] + objs, check=True)
    return lib


if __name__ == "__main__":
    import sys
    print(build(sys.argv[1]))
