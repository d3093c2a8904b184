"""Builds trace_amd/lib/libtrace_hip.so with hipcc for gfx950 (cross-compiles without a GPU).

    python -m trace_amd.build            # rebuild if sources are newer
    python -m trace_amd.build --force
"""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIBDIR = os.path.join(HERE, "lib")
LIB = os.path.join(LIBDIR, "libtrace_hip.so")

# (source, extra flags).  steps/guidance hold the op-exact elementwise chains: no FMA contraction.
# unet.hip: no SLP vectorisation.  With it the two GroupNorm rows a thread owns are summed as v_pk_add_f32
# chains whose operands are v_mov pairs of LDS-returned registers, and on gfx950 lanes 48..63 of those
# sums then differed from run to run (five build variants A/B'd on the box).
# The row sums are additionally fenced in the source (conv_kernels.h), so either guard alone is enough;
# packed fp32 is also an anti-lever beside MFMAs (MI355X_MICROARCH.md).
SOURCES = [
    ("unet.hip", ["-fno-slp-vectorize"]),
    ("steps.hip", ["-ffp-contract=off"]),
    ("guidance.hip", ["-ffp-contract=off"]),
    ("conv2d.hip", ["-fno-slp-vectorize"]),
    ("attention.hip", ["-fno-slp-vectorize"]),
    ("attn_f32.hip", ["-fno-slp-vectorize"]),
    ("attn_bf16.hip", ["-fno-slp-vectorize"]),
    ("attn_f16.hip", ["-fno-slp-vectorize"]),
    ("norm.hip", ["-fno-slp-vectorize"]),
    ("rotary.hip", ["-fno-slp-vectorize"]),
]
# No packed fp32 arithmetic anywhere (v_pk_add / mul / fma_f32): some of its forms give wrong results now and then on
# gfx950, see above.  hipcc's host pass does not know the feature and says so; that warning means nothing.
COMMON = ["--offload-arch=gfx950", "-O3", "-fPIC", "-std=c++17", "-Wall", "-Wno-unused-function",
          "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
          "-I", os.path.join(ROOT, "include"), "-I", CSRC]


def _hipcc():
    for c in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", "hipcc"):
        if c and (os.path.isabs(c) and os.path.exists(c) or not os.path.isabs(c)):
            return c
    raise RuntimeError("hipcc not found")


def _newer(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(not os.path.exists(d) or os.path.getmtime(d) > t for d in deps)


def _stale_object(obj, src):
    """Whether `obj` is older than a file it was made from (the compiler wrote their names beside it)."""
    made_from = obj[:-2] + ".d"
    if not os.path.exists(made_from):
        return True
    names = open(made_from).read().replace("\\\n", " ").split()
    return _newer(obj, [src, os.path.abspath(__file__)] + [n for n in names if n.startswith(ROOT) and n[-1] != ":"])


def build(force=False, verbose=True):
    os.makedirs(LIBDIR, exist_ok=True)
    objdir = os.path.join(LIBDIR, "obj")
    os.makedirs(objdir, exist_ok=True)
    hipcc = _hipcc()
    objs = []
    procs = []
    for src, extra in SOURCES:
        obj = os.path.join(objdir, src.replace(".hip", ".o"))
        objs.append(obj)
        if not force and not _stale_object(obj, os.path.join(CSRC, src)):
            continue
        cmd = [hipcc] + COMMON + extra + ["-MMD", "-MF", obj[:-2] + ".d", "-c", os.path.join(CSRC, src), "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        procs.append((cmd, subprocess.Popen(cmd)))
    for cmd, p in procs:
        if p.wait() != 0:
            raise RuntimeError("compile failed: " + " ".join(cmd))
    if not procs and not _newer(LIB, objs):
        return LIB
    cmd = [hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB] + objs
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv)
    print(LIB)
