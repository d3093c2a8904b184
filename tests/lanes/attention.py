"""Attention and its backward pass on the CPU's lanes (hip/hip_runtime.h), every tensor in memory that ends where it may not be
touched.  usage: attention.py LIBRARY, one case a line on stdin as JSON; ends at the first that reads elsewhere or is wrong."""
import ctypes as C
import json
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
sys.path[:0] = [ROOT, os.path.join(ROOT, "tests")]

import test_gpu_layers as formulas
from attention_formulas import backward64, forward64
from trace_amd import _cabi

formulas.DEV = "cpu"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


class Lanes:
    def __init__(self, path):
        self.lib = C.CDLL(path)
        self.lib.lanes_alloc.restype, self.lib.lanes_alloc.argtypes = C.c_void_p, [C.c_size_t, C.c_int]
        self.lib.lanes_error.restype = C.c_char_p
        for name in ("trace_attention_workspace_bytes", "trace_attention", "trace_attention_backward"):
            fn = getattr(self.lib, name)
            fn.restype, fn.argtypes = _cabi.PROTOTYPES[name]
        self.lib.lanes_watch()

    def empty(self, n, dtype, front=False):
        """n elements between guards, NaN (or the highest integer)."""
        es = torch.empty(0, dtype=dtype).element_size()
        if not n:
            return torch.empty(0, dtype=dtype)
        p = self.lib.lanes_alloc(n * es, int(front))
        t = torch.frombuffer((C.c_char * (n * es)).from_address(p), dtype=dtype)
        t.view(torch.uint8).fill_(0xff)
        return t

    def tensor(self, shape, dtype, off=0, pad=0, front=False):
        """(B, L, H, D) with `pad` elements between tokens, `off` before the first; the memory ends with the last head."""
        B, L, H, D = shape
        token = H * D + pad
        n = off + (B * L - 1) * token + H * D if B * L else 0
        return self.empty(n, dtype, front).as_strided(shape, (L * token, token, D, 1), off)

    def call(self, name, *args):
        if getattr(self.lib, name)(*args):
            raise RuntimeError("%s: %s" % (name, self.lib.lanes_error().decode()))


def run(lanes, case):
    dtype = TYPES[case["dtype"]]
    B, Lq, Lk, Hq, Hk, D = case["size"]
    off, pad, front = case.get("off", 0), case.get("pad", 0), case.get("front", False)
    g = torch.Generator().manual_seed(case.get("seed", 0))

    def filled(shape, size=1.0):
        t = lanes.tensor(shape, dtype, off, pad, front)
        t.copy_(torch.randn(shape, generator=g) * size)
        return t

    q, k = filled((B, Lq, Hq, D), case.get("q", 1.0)), filled((B, Lk, Hk, D), case.get("k", 1.0))
    v, dout = filled((B, Lk, Hk, D), case.get("v", 1.0)), filled((B, Lq, Hq, D), case.get("dout", 1.0))
    masks = {"causal": case.get("causal", False)}
    start = lengths = mask = None
    if "query_start" in case:
        masks["query_start"] = start = lanes.empty(B, torch.int32).copy_(torch.tensor(case["query_start"]))
    if "key_lengths" in case:
        masks["key_lengths"] = lengths = lanes.empty(B, torch.int32).copy_(torch.tensor(case["key_lengths"]))
    if "masked" in case:
        masks["key_mask"] = mask = (lanes.empty(B * Lk, torch.uint8).view(B, Lk)
                                    .copy_(torch.rand(B, Lk, generator=g) >= case["masked"]).view(torch.bool))
    out, dq = (lanes.tensor((B, Lq, Hq, D), dtype, front=front) for _ in range(2))
    dk, dv = (lanes.tensor((B, Lk, Hk, D), dtype, front=front) for _ in range(2))
    lse = lanes.empty(B * Hq * Lq, torch.float32).view(B, Hq, Lq)
    at = lambda t: None if t is None else t.data_ptr()
    strides = [s for t in (q, k, v, out, dout, dq, dk, dv) for s in t.stride()[:3]]
    desc = _cabi.AttentionDesc(list(TYPES).index(case["dtype"]), B, Lq, Lk, Hq, Hk, D, D ** -0.5, int(masks["causal"]), at(start),
                               at(lengths), at(mask), Lk, *strides)
    for back in (0, 1):
        n = lanes.lib.trace_attention_workspace_bytes(C.byref(desc), back)
        room = lanes.empty((n + 3) // 4, torch.float32)
        work = (at(room) if n else None, n, None)
        if back:
            lanes.call("trace_attention_backward", C.byref(desc), *map(at, (dout, q, k, v, out, lse, dq, dk, dv)), *work)
        else:
            lanes.call("trace_attention", C.byref(desc), *map(at, (q, k, v, out, lse)), *work)
    want = {"lse": formulas.attention64(q, k, v, **masks)["lse"], **forward64(q, k, v, **masks),
            **backward64(dout, q, k, v, out, lse, **masks)}
    for name, got in (("out", out), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv)):
        formulas.near(got, *want[name], what=name)


if __name__ == "__main__":
    torch.set_num_threads(1)
    lanes = Lanes(sys.argv[1])
    for line in sys.stdin:
        print(line.strip(), flush=True)
        run(lanes, json.loads(line))
    print("done")
