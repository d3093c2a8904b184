"""The attention kernels run lane by lane on the CPU (tests/lanes): every access stays within the tensors, which end at memory that may
not be touched, and results are within the bounds of attention_formulas.py."""
import itertools
import json
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, os.path.join(HERE, "lanes"))

import build as lanes_build  # noqa: E402


@pytest.fixture(scope="session")
def lanes(tmp_path_factory):
    return lanes_build.build(str(tmp_path_factory.mktemp("lanes")))


def run(lanes, cases, at_once=4):
    """The cases, dealt to a few processes; each ends at its first that fails, with the case's line as its last."""
    cmd = [sys.executable, os.path.join(HERE, "lanes", "attention.py"), lanes]
    jobs = [subprocess.Popen(cmd, stdin=subprocess.PIPE, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)
            for _ in range(min(at_once, len(cases)))]
    with ThreadPoolExecutor(len(jobs)) as pool:
        said = list(pool.map(lambda n: jobs[n].communicate("\n".join(json.dumps(c) for c in cases[n::len(jobs)]), timeout=600),
                             range(len(jobs))))
    for job, (out, err) in zip(jobs, said):
        assert job.returncode == 0 and out.endswith("done\n"), out[-300:] + err[-2000:]


SHORT = ((1, 1), (1, 2), (31, 33), (32, 32), (33, 1), (33, 31), (64, 50), (2, 63), (63, 64))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_short_sequences_read_nothing_behind_their_last_token(lanes, dtype):
    """Element-wise loads (a head size, window or stride off the 16-byte grid) and 16-byte ones, of every tile shape."""
    forms = (dict(D=17), dict(D=20), dict(D=8, off=1), dict(D=32, pad=3), dict(D=24))
    run(lanes, [dict(dtype=dtype, size=[1, Lq, Lk, 2, 1, f["D"]], **f) for f in forms for Lq, Lk in SHORT])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_accesses_stay_within_the_tensors(lanes, dtype):
    """Every kernel: few queries with and without joins, long sequences, shares, shared heads, masks, lengths, empty ranges."""
    run(lanes, [dict(dtype=dtype, front=front, **c) for front, c in itertools.product((False, True), (
        dict(size=[2, 1, 300, 4, 1, 20], off=1, pad=2, key_lengths=[300, 33]),
        dict(size=[2, 3, 150, 4, 2, 64], causal=True, key_lengths=[0, 150], query_start=[5, 147]),
        dict(size=[1, 16, 70, 2, 2, 128], masked=0.5),
        dict(size=[1, 70, 130, 2, 1, 40], pad=1, causal=True),
        dict(size=[2, 129, 67, 2, 1, 24], masked=0.3),
        dict(size=[1, 65, 200, 1, 1, 72], key_lengths=[131]),
        dict(size=[1, 33, 1, 1, 1, 128]), dict(size=[2, 1, 90, 1, 1, 17]),
        dict(size=[3, 52, 52, 2, 1, 64], causal=True, masked=0.2)))])


@pytest.mark.parametrize("size", [[1, 40, 40, 2, 1, 64], [1, 64, 20, 4, 1, 128], [2, 30, 33, 2, 2, 20], [1, 100, 70, 4, 2, 64],
                                  [1, 65, 200, 2, 1, 128], [1, 20, 300, 1, 1, 32], [1, 65, 6, 4, 1, 80]])
def test_large_fp16_gradients(lanes, size):
    """dout of a scaled loss: dout . v far above what fp16 holds, gradients that it holds."""
    run(lanes, [dict(dtype="f16", size=size, v=4.0, dout=1000.0),
                dict(dtype="f16", size=size, v=8.0, dout=8000.0, q=0.05, k=0.01, causal=True)])
