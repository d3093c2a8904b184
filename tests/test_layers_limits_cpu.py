"""The plans of the attention-block operators at the largest sizes their entries take (include/trace_hip.h): workspaces as large as the
sizes ask for, from arithmetic that does not wrap.  Nothing is launched."""
import ctypes as C

import pytest

from trace_amd import _cabi

ROWS = 2 ** 31 - 1


@pytest.mark.parametrize("columns, waves", [(1, 4096), (1000, 4096), (4096, 1024), (16384, 512)])
@pytest.mark.parametrize("rows, per", [(ROWS, ROWS), (ROWS, ROWS - 1), (ROWS - 5000, ROWS), (2 ** 30 + 1, 2 ** 30), (ROWS, 2 ** 20), (ROWS, 1)])
@pytest.mark.parametrize("cond", [0, 1])
def test_norm_workspace_of_the_most_rows(columns, waves, rows, per, cond):
    """Four tables of a row for each workgroup (four waves of 64 lanes, or one row's lanes); with conditioning, three of a row for each
    chunk of a group that is cut."""
    d = _cabi.NormDesc(0, 0, rows, columns, per, cond, cond, 0, 1.0, 1e-5, columns, columns, columns, columns)
    n = _cabi.lib().trace_residual_norm_workspace_bytes(C.byref(d))
    teams = 4 if columns <= 1024 else 1
    groups = -(-rows // per)
    most = max(waves, groups)
    assert 0 < n <= 4 * columns * (4 * (waves // teams + 1) + 3 * most * cond)
    if groups < waves // 2:                               # enough chunks for every team, give or take a rounding
        assert n >= 4 * columns * 4 * (waves // teams) // 2


def test_attention_backward_refuses_more_query_tiles_than_it_counts():
    """Tiles of 32 queries of the heads that share a key head, counted in 32 bits; the forward pass has no such count."""
    L = _cabi.lib()
    for Lq, Hq, Hk, ok in ((2 ** 30, 64, 1, False), (2 ** 30, 64, 2, True), (2 ** 30, 128, 2, False), (2 ** 20, 2 ** 16, 1, False),
                           (2 ** 20, 65535, 1, True)):
        d = _cabi.AttentionDesc(0, 1, Lq, 1, Hq, Hk, 1, 1.0)
        got = [L.trace_attention_workspace_bytes(C.byref(d), b) for b in (0, 1)]
        assert got[0] >= 0 and (got[1] >= 0) == ok, (Lq, Hq, Hk)
        if not ok:
            assert got[1] == -1 and "tiles" in L.trace_last_error().decode()
            assert L.trace_attention_backward(C.byref(d), *[None] * 10, 0, None) == -1 and "tiles" in L.trace_last_error().decode()
