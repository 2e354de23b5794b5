"""Gated delta rule: alignments that the C entry points ask for, without a GPU."""
import pytest

from fpscan_b200 import _lib

SIZES = (2, 3, 2, 4, 16, 24)  # batch, seqlen, key heads, heads, dk, dv


@pytest.mark.parametrize("dtype, size", [(0, 4), (1, 2), (2, 2)])
def test_a_step_refuses_what_its_loads_cannot_take(dtype, size):
    lib = _lib.load()
    # q, k, v, log_decay, beta, initial, out, final_state; v, the decays and out one element at a time
    for i, by in ((0, 8), (1, 8), (2, 1), (3, 1), (4, 1), (5, 4), (6, 1), (7, 4), (2, size // 2)):
        p = [(j + 1) << 20 for j in range(8)]
        p[i] += by
        if i in (5, 7):
            p[5] = p[7] = p[i]  # in place
        assert lib.fpscan_delta_step(*p, *SIZES, 1.0, dtype, None) == 1
        assert b"aligned" in lib.fpscan_last_error()
