"""CPU: calls of the attention-conditioning operators that their checks and plans have to take or refuse before anything is launched."""
import ctypes

import pytest


def _lib():
    from layout2img_amd import _lib as L
    return L.load()


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("D", [8, 32, 40, 64, 72, 96, 128])
def test_cross_attention_plans_a_list_without_states(D, dtype):
    """Forward and backward, whatever the number of queries: a plan that divides by the number of the states' tiles would end the process."""
    n = (ctypes.c_longlong * 1)()
    for B, Lq, Hk, G in ((1, 1, 1, 1), (1, 64, 1, 1), (1, 65, 1, 1), (2, 65, 2, 4), (1, 100000, 1, 1), (600, 65, 1, 1)):
        for bwd in (0, 1):
            assert _lib().l2i_cross_attention_scratch(B, Lq, 0, Hk, G, D, dtype, bwd, n) == 0, (B, Lq, Hk, G, bwd)
            assert n[0] == (B * Hk * Lq * G + 3) // 4 * 4 * bwd   # (the rows' D alone: nothing is cut in ranges)
        assert _lib().l2i_cross_attention_wants_lo(B, Lq, 0, Hk, G, D, dtype) in (0, 1)
