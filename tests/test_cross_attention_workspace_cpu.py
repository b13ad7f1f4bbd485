"""Workspace sizes of calls that the entry points refuse: 0, not the size of what their row count leaves in 32 bits (a negative one reached the allocator's error).  And what the plan of a backward asks
for tells whether it cuts the keys."""
import pytest

import lightly_train_amd  # noqa: F401
from lightly_train_amd import _lib


@pytest.mark.parametrize("B,Nq,Nk,H,Hkv", [(1, 1 << 29, 5000, 4, 1), (1, (1 << 30) + 100, 5000, 4, 1), (1, 1 << 28, 5000, 24, 1), (2, 4, 1 << 24, 1, 1), (1 << 20, 4, 64, 1, 1)])
def test_workspace_sizes_of_calls_that_are_refused_are_zero(B, Nq, Nk, H, Hkv):
    lib = _lib.load()
    for fn in (lib.lt_cross_attention_fwd_ws_floats, lib.lt_cross_attention_bwd_ws_floats):
        assert fn(B, Nq, Nk, H, Hkv, 64) == 0
    assert lib.lt_cross_attention_fwd_ws_floats(1, 40, 5000, 1, 1, 64) > 0 and lib.lt_cross_attention_bwd_ws_floats(1, 40, 0, 1, 1, 64) > 0


def test_a_backward_that_one_round_of_workgroups_holds_is_not_cut():
    """head_dim 128: a CU holds one workgroup of the dQ kernel.  192 of them fit the card uncut (the workspace is D alone); cut in two they would take two rounds."""
    rows = 8 * 12 * 196
    assert _lib.load().lt_cross_attention_bwd_ws_floats(8, 196, 1370, 12, 12, 128) == rows
    assert _lib.load().lt_cross_attention_bwd_ws_floats(8, 196, 1370, 12, 12, 64) > rows      # (three to a CU: there the cut pays)
