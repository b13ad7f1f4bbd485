"""Scales for which the kernels' fp32 arithmetic on lse / scale and scale * log2(e) * score has no room are refused by name (no device needed)."""
import ctypes as C

import pytest
import torch

import lightly_train_amd  # noqa: F401
from lightly_train_amd import _lib, ops
from test_cross_attention_cpu import _args, _desc


@pytest.mark.parametrize("scale", [1e-38, 2.0 ** -101, 2.0 ** 101, 3e38])
def test_scales_past_the_range_are_refused(scale):
    lib = _lib.load()
    for fn in (lib.lt_cross_attention_fwd, lib.lt_cross_attention_bwd):
        assert fn(C.byref(_desc(scale=scale)), None) == -22 and b"scale" in lib.lt_last_error()
    with pytest.raises(ValueError, match="scale"):
        ops.cross_attention_fwd(**_args(scale=scale))
