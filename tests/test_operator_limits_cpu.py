"""Sizes and strides past what the strided operators' launches and 32-bit offsets hold are refused by name before anything is launched."""
import ctypes as C

import pytest

import lightly_train_amd  # noqa: F401
from lightly_train_amd import _lib


def _attention(**kw):
    d = _lib.CrossAttentionDesc()
    d.q = d.k = d.v = d.out = d.lse = d.dout = d.dq = d.dk = d.dv = 4096
    for n in ("sq", "so", "sdo", "sdq", "sk", "sv", "sdk", "sdv"):
        getattr(d, n)[:] = (1 << 14, 256, 64)
    d.B, d.Nq, d.Nk, d.H, d.Hkv, d.dh, d.dtype, d.scale = 2, 3, 5, 4, 4, 64, 0, 0.125
    for n, v in kw.items():
        if isinstance(v, tuple):
            getattr(d, n)[:] = v
        else:
            setattr(d, n, v)
    return d


@pytest.mark.parametrize("name", ["sq", "sk", "sv", "so"])
def test_token_strides_of_2_to_the_24_are_refused(name):
    lib = _lib.load()
    for fn in (lib.lt_cross_attention_fwd, lib.lt_cross_attention_bwd):
        assert fn(C.byref(_attention(**{name: (1 << 30, 1 << 24, 64)})), None) == -22
        assert b"2^24" in lib.lt_last_error()


@pytest.mark.parametrize("name", ["sdo", "sdq", "sdk", "sdv"])
def test_token_strides_of_gradients_are_refused(name):
    lib = _lib.load()
    assert lib.lt_cross_attention_bwd(C.byref(_attention(**{name: (1 << 30, 1 << 24, 64)})), None) == -22
    assert b"2^24" in lib.lt_last_error()


def test_more_workgroups_than_a_launch_holds_are_refused():
    lib = _lib.load()
    d = _attention(B=1 << 17, Nq=8192, Nk=64, ws=4096, ws_floats=1 << 62)
    assert lib.lt_cross_attention_fwd(C.byref(d), None) == -22 and b"workgroups" in lib.lt_last_error()
    assert lib.lt_cross_attention_bwd(C.byref(d), None) == -22 and b"workgroups" in lib.lt_last_error()
    r = _lib.RopeAxesDesc()
    r.x = r.out = r.pos = r.freqs = r.axis = 4096
    r.sx[:] = r.so[:] = (1 << 16, 64, 64)
    r.B, r.N, r.H, r.dh, r.axes = 1 << 20, 1 << 10, 1, 64, 1
    assert lib.lt_rope_axes(C.byref(r), None) == -22 and b"tokens" in lib.lt_last_error()
