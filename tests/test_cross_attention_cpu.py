"""Refusals of the cross-attention front end and its C entry points that need no device, and the 64-bit definition the GPU tests compare against."""
import ctypes as C

import pytest
import torch

import lightly_train_amd  # noqa: F401
from lightly_train_amd import _lib, ops

BF = torch.bfloat16


def _args(**kw):
    q, k = torch.zeros(2, 3, 4, 64, dtype=BF), torch.zeros(2, 5, 2, 64, dtype=BF)
    a = dict(q=q, k=k, v=k.clone(), out=torch.zeros_like(q), lse=torch.zeros(2, 4, 3), scale=0.125)
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,text", [
    (dict(q=torch.zeros(2, 3, 4, 64)), "bfloat16 or float16"), (dict(q=torch.zeros(6, 4, 64, dtype=BF)), "views"),
    (dict(k=torch.zeros(2, 5, 3, 64, dtype=BF)), "multiple of the key heads"), (dict(scale=0.0), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(q=torch.zeros(2, 3, 4, 60, dtype=BF)), "head_dim"), (dict(q=torch.zeros(2, 3, 4, 136, dtype=BF)), "head_dim"), ({}, "current device"),
])
def test_front_end_refuses(kw, text):
    if torch.cuda.is_available() and text == "current device":
        pytest.skip("needs a machine without a device")
    with pytest.raises((ValueError, AssertionError, RuntimeError), match=text if text != "current device" else None):
        ops.cross_attention_fwd(**_args(**kw))


def _desc(**kw):
    d = _lib.CrossAttentionDesc()
    d.q = d.k = d.v = d.out = d.lse = d.dout = d.dq = d.dk = d.dv = 4096
    for n in ("sq", "so", "sdo", "sdq"):
        getattr(d, n)[:] = (3 * 256, 256, 64)
    for n in ("sk", "sv", "sdk", "sdv"):
        getattr(d, n)[:] = (5 * 128, 128, 64)
    d.B, d.Nq, d.Nk, d.H, d.Hkv, d.dh, d.dtype, d.scale = 2, 3, 5, 4, 2, 64, 0, 0.125
    for n, v in kw.items():
        if isinstance(v, tuple):
            getattr(d, n)[:] = v
        else:
            setattr(d, n, v)
    return d


@pytest.mark.parametrize("kw", [dict(q=4100), dict(k=None), dict(out=None), dict(H=3), dict(Hkv=0), dict(dh=60), dict(dh=136), dict(dh=0), dict(dtype=2), dict(scale=0.0),
                                dict(scale=-1.0), dict(scale=float("nan")), dict(B=-1), dict(Nq=-1), dict(Nk=-1), dict(sq=(768, 252, 64)), dict(sk=(640, -128, 64)),
                                dict(Nq=1 << 24), dict(Nk=1 << 24)])
def test_c_entry_points_refuse_and_say_why(kw):
    lib = _lib.load()
    for fn in (lib.lt_cross_attention_fwd, lib.lt_cross_attention_bwd):
        assert fn(C.byref(_desc(**kw)), None) == -22
        assert b"lt_cross_attention" in lib.lt_last_error()
    assert lib.lt_cross_attention_fwd(None, None) == -22 and lib.lt_cross_attention_bwd(None, None) == -22


@pytest.mark.parametrize("kw", [dict(lse=None), dict(dout=None), dict(dk=4104), dict(sdq=(768, 250, 64))])
def test_backward_refuses_missing_or_misaligned_gradients(kw):
    assert _lib.load().lt_cross_attention_bwd(C.byref(_desc(**kw)), None) == -22


def test_too_small_workspace_is_refused():
    lib = _lib.load()
    need = lib.lt_cross_attention_fwd_ws_floats(1, 40, 5000, 1, 1, 64)
    assert need > 0
    d = _desc(B=1, Nq=40, Nk=5000, H=1, Hkv=1, ws=4096, ws_floats=need - 1)
    assert lib.lt_cross_attention_fwd(C.byref(d), None) == -22
    d.ws, d.ws_floats = 4100, need
    assert lib.lt_cross_attention_fwd(C.byref(d), None) == -22
    assert lib.lt_cross_attention_bwd_ws_floats(2, 40, 70, 4, 2, 64) >= 2 * 40 * 4


def test_nothing_to_do_is_no_error():
    lib = _lib.load()
    assert lib.lt_cross_attention_fwd(C.byref(_desc(B=0)), None) == 0
    assert lib.lt_cross_attention_fwd(C.byref(_desc(Nq=0)), None) == 0
    assert lib.lt_cross_attention_bwd(C.byref(_desc(B=0)), None) == 0
