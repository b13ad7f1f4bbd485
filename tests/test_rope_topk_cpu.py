"""Refusals of the rotary and top-logit front ends and C entry points that need no device, and the rotary tables."""
import ctypes as C

import pytest
import torch

import lightly_train_amd  # noqa: F401
from lightly_train_amd import _lib, ops

BF = torch.bfloat16


def _rope(**kw):
    x = torch.zeros(2, 5, 3, 64, dtype=BF)
    a = dict(x=x, out=x.clone(), pos=torch.zeros(4, 2, dtype=torch.int32), freqs=torch.ones(32), axis=torch.zeros(32, dtype=torch.int32), prefix=1)
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,text", [(dict(x=torch.zeros(2, 5, 3, 64, dtype=torch.float64)), "rope_axes.x"), (dict(x=torch.zeros(2, 5, 64, dtype=BF)), "rope_axes.x"),
                                     (dict(x=torch.zeros(2, 5, 3, 60, dtype=BF)), "head_dim"), (dict(prefix=6), "prefix"), (dict(prefix=-1), "prefix"),
                                     (dict(x2=torch.zeros(2, 5, 3, 64, dtype=BF)), "come together"), (dict(out=torch.zeros(2, 5, 3, 64)), "rope_axes.out|current device|cuda")])
def test_rope_front_end_refuses(kw, text):
    with pytest.raises(ValueError, match=text):
        ops.rope_axes(**_rope(**kw))


def test_rope_tables_and_grid():
    f, a = ops.rope_axes_tables(64, [8, 12, 12])
    assert a.tolist() == [0] * 8 + [1] * 12 + [2] * 12
    assert torch.allclose(f[8:20], 10000.0 ** (-torch.arange(12) / 12.0)) and f[0] == 1
    f, a = ops.rope_axes_tables(32, [4, 8], base=100.0, shared_spectrum=True)
    assert a.tolist() == [0] * 4 + [1] * 8 + [-1] * 4
    assert torch.allclose(f[:12], 100.0 ** (-torch.arange(12) / 16.0)) and (f[12:] == 0).all()
    for bad in ([20, 20], [], [1] * 5, [-1, 4]):
        with pytest.raises(ValueError):
            ops.rope_axes_tables(64, bad)
    g = ops.rope_grid(2, 3, 4)
    assert g.shape == (24, 3) and g[-1].tolist() == [1, 2, 3] and g[5].tolist() == [0, 1, 1]
    assert ops.rope_grid(3).tolist() == [[0], [1], [2]]


def _desc(**kw):
    d = _lib.RopeAxesDesc()
    d.x = d.out = d.pos = d.freqs = d.axis = 4096
    for n in ("sx", "so", "sx2", "so2"):
        getattr(d, n)[:] = (960, 192, 64)
    d.B, d.N, d.H, d.dh, d.axes = 2, 5, 3, 64, 2
    for n, v in kw.items():
        if isinstance(v, tuple):
            getattr(d, n)[:] = v
        else:
            setattr(d, n, v)
    return d


@pytest.mark.parametrize("kw", [dict(x=None), dict(out=4104), dict(pos=None), dict(freqs=None), dict(axis=None), dict(dh=60), dict(dh=264), dict(dh=0), dict(axes=0), dict(axes=5),
                                dict(H=0), dict(H2=-1), dict(H2=2), dict(prefix=6), dict(prefix=-1), dict(dtype=3), dict(sx=(960, 190, 64)), dict(B=-1)])
def test_rope_c_entry_refuses(kw):
    lib = _lib.load()
    assert lib.lt_rope_axes(C.byref(_desc(**kw)), None) == -22 and b"lt_rope_axes" in lib.lt_last_error()
    assert lib.lt_rope_axes(None, None) == -22
    assert lib.lt_rope_axes(C.byref(_desc(B=0)), None) == 0 and lib.lt_rope_axes(C.byref(_desc(N=0)), None) == 0


def _topk(**kw):
    a = dict(s=torch.zeros(3, 50), t_val=torch.zeros(3, 4), t_idx=torch.zeros(3, 4, dtype=torch.int64), inv_temp=1.0, coef=1.0, loss_rows=torch.zeros(3))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,text", [(dict(s=torch.zeros(3, 50, dtype=torch.float64)), "rows, K"), (dict(s=torch.zeros(150)), "rows, K"), (dict(t_val=torch.zeros(3, 51)), "min"),
                                     (dict(t_val=torch.zeros(3, 0)), "min"), (dict(inv_temp=0.0), "inv_temp"), (dict(inv_temp=float("nan")), "inv_temp"),
                                     (dict(s=torch.zeros(50, 3).t()), "topk_kl_fwd_bwd.s"), (dict(s=torch.zeros(1, 50).expand(3, 50)), "topk_kl_fwd_bwd.s")])
def test_topk_front_end_refuses(kw, text):
    with pytest.raises(ValueError, match=text):
        ops.topk_kl_fwd_bwd(**_topk(**kw))


@pytest.mark.parametrize("at,v", [(0, None), (1, 3), (2, 49), (3, None), (5, 3), (6, None), (8, 3), (11, 0.0), (11, float("inf")), (13, None), (16, 2), (17, 49), (19, 0), (19, 1 << 18 | 1),
                                  (20, 0), (20, 51), (20, 1025), (18, -1)])
def test_topk_c_entry_refuses(at, v):
    #       s  dt ld  val dt ldv idx 64 ldi lse w  it   coef rows loss d   dd ldd rows K  k
    args = [64, 0, 50, 64, 2, 4, 64, 1, 4, None, None, 1.0, 1.0, 64, None, 64, 0, 50, 3, 50, 4, None]
    args[at] = v
    if at == 19 and v:
        args[2] = args[17] = v
    assert _lib.load().lt_topk_kl_fwd_bwd(*args) == -22 and b"lt_topk_kl" in _lib.load().lt_last_error()


def test_topk_without_rows_is_no_error():
    assert _lib.load().lt_topk_kl_fwd_bwd(None, 0, 50, None, 2, 4, None, 1, 4, None, None, 1.0, 1.0, None, None, None, 0, 50, 0, 50, 4, None) == 0


def test_packed_descriptors_match_the_structures():
    """The front ends hand over packed bytes: same size and order as the declared structures."""
    for packer, cls, n in ((ops._ROPE, _lib.RopeAxesDesc, 31), (ops._XATTN, _lib.CrossAttentionDesc, 45)):
        assert packer.size == C.sizeof(cls)
        vals = list(range(1, n + 1))
        d = cls.from_buffer_copy(packer.pack(*vals))
        got = []
        for name, _ in cls._fields_:
            v = getattr(d, name)
            got += list(v) if hasattr(v, "__len__") else [v]
        assert got == vals
