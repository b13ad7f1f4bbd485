"""-m gpu: cross attention whose scores are large (probabilities from all of a row to nothing, a running maximum that moves in every tile), forward and backward, and
scales at the ends of the accepted range.

Bounds: a score is a sum of dh products in fp32 that the backward starts at -lse / scale, and its exponent rounds a few more times at the size of the score: with
X = scale sum |q k| (the size of the partial sums) + |lse|, |dS| <= 8 * 2^-24 X, so P is off by that relative (X <= 700 here: 3.4e-4).  The elementwise bounds are those of
test_gpu_cross_attention.py with this in the place of SLACK."""
import math

import pytest
import torch

from test_gpu_cross_attention import BF, HF, _exact, _inputs, _run
import test_gpu_cross_attention as base

pytestmark = pytest.mark.gpu


def _check(o, r, q, k, dt, scale, seen):
    P, dS, Q, K, V, DO, O, grp = r["parts"]
    u, tiny = torch.finfo(dt).eps / 2, (2.0 ** -25 if dt == HF else 0.0)
    T = lambda x: x.transpose(2, 3).contiguous()
    live = torch.isfinite(r["lse"])
    X = scale * torch.matmul(Q.abs(), T(K.abs())) + torch.where(live, r["lse"], 0.0).abs()[..., None]
    W = P * (8 * 2.0 ** -24 * X + 1e-6)                                   # |error of P|
    eo = u * torch.matmul(P, V.abs()) + 2 * torch.matmul(W, V.abs()) + u * O.abs() + tiny
    eD = (DO.abs() * eo).sum(3, keepdim=True)
    mag = torch.matmul(DO.abs(), T(V.abs())) + (DO * O).abs().sum(3, keepdim=True)
    eS = u * dS.abs() + W * mag + P * eD + 2.0 ** -24 * 8 * P * mag
    b = dict(out=eo.permute(0, 2, 1, 3), dq=scale * torch.matmul(eS, K.abs()).permute(0, 2, 1, 3), dk=scale * grp(torch.matmul(T(eS), Q.abs())),
             dv=grp(torch.matmul(T(P * u + W), DO.abs())))
    assert ((o["lse"].double() - r["lse"])[live].abs() <= 8 * 2.0 ** -24 * X.amax(3)[live] + 1e-6).all()
    for n in ("out", "dq", "dk", "dv"):
        assert torch.isfinite(o[n]).all(), n
        e = (o[n].double() - r[n]).abs() - (b[n] + u * r[n].abs() + tiny + 1e-30)
        assert (e <= 0).all(), (n, float(e.max()))


@pytest.mark.parametrize("Nq,Nk,H,Hkv,dh", [(2, 700, 2, 1, 64), (40, 700, 2, 2, 64), (200, 90, 2, 1, 64), (300, 700, 2, 2, 128), (70, 3001, 1, 1, 32), (260, 333, 2, 2, 96)])
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("spread", [4.0, 40.0])
def test_both_directions_of_peaked_rows(Nq, Nk, H, Hkv, dh, dt, spread):
    """Scores spread over about +-3 `spread`, rising along the keys, some keys hidden."""
    q, k, v, do, lens, km, seen = _inputs(2, Nq, Nk, H, Hkv, dh, dt, "mask", seed=11)
    km[1, :3], seen[1, :3] = True, True                                   # (entry 1 of _inputs sees nothing: give it three keys)
    k[1, :3], v[1, :3] = k[0, :3].nan_to_num(0.5), v[0, :3].nan_to_num(0.5, posinf=0.5)
    scale = spread / (1.5 * dh ** 0.5)
    ramp = torch.linspace(-1, 1, Nk, device="cuda")[None, :, None, None] * q[:, :1, :Hkv].float() * (2.0 / dh ** 0.5)
    k = torch.where(seen[:, :, None, None], (k.float() + ramp).to(dt), k)
    o = _run(q, k, v, do, scale, lens, km)
    _check(o, _exact(q, k, v, do, seen, scale), q, k, dt, scale, seen)


@pytest.mark.parametrize("Nq,Nk", [(2, 400), (100, 400)])
@pytest.mark.parametrize("scale", [2.0 ** -90, 1e-9, 1e9, 2.0 ** 60])
def test_scales_far_from_one_with_hidden_keys_first(Nq, Nk, scale):
    """The scores are of size 1; the first 200 keys are hidden (the running maximum still holds no key after three chunks)."""
    g = torch.Generator(device="cuda").manual_seed(2)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)
    h = (1.0 / (8 * scale)) ** 0.5                                        # q and k take half of 1 / scale each
    q, k, v, do = (rnd(1, Nq, 2, 64) * h).to(BF), (rnd(1, Nk, 2, 64) * h).to(BF), rnd(1, Nk, 2, 64).to(BF), rnd(1, Nq, 2, 64).to(BF)
    km = torch.ones(1, Nk, dtype=torch.bool, device="cuda")
    km[:, :200] = False
    o = _run(q, k, v, do, scale, None, km)
    r = _exact(q, k, v, do, km, scale)
    for n, size in (("out", 1.0), ("dq", scale * h), ("dk", scale * h), ("dv", 1.0)):      # compared at the size that the scale leaves them
        r[n], o[n] = r[n] / size, o[n].double() / size
    assert ((o["lse"].double() - r["lse"]).abs() < 1e-5).all()
    for n in ("out", "dq", "dk", "dv"):      # four roundings of P / dS, out in D and the result, norm-wise
        assert torch.isfinite(o[n]).all(), n
        assert float((o[n] - r[n]).norm()) <= 4 * 2.0 ** -8 * float(r[n].norm()), n
