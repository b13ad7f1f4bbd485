"""-m gpu: rotary positions with several axes (lt_rope_axes) against complex rotations in 64 bits.

Bound: the angle is reduced in 64 bits and rounded once to fp32 within a quarter turn (pi / 2 * 2^-25 = 4.7e-8), sine and cosine are off by at most
2 ulp (1.2e-7), the two products and their sum add 2^-24 each: |error| <= 3e-7 (|a| + |b|) + u |result|, u the half step of the output type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _ops():
    import lightly_train_amd  # noqa: F401
    from lightly_train_amd import ops
    return ops


def _exact(x, pos, freqs, axis, prefix=0, interleaved=False, inverse=False):
    A, half = pos.shape[-1], x.shape[-1] // 2
    ax = axis.long()
    on = (ax >= 0) & (ax < A)
    ang = pos.double()[..., ax.clamp(0, A - 1)] * freqs.double() * on
    if ang.dim() == 2:
        ang = ang[None]
    w = torch.polar(torch.ones_like(ang), -ang if inverse else ang)[:, :, None]
    z = x.double().clone()
    t = z[:, prefix:]
    a, b = (t[..., 0::2], t[..., 1::2]) if interleaved else (t[..., :half], t[..., half:])
    r = torch.complex(a, b) * w
    mag = torch.zeros_like(z)
    m = a.abs() + b.abs()
    if interleaved:
        z[:, prefix:] = torch.view_as_real(r).flatten(-2)
        mag[:, prefix:] = m.repeat_interleave(2, -1)
    else:
        z[:, prefix:] = torch.cat((r.real, r.imag), -1)
        mag[:, prefix:] = torch.cat((m, m), -1)
    return z, mag


def _check(got, x, *args, **kw):
    want, mag = _exact(x, *args, **kw)
    u = torch.finfo(got.dtype).eps / 2
    err = (got.double() - want).abs()
    bound = 3e-7 * mag + u * want.abs() + (2.0 ** -25 if got.dtype == HF else 0.0)
    assert (err <= bound).all(), (err - bound).max().item()


def _inputs(B, N, H, dh, A, dt, prefix, own, span=1000, seed=0, fl=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(B, N, H, dh, device="cuda", generator=g).to(dt)
    shape = (B, N - prefix, A) if own else (N - prefix, A)
    pos = torch.randint(-span, span + 1, shape, device="cuda", generator=g, dtype=torch.int32)
    if fl:
        pos = torch.randn(shape, device="cuda", generator=g) * span
    ops = _ops()
    n = dh // 2
    freqs, axis = ops.rope_axes_tables(dh, [n // A] * A, device="cuda")
    return x, pos, freqs, axis


CASES = [   # B, N, H, dh, axes, dtype, prefix, per sample, interleaved, inverse, float positions
    (1, 1, 1, 64, 1, BF, 0, False, False, False, False), (16, 1, 12, 64, 3, BF, 0, True, False, False, False),
    (2, 197, 12, 64, 2, BF, 1, False, False, False, True), (3, 201, 6, 64, 3, HF, 5, True, True, True, False),
    (2, 65, 3, 128, 4, F32, 0, False, True, False, False), (2, 33, 5, 72, 2, BF, 0, True, False, True, False),
    (2, 33, 5, 72, 3, HF, 1, False, True, False, True), (1, 1000, 2, 8, 1, BF, 0, False, False, False, False),
    (2, 50, 17, 256, 2, BF, 0, True, True, False, False), (3, 21, 4, 80, 3, F32, 2, True, False, True, True),
    (2, 40, 4, 24, 2, F32, 40, False, False, False, False), (5, 7, 9, 32, 4, BF, 0, True, False, False, False),
]


@pytest.mark.parametrize("B,N,H,dh,A,dt,prefix,own,il,inv,fl", CASES)
def test_against_the_definition(B, N, H, dh, A, dt, prefix, own, il, inv, fl):
    x, pos, freqs, axis = _inputs(B, N, H, dh, A, dt, prefix, own, fl=fl)
    out = torch.full_like(x, 9.0)
    _ops().rope_axes(x, out, pos, freqs, axis, prefix=prefix, interleaved=il, inverse=inv)
    _check(out, x, pos, freqs, axis, prefix, il, inv)
    assert torch.equal(out[:, :prefix], x[:, :prefix])


@pytest.mark.parametrize("fl", [False, True])
def test_far_positions_keep_their_angle(fl):
    x, pos, freqs, axis = _inputs(2, 300, 4, 64, 2, F32, 0, True, span=2 ** 24, fl=fl)
    if not fl:
        pos[0, 0], pos[0, 1] = 2 ** 31 - 1, -2 ** 31
    out = torch.empty_like(x)
    _ops().rope_axes(x, out, pos, freqs, axis)
    _check(out, x, pos, freqs, axis)


def test_q_and_k_of_a_packed_projection_in_place_and_back():
    """One launch over both, inside the packed activation; v stays as it was; the inverse returns the input to rounding; pairs without an axis and
    values that are not finite pass through."""
    ops = _ops()
    B, N, H, dh = 2, 58, 6, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    qkv = torch.randn(B, N, 3, H, dh, device="cuda", generator=g).to(BF)
    pos = torch.cat([ops.rope_grid(3, 19, 1, device="cuda")])
    freqs, axis = ops.rope_axes_tables(dh, [4, 10, 10], device="cuda")
    qkv[:, :, 0, :, 30] = float("inf")       # pair 30 has no axis
    was = qkv.clone()
    q, k = qkv[:, :, 0], qkv[:, :, 1]
    ops.rope_axes(q, q, pos, freqs, axis, prefix=1, x2=k, out2=k)
    fin = [i for i in range(dh) if i % 32 != 30]
    for got, x in ((q, was[:, :, 0]), (k, was[:, :, 1])):
        want, mag = _exact(torch.where(x.isinf(), 0.0, x.float()), pos, freqs, axis, 1)
        assert ((got.double() - want)[..., fin].abs() <= (2.0 ** -8 * want.abs() + 3e-7 * mag)[..., fin]).all()
    assert torch.equal(q[..., [30, 62]], was[:, :, 0][..., [30, 62]])
    assert torch.equal(qkv[:, :, 2], was[:, :, 2])
    ops.rope_axes(q, q, pos, freqs, axis, prefix=1, inverse=True, x2=k, out2=k)
    back = (qkv[..., fin].float() - was[..., fin].float()).abs()
    # two roundings of each of the two values that meet: u |r| first, turned back, then u |x|
    pair = (was[..., fin].float().abs() + was[..., [(i + 32) % 64 for i in fin]].float().abs())
    assert (back <= 2.0 ** -8 * (2 * pair) + 1e-6).all()


def test_gradient_is_the_inverse_rotation():
    """<R x, y> = <x, R^T y> in exact arithmetic; and against differences of the 64-bit definition along a direction (the map is linear)."""
    ops = _ops()
    x, pos, freqs, axis = _inputs(2, 30, 4, 64, 3, F32, 1, True)
    y = torch.randn_like(x)
    rx, ry = torch.empty_like(x), torch.empty_like(x)
    ops.rope_axes(x, rx, pos, freqs, axis, prefix=1)
    ops.rope_axes(y, ry, pos, freqs, axis, prefix=1, inverse=True)
    a, b = (rx.double() * y.double()).sum(), (x.double() * ry.double()).sum()
    assert abs(a - b) <= 1e-6 * (rx.double().abs() * y.double().abs()).sum()
    d = torch.randn(x.shape, device="cuda", dtype=torch.float64)
    f = lambda s: (_exact(x.double() + s * d, pos, freqs, axis, 1)[0] * y.double()).sum()
    assert abs((f(0.5) - f(-0.5)) - (ry.double() * d).sum()) <= 1e-6 * (ry.double().abs() * d.abs()).sum()


def test_streams_graphs_and_plans():
    ops = _ops()
    x, pos, freqs, axis = _inputs(4, 100, 6, 64, 3, BF, 0, True)
    want = torch.empty_like(x)
    ops.rope_axes(x, want, pos, freqs, axis)
    torch.cuda.synchronize()
    out = torch.zeros_like(x)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.rope_axes(x, out, pos, freqs, axis)
    side.synchronize()
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ops.rope_axes(x, out, pos, freqs, axis)
    p0 = pos.clone()
    for shift in (3, 0, 5):
        pos.copy_(p0 + shift)
        ops.rope_axes(x, want, pos, freqs, axis)
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    with ops.record_plan() as plan:
        ops.rope_axes(x, out, pos, freqs, axis)
    out.zero_()
    plan.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_writes_nothing_but_its_output():
    x, pos, freqs, axis = _inputs(2, 13, 3, 72, 2, BF, 0, False)
    wide = torch.full((2, 15, 5, 72), 7.0, device="cuda", dtype=BF)
    out = wide[:, 1:14, 1:4]
    _ops().rope_axes(x, out, pos, freqs, axis)
    _check(out, x, pos, freqs, axis)
    out.fill_(7.0)
    assert (wide == 7.0).all()
    e = torch.empty(0, 13, 3, 72, device="cuda", dtype=BF)
    _ops().rope_axes(e, torch.empty_like(e), pos, freqs, axis)
