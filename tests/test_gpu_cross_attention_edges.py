"""-m gpu: cross attention where its documentation promises a result and the values or layouts are the odd ones: entries without a visible key whose queries hold NaN,
row counts at the borders between the kernels, sequence-first memory, two calls at once, offsets past 32 bits.

Tolerances: u = finfo(dtype).eps / 2 is one rounding.  Forward: P and out are rounded once each -> 2 u of the largest |v| a row can mix.  Backward: P / dS, the out in
D and the gradient itself, over sums whose terms cancel; norm-wise 3 u, asserted 4 u of the gradient's norm (f32 statistics are below u / 100)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _definition(q, k, v, scale, seen=None, dout=None):
    q, k, v = (x.double().requires_grad_(True) for x in (q, k, v))
    G = q.shape[2] // k.shape[2]
    K, V = (x.repeat_interleave(G, 2).permute(0, 2, 1, 3) for x in (k, v))
    S = (q.permute(0, 2, 1, 3) @ K.transpose(2, 3)) * scale
    if seen is not None:
        S = S.masked_fill(~seen[:, None, None, :], float("-inf"))
    out = (torch.softmax(S, 3) @ V).permute(0, 2, 1, 3)
    if dout is None:
        return out.detach(), torch.logsumexp(S, 3).detach()
    return (out.detach(),) + torch.autograd.grad(out, (q, k, v), dout.double())


def _run(q, k, v, scale, dout, **kw):
    from lightly_train_amd import ops

    B, Nq, H, _ = q.shape
    out, lse = torch.empty_like(q), torch.empty(B, H, Nq, device="cuda")
    ops.cross_attention_fwd(q, k, v, out, lse, scale, **kw)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    ops.cross_attention_bwd(q, k, v, out, dout, lse, dq, dk, dv, scale, **kw)
    return out, lse, dq, dk, dv


def _rel(a, b):
    return float((a.double() - b).norm() / b.norm().clamp(min=1e-30))


@pytest.mark.parametrize("Nq,Nk", [(1, 70), (3, 2000), (200, 70), (200, 2000), (700, 130)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("how", ["mask", "lens"])
def test_an_entry_without_visible_keys_is_zero_whatever_its_tensors_hold(Nq, Nk, bad, how):
    g = torch.Generator(device="cuda").manual_seed(5)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g).to(BF)
    q, k, v, do = rnd(2, Nq, 2, 64), rnd(2, Nk, 2, 64), rnd(2, Nk, 2, 64), rnd(2, Nq, 2, 64)
    for t in (q, k, v, do):
        t[1] = bad
    kw = (dict(key_mask=torch.tensor([[True], [False]], device="cuda").expand(2, Nk).contiguous()) if how == "mask"
          else dict(key_lens=torch.tensor([Nk, 0], device="cuda", dtype=torch.int32)))
    out, lse, dq, dk, dv = _run(q, k, v, 0.125, do, **kw)
    assert (out[1] == 0).all() and (lse[1] == float("-inf")).all()
    assert (dq[1] == 0).all() and (dk[1] == 0).all() and (dv[1] == 0).all()
    want = _definition(q[:1], k[:1], v[:1], 0.125, dout=do[:1])
    for a, b in zip((out, dq, dk, dv), want):
        assert _rel(a[:1], b) < 4 * 2.0 ** -8


@pytest.mark.parametrize("dh", [32, 64, 72, 96, 128])
@pytest.mark.parametrize("Nq,H,Hkv", [(32, 2, 2), (33, 2, 2), (16, 4, 2), (17, 4, 2), (63, 2, 2), (128, 2, 2), (129, 2, 2), (224, 2, 2), (225, 2, 2), (75, 6, 2)])
def test_row_counts_around_the_borders_between_the_kernels(dh, Nq, H, Hkv):
    g = torch.Generator(device="cuda").manual_seed(Nq * 131 + dh)
    dt = HF if Nq % 2 else BF
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dt)
    Nk = 333
    q, do, k, v = rnd(2, Nq, H, dh), rnd(2, Nq, H, dh), rnd(2, Nk, Hkv, dh), rnd(2, Nk, Hkv, dh)
    lens = torch.tensor([Nk, 97], device="cuda", dtype=torch.int32)
    mask = torch.rand(2, Nk, device="cuda", generator=g) < 0.7
    mask[:, 0] = True
    seen = mask & (torch.arange(Nk, device="cuda")[None] < lens[:, None])
    out, _, dq, dk, dv = _run(q, k, v, dh ** -0.5, do, key_lens=lens, key_mask=mask)
    want = _definition(q, k, v, dh ** -0.5, seen, do)
    u = torch.finfo(dt).eps / 2
    for name, a, b in zip(("out", "dq", "dk", "dv"), (out, dq, dk, dv), want):
        assert _rel(a, b) < 4 * u, name
    assert (dk[~seen] == 0).all() and (dv[~seen] == 0).all()


@pytest.mark.parametrize("Nq,Nk", [(1, 1), (5, 300), (150, 300)])
def test_sequence_first_memory(Nq, Nk):
    g = torch.Generator(device="cuda").manual_seed(9)
    rnd = lambda n, h: torch.randn(n, 3, h, 64, device="cuda", generator=g).to(BF).transpose(0, 1)
    q, do, k, v = rnd(Nq, 4), rnd(Nq, 4), rnd(Nk, 2), rnd(Nk, 2)
    got = _run(q, k, v, 0.125, do)
    want = _run(*(x.contiguous() for x in (q, k, v)), 0.125, do.contiguous())
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_two_calls_at_once_with_their_own_scratch():
    g = torch.Generator(device="cuda").manual_seed(3)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g).to(BF)
    sets = [(rnd(2, n, 4, 64), rnd(2, 3001, 2, 64), rnd(2, 3001, 2, 64), rnd(2, n, 4, 64)) for n in (1, 250)]
    want = [_run(q, k, v, 0.125, do) for q, k, v, do in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(3):
        for i, (q, k, v, do) in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                got[i].append(_run(q, k, v, 0.125, do))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            for a, b in zip(r, want[i]):
                assert torch.equal(a, b)


@pytest.mark.parametrize("Nq", [2, 70])
def test_offsets_past_32_bits_in_a_long_cache(Nq):
    """A view into a cache whose tokens lie 2^20 elements apart: the last of 2100 tokens begins past 2^31 elements (4.4 GB)."""
    step, Nk = 1 << 20, 2100
    cache = torch.zeros(Nk * step, device="cuda", dtype=BF)
    k, v = (cache.as_strided((1, Nk, 1, 64), (0, step, 64, 1), at) for at in (0, 64))
    g = torch.Generator(device="cuda").manual_seed(2)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g).to(BF)
    k.copy_(rnd(1, Nk, 1, 64)); v.copy_(rnd(1, Nk, 1, 64))
    q, do = rnd(1, Nq, 1, 64), rnd(1, Nq, 1, 64)
    from lightly_train_amd import ops

    def both(k, v):
        out, lse, dq = torch.empty_like(q), torch.empty(1, 1, Nq, device="cuda"), torch.empty_like(q)
        dk, dv = torch.empty(1, Nk, 1, 64, device="cuda", dtype=BF), torch.empty(1, Nk, 1, 64, device="cuda", dtype=BF)
        ops.cross_attention_fwd(q, k, v, out, lse, 0.125)
        ops.cross_attention_bwd(q, k, v, out, do, lse, dq, dk, dv, 0.125)
        return out, lse, dq, dk, dv

    for a, b in zip(both(k, v), both(k.contiguous(), v.contiguous())):
        assert torch.equal(a, b)
