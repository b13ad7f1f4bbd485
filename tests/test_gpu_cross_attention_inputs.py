"""-m gpu: inputs that the documentation of cross attention allows and that come from broadcasting: keys, values, queries and upstream gradients with stride 0 along the batch, the
tokens or the heads; uint8 masks of any value; no lse; integer lengths past both ends.  A broadcast input gives bitwise what its copy gives."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _both(q, k, v, do, **kw):
    from lightly_train_amd import ops

    B, Nq, H, dh = q.shape
    new = lambda t: torch.full(t.shape, float("nan"), device="cuda", dtype=t.dtype)
    out, lse, dq, dk, dv = new(q), torch.full((B, H, Nq), float("nan"), device="cuda"), new(q), new(k), new(v)
    ops.cross_attention_fwd(q, k, v, out, lse, dh ** -0.5, **kw)
    alone = new(q)
    ops.cross_attention_fwd(q, k, v, alone, None, dh ** -0.5, **kw)
    assert torch.equal(alone, out)
    ops.cross_attention_bwd(q, k, v, out, do, lse, dq, dk, dv, dh ** -0.5, **kw)
    return out, lse, dq, dk, dv


@pytest.mark.parametrize("Nq,Nk,dh,dt", [(1, 70, 64, BF), (1, 3000, 64, HF), (9, 300, 32, HF), (50, 130, 128, BF), (200, 1000, 64, HF), (300, 3000, 96, BF)])
def test_broadcast_inputs_give_what_their_copies_give(Nq, Nk, dh, dt):
    g = torch.Generator(device="cuda").manual_seed(Nq + Nk)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dt)
    B, H, Hkv = 3, 6, 3
    q, k, v, do = rnd(B, Nq, H, dh), rnd(B, Nk, Hkv, dh), rnd(B, Nk, Hkv, dh), rnd(B, Nq, H, dh)
    one = dict(batch=lambda t: t[:1].expand_as(t), token=lambda t: t[:, :1].expand_as(t), head=lambda t: t[:, :, :1].expand_as(t), all=lambda t: t[:1, :1, :1].expand_as(t))
    for f in one.values():
        for pick in ("q", "k", "v", "do", "qkvdo"):
            args = [f(t) if n in pick or pick == "qkvdo" else t for n, t in (("q", q), ("k", k), ("v", v), ("do", do))]
            for a, b in zip(_both(*args), _both(*(t.contiguous() for t in args))):
                assert torch.equal(a, b) and not a.isnan().any()


@pytest.mark.parametrize("Nq", [2, 90])
def test_masks_and_lengths_of_any_value(Nq):
    g = torch.Generator(device="cuda").manual_seed(1)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g).to(BF)
    B, Nk = 5, 333
    q, k, v, do = rnd(B, Nq, 2, 64), rnd(B, Nk, 2, 64), rnd(B, Nk, 2, 64), rnd(B, Nq, 2, 64)
    m = torch.randint(0, 256, (B, Nk), device="cuda", generator=g, dtype=torch.int32)
    m = torch.where(m < 128, 0, m).to(torch.uint8)
    low, high = torch.iinfo(torch.int32).min, torch.iinfo(torch.int32).max
    lens = torch.tensor([low, -1, high, Nk, 7], device="cuda", dtype=torch.int32)
    want = _both(q, k, v, do, key_mask=m != 0, key_lens=lens.clamp(0, Nk))
    for a, b in zip(_both(q, k, v, do, key_mask=m, key_lens=lens), want):
        assert torch.equal(a, b)
