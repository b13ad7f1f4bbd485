"""-m gpu: f16 cross attention where the factors of the second products are small: probabilities far below a row's largest (an attention sink before a long tail) and
gradients of a small upstream scale.  f16 has 2^-14 as its smallest normal number, so what a product rounds to 16 bits has to be brought into its range first.

Forward bound: P is rounded once (u relative, u = 2^-11, or 2^-36 of the row's largest where that is more) and out once.  With V >= 0 the sum of |P V| is out itself, so
the error is at most 2 u out + (keys / sum of exponentials) 2^-36 max|V|, plus fp32 statistics (1e-5) and half a step of f16's subnormal numbers."""
import pytest
import torch

from test_gpu_cross_attention_edges import HF, _definition

pytestmark = pytest.mark.gpu
U = 2.0 ** -11


def _ops():
    import lightly_train_amd  # noqa: F401
    from lightly_train_amd import ops
    return ops


def _sinks(B, Nq, Nk, H, Hkv, dh, gap, seed=0):
    """Every 97th key is a sink: its score lies `gap` above the others' (spread 1) and its value is 0; the others' values are 512 .. 1536 (their weighted mean is then no
    subnormal number, whose own rounding would hide what is lost)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randn(B, Nq, H, dh, device="cuda", generator=g) * 0.25
    q[..., 0] = 8.0
    k = torch.randn(B, Nk, Hkv, dh, device="cuda", generator=g) * (4.0 / dh ** 0.5)
    k[..., 0] = 0.0
    v = (torch.rand(B, Nk, Hkv, dh, device="cuda", generator=g) + 0.5) * 1024
    k[:, ::97, :, 0] = gap / 8.0
    v[:, ::97] = 0.0
    return q.to(HF), k.to(HF), v.to(HF)


@pytest.mark.parametrize("Nq,Nk,B,H,Hkv,dh", [(1, 1370, 2, 2, 2, 64), (1, 25088, 1, 2, 1, 64), (8, 6273, 2, 8, 2, 128), (20, 25088, 1, 1, 1, 32), (200, 6273, 1, 4, 2, 64), (784, 25088, 1, 2, 1, 64),
                                              (300, 25088, 1, 1, 1, 128), (900, 3000, 2, 2, 2, 32), (40, 200000, 1, 1, 1, 64)])
@pytest.mark.parametrize("gap", [16.0, 18.0])
def test_the_tail_behind_a_sink_is_not_lost(Nq, Nk, B, H, Hkv, dh, gap):
    q, k, v = _sinks(B, Nq, Nk, H, Hkv, dh, gap)
    out, lse = torch.empty_like(q), torch.empty(B, H, Nq, device="cuda")
    _ops().cross_attention_fwd(q, k, v, out, lse, 1.0)
    want, wl = _definition(q, k, v, 1.0)
    assert float(want.min()) > 2.0 ** -13
    err = (out.double() - want).abs()
    bound = (2 * U + 1e-5) * want + 97 * 2.0 ** -36 * 1536 + 2.0 ** -25
    assert (err <= bound).all(), float((err / bound).max())
    assert (lse.double() - wl).abs().max() < 1e-5


def _gradients(q, k, v, do, scale):
    """out, dq, dk, dv of the definition in 64 bits (products written out, heads shared by groups)."""
    G = q.shape[2] // k.shape[2]
    Q, DO = (x.double().permute(0, 2, 1, 3).contiguous() for x in (q, do))
    K, V = (x.double().repeat_interleave(G, 2).permute(0, 2, 1, 3).contiguous() for x in (k, v))
    T = lambda x: x.transpose(2, 3).contiguous()
    S = torch.matmul(Q, T(K)) * scale
    P = torch.softmax(S, 3)
    O = torch.matmul(P, V)
    dS = P * (torch.matmul(DO, T(V)) - (DO * O).sum(3, keepdim=True)) * scale
    grp = lambda x: x.unflatten(1, (k.shape[2], G)).sum(2)
    back = lambda x: x.permute(0, 2, 1, 3)
    return back(O), back(torch.matmul(dS, K)), back(grp(torch.matmul(T(dS), Q))), back(grp(torch.matmul(T(P), DO)))


def _backward(q, k, v, do, scale):
    ops = _ops()
    out, lse = torch.empty_like(q), torch.empty(q.shape[0], q.shape[2], q.shape[1], device="cuda")
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    ops.cross_attention_fwd(q, k, v, out, lse, scale)
    ops.cross_attention_bwd(q, k, v, out, do, lse, dq, dk, dv, scale)
    return out, dq, dk, dv


def _assert_roundings(got, want):
    """4 u of the gradient's norm (P / dS, out in D, the result: three roundings) and one half step of the subnormal numbers for each output."""
    for name, a, b in zip(("out", "dq", "dk", "dv"), got, want):
        assert torch.isfinite(a).all(), name
        err, allowed = float((a.double() - b).norm()), 4 * U * float(b.norm()) + 2.0 ** -25 * b.numel() ** 0.5
        assert err <= allowed, (name, err / float(b.norm()), allowed / float(b.norm()))


SHAPES = [(1, 1370, 4, 2, 2, 64), (20, 6273, 1, 2, 1, 128), (30, 100, 3, 2, 2, 72), (784, 25088, 1, 1, 1, 64), (196, 1370, 2, 2, 2, 64), (500, 6273, 1, 2, 1, 128), (64, 100, 2, 4, 2, 32),
          (300, 2000, 1, 2, 2, 96)]


@pytest.mark.parametrize("Nq,Nk,B,H,Hkv,dh", SHAPES)
@pytest.mark.parametrize("size", [1e-4, 1e-3, 1e-2, 1.0, 1e3])
def test_gradients_keep_their_bits_at_every_upstream_scale(Nq, Nk, B, H, Hkv, dh, size):
    g = torch.Generator(device="cuda").manual_seed(Nq + dh)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)
    q, k, v, do = rnd(B, Nq, H, dh).to(HF), rnd(B, Nk, Hkv, dh).to(HF), rnd(B, Nk, Hkv, dh).to(HF), (rnd(B, Nq, H, dh) * size).to(HF)
    got, want = _backward(q, k, v, do, dh ** -0.5), _gradients(q, k, v, do, dh ** -0.5)
    _assert_roundings(got, want)


@pytest.mark.parametrize("Nq,Nk,B,H,Hkv,dh", SHAPES)
def test_scales_that_differ_from_row_to_row_and_grow_along_the_axes(Nq, Nk, B, H, Hkv, dh):
    """Upstream rows from 2^-12 to 2^10 in ascending and in mixed order, values that grow along the keys: every row and key meets its largest dS late."""
    g = torch.Generator(device="cuda").manual_seed(Nq + dh + 1)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)
    q, k = rnd(B, Nq, H, dh).to(HF), rnd(B, Nk, Hkv, dh).to(HF)
    v = (rnd(B, Nk, Hkv, dh) * torch.logspace(-8, 3, Nk, base=2.0, device="cuda")[None, :, None, None]).to(HF)
    for order in (torch.arange(Nq, device="cuda"), torch.randperm(Nq, device="cuda", generator=g)):
        size = torch.logspace(-12, 10, Nq, base=2.0, device="cuda")[order]
        do = (rnd(B, Nq, H, dh) * size[None, :, None, None]).to(HF)
        got, want = _backward(q, k, v, do, dh ** -0.5), _gradients(q, k, v, do, dh ** -0.5)
        _assert_roundings(got, want)
        for a, b, s in zip(got[1].unbind(1), want[1].unbind(1), size.tolist()):      # row by row: no row hides behind a larger one
            # (its own roundings, and out's in D: u |dO . O| P K, at most as large as dQ's terms)
            assert float((a.double() - b).norm()) <= 6 * U * float(b.norm()) + 2.0 ** -25 * b.numel() ** 0.5, s


@pytest.mark.parametrize("Nq,Nk,dh", [(3, 400, 64), (100, 400, 64), (100, 90, 128), (300, 400, 128)])
def test_products_past_the_largest_f16_number_are_no_infinities(Nq, Nk, dh):
    """The last row's upstream gradient points along the value of the key that holds half of its probability: its dS is past 65504, no gradient is."""
    g = torch.Generator(device="cuda").manual_seed(7)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)
    q, k, v = (rnd(1, Nq, 1, dh) * 0.02).to(HF), (rnd(1, Nk, 1, dh) * 0.02).to(HF), rnd(1, Nk, 1, dh).to(HF)
    q[..., 0], k[..., 0] = 16.0, 0.0
    k[0, 3, 0, 0] = 32.0
    scale = 6.0 / 512                                # the score of key 3 lies 6 above the others
    do = (rnd(1, Nq, 1, dh) * 8).to(HF)
    do[0, -1, 0] = v[0, 3, 0].sign() * 6144
    want = _gradients(q, k, v, do, scale)
    P = torch.softmax(torch.matmul(q[0, -1:, 0].double(), k[0, :, 0].double().t().contiguous()) * scale, 1)[0]
    dP = torch.matmul(v[0, :, 0].double(), do[0, -1, 0].double())
    assert (P * (dP - (P * dP).sum())).abs().max() > 65504 and all(x.abs().max() < 60000 for x in want)
    _assert_roundings(_backward(q, k, v, do, scale), want)


@pytest.mark.parametrize("Nq,Nk", [(2, 900), (100, 900), (300, 2000)])
def test_replayed_graphs_find_their_scales_anew(Nq, Nk):
    """One captured pass, replayed over upstream gradients of other sizes with eager calls between: nothing of one replay's powers of two reaches the next."""
    ops = _ops()
    g = torch.Generator(device="cuda").manual_seed(4)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)
    q, k, v, do = rnd(2, Nq, 2, 64).to(HF), rnd(2, Nk, 2, 64).to(HF), rnd(2, Nk, 2, 64).to(HF), rnd(2, Nq, 2, 64).to(HF)
    o = [torch.empty_like(q), torch.empty(2, 2, Nq, device="cuda"), torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)]
    ws = torch.empty(max(ops.cross_attention_fwd_ws_floats(2, Nq, Nk, 2, 2, 64), ops.cross_attention_bwd_ws_floats(2, Nq, Nk, 2, 2, 64)), device="cuda")

    def run():
        ops.cross_attention_fwd(q, k, v, o[0], o[1], 0.125, ws=ws)
        ops.cross_attention_bwd(q, k, v, o[0], do, o[1], o[2], o[3], o[4], 0.125, ws=ws)

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    base = do.float()
    for size in (1e3, 1e-3, 1.0, 1e3, 1e-4):
        do.copy_((base * size).to(HF))
        want = _backward(q, k, v, do, 0.125)
        for t in (*o, ws):
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((o[0], *o[2:]), want):
            assert torch.equal(a, b), size
