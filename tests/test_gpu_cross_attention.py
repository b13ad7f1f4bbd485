"""-m gpu: cross attention to a sequence of another length (lt_cross_attention_fwd / _bwd) against its definition in 64 bits.

Bounds (u = half a step of the 16-bit type, 2^-8 bf16 / 2^-11 f16): the kernels round P (relative u) before P V, dS before dS K / dS^T Q and P before
P^T dO, and every output once; scores, statistics and sums are fp32, which SLACK covers (a score is a sum of dh products: |error| <= a few
2^-24 * sum |q k| ~ 1e-5 at these sizes, and lse carries 2^-24 * |lse|).  D = rowsum(dO * O) uses the rounded O.  So, elementwise,
  |dO_ut|  <= u (P |V|) + u |O|                          |dD| <= |dO| . |error of O|
  |ddS|    <= u |dS| + P |dD|                            |ddQ| <= scale |ddS| |K| + u |dQ|, |ddK| <= scale |ddS|^T |Q| + u |dK|
  |ddV|    <= u (P^T |dO|) + u |dV|
and f16 adds its smallest step (2^-24) / 2 per rounded factor."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
SLACK = 2e-4
BF, HF = torch.bfloat16, torch.float16


def _ops():
    import lightly_train_amd  # noqa: F401
    from lightly_train_amd import ops
    return ops


def _inputs(B, Nq, Nk, H, Hkv, dh, dt, mask="none", packed=False, seed=0, poison=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = (torch.randn(B, Nq, H, dh, device="cuda", generator=g) * 1.5).to(dt)
    if packed:
        kv = torch.randn(B, Nk, 2, Hkv, dh, device="cuda", generator=g).to(dt)
        k, v = kv[:, :, 0], kv[:, :, 1]
    else:
        k, v = (torch.randn(B, Nk, Hkv, dh, device="cuda", generator=g).to(dt) for _ in range(2))
    do = torch.randn(B, Nq, H, dh, device="cuda", generator=g).to(dt)
    lens = km = None
    seen = torch.ones(B, Nk, dtype=torch.bool, device="cuda")
    if mask in ("lens", "both"):
        lens = torch.randint(0, Nk + 1, (B,), device="cuda", generator=g).int()
        lens[0] = Nk
        if B > 1:
            lens[1] = 0
        if B > 2:
            lens[2] = -3                   # clamped
        if B > 3:
            lens[3] = Nk + 7               # clamped
        seen &= torch.arange(Nk, device="cuda")[None] < lens[:, None]
    if mask in ("mask", "both"):
        km = torch.rand(B, Nk, device="cuda", generator=g) < 0.7
        if B > 1:
            km[B - 1] = False
        seen &= km
    if poison and mask != "none":
        k[~seen] = float("nan")
        v[~seen] = float("inf")
    return q, k, v, do, lens, km, seen


def _exact(q, k, v, do, seen, scale):
    """out, lse, dq, dk, dv and the sums the bounds need, in 64 bits, [B, ..] layouts of the operator."""
    B, Nq, H, dh = q.shape
    Nk, Hkv = k.shape[1:3]
    G = H // Hkv
    z = lambda x: torch.where(seen[:, :, None, None], x.double(), 0.0)
    hd = lambda x: x.double().permute(0, 2, 1, 3).contiguous()                                 # [B, H, N, dh]
    K, V = (z(x).permute(0, 2, 1, 3).repeat_interleave(G, 1).contiguous() for x in (k, v))     # [B, H, Nk, dh]
    Q, DO = hd(q), hd(do)
    T = lambda x: x.transpose(2, 3).contiguous()
    S = torch.matmul(Q, T(K)) * scale
    S = S.masked_fill(~seen[:, None, None, :], -math.inf)
    lse = torch.logsumexp(S, 3) if Nk else torch.full((B, H, Nq), -math.inf, device=q.device, dtype=torch.float64)
    live = (lse > -math.inf)[..., None]
    P = torch.where(live, torch.exp(S - torch.where(live, lse[..., None], 0.0)), 0.0)
    O = torch.matmul(P, V)
    DO = torch.where(live, DO, 0.0)
    D = (DO * O).sum(3, keepdim=True)
    dS = P * (torch.matmul(DO, T(V)) - D)
    grp = lambda x: x.view(B, Hkv, G, Nk, dh).sum(2).permute(0, 2, 1, 3)
    r = dict(out=O.permute(0, 2, 1, 3), lse=lse, dq=(torch.matmul(dS, K) * scale).permute(0, 2, 1, 3), dk=grp(torch.matmul(T(dS), Q)) * scale,
             dv=grp(torch.matmul(T(P), DO)))
    r["parts"] = (P, dS, Q, K, V, DO, O, grp)
    return r


def _bounds(r, dt, scale):
    P, dS, Q, K, V, DO, O, grp = r["parts"]
    u, tiny = torch.finfo(dt).eps / 2, (2.0 ** -25 if dt == HF else 0.0)
    T = lambda x: x.transpose(2, 3).contiguous()
    eo = (u + SLACK) * torch.matmul(P, V.abs()) + tiny * V.abs().sum(2, keepdim=True)
    eo_r = eo + u * O.abs() + tiny
    eD = (DO.abs() * eo_r).sum(3, keepdim=True)
    mag = P * (torch.matmul(DO.abs(), T(V.abs())) + (DO * O).abs().sum(3, keepdim=True))     # what dS is the difference of
    eS = (u * dS.abs() + SLACK * mag + P * eD) + tiny
    b = dict(out=eo_r.permute(0, 2, 1, 3), dq=scale * torch.matmul(eS, K.abs()).permute(0, 2, 1, 3), dk=scale * grp(torch.matmul(T(eS), Q.abs())),
             dv=grp(torch.matmul(T(P * (u + SLACK) + tiny / 4096), DO.abs())))
    for n in ("dq", "dk", "dv"):
        b[n] = b[n] + u * r[n].abs() + tiny
    return b


def _run(q, k, v, do, scale, lens=None, km=None, outs=None, ws=None, bwd=True):
    ops = _ops()
    B, Nq, H, dh = q.shape
    o = outs or dict(out=torch.empty(B, Nq, H, dh, device="cuda", dtype=q.dtype), dq=torch.empty(B, Nq, H, dh, device="cuda", dtype=q.dtype),
                     dk=torch.empty(k.shape, device="cuda", dtype=q.dtype), dv=torch.empty(k.shape, device="cuda", dtype=q.dtype),
                     lse=torch.empty(B, H, Nq, device="cuda"))
    ops.cross_attention_fwd(q, k, v, o["out"], o["lse"], scale, key_lens=lens, key_mask=km, ws=ws)
    if bwd:
        ops.cross_attention_bwd(q, k, v, o["out"], do, o["lse"], o["dq"], o["dk"], o["dv"], scale, key_lens=lens, key_mask=km, ws=ws)
    return o


def _compare(o, r, dt, scale, names=("out", "dq", "dk", "dv")):
    b = _bounds(r, dt, scale)
    assert torch.equal(o["lse"].isinf(), r["lse"].isinf())
    fin = ~r["lse"].isinf()
    assert (o["lse"].double() - r["lse"])[fin].abs().max().item() < 5e-5 if fin.any() else True
    for n in names:
        e = (o[n].double() - r[n]).abs()
        assert torch.isfinite(o[n]).all(), n
        over = e > b[n] + 1e-12
        assert not over.any(), (n, e[over].max().item(), b[n][over].min().item(), over.sum().item())


CASES = [   # B, Nq, Nk, H, Hkv, dh, dtype, mask, packed
    (1, 1, 1, 1, 1, 64, BF, "none", False), (1, 1, 197, 12, 12, 64, BF, "none", False), (3, 1, 1370, 4, 4, 64, BF, "none", True),
    (4, 1, 33, 2, 1, 64, HF, "both", False), (2, 7, 65, 8, 2, 64, BF, "mask", True), (5, 4, 31, 8, 1, 32, BF, "lens", False),
    (1, 32, 64, 1, 1, 64, BF, "none", False), (1, 33, 64, 1, 1, 64, BF, "none", False), (2, 11, 257, 6, 2, 128, HF, "mask", False),
    (4, 100, 129, 2, 2, 64, HF, "both", True), (2, 196, 197, 3, 3, 64, BF, "none", True), (2, 65, 130, 4, 2, 128, BF, "lens", False),
    (5, 50, 63, 2, 1, 40, BF, "both", False), (2, 129, 96, 1, 1, 96, BF, "mask", False), (2, 70, 200, 2, 2, 72, HF, "none", True),
    (2, 40, 77, 2, 2, 8, BF, "none", False), (2, 45, 90, 4, 4, 24, HF, "lens", False), (1, 257, 300, 2, 2, 80, BF, "mask", True),
    (1, 40, 5003, 1, 1, 64, BF, "none", False), (1, 3, 9001, 1, 1, 64, HF, "mask", False), (1, 2500, 40, 2, 1, 64, BF, "none", False),
    (1, 1100, 5, 1, 1, 128, HF, "none", True), (1, 64, 4100, 3, 3, 128, BF, "lens", False), (2, 513, 700, 4, 2, 32, BF, "none", False),
    (9, 2, 40, 3, 3, 64, BF, "both", True), (1, 1, 20000, 2, 2, 128, BF, "none", True),
]


@pytest.mark.parametrize("B,Nq,Nk,H,Hkv,dh,dt,mask,packed", CASES)
def test_against_the_definition(B, Nq, Nk, H, Hkv, dh, dt, mask, packed):
    q, k, v, do, lens, km, seen = _inputs(B, Nq, Nk, H, Hkv, dh, dt, mask, packed)
    scale = dh ** -0.5
    o = _run(q, k, v, do, scale, lens, km)
    _compare(o, _exact(q, k, v, do, seen, scale), dt, scale)


def test_rows_without_keys_and_hidden_keys_give_exact_zeros():
    q, k, v, do, lens, km, seen = _inputs(6, 40, 150, 4, 2, 64, BF, "both")
    do[1] = float("nan")                       # (entry 1 sees no key: its upstream gradient is not read)
    for Nq in (40, 3):
        o = _run(q[:, :Nq], k, v, do[:, :Nq], 0.125, lens, km)
        empty = ~seen.any(1)
        assert empty.sum() >= 2
        assert (o["out"][empty] == 0).all() and (o["dq"][empty] == 0).all() and (o["lse"][empty] == -math.inf).all()
        assert (o["dk"][~seen] == 0).all() and (o["dv"][~seen] == 0).all()
        assert torch.isfinite(o["dk"]).all() and torch.isfinite(o["dq"]).all()


@pytest.mark.parametrize("Nq,Nk", [(0, 5), (5, 0), (40, 0), (0, 0)])
def test_no_queries_or_no_keys(Nq, Nk):
    q, k, v, do, *_ = _inputs(2, Nq, Nk, 2, 2, 64, BF)
    o = _run(q, k, v, do, 0.125)
    assert (o["out"] == 0).all() and (o["dq"] == 0).all() and (o["dk"] == 0).all() and (o["dv"] == 0).all() and (o["lse"] == -math.inf).all()


@pytest.mark.parametrize("Nq,Nk,dh", [(1, 77, 64), (50, 77, 64), (50, 1200, 128), (130, 70, 40)])
def test_views_are_read_and_written_in_place_and_nothing_else_is(Nq, Nk, dh):
    """Outputs inside wider buffers (a packed dkv, token rows behind the last one, a head slice), a query broadcast over the batch."""
    B, H, dt = 3, 4, BF
    q, k, v, do, lens, km, seen = _inputs(B, Nq, Nk, H, 2, dh, dt, "lens", True)
    q = q[:1].expand(B, Nq, H, dh)
    wide_q, wide_o = (torch.full((B, Nq + 3, H + 2, dh), 7.0, device="cuda", dtype=dt) for _ in range(2))
    wide_kv = torch.full((B, Nk + 2, 2, 2, dh), 7.0, device="cuda", dtype=dt)
    o = dict(out=wide_o[:, 1:Nq + 1, 1:H + 1], dq=wide_q[:, 2:Nq + 2, 2:], dk=wide_kv[:, 1:Nk + 1, 0], dv=wide_kv[:, 1:Nk + 1, 1],
             lse=torch.empty(B, H, Nq, device="cuda"))
    _run(q, k, v, do, dh ** -0.5, lens, km, outs=o)
    _compare(o, _exact(q, k, v, do, seen, dh ** -0.5), dt, dh ** -0.5)
    for w, n in ((wide_o, "out"), (wide_q, "dq")):
        o[n].fill_(7.0)
        assert (w == 7.0).all(), n
    o["dk"].fill_(7.0); o["dv"].fill_(7.0)
    assert (wide_kv == 7.0).all()


@pytest.mark.parametrize("Nq,Nk,H,Hkv,dh,dt", [(4, 60, 2, 1, 64, BF), (60, 200, 2, 2, 32, HF)])
def test_gradients_against_differences(Nq, Nk, H, Hkv, dh, dt):
    """<gradient, direction> against the central difference of sum(out * dout) of the 64-bit definition."""
    q, k, v, do, lens, km, seen = _inputs(2, Nq, Nk, H, Hkv, dh, dt, "mask", poison=False)
    scale = dh ** -0.5
    o = _run(q, k, v, do, scale, lens, km)
    r = _exact(q, k, v, do, seen, scale)
    b = _bounds(r, dt, scale)
    g = torch.Generator(device="cuda").manual_seed(5)
    x = dict(q=q.double(), k=k.double(), v=v.double())
    for n in "qkv":
        d = torch.randn(x[n].shape, device="cuda", generator=g, dtype=torch.float64)
        f = lambda s: (_exact(*[x[m] + s * d if m == n else x[m] for m in "qkv"], do, seen, scale)["out"] * do.double() * seen.any(1)[:, None, None, None]).sum()
        h = 1e-5
        diff = (f(h) - f(-h)) / (2 * h)
        got = (o["d" + n].double() * d).sum()
        assert abs(got - diff) <= (b["d" + n] * d.abs()).sum() + 1e-6 * abs(diff), n


def test_large_scores_and_a_far_away_maximum():
    """Scores of a few hundred, ascending along the keys: the running maximum moves in every tile, early tiles end at weight 0."""
    B, Nq, Nk, H, dh = 1, 40, 700, 1, 64
    q, k, v, do, lens, km, seen = _inputs(B, Nq, Nk, H, H, dh, BF)
    k = (k.float() * 0.1 + torch.linspace(-8, 8, Nk, device="cuda")[None, :, None, None] * q[:, :1].float().mean((0, 1), keepdim=True)).to(BF)
    for n in (40, 2):
        o = _run(q[:, :n], k, v, do[:, :n], 1.0)
        _compare(o, _exact(q[:, :n], k, v, do[:, :n], seen, 1.0), BF, 1.0, names=("out",))
    z = torch.zeros_like(q)
    o = _run(z, k, v, do, 1.0)
    _compare(o, _exact(z, k, v, do, seen, 1.0), BF, 1.0)


@pytest.mark.parametrize("Nq,Nk", [(1, 3000), (200, 3000), (900, 48)])
def test_results_are_bitwise_reproducible_on_another_stream_and_in_a_replayed_graph(Nq, Nk):
    ops = _ops()
    args = [_inputs(2, Nq, Nk, 2, 1, 64, BF, "mask", seed=s) for s in (1, 2)]
    scale = 0.125
    want = [_run(*a[:4], scale, None, a[5]) for a in args]
    torch.cuda.synchronize()
    n = max(ops.cross_attention_fwd_ws_floats(2, Nq, Nk, 2, 1, 64), ops.cross_attention_bwd_ws_floats(2, Nq, Nk, 2, 1, 64))
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for st, a in zip(streams, args):           # at the same time, a workspace each
        with torch.cuda.stream(st):
            got.append(_run(*a[:4], scale, None, a[5], ws=torch.full((n,), float("nan"), device="cuda")))
    torch.cuda.synchronize()
    for w, o in zip(want, got):
        for name in w:
            assert torch.equal(w[name], o[name]), name
    static = [x.clone() if torch.is_tensor(x) else x for x in args[0]]
    outs = {k_: torch.zeros_like(x) for k_, x in want[0].items()}
    ws = torch.zeros(n, device="cuda")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        _run(*static[:4], scale, None, static[5], outs=outs, ws=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        _run(*static[:4], scale, None, static[5], outs=outs, ws=ws)
    for i in (1, 0, 1, 0):
        for s_, x in zip(static, args[i]):
            if torch.is_tensor(s_):
                s_.copy_(x)
        ws.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for name in outs:
            assert torch.equal(outs[name], want[i][name]), (i, name)


def test_recorded_launch_plan_replays_both_directions():
    ops = _ops()
    a = _inputs(2, 50, 300, 2, 2, 64, BF)
    outs = _run(*a[:4], 0.125)
    want = {n: x.clone() for n, x in outs.items()}
    with ops.record_plan() as plan:
        _run(*a[:4], 0.125, outs=outs)
    assert plan.counts()["launches"] == 2
    for x in outs.values():
        x.zero_()
    plan.replay()
    torch.cuda.synchronize()
    for n in want:
        assert torch.equal(outs[n], want[n]), n


def test_refusals_on_the_device():
    ops = _ops()
    q, k, v, do, *_ = _inputs(2, 40, 600, 2, 2, 64, BF)
    out, lse = torch.empty_like(q), torch.empty(2, 2, 40, device="cuda")
    bad = [dict(q=torch.empty(2, 40, 2, 68, device="cuda", dtype=BF)[..., 2:66]), dict(out=torch.empty(1, 40, 2, 64, device="cuda", dtype=BF).expand(2, 40, 2, 64)),
           dict(lse=torch.empty(2, 40, 2, device="cuda").transpose(1, 2)), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
           dict(key_lens=torch.zeros(2, dtype=torch.int64, device="cuda")), dict(key_mask=torch.ones(2, 600, device="cuda")),
           dict(key_mask=torch.ones(2, 599, device="cuda", dtype=torch.bool)), dict(v=v.half()), dict(k=k[:, :, :, :32]),
           dict(ws=torch.empty(0, device="cuda", dtype=torch.float64)), dict(key_lens=torch.zeros(2, dtype=torch.int32))]
    for x in bad:
        a = dict(q=q, k=k, v=v, out=out, lse=lse, scale=0.125)
        a.update(x)
        with pytest.raises(ValueError):
            ops.cross_attention_fwd(**a)
    small = torch.empty(ops.cross_attention_bwd_ws_floats(2, 40, 600, 2, 2, 64) - 1, device="cuda")
    with pytest.raises(ValueError):
        ops.cross_attention_bwd(q, k, v, out, do, lse, torch.empty_like(q), torch.empty_like(k), torch.empty_like(v), 0.125, ws=small)
