"""-m gpu: captured graphs of the encoder-reading operators as a user would keep them: two graphs over the same tensors with scratch of their own, replayed in turn with
eager calls between; scratch made inside the capture; scratch that holds NaN; rotary positions and the loss in the same graph; inputs changed between replays."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _ops():
    import lightly_train_amd  # noqa: F401
    from lightly_train_amd import ops
    return ops


def _set(Nq, Nk, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g).to(BF)
    return dict(q=rnd(2, Nq, 4, 64), k=rnd(2, Nk, 2, 64), v=rnd(2, Nk, 2, 64), do=rnd(2, Nq, 4, 64), lens=torch.tensor([Nk, Nk // 2], device="cuda", dtype=torch.int32))


def _outs(x):
    return dict(out=torch.empty_like(x["q"]), lse=torch.empty(2, 4, x["q"].shape[1], device="cuda"), dq=torch.empty_like(x["q"]), dk=torch.empty_like(x["k"]),
                dv=torch.empty_like(x["v"]))


def _both(x, o, fws=None, bws=None):
    ops = _ops()
    ops.cross_attention_fwd(x["q"], x["k"], x["v"], o["out"], o["lse"], 0.125, key_lens=x["lens"], ws=fws)
    ops.cross_attention_bwd(x["q"], x["k"], x["v"], o["out"], x["do"], o["lse"], o["dq"], o["dk"], o["dv"], 0.125, key_lens=x["lens"], ws=bws)


@pytest.mark.parametrize("own", [True, False])
@pytest.mark.parametrize("Nq,Nk", [(1, 5000), (60, 5000), (700, 130)])
def test_two_graphs_and_eager_calls_in_turn(Nq, Nk, own):
    ops = _ops()
    x = _set(Nq, Nk, 1)
    sizes = (ops.cross_attention_fwd_ws_floats(2, Nq, Nk, 4, 2, 64), ops.cross_attention_bwd_ws_floats(2, Nq, Nk, 4, 2, 64))
    nan = lambda n: torch.full((n,), float("nan"), device="cuda")
    graphs, outs = [], []
    for _ in range(2):
        o = _outs(x)
        fw, bw = (nan(sizes[0]), nan(sizes[1])) if own else (None, None)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            _both(x, o, fw, bw)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            _both(x, o, fw, bw)
        graphs.append((graph, fw, bw))
        outs.append(o)
    for step in range(4):
        fresh = _set(Nq, Nk, 10 + step)
        for n in x:
            x[n].copy_(fresh[n])
        want = _outs(x)
        _both(x, want, nan(sizes[0]), nan(sizes[1]))
        for i in (0, 1) if step % 2 else (1, 0):
            for t in outs[i].values():
                t.fill_(float("nan"))
            graphs[i][0].replay()
        torch.cuda.synchronize()
        for o in outs:
            for n in want:
                assert torch.equal(o[n], want[n]), (step, n)


def test_rotary_positions_and_loss_in_one_graph():
    ops = _ops()
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(2, 50, 3, 64, device="cuda", generator=g)
    freqs, axis = ops.rope_axes_tables(64, [8, 12, 12], device="cuda")
    pos = torch.randint(0, 1000, (2, 50, 3), device="cuda", generator=g, dtype=torch.int32)
    s = torch.randn(300, 20000, device="cuda", generator=g)
    val, idx = torch.topk(torch.randn(300, 20000, device="cuda", generator=g), 40, 1)

    def run(o):
        ops.rope_axes(x, o["rot"], pos, freqs, axis)
        o["loss"].zero_()
        ops.topk_kl_fwd_bwd(s, val, idx, 0.5, 0.1, o["rows"], o["d"], loss=o["loss"])

    make = lambda: dict(rot=torch.empty_like(x), loss=torch.zeros(1, device="cuda"), rows=torch.empty(300, device="cuda"), d=torch.empty(300, 20000, device="cuda", dtype=BF))
    o = make()
    run(o)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(o)
    for step in range(3):
        x.normal_(generator=g); s.normal_(generator=g)
        idx.copy_(idx.roll(1, 0))
        want = make()
        run(want)
        for t in o.values():
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for n in want:
            assert torch.equal(o[n], want[n]), (step, n)
