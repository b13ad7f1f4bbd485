"""-m gpu: distillation from a teacher's top logits (lt_topk_kl_fwd_bwd) against its definition in 64 bits.

Bounds: an exponent z = s * inv_temp in base 2 is off by a few 2^-24 |z|, |z| <= 60 here, so a student probability is off by REL = 2e-5 relative and a
logarithm by as much; p without t_lse likewise, with t_lse it is exact to fp32.  Hence
  |dloss| <= 2 REL w sum p (1 + |log p| + |log q|) (bucket included),  |ddlogits| <= REL g (q + p) (others: REL g (q + p_rest q / q_rest)) + u |dlogits|."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
REL = 2e-5
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _ops():
    import lightly_train_amd  # noqa: F401
    from lightly_train_amd import ops
    return ops


def _exact(s, t_val, t_idx, it, coef, t_lse=None, weight=None):
    rows, K = s.shape
    loss, eloss = torch.zeros(rows, dtype=torch.float64), torch.zeros(rows, dtype=torch.float64)
    d, ed = torch.zeros(rows, K, dtype=torch.float64), torch.zeros(rows, K, dtype=torch.float64)
    s, t_val, t_idx = s.cpu().double(), t_val.cpu().double(), t_idx.cpu().tolist()
    for r in range(rows):
        w = coef * (1.0 if weight is None else float(weight[r]))
        at, js = [], []
        for j, i in enumerate(t_idx[r]):
            if 0 <= i < K and i not in at:
                at.append(i)
                js.append(j)
        if not at or w == 0:
            continue
        t = t_val[r, js] * it
        if t_lse is None and t.max() == -math.inf:
            continue
        e = torch.exp(t - t.max())      # (t.max() + log(sum) would round the logarithm away next to the type's lowest value)
        p = e / e.sum() if t_lse is None else torch.exp(t - float(t_lse[r]))
        logq = torch.log_softmax(s[r] * it, 0)
        q = torch.exp(logq)
        keep = torch.zeros(K, dtype=torch.bool)
        keep[at] = True
        lp = torch.where(p > 0, torch.log(p), 0.0)
        lq = torch.where(p > 0, logq[at], 0.0)
        loss[r] = w * (p * (lp - lq)).sum()
        eloss[r] = abs(w) * (p * (1 + lp.abs() + lq.abs())).sum()
        g, mag = q.clone(), q.clone()
        if t_lse is not None and len(at) < K:
            rest = max(0.0, 1.0 - float(p.sum()))
            log_rest = torch.logsumexp(logq[~keep], 0)
            if rest > 0:
                loss[r] += w * rest * (math.log(rest) - log_rest)
                eloss[r] += abs(w) * rest * (1 + abs(math.log(rest)) + abs(log_rest))
                x = torch.where(logq > -math.inf, rest * torch.exp(logq - log_rest), 0.0)
                g, mag = q - x, q + x
        g[at], mag[at] = q[at] - p, q[at] + p
        d[r], ed[r] = w * it * g, abs(w) * it * mag
    return loss, d, 2 * REL * eloss, REL * ed


def _inputs(rows, K, k, dt=F32, vdt=F32, idt=torch.int64, spread=2.0, seed=0, gone=0.1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = torch.randn(rows, K, device="cuda", generator=g) * spread
    t = z * 0.5 + torch.randn(rows, K, device="cuda", generator=g) * spread
    val, idx = torch.topk(t, k, 1)
    idx = torch.where(torch.rand(rows, k, device="cuda", generator=g) < gone, torch.tensor(-1, device="cuda"), idx).to(idt)
    return z.to(dt), val.to(vdt), idx, torch.logsumexp(t.double() * 0.5, 1).float(), torch.rand(rows, device="cuda", generator=g) + 0.2


def _check(s, t_val, t_idx, loss, d, it=0.5, coef=0.3, t_lse=None, weight=None):
    want, wd, el, ed = _exact(s, t_val, t_idx, it, coef, t_lse, weight)
    fin = torch.isfinite(want)
    assert torch.equal(torch.isfinite(loss.cpu()), fin)
    assert ((loss.cpu().double() - want).abs()[fin] <= el[fin] + 1e-12).all(), ((loss.cpu().double() - want).abs() - el).max()
    if d is not None:
        u = torch.finfo(d.dtype).eps / 2
        bound = ed + u * wd.abs() + (2.0 ** -25 if d.dtype == HF else 1e-38)
        err = (d.cpu().double() - wd).abs()
        assert (err <= bound).all(), (err - bound).max()


CASES = [   # rows, K, k, type of s, of dlogits, of t_val, of t_idx, bucket, weights
    (1, 1, 1, F32, F32, F32, torch.int64, True, False), (3, 10, 10, F32, F32, F32, torch.int64, False, True), (3, 10, 10, F32, F32, F32, torch.int32, True, False),
    (7, 1000, 10, F32, BF, F32, torch.int64, True, True), (5, 1000, 100, BF, BF, BF, torch.int32, True, False), (4, 1003, 7, F32, F32, HF, torch.int64, True, False),
    (4, 1001, 33, HF, HF, HF, torch.int32, False, True), (2, 4096, 1024, F32, F32, F32, torch.int64, True, False), (3, 16384, 65, F32, BF, F32, torch.int64, True, True),
    (2, 16388, 65, BF, BF, F32, torch.int64, False, False), (2, 65536, 256, F32, BF, F32, torch.int64, True, True), (2, 65536, 20, HF, HF, F32, torch.int64, True, False),
    (1, 131072, 300, BF, BF, F32, torch.int64, True, False), (1, 131072, 64, F32, F32, F32, torch.int64, True, False), (2, 65540, 50, F32, F32, F32, torch.int64, False, False),
    (1, 50257, 50, BF, BF, F32, torch.int32, True, False), (1, 262144, 40, BF, BF, F32, torch.int64, True, False), (300, 257, 3, F32, BF, F32, torch.int64, True, True),
    (2, 20481, 30, HF, HF, F32, torch.int64, True, False), (2, 6000, 30, F32, F32, F32, torch.int64, False, False),
]


@pytest.mark.parametrize("rows,K,k,dt,ddt,vdt,idt,tail,weights", CASES)
def test_against_the_definition(rows, K, k, dt, ddt, vdt, idt, tail, weights):
    s, val, idx, lse, w = _inputs(rows, K, k, dt, vdt, idt)
    if rows > 2:
        idx[1] = -1                      # a row without entries
    lse, w = lse if tail else None, w if weights else None
    d, lr, total = torch.empty(rows, K, device="cuda", dtype=ddt), torch.empty(rows, device="cuda"), torch.full((1,), 2.0, device="cuda")
    _ops().topk_kl_fwd_bwd(s, val, idx, 0.5, 0.3, lr, d, t_lse=lse, row_weight=w, loss=total)
    _check(s, val, idx, lr, d, t_lse=lse, weight=w)
    assert abs(float(total) - 2.0 - float(lr.double().sum())) <= 1e-5 * (1 + float(lr.double().abs().sum()))
    only = torch.empty(rows, device="cuda")
    _ops().topk_kl_fwd_bwd(s, val, idx, 0.5, 0.3, only, t_lse=lse, row_weight=w)      # the loss alone
    assert torch.equal(only, lr)


@pytest.mark.parametrize("K", [40, 41, 5000])
@pytest.mark.parametrize("tail", [False, True])
def test_repeated_missing_and_outside_indices(K, tail):
    s, val, idx, lse, _ = _inputs(6, K, 20, gone=0.0)
    idx[0, 5:] = idx[0, 0]
    idx[1, 3], idx[1, 9], idx[1, 17] = idx[1, 12], idx[1, 12], idx[1, 12]
    idx[2, :] = K
    idx[3, ::2] = -7
    idx[4, 4] = 2 ** 40
    idx[5, 1:] = -1
    lse = lse if tail else None
    for _ in range(3):
        d, lr = torch.full((6, K), 5.0, device="cuda"), torch.empty(6, device="cuda")
        _ops().topk_kl_fwd_bwd(s, val, idx, 0.5, 0.3, lr, d, t_lse=lse)
        _check(s, val, idx, lr, d, t_lse=lse)
        assert (d[2] == 0).all() and lr[2] == 0


def test_masked_logits_and_rows_of_weight_zero():
    low = torch.finfo(F32).min
    s, val, idx, lse, w = _inputs(8, 600, 12, gone=0.0)
    s[0, :] = torch.where(torch.rand(600, device="cuda") < 0.5, -math.inf, s[0])      # classes the student may not take
    s[0, idx[0]] = 1.0
    val[1, 6:] = -math.inf
    val[2, 6:] = low
    val[3] = low                           # uniform over the kept
    val[4] = -math.inf                     # nothing known
    s[5], w[5] = float("nan"), 0.0
    s[6, idx[6]] += 200.0                  # the student is sure of the kept: q_rest ~ e^-100
    s[7] = torch.where(torch.arange(600, device="cuda") < 300, low, 0.0)
    for tail in (None, lse):
        d, lr = torch.empty(8, 600, device="cuda"), torch.empty(8, device="cuda")
        _ops().topk_kl_fwd_bwd(s, val, idx, 0.5, 0.3, lr, d, t_lse=tail, row_weight=w)
        rows = [0, 1, 2, 3, 4, 5, 6] if tail is None else [0, 1, 2, 5, 6]
        pick = torch.tensor(rows, device="cuda")
        _check(s[pick], val[pick], idx[pick], lr[pick], d[pick], t_lse=None if tail is None else tail[pick], weight=w[pick])
        assert (d[5] == 0).all() and lr[5] == 0
    s[6, :] = -math.inf
    s[6, idx[6]] = 0.0                     # q_rest is zero and the teacher's is not
    _ops().topk_kl_fwd_bwd(s, val, idx, 0.5, 0.3, lr, d, t_lse=lse, row_weight=w)
    assert lr[6] == math.inf and not d[6].isnan().any()


@pytest.mark.parametrize("dt,ddt,K", [(F32, BF, 1000), (F32, F32, 1001), (BF, BF, 70000), (HF, HF, 999)])
def test_row_strides_and_nothing_else_is_written(dt, ddt, K):
    s, val, idx, lse, w = _inputs(5, K, 9, dt)
    for off, pad in ((0, 8), (3, 5)):
        wide = torch.full((5, K + off + pad), 3.0, device="cuda", dtype=dt)
        wide[:, off:off + K] = s
        grad = torch.full((5, K + off + pad), 7.0, device="cuda", dtype=ddt)
        v2, i2 = torch.zeros(5, 20, device="cuda"), torch.zeros(5, 13, device="cuda", dtype=torch.int64)
        v2[:, 2:11], i2[:, 4:13] = val, idx
        lr = torch.empty(5, device="cuda")
        _ops().topk_kl_fwd_bwd(wide[:, off:off + K], v2[:, 2:11], i2[:, 4:13], 0.5, 0.3, lr, grad[:, off:off + K], t_lse=lse)
        _check(s, val, idx, lr, grad[:, off:off + K], t_lse=lse)
        grad[:, off:off + K] = 7.0
        assert (grad == 7.0).all()


@pytest.mark.parametrize("tail", [False, True])
def test_gradient_against_differences(tail):
    s, val, idx, lse, w = _inputs(4, 200, 12)
    lse = lse if tail else None
    d, lr = torch.empty(4, 200, device="cuda"), torch.empty(4, device="cuda")
    _ops().topk_kl_fwd_bwd(s, val, idx, 0.5, 0.3, lr, d, t_lse=lse, row_weight=w)
    g = torch.Generator(device="cuda").manual_seed(9)
    u = torch.randn(4, 200, device="cuda", generator=g, dtype=torch.float64)
    f = lambda h: _exact(s.double() + h * u, val, idx, 0.5, 0.3, lse, w)[0].sum()
    diff = (f(1e-4) - f(-1e-4)) / 2e-4
    _, wd, _, ed = _exact(s, val, idx, 0.5, 0.3, lse, w)
    assert abs(float((d.double() * u).sum()) - float(diff)) <= float(((ed + 2.0 ** -24 * wd.abs()) * u.cpu().abs()).sum()) + 1e-6 * abs(float(diff)) + 1e-7


def test_streams_graphs_and_plans_are_bitwise_equal():
    ops = _ops()
    s, val, idx, lse, w = _inputs(40, 5000, 60)
    run = lambda: ops.topk_kl_fwd_bwd(s, val, idx, 0.5, 0.3, lr, d, t_lse=lse, row_weight=w, loss=total)
    d, lr, total = torch.empty(40, 5000, device="cuda", dtype=BF), torch.empty(40, device="cuda"), torch.zeros(1, device="cuda")
    run()
    want = [x.clone() for x in (d, lr, total)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        total.zero_()
        run()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        run()
    with ops.record_plan() as plan:
        run()
    torch.cuda.synchronize()
    for replay in (graph.replay, plan.replay, graph.replay):
        for x in (d, lr, total):
            x.zero_()
        torch.cuda.synchronize()
        replay()
        torch.cuda.synchronize()
        for x, y in zip((d, lr, total), want):
            assert torch.equal(x, y)
