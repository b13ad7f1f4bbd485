"""-m gpu: the bucketed top-logit loss where the teacher's kept probabilities do not sum to 1 with the bucket: values stored in 16 bits next to a 32-bit log-sum-exp (a
sure teacher's pass 1), and rows of which every class is kept.  The gradient has to be the loss's own, w / T (q (sum p + p_rest) - p).

Bounds: those of test_gpu_topk_kl.py (REL covers the exponentials and logarithms in fp32), the gradient's formed by 64-bit autograd of the loss."""
import math

import pytest
import torch

from test_gpu_topk_kl import BF, F32, HF, REL, _ops

pytestmark = pytest.mark.gpu


def _loss(s, p, at, keep, it):
    """sum p (log p - log q) + p_rest (log p_rest - log q_rest), one row, from the logits in 64 bits."""
    logq = torch.log_softmax(s * it, 0)
    some = p > 0
    loss = (p[some] * (torch.log(p[some]) - logq[at][some])).sum()
    rest = max(0.0, 1.0 - float(p.sum())) if not keep.all() else 0.0
    if rest > 0:
        loss = loss + rest * (math.log(rest) - torch.logsumexp(logq[~keep], 0))
    return loss, rest


def _inputs(rows, K, k, vdt, dt, spread, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.randn(rows, K, device="cuda", generator=g) * spread
    s = (t * 0.5 + torch.randn(rows, K, device="cuda", generator=g) * 2).to(dt)
    val, idx = torch.topk(t, k, 1)
    return s, val.to(vdt), idx, t.double()


CASES = [   # rows, K, k, type of t_val, of s, of dlogits, spread of the teacher's logits
    (40, 1000, 10, BF, F32, F32, 8.0), (40, 1000, 10, HF, F32, F32, 8.0), (40, 1000, 10, BF, BF, BF, 8.0), (40, 1003, 10, BF, HF, HF, 8.0), (3, 65536, 64, BF, F32, BF, 8.0),
    (2, 131072, 64, BF, BF, BF, 8.0), (300, 16388, 20, BF, F32, F32, 8.0), (20, 12, 12, BF, F32, F32, 3.0), (20, 100, 100, HF, F32, F32, 3.0),
]


@pytest.mark.parametrize("rows,K,k,vdt,dt,ddt,spread", CASES)
def test_the_gradient_is_that_of_the_returned_loss(rows, K, k, vdt, dt, ddt, spread):
    it, coef = 1.0, 0.3
    s, val, idx, t = _inputs(rows, K, k, vdt, dt, spread)
    lse = torch.logsumexp(t * it, 1).float()
    d, lr = torch.empty(rows, K, device="cuda", dtype=ddt), torch.empty(rows, device="cuda")
    _ops().topk_kl_fwd_bwd(s, val, idx, it, coef, lr, d, t_lse=lse)
    u, tiny = torch.finfo(ddt).eps / 2, 2.0 ** -25 if ddt == HF else 1e-38
    away = 0.0
    for r in range(rows):
        x = s[r].double().cpu().requires_grad_(True)
        at = idx[r].cpu()
        p = torch.exp(val[r].double().cpu() * it - float(lse[r]))
        keep = torch.zeros(K, dtype=torch.bool)
        keep[at] = True
        loss, rest = _loss(x, p, at, keep, it)
        grad, = torch.autograd.grad(loss, x)
        logq = torch.log_softmax(x.detach() * it, 0)
        q, ps = torch.exp(logq), torch.zeros(K, dtype=torch.float64)
        ps[at] = p
        total = float(p.sum()) + rest
        away = max(away, abs(total - 1.0))
        side = rest * torch.exp(logq - torch.logsumexp(logq[~keep], 0)) * ~keep if rest > 0 else 0.0
        bound = coef * it * REL * (q * max(total, 1.0) + ps + side) + u * coef * it * grad.abs() + tiny
        err = (d[r].double().cpu() - coef * it * grad).abs()
        assert (err <= bound).all(), (r, total, float((err - bound).max()))
        mag = float((p * (1 + p.log().abs() + logq[at].abs())).sum()) + (rest * (1 + abs(math.log(rest)) + 60.0) if rest > 0 else 0.0)
        assert abs(float(lr[r]) - coef * float(loss.detach())) <= 2 * REL * coef * mag, r
    assert away > (1e-2 if vdt == BF else 1e-4)          # (otherwise the case does not reach what it is for)


@pytest.mark.parametrize("vdt", [BF, HF])
def test_gradient_against_differences_of_the_loss(vdt):
    it, coef, rows, K, k = 0.5, 0.3, 6, 300, 12
    s, val, idx, t = _inputs(rows, K, k, vdt, F32, 16.0, seed=3)
    lse = torch.logsumexp(t * it, 1).float()
    d, lr = torch.empty(rows, K, device="cuda"), torch.empty(rows, device="cuda")
    _ops().topk_kl_fwd_bwd(s, val, idx, it, coef, lr, d, t_lse=lse)
    dirs = torch.randn(rows, K, dtype=torch.float64, generator=torch.Generator().manual_seed(9))
    dirs[:, ::2] += 1.0                                  # (not across the constant direction alone: a push on all logits shows)
    for r in range(rows):
        at, p = idx[r].cpu(), torch.exp(val[r].double().cpu() * it - float(lse[r]))
        keep = torch.zeros(K, dtype=torch.bool)
        keep[at] = True
        f = lambda h: float(_loss(s[r].double().cpu() + h * dirs[r], p, at, keep, it)[0])
        diff = coef * (f(1e-4) - f(-1e-4)) / 2e-4
        got = float((d[r].double().cpu() * dirs[r]).sum())
        q = torch.softmax(s[r].double().cpu() * it, 0)
        bound = coef * it * (REL + 2.0 ** -23) * float((2 * q * dirs[r].abs()).sum() + 2 * (p * dirs[r][at].abs()).sum())
        assert abs(got - diff) <= bound + 1e-6 * abs(diff), r
