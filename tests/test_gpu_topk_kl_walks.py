"""-m gpu: top-logit distillation where a workgroup walks several rows: more rows than workgroups, rows wider than the registers, more kept entries than
threads, and what a row leaves behind for the next one (repeated entries, rows of weight 0 that hold NaN).  Bounds: those of test_gpu_topk_kl.py."""
import pytest
import torch

from test_gpu_topk_kl import BF, F32, HF, _check, _inputs, _ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("rows,K,k,dt,ddt,ld", [(520, 16388, 40, F32, BF, 0), (300, 20481, 600, F32, F32, 0), (300, 66000, 1024, BF, BF, 0), (270, 131080, 30, HF, HF, 0),
                                                (300, 68000, 700, F32, BF, 8), (270, 43000, 33, HF, HF, 1)])
def test_rows_after_rows(rows, K, k, dt, ddt, ld, tail):
    s, val, idx, lse, w = _inputs(rows, K, k, dt, seed=rows + K)
    if ld:       # rows of a wider matrix
        wide = torch.full((rows, K + ld), float("nan"), device="cuda", dtype=dt)
        wide[:, :K] = s
        s = wide[:, :K]
    idx[2] = idx[2, 0]                    # one class again and again
    idx[3, k // 2:] = idx[3, : k - k // 2].clone()
    idx[4] = -1
    w[5] = 0.0
    s[5] = float("nan")
    idx[256:] = idx[256:].flip(1)         # rows that follow others of the same workgroup
    d, lr = torch.full((rows, K), 7.0, device="cuda", dtype=ddt), torch.empty(rows, device="cuda")
    _ops().topk_kl_fwd_bwd(s, val, idx, 0.5, 0.3, lr, d, t_lse=lse if tail else None, row_weight=w)
    pick = torch.tensor([0, 1, 2, 3, 4, 5, 6, 255, 256, 257, 258, 259, 260, 261, 262, rows - 1], device="cuda")
    _check(s[pick], val[pick], idx[pick], lr[pick], d[pick], t_lse=lse[pick].cpu() if tail else None, weight=w[pick].cpu())
    half = torch.empty(rows - 200, device="cuda")      # the same rows from another first row (another workgroup's): the same bits
    _ops().topk_kl_fwd_bwd(s[200:], val[200:], idx[200:], 0.5, 0.3, half, None, t_lse=lse[200:].contiguous() if tail else None, row_weight=w[200:].contiguous())
    assert torch.equal(half, lr[200:])


@pytest.mark.parametrize("K", [8, 9])
def test_more_rows_than_a_launch_has_workgroups(K):
    rows, it = (1 << 20) + 1000, 0.5
    g = torch.Generator(device="cuda").manual_seed(K)
    s = torch.randn(rows, K, device="cuda", generator=g)
    t = torch.randn(rows, K, device="cuda", generator=g)
    val, idx = torch.topk(t, 3, 1)
    d, lr = torch.empty(rows, K, device="cuda"), torch.empty(rows, device="cuda")
    _ops().topk_kl_fwd_bwd(s, val, idx, it, 1.0, lr, d)
    p = torch.softmax(val.double() * it, 1)
    lq = torch.log_softmax(s.double() * it, 1)
    want = (p * (torch.log(p) - lq.gather(1, idx))).sum(1)
    grad = it * torch.exp(lq)
    grad.scatter_add_(1, idx, -it * p)
    assert (lr.double() - want).abs().max() < 4e-5 * 8      # 2 REL sum p (1 + |log p| + |log q|), the logarithms below 7
    assert (d.double() - grad).abs().max() < 2e-5 + 2.0 ** -24
