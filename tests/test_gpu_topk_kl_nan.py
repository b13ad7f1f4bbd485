"""-m gpu: a NaN in the teacher's kept values or in the student's row shows in that row's loss and gradient (a diverged teacher must not pass for a row without entries), and
nowhere else; a NaN of an entry that does not count (index missing or repeated) stays out."""
import pytest
import torch

from test_gpu_topk_kl import BF, F32, HF, _check, _inputs, _ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("K,dt,vdt", [(600, F32, F32), (601, BF, BF), (20000, HF, HF)])
@pytest.mark.parametrize("tail", [False, True])
def test_a_nan_shows_in_its_row_alone(K, dt, vdt, tail):
    nan, rows = float("nan"), 9
    s, val, idx, lse, w = _inputs(rows, K, 12, dt, vdt, gone=0.0)
    lse = lse if tail else None
    val[0] = nan
    val[1, 3] = nan
    val[2], val[2, 5] = -float("inf"), nan
    val[3, 4:], idx[3, 4:] = nan, -1                     # missing entries
    val[4, 7], idx[4, 7] = nan, idx[4, 2]                # a repeated one
    s[5, idx[5, 6]] = nan                                # the student, at a kept class
    free = [i for i in range(K) if i not in idx[6].tolist()][3]
    s[6, free] = nan                                     # and at another
    d, lr = torch.empty(rows, K, device="cuda", dtype=dt), torch.empty(rows, device="cuda")
    _ops().topk_kl_fwd_bwd(s, val, idx, 0.5, 0.3, lr, d, t_lse=lse, row_weight=w)
    for r in (0, 1, 2, 5, 6):
        assert lr[r].isnan(), r
        assert d[r, idx[r]].isnan().any(), r
    pick = torch.tensor([3, 4, 7, 8], device="cuda")
    _check(s[pick], val[pick].nan_to_num(0.0), idx[pick], lr[pick], d[pick], t_lse=None if lse is None else lse[pick], weight=w[pick])
