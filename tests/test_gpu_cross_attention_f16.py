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
