"""The norm on float32 rows that are whole 16 bytes but not whole eights of columns, and
on views whose neighbours must stay as they are (needs a B200)."""
import pytest
import torch

from tests import fp8_util as U

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from race_attention_b200 import _lib
    _lib.load()


@pytest.mark.parametrize("weight", [torch.float32, torch.bfloat16], ids=["wf32", "wbf16"])
@pytest.mark.parametrize("k", [4, 12, 36, 60, 92, 100, 156, 164, 252, 260, 300, 500, 508, 516, 700, 1004, 1020, 1028, 2500,
                               4092, 4100, 5004, 12292, 16380, 16388, 50004])
def test_rows_of_whole_fours(k, weight):
    """Results and gradients in float64, with bounds as derived beside the norm's other
    tests; the widths beside the row, in one wider tensor, are not read and not written."""
    from race_attention_b200.fp8 import rms_norm
    r = 21 if k > 4096 else 2500
    g = torch.Generator(device="cuda").manual_seed(k)
    wide = torch.full((r, k + 8), float("nan"), device="cuda")
    x = wide[:, 4:4 + k]
    x.copy_(torch.randn(r, k, generator=g, device="cuda"))
    res, dy, dh = (torch.randn(r, k, generator=g, device="cuda") for _ in range(3))
    w = (1 + 0.2 * torch.randn(k, generator=g, device="cuda")).to(weight)
    X, R, W = x.detach().requires_grad_(), res.clone().requires_grad_(), w.clone().requires_grad_()
    y, h = rms_norm(X, W, residual=R)
    assert torch.equal(h, x + res)
    hd = (x + res).double()
    rstd = (hd.square().mean(1, keepdim=True) + 1e-6).rsqrt()
    exact = x.double() + res.double()
    ref = exact * (exact.square().mean(1, keepdim=True) + 1e-6).rsqrt() * w.double()
    assert U.rel_l2(y, ref) < 8 * 2.0 ** -24
    dx, dr, dw = torch.autograd.grad((y, h), (X, R, W), (dy, dh))
    t = dy.double() * w.double()
    gh = dh.double() + rstd * (t - hd * rstd ** 2 * (t * hd).mean(1, keepdim=True))
    size = float(gh.norm()) + float((t * rstd).norm())
    assert float((dx.double() - gh).norm()) < 32 * 2.0 ** -24 * size and torch.equal(dx, dr)
    assert U.rel_l2(dw, (dy.double() * hd * rstd).sum(0)) < (64 * 2.0 ** -24 if weight == torch.float32 else 2.0 ** -8)
    q, h8 = rms_norm(x, w, residual=res, quantize=True)
    codes, scales = U.rows(y.detach().cpu())
    assert U.same_bits(q.codes, codes) and torch.equal(q.scales.cpu(), scales) and torch.equal(h8, h)
    assert U.rel_l2(rms_norm(x, w), x.double() * (x.double().square().mean(1, keepdim=True) + 1e-6).rsqrt() *
                    w.double()) < 8 * 2.0 ** -24
    assert bool(wide[:, :4].isnan().all()) and bool(wide[:, 4 + k:].isnan().all())
