"""The norm's backward pass in each of its forms (needs a B200): rows that wait in shared
memory or in registers, by type and width, with more rows than the grid has places."""
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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("r,k", [(9000, 64), (8000, 96), (7001, 104), (5000, 256), (3000, 264), (2500, 768),
                                 (1500, 1024), (1300, 1032), (901, 3000), (700, 4096), (400, 4104), (333, 6144),
                                 (301, 8192), (200, 12288), (170, 16384)])
@pytest.mark.parametrize("both", [True, False], ids=["dh", "alone"])
def test_gradients(r, k, dtype, both):
    """Bounds as derived beside the norm's other gradients: a few roundings of either
    term of dx in 32 bits, and for bfloat16 one of the result and one of the held h;
    dweight sums its rows in 32 bits, one after the other within a warp."""
    from race_attention_b200.fp8 import rms_norm
    g = torch.Generator(device="cuda").manual_seed(k)
    x, res, dy, dh = (torch.randn(r, k, generator=g, device="cuda").to(dtype) for _ in range(4))
    w = 1 + 0.2 * torch.randn(k, generator=g, device="cuda")
    h = (x.float() + res.float()).to(dtype).double()
    rstd = (h.square().mean(1, keepdim=True) + 1e-6).rsqrt()
    t = dy.double() * w.double()
    gh = rstd * (t - h * rstd ** 2 * (t * h).mean(1, keepdim=True))
    size = float((gh + dh.double()).norm()) + float((t * rstd).norm())
    if both:
        gh = gh + dh.double()
    gw = (dy.double() * h * rstd).sum(0)
    grads = []
    for _ in range(2):
        X, R, W = x.clone().requires_grad_(), res.clone().requires_grad_(), w.clone().requires_grad_()
        yy, hh = rms_norm(X, W, residual=R)
        torch.autograd.backward((yy, hh) if both else (yy,), (dy, dh) if both else (dy,))
        grads.append((X.grad, R.grad, W.grad))
    dx, dr, dw = grads[0]
    tol = 32 * 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -8
    assert float((dx.double() - gh).norm()) < tol * size and torch.equal(dx, dr)
    assert U.rel_l2(dw, gw) < (64 * 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -8)
    assert all(torch.equal(a, b) for a, b in zip(*grads))         # a fixed order of sums
