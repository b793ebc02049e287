"""8-bit operators on tensors of nothing (needs a B200)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from race_attention_b200 import _lib
    _lib.load()


NOTHING = [(lead, n, k) for lead in ((), (6,), (2, 3), (2, 0), (0,)) for n, k in ((5, 0), (0, 16), (0, 0), (5, 16))
           if 0 in (*lead, n, k)]


@pytest.mark.parametrize("lead,n,k", NOTHING, ids=str)
def test_linear(lead, n, k):
    """Sums over nothing are zero, forward and backward, whatever the leading axes."""
    from race_attention_b200.fp8 import fp8_linear, quantize_fp8
    x = torch.ones(*lead, k, device="cuda").requires_grad_()
    w = torch.ones(n, k, device="cuda").requires_grad_()
    y = fp8_linear(x, w)
    assert y.shape == (*lead, n) and bool((y == 0).all())
    dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
    rows = x.numel() // k if k else torch.Size(lead).numel()
    assert dx.shape == x.shape and bool((dx == 0).all())
    assert dw.shape == w.shape and bool((dw == 0).all())
    a, t = quantize_fp8(x, transposed=True)
    assert a.shape == (rows, k) and t.shape == (k, rows)
