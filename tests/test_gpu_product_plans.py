"""Products at the sides of each choice of kernel, ranks and splits (needs a B200)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from race_attention_b200 import _lib
    _lib.load()


@pytest.mark.parametrize("square", [True, False], ids=["square", "rows"])
@pytest.mark.parametrize("m,n,k", [(33, 768, 3000), (40, 512, 3000), (64, 4096, 4096), (128, 8192, 8192), (256, 4096, 4096),
                                   (2048, 512, 4096), (1000, 333, 5000), (300, 1000, 8192), (1800, 1536, 768),
                                   (2048, 1280, 768), (16384, 384, 384), (785, 2304, 768), (65, 1000, 16000)])
def test_products(m, n, k, square):
    """Against float64 of the same codes: 128 terms a block in 32 bits, 4e-6 in the 2-norm
    as derived beside the product's other tests, and one rounding of 2^-24 a block."""
    from race_attention_b200.fp8 import fp8_matmul, quantize_fp8
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    a = quantize_fp8(torch.randn(m, k, generator=g, device="cuda") * torch.rand(m, 1, generator=g, device="cuda").exp())
    b = quantize_fp8(torch.randn(n, k, generator=g, device="cuda") * 0.02, square=square)
    ref = a.dequantize().double() @ b.dequantize().double().t()
    y = fp8_matmul(a, b, torch.float32)
    tol = 4e-6 + (k / 128) ** 0.5 * 2.0 ** -24
    rows = (y.double() - ref).norm(dim=1) / ref.norm(dim=1)
    assert float((y.double() - ref).norm() / ref.norm()) < tol and float(rows.max()) < 2 * tol
    assert torch.equal(y, fp8_matmul(a, b, torch.float32))
    assert torch.equal(fp8_matmul(a, b), y.bfloat16())
