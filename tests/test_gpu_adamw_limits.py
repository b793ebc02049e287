"""The AdamW step at the ends of its range (needs a B200)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from race_attention_b200 import _lib
    _lib.load()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("large", [1.0, 1e10, 1e17])
def test_no_second_moment_above_zero_is_held_as_zero(large, dtype):
    """One large gradient in each block, the others down to where their square's
    average is the smallest float above zero: 1e-3 * (2e-21)^2 = 4e-45."""
    from race_attention_b200.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(256, device="cuda", dtype=dtype))
    opt = AdamW([p], lr=1e-3, betas=(0.9, 0.999), state_bits=8, weight_decay=0.0)
    p.grad = torch.logspace(-20.7, -3, 256, device="cuda").to(dtype)
    p.grad[::128] = large
    p.grad[5] = 0
    opt.step()
    codes = opt.exp_avg_sq.float()
    zero = torch.zeros(256, dtype=torch.bool, device="cuda")
    zero[5] = True                   # its second moment is zero
    assert torch.equal(codes == 0, zero) and float(codes.max()) == 448
    assert float(p.detach().float().abs().max()) < 1e-2
