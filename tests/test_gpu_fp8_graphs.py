"""The 8-bit operators in CUDA graphs (needs a B200): the passes can be captured, the
optimizer's step cannot."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from race_attention_b200 import _lib
    _lib.load()


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_a_captured_step_is_refused(bits, dtype):
    """A replay would repeat the captured step's count, rate and noise."""
    from race_attention_b200._lib import RaceError
    from race_attention_b200.optim import AdamW
    p = torch.nn.Parameter(torch.ones(300, device="cuda", dtype=dtype))
    twin = torch.nn.Parameter(p.detach().clone())
    opt, other = AdamW([p], state_bits=bits, seed=1), AdamW([twin], state_bits=bits, seed=1)
    p.grad, twin.grad = torch.ones_like(p), torch.ones_like(p)
    opt.step()
    other.step()
    held = torch.zeros(1, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held += 1                       # the capture goes on
        with pytest.raises(RaceError, match="capture"):
            opt.step()
    g.replay()
    torch.cuda.synchronize()
    assert float(held) == 1 and opt.state[p]["step"] == 1 and torch.equal(p, twin)
    opt.step()
    other.step()
    assert opt.state[p]["step"] == 2 and torch.equal(p, twin)


def captured(f, inputs):
    """f's results of other inputs, from a graph captured with these."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        f(*inputs)                      # what a first call sets up stays outside
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = f(*inputs)
    for x in inputs:
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, device="cuda") * 0.5 + 0.1)
    ref = [t.clone() for t in f(*inputs)]
    g.replay()
    torch.cuda.synchronize()
    return out, ref


@pytest.mark.parametrize("rows", [1, 40, 1000])
def test_serving_calls(rows):
    from race_attention_b200.fp8 import fp8_linear, quantize_fp8, rms_norm
    held = quantize_fp8(torch.randn(384, 256, device="cuda"), square=True)

    @torch.no_grad()
    def f(x, w):
        y, h = rms_norm(x, w, residual=x, quantize=True)
        a, t = quantize_fp8(x, transposed=True)
        return (y.codes.view(torch.uint8), y.scales, h, fp8_linear(y, held), fp8_linear(x, held), rms_norm(x, w),
                a.codes.view(torch.uint8), t.codes.view(torch.uint8), t.scales)

    got, ref = captured(f, [torch.randn(rows, 256, device="cuda"), torch.ones(256, device="cuda")])
    assert all(torch.equal(a, b) for a, b in zip(got, ref))


@pytest.mark.parametrize("rows", [5, 1000])
def test_training_passes(rows):
    from race_attention_b200.fp8 import fp8_linear, rms_norm

    def f(x, n, w, dy):
        y, h = rms_norm(x, n, residual=x)
        z = fp8_linear(y, w)
        return (z.detach(), *torch.autograd.grad((z, h), (x, n, w), (dy, x.detach())))

    x = torch.randn(rows, 256, device="cuda").requires_grad_()
    n = torch.ones(256, device="cuda").requires_grad_()
    w = torch.randn(384, 256, device="cuda").requires_grad_()
    got, ref = captured(f, [x, n, w, torch.randn(rows, 384, device="cuda")])
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
