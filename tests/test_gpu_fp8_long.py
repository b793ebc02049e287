"""The 8-bit operators on tens of millions of tokens and on long linear passes (needs
a B200): results against float64 of the same codes on the device."""
import pytest
import torch

pytestmark = pytest.mark.gpu

L2 = 4e-6                 # of one product of 128 terms, as derived beside the product's tests
LONG = 65535 * 128        # rows that one launch of the quantisation takes


@pytest.fixture(autouse=True, scope="module")
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from race_attention_b200 import _lib
    _lib.load()


def bits(a, b):
    return torch.equal(a.codes.view(torch.uint8), b.codes.view(torch.uint8)) and torch.equal(a.scales, b.scales)


def randn(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)


@pytest.mark.parametrize("extra", [0, 1, 300])
@pytest.mark.parametrize("square", [False, True], ids=["rows", "square"])
def test_quantize_more_rows_than_a_launch_takes(extra, square):
    """The same bits as the parts have that end on a block."""
    from race_attention_b200.fp8 import BlockFp8, quantize_fp8
    x = randn(LONG + extra, 17, dtype=torch.bfloat16)
    a, t = quantize_fp8(x, square=square, transposed=True)
    alone, only = quantize_fp8(x, square=square), quantize_fp8(x, square=square, transposed="only")
    assert bits(a, alone) and bits(t, only) and not bool((a.codes.view(torch.uint8) & 0x7f == 0x7f).any())
    block = 128 if square else 1
    for r0, r1 in ((0, 1280), (LONG - 1280, LONG), (LONG, LONG + extra)):
        if r0 == r1:
            continue
        p, q = quantize_fp8(x[r0:r1], square=square, transposed=True)
        assert bits(BlockFp8(a.codes[r0:r1], a.scales[r0 // block:-(-r1 // block)]), p) or (square and r1 - r0 == 1)
        assert torch.equal(a.codes[r0:r1].view(torch.uint8), p.codes.view(torch.uint8))
        assert torch.equal(t.codes[:, r0:r1].view(torch.uint8), q.codes.view(torch.uint8))
        assert torch.equal(t.scales[:, r0 // 128:-(-r1 // 128)], q.scales)


def close(got, ref, tol):
    return float((got.double() - ref).norm() / ref.norm()) < tol


@pytest.mark.parametrize("r,n,k,dtype", [
    (LONG + 300, 24, 16, torch.bfloat16),       # more rows than a launch quantises
    (65536, 2304, 768, torch.bfloat16),         # pairs of CTAs in all three products, dW's contraction cut
    (20001, 1000, 520, torch.float32),
    (3001, 4096, 1024, torch.float32)])
def test_long_linear_pass(r, n, k, dtype):
    """y, dx and dW against float64 products of what the quantisation gives (whose bits
    have tests of their own).  A contraction over j blocks adds j roundings in 32 bits."""
    from race_attention_b200.fp8 import fp8_linear, quantize_fp8
    x, w, dy = randn(r, k, dtype=dtype), randn(n, k, seed=1) * 0.05, randn(r, n, seed=2, dtype=dtype)
    X, W = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = fp8_linear(X, W)
    dx, dw = torch.autograd.grad(y, (X, W), dy)
    assert y.dtype == dx.dtype == dtype and dw.dtype == torch.float32
    tol = lambda length, t: L2 + (length / 128) ** 0.5 * 2.0 ** -24 + (2.0 ** -8 if t == torch.bfloat16 else 0)  # noqa: E731
    wv = quantize_fp8(w, square=True).dequantize().double()
    gw = torch.zeros(n, k, dtype=torch.float64, device="cuda")
    (xr, xt), (dr, dt) = quantize_fp8(x, transposed=True), quantize_fp8(dy, transposed=True)
    step = 1 << 20
    for r0 in range(0, r, step):
        s = slice(r0, min(r0 + step, r))
        b = slice(r0 // 128, -(-s.stop // 128))
        from race_attention_b200.fp8 import BlockFp8
        part = lambda q: BlockFp8(q.codes[s], q.scales[s]).dequantize().double()  # noqa: E731
        turned = lambda q: BlockFp8(q.codes[:, s], q.scales[:, b]).dequantize().double()  # noqa: E731
        assert close(y.detach()[s], part(xr) @ wv.t(), tol(k, dtype))
        assert close(dx[s], part(dr) @ wv, tol(n, dtype))
        gw += turned(dt) @ turned(xt).t()
    assert close(dw, gw, tol(r, torch.float32))
