"""The 8-bit operators beside torch's autograd (needs a B200): writes into a caller's
tensor are seen by its version check."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from race_attention_b200 import _lib
    _lib.load()


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda()


@pytest.mark.parametrize("bits", [8, 32])
def test_a_step_between_the_passes_is_seen(bits):
    from race_attention_b200.fp8 import rms_norm
    from race_attention_b200.optim import AdamW
    x, w, still = randn(4, 64), torch.nn.Parameter(torch.ones(64, device="cuda")), torch.nn.Parameter(randn(64))
    opt = AdamW([w, still], state_bits=bits)
    w.grad = torch.ones_like(w)
    kept = still._version
    y = rms_norm(x, w)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    assert still._version == kept           # it had no gradient and did not move
    opt.zero_grad()
    rms_norm(x, w).sum().backward()
    assert w.grad is not None


def test_a_product_into_a_saved_tensor_is_seen():
    from race_attention_b200.fp8 import fp8_matmul, quantize_fp8
    a, b = quantize_fp8(randn(8, 256)), quantize_fp8(randn(16, 256, seed=1))
    out = torch.ones(8, 16, device="cuda")
    x = randn(8, 16, seed=2).requires_grad_()
    y = (x * out).sum()
    assert fp8_matmul(a, b, torch.float32, out=out) is out
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_tangents_are_refused():
    """Without an input that requires grad no autograd function stands in the way: the
    call itself refuses, with gradients enabled or not."""
    import torch.autograd.forward_ad as fw
    from race_attention_b200.fp8 import fp8_linear, quantize_fp8, rms_norm
    x, w, n = randn(8, 256), randn(96, 256, seed=1), torch.ones(256, device="cuda")
    held = quantize_fp8(w, square=True)
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
        calls = [lambda: fp8_linear(dual(x), w), lambda: fp8_linear(x, dual(w)), lambda: fp8_linear(dual(x), held),
                 lambda: fp8_linear(dual(x).half(), w), lambda: rms_norm(dual(x), n), lambda: rms_norm(x, dual(n)),
                 lambda: rms_norm(x, n, residual=dual(x)), lambda: rms_norm(dual(x), n, quantize=True),
                 lambda: fp8_linear(dual(x).requires_grad_(), w)]
        for f in calls:
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode|jvp"):
                    f()
        with pytest.raises(ValueError, match="no gradient"):
            fp8_linear(quantize_fp8(x), dual(w))
        assert fp8_linear(x, w).shape == (8, 96) and rms_norm(x, n).shape == x.shape    # nothing to lose here


@pytest.mark.parametrize("lead", [(6,), (2, 3), ()], ids=["rows", "axes", "vector"])
def test_results_change_in_place(lead):
    """y += b, an in-place activation and a slice's assignment, with the gradients of
    the same steps out of place."""
    from race_attention_b200.fp8 import fp8_linear, rms_norm
    b = randn(96, seed=5)

    def leaves():
        return [t.requires_grad_() for t in (randn(*lead, 256), randn(96, 256, seed=1), 1 + 0.1 * randn(256, seed=2),
                                             randn(*lead, 256, seed=3))]

    def run(inplace):
        x, w, n, r = leaves()
        y, h = rms_norm(x, n, residual=r)
        u = rms_norm(x, n)
        if inplace:
            y *= 0.5
            torch.relu_(u)
        else:
            y, u = y * 0.5, torch.relu(u)
        z = fp8_linear(y + u, w)
        if inplace:
            z += b
            torch.nn.functional.relu(z, inplace=True)
        else:
            z = torch.relu(z + b)
        return (z.detach(), *torch.autograd.grad((z, h), (x, w, n, r), (torch.ones_like(z), randn(*lead, 256, seed=4))))

    for got, ref in zip(run(True), run(False)):
        assert torch.equal(got, ref)


def test_a_changed_residual_is_seen():
    """The backward pass reads h, so it has to refuse one that changed."""
    from race_attention_b200.fp8 import rms_norm
    x, n = randn(4, 256).requires_grad_(), torch.ones(256, device="cuda")
    y, h = rms_norm(x, n, residual=randn(4, 256, seed=1))
    h += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        (y.sum() + h.sum()).backward()


def test_results_hold_no_cycle():
    """A result that is dropped frees its memory at once, the graph with it."""
    import gc
    from race_attention_b200.fp8 import fp8_linear, rms_norm
    x, w, n = randn(512, 256).requires_grad_(), randn(96, 256, seed=1).requires_grad_(), torch.ones(256, device="cuda")
    gc.disable()
    try:
        for _ in range(2):
            torch.cuda.synchronize()
            before = torch.cuda.memory_allocated()
            y, h = rms_norm(x, n, residual=x)
            z = fp8_linear(h, w)
            del y, h, z
            after = torch.cuda.memory_allocated()
        assert after == before
    finally:
        gc.enable()
