"""A layer's weight held in 8 bits follows the weight (needs a B200)."""
import copy
import io

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from race_attention_b200 import _lib
    _lib.load()


def layer(seed):
    from race_attention_b200.fp8 import Fp8Linear
    torch.manual_seed(seed)
    return Fp8Linear(256, 96, device="cuda")


def fresh(m, x):
    """What a layer with this weight, held now, gives."""
    from race_attention_b200.fp8 import fp8_linear, quantize_fp8
    return fp8_linear(x, quantize_fp8(m.weight, square=True))


def step(m):
    from race_attention_b200.optim import AdamW
    m.weight.grad = torch.ones_like(m.weight)
    AdamW([m.weight], lr=0.1).step()
    m.weight.grad = None


def torch_step(m):
    m.weight.grad = torch.ones_like(m.weight)
    torch.optim.SGD([m.weight], lr=0.1).step()
    m.weight.grad = None


def trained(m):
    m.train()
    step(m)
    m.eval()


def replaced(m):
    m.weight = layer(5).weight


CHANGES = {"state": lambda m: m.load_state_dict(layer(1).state_dict()),
           "assigned state": lambda m: m.load_state_dict(layer(1).state_dict(), assign=True),
           "step": step, "torch's step": torch_step, "training": trained, "type": lambda m: m.bfloat16(),
           "in place": lambda m: m.weight.detach().mul_(2), "replaced": replaced,
           "host and back": lambda m: m.cpu().cuda()}


@pytest.mark.parametrize("change", CHANGES.values(), ids=CHANGES.keys())
@torch.no_grad()
def test_a_held_weight_follows(change):
    m, x = layer(0).eval().hold(), torch.randn(7, 256, device="cuda")
    before = m(x)
    held = m.held
    assert torch.equal(before, fresh(m, x)) and m(x) is not None and m.held is held     # laid out once
    change(m)
    got = m(x)
    assert torch.equal(got, fresh(m, x)) and m.held is not held
    again = m.held
    assert torch.equal(m(x), got) and m.held is again
    if change not in (CHANGES["host and back"],):
        assert not torch.equal(got, before)


@torch.no_grad()
def test_a_copy_follows_its_own_weight():
    m, x = layer(0), torch.randn(7, 256, device="cuda")
    for _ in range(3):
        m.weight.mul_(1.5)
    m.eval().hold()
    ref = m(x)
    f = io.BytesIO()
    torch.save(m, f)
    f.seek(0)
    for c in (copy.deepcopy(m), torch.load(f, weights_only=False)):
        assert torch.equal(c(x), ref)
        c = copy.deepcopy(m)
        for _ in range(3):
            c.weight.mul_(2)
        assert torch.equal(c(x), fresh(c, x)) and torch.equal(m(x), ref)


def test_a_weight_without_a_count():
    with torch.inference_mode():
        m, x = layer(0).eval().hold(), torch.randn(7, 256, device="cuda")
        held = m.held
        assert torch.equal(m(x), fresh(m, x)) and m.held is held


def test_one_row_serves_as_either_kind():
    """One row has the same scales by rows and by blocks: both are taken wherever one is."""
    from race_attention_b200.fp8 import BlockFp8, fp8_linear, fp8_matmul, quantize_fp8
    x, w = torch.randn(1, 300, device="cuda"), torch.randn(1, 300, device="cuda")
    a, s = quantize_fp8(x), quantize_fp8(x, square=True)
    h, t = quantize_fp8(w, square=True, transposed=True)
    again = BlockFp8(h.codes, h.scales)                       # as a program that stored both would
    ref = fp8_matmul(a, h, torch.float32)
    for left in (a, s):
        for right in (h, again, quantize_fp8(w)):
            assert torch.equal(fp8_matmul(left, right, torch.float32), ref)
    assert torch.equal(fp8_linear(x, again), ref) and torch.equal(fp8_linear(x, quantize_fp8(w)), ref)
    z = torch.randn(5, 1, device="cuda").requires_grad_()      # and as the transpose of one column
    v, u = quantize_fp8(torch.randn(300, 1, device="cuda"), square=True, transposed=True)
    grads = [torch.autograd.grad(fp8_linear(z, (v, q)), z, torch.ones(5, 300, device="cuda"))[0]
             for q in (u, BlockFp8(u.codes, u.scales.clone()))]
    assert grads[0].shape == z.shape and torch.equal(*grads)
    with pytest.raises(ValueError, match="square"):
        fp8_linear(x, quantize_fp8(torch.randn(2, 300, device="cuda")))
    with pytest.raises(ValueError, match="scale for each row"):
        fp8_matmul(quantize_fp8(torch.randn(2, 300, device="cuda"), square=True), h)


def test_gradients_in_eval_mode():
    """A held layer passes the gradients that it passes without its copy."""
    m, x = layer(0), torch.randn(7, 256, device="cuda", requires_grad=True)
    m.eval()
    ref = torch.autograd.grad(m(x).square().sum(), (x, m.weight))
    m.hold()
    got = torch.autograd.grad(m(x).square().sum(), (x, m.weight))
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    assert not m(x.detach()).requires_grad          # served


def test_a_held_decoder_in_eval_mode_has_gradients():
    from race_attention_b200.block8 import RACEDecoder8
    torch.manual_seed(0)
    model = RACEDecoder8(vocab=64, width=128, heads=4, layers=2, device="cuda").eval()
    tokens = torch.randint(0, 64, (2, 50), device="cuda")
    model(tokens).float().square().mean().backward()
    ref = {n: p.grad.clone() for n, p in model.named_parameters()}
    model.zero_grad()
    model.hold()
    model(tokens).float().square().mean().backward()
    for n, p in model.named_parameters():
        assert torch.equal(p.grad, ref[n]), n
