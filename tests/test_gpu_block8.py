"""The 8-bit operators together (needs a B200): a RACE block and a small decoder,
trained and served."""
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


def plain_block(block, x, residual):
    """The same block with float32 linear layers and norms written out."""
    norm = lambda z, w: z * (z.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w  # noqa: E731
    B, T, W = x.shape
    h = x + residual
    q, k, v = (norm(h, block.norm1.weight) @ block.qkv.weight.t()).view(B, T, 3, block.heads, block.d_k).unbind(2)
    a = block.ace(*(z.unsqueeze(0).contiguous() for z in (k, v, q)))[0].reshape(B, T, W)
    h = h + a @ block.out.weight.t()
    z = torch.nn.functional.gelu(norm(h, block.norm2.weight) @ block.up.weight.t())
    return z @ block.down.weight.t(), h


def test_block_against_float32():
    """A code is off by at most 2^-4 of itself, 2^-4 / sqrt(3) = 3.6 % in the 2-norm;
    a product of two such operands by 5.1 %, and the block's branch passes
    through four of them: below 4 * 5.1 %."""
    from race_attention_b200.block8 import RACEBlock8
    torch.manual_seed(1)
    block = RACEBlock8(384, 6, device="cuda")
    x, r = torch.randn(2, 200, 384, device="cuda"), torch.randn(2, 200, 384, device="cuda")
    leaves = []
    grads = []
    outs = []
    for f in (lambda a, b: block(a, b), lambda a, b: plain_block(block, a, b)):
        a, b = x.clone().requires_grad_(), r.clone().requires_grad_()
        z, h = f(a, b)
        block.zero_grad()
        (z.square().mean() + h.square().mean()).backward()
        outs.append((z.detach(), h.detach()))
        grads.append({n: p.grad.clone() for n, p in block.named_parameters()} | {"x": a.grad, "r": b.grad})
        leaves.append((a, b))
    for got, ref in zip(*outs):
        assert U.rel_l2(got, ref) < 4 * 0.051
    for n in grads[0]:
        # backwards through as many products again
        assert U.rel_l2(grads[0][n], grads[1][n]) < 8 * 0.051, n


def test_decoder_trains_and_serves():
    from race_attention_b200 import _lib
    from race_attention_b200.block8 import RACEDecoder8, train
    torch.manual_seed(2)
    model = RACEDecoder8(vocab=64, width=128, heads=4, layers=2, device="cuda")
    losses = train(model, steps=60, batch=8, tokens=96, lr=3e-3)
    assert losses[-1] < 0.6 * losses[0], losses
    tokens = torch.randint(0, 64, (2, 50), device="cuda")
    with torch.no_grad():
        ref = model(tokens)
        model.eval().hold()
        got = model(tokens)
        kernels = _lib.last_kernels()
        assert kernels and kernels[0].startswith("mm_")
        # served rows skip one rounding to bfloat16 before they are quantised: as far
        # as two quantisations of the same rows can be apart, through nine products
        assert U.rel_l2(got, ref) < 9 * 0.051
        one = model(tokens[:1, :1])
        assert one.shape == (1, 1, 64) and bool(one.isfinite().all())
        model.train().release()
        again = model(tokens)
    assert torch.equal(again, ref)


def test_one_launch_list_for_mixed_types():
    """float32 and bfloat16 parameters of one optimizer move as they do alone."""
    from race_attention_b200.optim import AdamW
    for bits in (8, 32):
        a = [torch.nn.Parameter(torch.randn(n, device="cuda").to(t)) for n, t in
             ((300, torch.float32), (5000, torch.bfloat16), (129, torch.float32), (64, torch.bfloat16))]
        b = [torch.nn.Parameter(p.detach().clone()) for p in a]
        for p, q in zip(a, b):
            p.grad = torch.randn_like(p)
            q.grad = p.grad.clone()
        both = AdamW(a, state_bits=bits, seed=3)
        one = AdamW(b, state_bits=bits, seed=3)
        for _ in range(2):
            both.step()
            for i in range(4):                       # one tensor at a time
                grads = [q.grad for q in b]
                for j, q in enumerate(b):
                    q.grad = grads[j] if j == i else None
                one.step()
                for q, g in zip(b, grads):
                    q.grad = g
        assert all(torch.equal(p, q) for p, q in zip(a, b))
