"""bfloat16 parameters with 32-bit states against the formula in float64 (needs a B200)."""
import pytest
import torch

from tests import fp8_util as U

pytestmark = pytest.mark.gpu

LR, B1, B2, EPS, WD, SEED = 1e-2, 0.9, 0.95, 1e-8, 0.1, 77


@pytest.fixture(autouse=True, scope="module")
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from race_attention_b200 import _lib
    _lib.load()


@pytest.mark.parametrize("sizes", [[(1,), (7, 3), (129,), (2049,)], [(64, 96), (33, 333), (5000,)]], ids=["small", "more"])
def test_three_steps(sizes):
    """m and v: fewer than 32 roundings of 2^-24.  A parameter is its value in 64 bits cut to
    8 bits of mantissa, one step up where the part cut off and the element's noise reach a
    whole step.  The value in 32 bits is off by fewer than 16 roundings of 2^-24, 2^-12 of
    such a step: nearer than that to a whole one either neighbour is right."""
    from race_attention_b200.optim import AdamW
    g = torch.Generator().manual_seed(1)
    ps = [torch.nn.Parameter(torch.randn(*s, generator=g).bfloat16().cuda()) for s in sizes]
    opt = AdamW(ps, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, seed=SEED)
    states = [[0.0, 0.0] for _ in ps]
    for t in range(1, 4):
        before = [p.detach().cpu().double() for p in ps]
        grads = [(torch.randn(*s, generator=g) * 10.0 ** -t).bfloat16() for s in sizes]
        for p, x in zip(ps, grads):
            p.grad = x.cuda()
        opt.step()
        for p, old, x, s in zip(ps, before, grads, states):
            x = x.double()
            s[0], s[1] = B1 * s[0] + (1 - B1) * x, B2 * s[1] + (1 - B2) * x * x
            want = old * (1 - LR * WD) - LR / (1 - B1 ** t) * s[0] / ((s[1] / (1 - B2 ** t)).sqrt() + EPS)
            at, n = opt.offsets[p], p.numel()
            assert U.rel_l2(opt.exp_avg[at:at + n].view(p.shape), s[0]) < 32 * 2.0 ** -24
            assert U.rel_l2(opt.exp_avg_sq[at:at + n].view(p.shape), s[1]) < 32 * 2.0 ** -24
            unit = torch.exp2((torch.frexp(want)[1] - 8).double())        # of 8 bits of mantissa
            noise = (U.noise(torch.arange(n) + at, SEED, t, 1) & 0xFFFF).double().view(p.shape) / 65536
            reach = want.abs() / unit + noise
            fixed = (reach - reach.round()).abs() > 2.0 ** -12
            got = p.detach().cpu().double()
            assert torch.equal(got[fixed], (want.sign() * reach.floor() * unit)[fixed])
            assert bool(((got - want).abs() <= unit * (1 + 2.0 ** -12)).all())
            assert n < 100 or float(fixed.double().mean()) > 0.99
