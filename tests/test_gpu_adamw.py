"""The AdamW step on the GPU (needs a B200): 32-bit states against float64 and
torch.optim.AdamW, 8-bit states bit for bit against a restatement in 32-bit
operations."""
import math

import pytest
import torch

from tests import fp8_util as U

pytestmark = pytest.mark.gpu

LR, B1, B2, EPS, WD = 1e-2, 0.9, 0.95, 1e-8, 0.1


@pytest.fixture(autouse=True, scope="module")
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from race_attention_b200 import _lib
    _lib.load()


SIZES = [(1,), (7, 3), (128,), (129,), (64, 96), (2048,), (2049,), (0,), (33, 333)]


def model(dtype, seed=0, sizes=SIZES):
    g = torch.Generator().manual_seed(seed)
    ps = [torch.nn.Parameter(torch.randn(*s, generator=g).to(dtype).cuda()) for s in sizes]
    grads = [[(torch.randn(*s, generator=g) * 10.0 ** -i).to(dtype) for s in sizes] for i in range(3)]
    return ps, grads


def test_states_in_32_bits():
    """Three steps against the formula in float64: each operation rounds once,
    2^-24 of its result, fewer than 32 of them in three steps."""
    from race_attention_b200.optim import AdamW
    ps, grads = model(torch.float32)
    ref = [[p.detach().cpu().double(), 0.0, 0.0] for p in ps]
    opt = AdamW(ps, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD)
    twin = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    other = torch.optim.AdamW(twin, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD)
    for t, gs in enumerate(grads, 1):
        for p, q, g in zip(ps, twin, gs):
            p.grad, q.grad = g.cuda(), g.cuda()
        opt.step()
        other.step()
        for r, g in zip(ref, gs):
            g = g.double()
            r[1] = B1 * r[1] + (1 - B1) * g
            r[2] = B2 * r[2] + (1 - B2) * g * g
            r[0] = r[0] * (1 - LR * WD) - LR / (1 - B1 ** t) * r[1] / ((r[2] / (1 - B2 ** t)).sqrt() + EPS)
    tol = 32 * 2.0 ** -24
    for p, q, r in zip(ps, twin, ref):
        if not p.numel():
            continue
        assert U.rel_l2(p, r[0]) < tol and U.rel_l2(p, q) < 2 * tol
        at = opt.offsets[p]
        m, v = (s[at:at + p.numel()].view(p.shape) for s in (opt.exp_avg, opt.exp_avg_sq))
        assert U.rel_l2(m, r[1]) < tol and U.rel_l2(v, r[2]) < tol


def plain_step(p, m, v, g, t, seed, first, bits, held):
    """One step of one flat tensor padded to 128, in 32-bit operations on the CPU."""
    f = lambda x: torch.tensor(x, dtype=torch.float32)  # noqa: E731
    if bits == 8:
        m = held[0].float() * held[1].repeat_interleave(128)
        v = (held[2].float() * held[3].repeat_interleave(128)).square()
    m = f(B1) * m + f(1 - B1) * g
    v = f(B2) * v + f(1 - B2) * g * g
    root = v.sqrt()
    q = p.double() * (1 - LR * WD) - LR / (1 - B1 ** t) * m.double() / (root.double() / math.sqrt(1 - B2 ** t) + EPS)
    i = torch.arange(p.numel()) + first
    r = U.noise(i, seed, t, 0)
    return q, m, v, (*U.hold(m, r & 0xFFFF, False), *U.hold(root, r >> 16, True))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_states_in_8_bits(dtype):
    """Codes and scales equal the restatement's bit for bit after each of three steps."""
    from race_attention_b200.optim import AdamW
    ps, grads = model(dtype, seed=3)
    opt = AdamW(ps, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, state_bits=8, seed=77)
    pad = lambda x: torch.nn.functional.pad(x.reshape(-1).float(), (0, (-x.numel()) % 128))  # noqa: E731
    held = [[torch.zeros(pad(p.detach().cpu()).numel()).to(U.F8), torch.zeros(-(-p.numel() // 128)),
             torch.zeros(pad(p.detach().cpu()).numel()).to(U.F8), torch.zeros(-(-p.numel() // 128))] for p in ps]
    for t, gs in enumerate(grads, 1):
        before = [pad(p.detach().cpu()) for p in ps]
        for p, g in zip(ps, gs):
            p.grad = g.cuda()
        opt.step()
        for i, (p, g) in enumerate(zip(ps, gs)):
            n = p.numel()
            if not n:
                continue
            at = opt.offsets[p]
            q, m, v, held[i] = plain_step(before[i], None, None, pad(g), t, 77, at, 8, held[i])
            cm, sm, cv, sv = held[i]
            e = at + cm.numel()
            assert U.same_bits(opt.exp_avg[at:e], cm) and U.same_bits(opt.exp_avg_sq[at:e], cv)
            assert torch.equal(opt.exp_avg_scale[at // 128:e // 128].cpu(), sm)
            assert torch.equal(opt.exp_avg_sq_scale[at // 128:e // 128].cpu(), sv)
            if dtype == torch.float32:
                assert U.rel_l2(p.reshape(-1), q[:n]) < 16 * 2.0 ** -24
            else:
                # up or down: within a step of the format (2^-7 of itself), right on average
                d = p.detach().cpu().double().reshape(-1) - q[:n]
                assert bool((d.abs() <= 2.0 ** -7 * q[:n].abs() * 1.01).all())


def test_rounding_is_right_on_average():
    """bfloat16 parameters and 8-bit states move by their mean even where a single
    change is far below a step.  n elements of one value: the mean of their
    roundings is off by a step / sqrt(12 n) or so; 6 of those are allowed."""
    from race_attention_b200.optim import AdamW
    n = 1 << 16
    p = torch.nn.Parameter(torch.full((n,), 1.0, dtype=torch.bfloat16, device="cuda"))
    opt = AdamW([p], lr=1e-4, betas=(0.9, 0.999), eps=0.0, weight_decay=0.0, state_bits=8, seed=5)
    p.grad = torch.ones_like(p)
    for _ in range(20):
        opt.step()
    # m / sqrt(v) = 1 up to the states' own rounding (each right on average), 20 steps of 1e-4
    step = 2.0 ** -8          # spacing just below 1
    assert abs(float(p.double().mean()) - (1 - 20e-4)) < 6 * step * 20 ** 0.5 / (12 * n) ** 0.5 + 0.02 * 20e-4
    big = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    opt = AdamW([big], lr=0.0, betas=(0.9, 0.999), state_bits=8, seed=6)
    big.grad = torch.full_like(big, 0.37)
    big.grad[::128] = 1.0     # one element of each block sets its scale
    opt.step()
    root0 = math.sqrt(0.001) * 0.37
    keep = torch.ones(n, dtype=torch.bool)
    keep[::128] = False
    for t in range(2, 30):    # only decay from here on: 0.05 % of the root a step
        big.grad.zero_()
        opt.step()
    v = opt.exp_avg_sq.float() * opt.exp_avg_sq_scale.repeat_interleave(128)
    got, want = float(v.cpu()[keep].double().mean()), root0 * 0.999 ** 14
    # 29 roundings of codes 1/8 to 1/16 apart: each right on average
    assert abs(got / want - 1) < 6 * (1 / 8) * 29 ** 0.5 / (12 * n) ** 0.5


def test_small_second_moment_is_not_held_as_zero():
    from race_attention_b200.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(128, device="cuda"))
    opt = AdamW([p], lr=1e-3, state_bits=8, weight_decay=0.0)
    g = torch.full((128,), 1e-9, device="cuda")
    g[0] = 1.0
    p.grad = g
    for _ in range(5):
        opt.step()
    assert float(opt.exp_avg_sq.float().min()) >= 2.0 ** -9
    assert float(p.detach().abs().max()) < 6e-3


def test_many_tensors_and_skipped_ones():
    """More tensors than one launch carries; none without a gradient moves."""
    from race_attention_b200 import _lib
    from race_attention_b200.optim import AdamW
    ps = [torch.nn.Parameter(torch.full((5 + i % 200,), float(i), device="cuda")) for i in range(800)]
    opt = AdamW(ps, lr=1.0, eps=0.0, weight_decay=0.0)
    for i, p in enumerate(ps):
        if i % 3:
            p.grad = torch.ones_like(p)
    opt.step()
    assert len(_lib.last_kernels()) >= 2 and set(_lib.last_kernels()) == {"adamw"}
    for i, p in enumerate(ps):
        # m / sqrt(v) of the first step is the gradient's sign, up to four roundings
        want = float(i) - (1.0 if i % 3 else 0.0)
        assert bool(((p.detach() - want).abs() <= 2.0 ** -21 * (abs(want) + 1)).all())
        assert opt.state[p]["step"] == (1 if i % 3 else 0)
    opt.zero_grad(set_to_none=True)
    before = [p.detach().clone() for p in ps]
    opt.step()
    assert all(torch.equal(a, p) for a, p in zip(before, ps))


def test_odd_addresses_strided_gradients_and_groups():
    from race_attention_b200.optim import AdamW
    flat = torch.randn(5000, device="cuda")
    views = [torch.nn.Parameter(flat[1:1000]), torch.nn.Parameter(flat[1003:1003 + 60 * 50].view(60, 50))]
    twins = [torch.nn.Parameter(v.detach().clone()) for v in views]
    for v, w in zip(views, twins):
        g = torch.randn(*reversed(v.shape), device="cuda")
        v.grad = g.permute(*reversed(range(v.dim())))
        w.grad = v.grad.contiguous()
    a = AdamW([{"params": views[:1], "lr": 0.1}, {"params": views[1:], "weight_decay": 0.0}], lr=LR)
    b = AdamW([{"params": twins[:1], "lr": 0.1}, {"params": twins[1:], "weight_decay": 0.0}], lr=LR)
    for _ in range(2):
        a.step()
        b.step()
    for v, w in zip(views, twins):
        assert torch.equal(v, w)


@pytest.mark.parametrize("bits", [8, 32])
def test_nan_stays_in_its_block(bits):
    from race_attention_b200.optim import AdamW
    for dtype in (torch.float32, torch.bfloat16):
        p = torch.nn.Parameter(torch.ones(512, device="cuda", dtype=dtype))
        opt = AdamW([p], state_bits=bits)
        p.grad = torch.ones_like(p)
        p.grad[200] = float("nan")
        opt.step()
        bad = torch.zeros(512, dtype=torch.bool)
        bad[200] = True
        assert torch.equal(p.detach().isnan().cpu(), bad)
        opt.step()
        if bits == 8:
            bad[128:256] = True
        assert torch.equal(p.detach().isnan().cpu(), bad)


@pytest.mark.parametrize("bits", [8, 32])
def test_state_dict(bits):
    from race_attention_b200.optim import AdamW
    def run(split):
        ps, grads = model(torch.float32, seed=9)
        opt = AdamW(ps, lr=LR, state_bits=bits, seed=4)
        for i, gs in enumerate(grads):
            if split and i == 1:
                import io
                f = io.BytesIO()
                torch.save(opt.state_dict(), f)
                f.seek(0)
                opt = AdamW(ps, lr=0.5, state_bits=bits, seed=0)
                opt.load_state_dict(torch.load(f))
            for p, g in zip(ps, gs):
                p.grad = g.cuda()
            opt.step()
        return ps
    for a, b in zip(run(False), run(True)):
        assert torch.equal(a, b)
    ps, _ = model(torch.float32)
    with pytest.raises(ValueError, match="bits"):
        AdamW(ps, state_bits=40 - bits).load_state_dict(AdamW(ps, state_bits=bits).state_dict())
    with pytest.raises(ValueError, match="sizes|groups"):
        AdamW(ps, state_bits=bits).load_state_dict(AdamW(ps[4:], state_bits=bits).state_dict())


def test_refusals():
    from race_attention_b200.optim import AdamW
    p = torch.nn.Parameter(torch.ones(4, 4, device="cuda"))
    for kw in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(weight_decay=-0.1), dict(state_bits=16)):
        with pytest.raises(ValueError):
            AdamW([p], **kw)
    with pytest.raises(ValueError, match="CUDA"):
        AdamW([torch.nn.Parameter(torch.ones(3))])
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        AdamW([torch.nn.Parameter(torch.ones(3, device="cuda", dtype=torch.float16))])
    with pytest.raises(ValueError, match="contiguous"):
        AdamW([torch.nn.Parameter(torch.ones(4, 6, device="cuda").t())])
    opt = AdamW([p])
    p.grad = torch.ones(4, 4, device="cuda")
    p.data = torch.ones(40, 40, device="cuda")
    p.grad = torch.ones(40, 40, device="cuda")
    with pytest.raises(ValueError, match="changed"):
        opt.step()
