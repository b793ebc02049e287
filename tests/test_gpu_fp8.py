"""The 8-bit operators on the GPU (needs a B200): quantisation, the product of
8-bit operands, the linear layer trained through it and the norm.

Quantisation is compared bit for bit with a restatement in 32-bit operations.
The product is compared with float64 on the same codes: the tensor core adds
128 products at a time in 32 bits, each addition off by at most 2^-22 of
the terms' magnitudes, so 128 * 2^-22 = 2^-15 of sum |a||b| bounds every element
and, errors being independent, sqrt(128) * 2^-22 < 4e-6 the relative 2-norm;
a bfloat16 result adds 2^-8 of itself at most."""
import pytest
import torch

from tests import fp8_util as U

pytestmark = pytest.mark.gpu

L2 = 4e-6
BF16 = 2.0 ** -8


@pytest.fixture(autouse=True, scope="module")
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from race_attention_b200 import _lib
    _lib.load()


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=gen(seed)).to(dtype)


# ------------------------------------------------------------------ quantisation

SHAPES = [(1, 1), (1, 128), (3, 5), (7, 130), (127, 129), (128, 128), (130, 257), (300, 1000),
          (513, 48)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("r,k", SHAPES)
def test_quantize_rows_and_transpose(r, k, dtype):
    from race_attention_b200.fp8 import quantize_fp8
    x = (randn(r, k, seed=r + k) * randn(r, 1, seed=1).exp()).to(dtype)
    a, t = quantize_fp8(x.cuda(), transposed=True)
    for got, src in ((a, x), (t, x.t())):
        codes, scales = U.rows(src)
        assert got.codes.shape == codes.shape and torch.equal(got.scales.cpu(), scales)
        assert U.same_bits(got.codes, codes)
    alone, only = quantize_fp8(x.cuda()), quantize_fp8(x.cuda(), transposed="only")
    assert U.same_bits(alone.codes, a.codes) and U.same_bits(only.codes, t.codes)
    assert torch.equal(alone.scales, a.scales) and torch.equal(only.scales, t.scales)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("r,k", SHAPES)
def test_quantize_square(r, k, dtype):
    from race_attention_b200.fp8 import quantize_fp8
    x = randn(r, k, seed=r * 3 + k).to(dtype)
    a, t = quantize_fp8(x.cuda(), square=True, transposed=True)
    codes, scales = U.square(x)
    assert torch.equal(a.scales.cpu(), scales) and U.same_bits(a.codes, codes)
    assert torch.equal(t.scales.cpu(), scales.t()) and U.same_bits(t.codes, codes.t())
    only = quantize_fp8(x.cuda(), square=True, transposed="only")
    assert torch.equal(only.scales.cpu(), scales.t()) and U.same_bits(only.codes, codes.t())


def test_quantize_layouts():
    """Row strides, a base off 16 bytes, transposed and broadcast inputs, leading axes."""
    from race_attention_b200.fp8 import quantize_fp8
    big = randn(70, 300, seed=4).cuda()
    views = [big[:, 3:200], big[::2, :256], big.t(), big[:1].expand(5, 300), big[:, :256][:, 1:2],
             big.view(7, 10, 300), big[:, ::2]]
    for v in views:
        got = quantize_fp8(v)
        codes, scales = U.rows(v.reshape(-1, v.shape[-1]).cpu())
        assert torch.equal(got.scales.cpu(), scales) and U.same_bits(got.codes, codes)


def test_quantize_extreme_values():
    from race_attention_b200.fp8 import quantize_fp8
    x = randn(8, 384, seed=5)
    x[0, :128] = 0
    x[1, :128] *= 1e-42          # below the smallest scale
    x[2] *= 3e37
    x[3, 5] = float("nan")
    x[4, 130] = float("inf")
    x[5, 300] = float("-inf")
    x[6, 7] = 1e30               # one large value, the rest vanish beside it
    got = quantize_fp8(x.cuda())
    codes, scales = U.rows(x)
    assert U.same_bits(got.scales, scales) and U.same_bits(got.codes, codes)
    v = got.dequantize().cpu()
    bad = ~v.isfinite().view(8, 3, 128)
    whole = torch.zeros(8, 3, dtype=torch.bool)
    whole[3, 0] = whole[4, 1] = whole[5, 2] = True      # a block is non-finite throughout, or nowhere
    assert torch.equal(bad.all(2), whole) and torch.equal(bad.any(2), whole)
    assert not v[0, :128].any()


def test_quantize_empty():
    from race_attention_b200.fp8 import quantize_fp8
    a, t = quantize_fp8(torch.empty(0, 64, device="cuda"), transposed=True)
    assert a.codes.shape == (0, 64) and t.codes.shape == (64, 0)


# ------------------------------------------------------------------ product


def operands(m, n, k, square, seed=0):
    """Codes and scales on the CPU, values spread over many powers of two."""
    a = U.rows(randn(m, k, seed=seed) * randn(m, 1, seed=seed + 1).exp())
    w = randn(n, k, seed=seed + 2) * 0.02
    return a, (U.square(w) if square else U.rows(w))


def held(codes, scales):
    from race_attention_b200.fp8 import BlockFp8
    return BlockFp8(codes.cuda(), scales.cuda())


def check_product(y, a, b, bf16):
    va, vb = U.values(*a), U.values(*b)
    ref, mass = va @ vb.t(), va.abs() @ vb.abs().t()
    y = y.double().cpu()
    assert U.rel_l2(y, ref) < (BF16 if bf16 else L2)
    bound = 2.0 ** -15 * mass + (BF16 * ref.abs() if bf16 else 0) + 1e-37
    assert bool(((y - ref).abs() <= bound).all())


PRODUCTS = [(1, 1, 1), (1, 128, 128), (1, 2304, 768), (2, 130, 1000), (15, 512, 257), (16, 257, 640),
            (17, 384, 96), (33, 100, 384), (64, 129, 130), (65, 1536, 384), (100, 1, 50),
            (128, 128, 128), (129, 127, 255), (255, 256, 256), (256, 257, 384), (257, 640, 129),
            (785, 1160, 776), (1001, 520, 1048), (1024, 1024, 1024)]


@pytest.mark.parametrize("square", [True, False], ids=["square", "rows"])
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product(m, n, k, square):
    from race_attention_b200.fp8 import fp8_matmul
    a, b = operands(m, n, k, square, seed=m + n + k)
    A, B = held(*a), held(*b)
    check_product(fp8_matmul(A, B, torch.float32), a, b, False)
    check_product(fp8_matmul(A, B, torch.bfloat16), a, b, True)


@pytest.mark.parametrize("square", [True, False], ids=["square", "rows"])
@pytest.mark.parametrize("m,n,k", [(4096, 2304, 768), (5000, 1111, 700), (2304, 768, 20000),
                                   (300, 200, 33000), (9000, 260, 130), (2049, 4097, 385)])
def test_product_large(m, n, k, square):
    """Shapes that spread over every SM, and long contractions that are cut."""
    from race_attention_b200.fp8 import BlockFp8, fp8_matmul, quantize_fp8
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    x = torch.randn(m, k, generator=g, device="cuda")
    w = torch.randn(n, k, generator=g, device="cuda") * 0.02
    A, B = quantize_fp8(x), quantize_fp8(w, square=square)
    va, vb = A.dequantize().double(), B.dequantize().double()
    ref = va @ vb.t()
    # the long sum over blocks adds one rounding for each, 2^-24 of a running sum
    tol = L2 + (k / 128) ** 0.5 * 2.0 ** -24
    for dtype, t in ((torch.float32, tol), (torch.bfloat16, BF16)):
        y = fp8_matmul(A, B, dtype)
        assert float((y.double() - ref).norm() / ref.norm()) < t
        assert torch.equal(y, fp8_matmul(A, B, dtype))          # a fixed order of summation
    # the last rows and columns, where tiles are ragged
    y = fp8_matmul(A, B, torch.float32).double()
    for s in ((slice(-130, None), slice(None)), (slice(None), slice(-130, None))):
        assert float((y[s] - ref[s]).norm() / ref[s].norm()) < tol
    assert isinstance(B, BlockFp8)


def test_product_of_millions_of_rows():
    """More row tiles than a grid has along its second axis, with few columns."""
    from race_attention_b200.fp8 import fp8_matmul, quantize_fp8
    m = 65536 * 64 + 5
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(m, 32, generator=g, device="cuda").bfloat16()
    w = torch.randn(8, 32, generator=g, device="cuda")
    A, B = quantize_fp8(x), quantize_fp8(w, square=True)
    y = fp8_matmul(A, B, torch.float32)
    ref = A.dequantize() @ B.dequantize().t()
    assert float((y - ref).norm() / ref.norm()) < L2 + 32 * 2.0 ** -24     # the reference sums in 32 bits too
    assert float((y[-70:] - ref[-70:]).norm() / ref[-70:].norm()) < L2 + 32 * 2.0 ** -24


def test_product_layouts():
    """Scales of either order, codes off 16 bytes or with strided columns, a strided result."""
    from race_attention_b200.fp8 import BlockFp8, fp8_matmul
    a, b = operands(40, 70, 200, True, seed=9)
    ref = fp8_matmul(held(*a), held(*b), torch.float32)
    wide = torch.zeros(40, 331, dtype=torch.uint8, device="cuda").view(U.F8)
    wide.view(torch.uint8)[:, 7:207] = a[0].cuda().view(torch.uint8)
    cols = a[0].cuda().view(torch.uint8).t().contiguous().t().view(U.F8)
    sc = a[1].cuda()
    for codes in (wide[:, 7:207], cols):
        for s in (sc, sc.t().contiguous().t(), sc.repeat(1, 3)[:, ::1][:, :2]):
            assert torch.equal(fp8_matmul(BlockFp8(codes, s), held(*b), torch.float32), ref)
    big = torch.full((40, 101), 7.0, device="cuda")
    out = fp8_matmul(held(*a), held(*b), torch.float32, out=big[:, 5:75])
    assert torch.equal(out, ref) and float(big[:, :5].min()) == 7 and float(big[:, 75:].min()) == 7


def test_product_empty():
    from race_attention_b200.fp8 import fp8_matmul, quantize_fp8
    q = lambda r, k: quantize_fp8(torch.ones(r, k, device="cuda"))  # noqa: E731
    assert fp8_matmul(q(0, 64), q(5, 64)).shape == (0, 5)
    assert fp8_matmul(q(5, 64), q(0, 64)).shape == (5, 0)
    e = held(torch.empty(3, 0, dtype=U.F8), torch.empty(3, 0))
    f = held(torch.empty(4, 0, dtype=U.F8), torch.empty(4, 0))
    assert torch.equal(fp8_matmul(e, f, torch.float32), torch.zeros(3, 4, device="cuda"))


@pytest.mark.parametrize("m", [3, 300])
def test_product_non_finite(m):
    """A non-finite block shows in every result that it enters, and in no other."""
    from race_attention_b200.fp8 import fp8_matmul, quantize_fp8
    x, w = randn(m, 300, seed=1), randn(260, 300, seed=2)
    x[1, 130] = float("inf")
    w[258, 5] = float("nan")
    y = fp8_matmul(quantize_fp8(x.cuda()), quantize_fp8(w.cuda()), torch.float32).cpu()
    bad = torch.zeros(m, 260, dtype=torch.bool)
    bad[1] = True
    bad[:, 258] = True
    assert torch.equal(~y.isfinite(), bad)


def test_product_on_another_stream_and_in_a_graph():
    from race_attention_b200.fp8 import fp8_matmul
    a, b = operands(50, 300, 400, True, seed=3)
    A, B = held(*a), held(*b)
    ref = fp8_matmul(A, B)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = fp8_matmul(A, B)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, ref)
    g = torch.cuda.CUDAGraph()
    out = torch.zeros_like(ref)
    with torch.cuda.graph(g):
        fp8_matmul(A, B, out=out)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ref)


@pytest.mark.parametrize("rows", [1, 20, 100])
def test_products_in_a_row(rows):
    """Launches that prepare while the one before them ends still see its results:
    each product's input is the last one's, and the run is the same with a
    synchronisation after each call."""
    from race_attention_b200.fp8 import fp8_matmul, quantize_fp8
    w = [quantize_fp8((randn(512, 512, seed=s) / 512 ** 0.5).cuda(), square=True) for s in range(3)]

    def run(sync):
        x = quantize_fp8(randn(rows, 512, seed=9).cuda())
        outs = []
        for i in range(60):
            y = fp8_matmul(x, w[i % 3])
            # a product of the same inputs right behind it, into memory that is reused
            fp8_matmul(x, w[(i + 1) % 3])
            x = quantize_fp8(y)
            outs.append(y)
            if sync:
                torch.cuda.synchronize()
        return torch.stack(outs)

    assert torch.equal(run(False), run(True))


@pytest.mark.parametrize("m", [8, 1000])
def test_product_wait_limit(m):
    """A wait that runs out is reported, and the next call is whole again."""
    from race_attention_b200 import _lib
    from race_attention_b200.fp8 import fp8_matmul
    a, b = operands(m, 640, 1280, True, seed=6)
    A, B = held(*a), held(*b)
    ref = fp8_matmul(A, B)
    out = torch.empty_like(ref)
    word = torch.zeros(1, dtype=torch.int32, pin_memory=True)
    lib = _lib.load()
    desc = _lib.RaceMatmulDesc(_lib.RACE_BF16, 1, m, 640, 1280, 1, 0)
    need = lib.race_scaled_matmul_workspace(desc)
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    blocks = lambda b: _lib.RaceBlocks(b.codes.data_ptr(), b.codes.stride(0), b.scales.data_ptr(),  # noqa: E731
                                       *b.scales.stride())
    _lib.check(lib.race_scaled_matmul(desc, blocks(A), blocks(B), _lib.RaceRows(out.data_ptr(), 640),
                                      word.data_ptr(), ws.data_ptr(), need,
                                      torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert int(word) & _lib.RACE_DEV_TIMEOUT and not int(word) & _lib.RACE_DEV_STUCK
    assert torch.equal(fp8_matmul(A, B), ref)


def test_product_refusals():
    from race_attention_b200.fp8 import BlockFp8, fp8_matmul
    a, b = operands(8, 16, 256, True, seed=7)
    A, B = held(*a), held(*b)
    with pytest.raises(ValueError, match="same number of columns"):
        fp8_matmul(A, held(*operands(8, 16, 128, True)[1]))
    with pytest.raises(ValueError, match="scale for each row"):
        fp8_matmul(B, A)
    with pytest.raises(ValueError, match="out_dtype"):
        fp8_matmul(A, B, torch.float16)
    with pytest.raises(ValueError, match="contiguous columns"):
        fp8_matmul(A, B, out=torch.empty(16, 8, device="cuda", dtype=torch.bfloat16).t())
    with pytest.raises(ValueError, match="same device"):
        fp8_matmul(A, BlockFp8(*b))


# ------------------------------------------------------------------ linear layer


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("r,n,k", [(1, 130, 64), (77, 96, 257), (200, 640, 384), (1001, 1048, 520)])
def test_linear_against_the_formula(r, n, k, dtype):
    from race_attention_b200.fp8 import fp8_linear
    x, w = randn(r, k, seed=1).to(dtype), randn(n, k, seed=2) * 0.05
    dy = (randn(r, n, seed=3) * randn(r, 1, seed=4).exp()).to(dtype)
    X, W = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    y = fp8_linear(X, W)
    y.backward(dy.cuda())
    assert y.dtype == dtype and X.grad.dtype == dtype and W.grad.dtype == torch.float32
    wv = U.values(*U.square(w))
    tol = L2 if dtype == torch.float32 else BF16
    assert U.rel_l2(y, U.values(*U.rows(x)) @ wv.t()) < tol
    assert U.rel_l2(X.grad, U.values(*U.rows(dy)) @ wv) < tol
    assert U.rel_l2(W.grad, U.values(*U.rows(dy.t())) @ U.values(*U.rows(x.t())).t()) < L2


def test_linear_against_differences():
    """On values that the format holds exactly the layer is linear: moving one
    element to a neighbour that is held too changes the loss by gradient times step."""
    from race_attention_b200.fp8 import fp8_linear
    pick = torch.tensor([-448.0, -16.0, -2.0, 0.0, 1.0, 8.0, 20.0, 448.0])
    ints = lambda r, c, s: pick[torch.randint(0, 8, (r, c), generator=gen(s))]  # noqa: E731
    x, w, dy = ints(130, 256, 1), ints(140, 256, 2), ints(130, 140, 3)
    for t in (x, w, dy):           # every block, of rows and of columns, reaches 448
        t[:, ::128] = 448.0
        t[::128, :] = 448.0
    X, W, D = (t.cuda() for t in (x, w, dy))
    Xg, Wg = X.clone().requires_grad_(), W.clone().requires_grad_()
    fp8_linear(Xg, Wg, torch.float32).backward(D)
    loss = lambda a, b: float((fp8_linear(a, b, torch.float32).double() * D.double()).sum())  # noqa: E731
    with torch.no_grad():
        for T, grad, other in ((0, Xg.grad, W), (1, Wg.grad, X)):
            for i, j in ((3, 5), (77, 200), (129, 131)):
                base = (X, W)[T]
                moved, before = base.clone(), base.clone()
                before[i, j], moved[i, j] = 16.0, 18.0
                args = [(before, other), (moved, other)] if T == 0 else [(other, before), (other, moved)]
                diff = (loss(*args[1]) - loss(*args[0])) / 2.0
                # sums of integers below 2^24 steps are exact in 32 bits up to their last places
                assert abs(diff - float(grad[i, j])) <= 2.0 ** -20 * 448 * 448 * 256


def test_linear_leading_axes_frozen_weight_and_held_inputs():
    from race_attention_b200.fp8 import Fp8Linear, fp8_linear, quantize_fp8, rms_norm
    w = (randn(96, 192, seed=1) * 0.1).cuda()
    x = randn(2, 5, 192, seed=2).cuda()
    y = fp8_linear(x, w)
    assert y.shape == (2, 5, 96) and not y.requires_grad
    pair = quantize_fp8(w, square=True, transposed=True)
    xg = x.clone().requires_grad_()
    z = fp8_linear(xg, pair)
    z.backward(torch.ones_like(z))
    xh = x.clone().requires_grad_()
    z2 = fp8_linear(xh, w)
    z2.backward(torch.ones_like(z2))
    assert torch.equal(y, z.detach()) and torch.equal(xg.grad, xh.grad)
    with pytest.raises(ValueError, match="transpose"):
        fp8_linear(xg, pair[0])
    wt = w.clone().requires_grad_()                # x needs no gradient
    fp8_linear(x, wt).sum().backward()
    assert wt.grad.shape == w.shape
    weight = torch.ones(192, device="cuda")
    n8 = rms_norm(x, weight, quantize=True)
    n = rms_norm(x, weight)
    assert torch.equal(fp8_linear(n8, pair[0], torch.float32), fp8_linear(n, w).view(10, 96))
    with pytest.raises(ValueError, match="no gradient"):
        fp8_linear(n8, wt)
    layer = Fp8Linear(192, 96, device="cuda")
    a = layer(x)
    layer.eval()
    layer.hold()
    assert torch.equal(layer(x), a.detach()) and layer(n8).dtype == torch.bfloat16
    assert layer.release().held is None
    with pytest.raises(ValueError, match="columns"):
        fp8_linear(x[..., :100], w)
    with pytest.raises(RuntimeError, match="CUDA"):
        fp8_linear(x.cpu(), w)


# ------------------------------------------------------------------ norm


def norm_ref(x, w, res, eps):
    h = x.double() if res is None else x.double() + res.double()
    return h * (h.square().mean(1, keepdim=True) + eps).rsqrt() * w.double(), h


# A result in 32 bits carries the sum's, the root's and three products' roundings:
# below 8 * 2^-24 relative to itself; bfloat16 adds 2^-9 in the 2-norm's worst case.
F32_NORM = 8 * 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("r,k", [(1, 1), (3, 7), (5, 128), (9, 256), (4, 384), (130, 768), (2, 1000),
                                 (7, 1001), (3, 1024), (2, 1025), (2, 4096), (3, 5003), (2, 16384),
                                 (1, 16390), (2, 65536)])
def test_norm(r, k, dtype):
    from race_attention_b200.fp8 import rms_norm
    x, res = randn(r, k, seed=k).to(dtype), randn(r, k, seed=k + 1).to(dtype)
    w = 1 + 0.2 * randn(k, seed=2)
    tol = F32_NORM if dtype == torch.float32 else 2.0 ** -9
    for rr in (None, res):
        ref, h = norm_ref(x, w, rr, 1e-6)
        got = rms_norm(x.cuda(), w.cuda(), residual=None if rr is None else rr.cuda())
        y = got if rr is None else got[0]
        assert y.dtype == dtype and U.rel_l2(y, ref) < tol
        if rr is not None:
            assert torch.equal(got[1].cpu(), (x.float() + res.float()).to(dtype))
        q = rms_norm(x.cuda(), w.cuda(), residual=None if rr is None else rr.cuda(), quantize=True)
        q = q if rr is None else q[0]
        # a code is off by half a step (2^-4 of itself, or 2^-10 below 2^-6) plus the
        # 32-bit value's own rounding; scales are held in 32 bits
        s = q.scales.cpu().double().repeat_interleave(128, 1)[:, :k]
        v = U.values(q.codes.cpu(), q.scales.cpu())
        assert bool(((v - ref).abs() <= (2.0 ** -4 + 1e-5) * ref.abs() + (2.0 ** -10 + 1e-6) * s).all())
        amax = torch.nn.functional.pad(ref.abs(), (0, (-k) % 128)).view(r, -1, 128).amax(2)
        assert U.rel_l2(q.scales, amax / 448) < 1e-6
        if dtype == torch.float32:       # the 8-bit form of the same 32-bit result
            codes, scales = U.rows(y.cpu())
            assert U.same_bits(q.codes, codes) and torch.equal(q.scales.cpu(), scales)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("r,k", [(1, 1), (3, 7), (700, 384), (4099, 129), (2000, 768), (64, 1001),
                                 (300, 2304), (40, 5003), (9, 16390)])
def test_norm_gradients(r, k, dtype):
    from race_attention_b200.fp8 import rms_norm
    x, res, dy, dh = (randn(r, k, seed=s).to(dtype) for s in range(4))
    w = 1 + 0.2 * randn(k, seed=5)
    h = (x.float() + res.float()).to(dtype).double().requires_grad_()
    wd = w.double().requires_grad_()
    rstd = (h.square().mean(1, keepdim=True) + 1e-6).rsqrt()
    y = h * rstd * wd
    gh, gw = torch.autograd.grad(y, (h, wd), dy.double())
    # both terms of dx round, and h held in bfloat16 against rstd of the sum before that
    # rounding leaves 2^-9 of the first where it cancels
    size = float((gh + dh.double()).norm()) + float((dy.double() * wd * rstd).detach().norm())
    gh = gh + dh.double()
    X, R, W = x.cuda().requires_grad_(), res.cuda().requires_grad_(), w.cuda().requires_grad_()
    yy, hh = rms_norm(X, W, residual=R)
    torch.autograd.backward((yy, hh), (dy.cuda(), dh.cuda()))
    # dx sums its row in 32 bits (pairwise over lanes): a few roundings of either term;
    # dweight sums rows one after the other within a warp, then pairwise
    tol = 32 * 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -8
    assert float((X.grad.double().cpu() - gh).norm()) < tol * size and torch.equal(X.grad, R.grad)
    # held h and rstd of the unrounded sum differ by a rounding of h: 2^-9 at most of a row's norm
    assert U.rel_l2(W.grad, gw) < (64 * 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -8)
    # without a residual, and with only one of the two results used
    X2, W2 = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    rms_norm(X2, W2).backward(dy.cuda())
    xd = x.double().requires_grad_()
    (gx,) = torch.autograd.grad(xd * (xd.square().mean(1, keepdim=True) + 1e-6).rsqrt() * w.double(), xd,
                                dy.double())
    assert float((X2.grad.double().cpu() - gx).norm()) < tol * (float(gx.norm()) + size)
    X3, R3 = x.cuda().requires_grad_(), res.cuda().requires_grad_()
    rms_norm(X3, w.cuda(), residual=R3)[1].backward(dh.cuda())
    assert torch.equal(X3.grad.cpu(), dh) and torch.equal(R3.grad.cpu(), dh)


def test_norm_against_differences():
    """Central differences of the 32-bit kernel along random directions, summed in 64 bits.
    Step 2^-6: the third derivative adds about 2^-12 of the slope, rounding
    2^-24 sqrt(n) / 2^-6 of a unit-sized sum."""
    from race_attention_b200.fp8 import rms_norm
    r, k = 6, 200
    x, w, dy = randn(r, k, seed=1).cuda(), (1 + 0.2 * randn(k, seed=2)).cuda(), randn(r, k, seed=3).cuda()
    X, W = x.clone().requires_grad_(), w.clone().requires_grad_()
    rms_norm(X, W).backward(dy)
    f = lambda a, b: float((rms_norm(a, b).double() * dy.double()).sum())  # noqa: E731
    e = 2.0 ** -6
    for s in range(4):
        u, z = randn(r, k, seed=10 + s).cuda(), randn(k, seed=20 + s).cuda()
        du = (f(x + e * u, w) - f(x - e * u, w)) / (2 * e)
        dz = (f(x, w + e * z) - f(x, w - e * z)) / (2 * e)
        size = float(dy.norm()) * 2.0 ** -10
        assert abs(du - float((X.grad.double() * u.double()).sum())) < size * float(u.norm()) / r ** 0.5
        assert abs(dz - float((W.grad.double() * z.double()).sum())) < size * float(z.norm())


def test_norm_layouts_types_and_edges():
    from race_attention_b200.fp8 import RMSNorm, rms_norm
    base = randn(40, 600, seed=1).cuda()
    w = (1 + 0.1 * randn(256, seed=2)).cuda()
    for v in (base[:, 3:259], base[::3, :256], base[:, :512:2], base.view(5, 8, 600)[..., 100:356]):
        ref, _ = norm_ref(v.reshape(-1, 256).cpu(), w.cpu(), None, 1e-6)
        assert U.rel_l2(rms_norm(v, w).reshape(-1, 256), ref) < F32_NORM
    wb = w.bfloat16()
    ref, _ = norm_ref(base[:, :256].cpu(), wb.cpu().float(), None, 1e-6)
    assert U.rel_l2(rms_norm(base[:, :256], wb), ref) < F32_NORM
    W = wb.clone().requires_grad_()
    rms_norm(base[:, :256].bfloat16(), W).sum().backward()
    assert W.grad.dtype == torch.bfloat16
    # dy that is broadcast (a sum's gradient) and rows of nothing
    z = torch.zeros(3, 256, device="cuda", requires_grad=True)
    rms_norm(z, w).sum().backward()
    assert bool(z.grad.isfinite().all())
    q = rms_norm(z.detach(), w, quantize=True)
    assert not bool(q.codes.float().any())
    e = torch.empty(0, 256, device="cuda", requires_grad=True)
    W = w.clone().requires_grad_()
    y = rms_norm(e, W)
    y.sum().backward()
    assert y.shape == (0, 256) and torch.equal(W.grad, torch.zeros_like(w))
    bad = base[:4, :256].clone()
    bad[2, 100] = float("nan")
    assert torch.equal((~rms_norm(bad, w).isfinite()).all(1).cpu(), torch.tensor([False, False, True, False]))
    m = RMSNorm(256, device="cuda")
    assert m(base[:, :256]).shape == (40, 256)
    # the sum of gradients is taken in a fixed order
    X = randn(3000, 256, seed=8).cuda()
    grads = []
    for _ in range(2):
        W = w.clone().requires_grad_()
        rms_norm(X, W).backward(X)
        grads.append(W.grad)
    assert torch.equal(*grads)


def test_no_second_derivatives():
    from race_attention_b200.fp8 import fp8_linear, rms_norm
    x, w = torch.ones(4, 64, device="cuda", requires_grad=True), torch.ones(32, 64, device="cuda", requires_grad=True)
    for y in (fp8_linear(x, w), rms_norm(x, w[0])):
        with pytest.raises(RuntimeError, match="second derivatives"):
            torch.autograd.grad(y.sum(), x, create_graph=True)


def test_norm_refusals():
    from race_attention_b200.fp8 import rms_norm
    x, w = torch.ones(2, 64, device="cuda"), torch.ones(64, device="cuda")
    with pytest.raises(ValueError, match="weight must be"):
        rms_norm(x, w[:32])
    with pytest.raises(ValueError, match="residual"):
        rms_norm(x, w, residual=x.bfloat16())
    with pytest.raises(ValueError, match="no gradient"):
        rms_norm(x.requires_grad_(), w, quantize=True)
    with pytest.raises(RuntimeError, match="CUDA"):
        rms_norm(torch.ones(2, 64), w.cpu())
    from race_attention_b200._lib import RaceError
    with pytest.raises(RaceError, match="65536"):
        rms_norm(torch.ones(1, 65537, device="cuda"), torch.ones(65537, device="cuda"))
