"""Host side of the 8-bit operators: what the C entry points and the Python
layer refuse, without a GPU."""
import ctypes

import pytest
import torch

from race_attention_b200 import _lib
from race_attention_b200._lib import RaceBlocks, RaceMatmulDesc, RaceNormDesc, RaceRows
from tests import fp8_util as U

INVALID, UNSUPPORTED, ALIGN, WORKSPACE = 1, 2, 3, 4
NOROWS, NOBLOCKS = RaceRows(None, 0), RaceBlocks(None, 0, None, 0, 0)


@pytest.fixture(scope="module")
def lib():
    import os
    if not os.path.exists(_lib.LIB_PATH):
        from race_attention_b200.build import build
        build()
    return _lib.load()


# host addresses that the entry points only look at
ADDR = 0x7000000000


def rows(ld=64, at=ADDR):
    return RaceRows(at, ld)


def blocks(ld=64, at=ADDR, scales=ADDR):
    return RaceBlocks(at, ld, scales, 1, 64)


def test_quantize_arguments(lib):
    q = lib.race_quantize
    assert q(rows(), 0, 4, 64, 0, NOBLOCKS, NOBLOCKS, None) == INVALID
    assert q(rows(), 5, 4, 64, 0, blocks(), NOBLOCKS, None) == INVALID
    assert q(rows(), 0, -1, 64, 0, blocks(), NOBLOCKS, None) == INVALID
    assert q(NOROWS, 0, 4, 64, 0, blocks(), NOBLOCKS, None) == INVALID
    assert q(rows(), 0, 4, 64, 0, blocks(scales=None), NOBLOCKS, None) == INVALID
    assert q(rows(), 0, 4, 64, 0, blocks(ld=40), NOBLOCKS, None) == ALIGN
    assert q(rows(), 0, 4, 64, 0, blocks(ld=48), NOBLOCKS, None) == INVALID
    assert q(rows(), 0, 4, 64, 0, blocks(at=ADDR + 8), NOBLOCKS, None) == ALIGN
    assert q(rows(at=ADDR + 2), 0, 4, 64, 0, blocks(), NOBLOCKS, None) == ALIGN
    assert q(rows(), 0, 9_000_000, 64, 0, blocks(), NOBLOCKS, None) == UNSUPPORTED
    assert q(NOROWS, 0, 0, 64, 0, blocks(), NOBLOCKS, None) == 0


def test_norm_arguments(lib):
    d = lambda **k: RaceNormDesc(**{**dict(dtype=0, weight_dtype=0, rows=4, width=64, eps=1e-6), **k})  # noqa: E731
    f = lambda desc, x=rows(), res=NOROWS, w=ADDR, y=rows(), y8=NOBLOCKS, h=NOROWS: lib.race_rms_norm(  # noqa: E731
        desc, x, res, w, y, y8, h, None, None)
    assert f(None) == INVALID and f(d(dtype=3)) == INVALID and f(d(weight_dtype=-1)) == INVALID
    assert f(d(width=0)) == INVALID and f(d(rows=-1)) == INVALID
    assert f(d(width=65537)) == UNSUPPORTED
    assert f(d(), w=None) == INVALID and f(d(), x=NOROWS) == INVALID
    assert f(d(), y=NOROWS) == INVALID and f(d(), y8=blocks()) == INVALID
    assert f(d(), res=rows()) == INVALID                      # h has to be given
    assert f(d(), y=rows(ld=32)) == INVALID                   # rows of the result overlap
    assert f(d(), y=NOROWS, y8=blocks(ld=72)) == ALIGN
    assert f(d(), x=rows(at=ADDR + 1)) == ALIGN
    assert f(d(rows=0), x=NOROWS, y=rows()) == 0
    b = lambda desc, ws=ADDR, n=1 << 30: lib.race_rms_norm_backward(  # noqa: E731
        desc, rows(), NOROWS, rows(), ADDR, ADDR, rows(), ADDR, ws, n, None)
    assert b(None) == INVALID
    assert lib.race_rms_norm_workspace(d()) >= 4 * 64
    assert lib.race_rms_norm_workspace(d(width=0)) == 0


def test_matmul_arguments(lib):
    d = lambda **k: RaceMatmulDesc(**{**dict(out_dtype=1, b_square=1, m=4, n=8, k=64, wait_polls=0, reserved=0), **k})  # noqa: E731
    f = lambda desc, a=blocks(), b=blocks(), y=rows(): lib.race_scaled_matmul(desc, a, b, y, None, None, 0, None)  # noqa: E731
    assert f(None) == INVALID and f(d(m=-1)) == INVALID and f(d(out_dtype=2)) == INVALID
    assert f(d(wait_polls=-1)) == INVALID
    assert f(d(), y=NOROWS) == INVALID and f(d(), y=rows(ld=4)) == INVALID
    assert f(d(), y=rows(at=ADDR + 1)) == ALIGN
    assert f(d(n=(1 << 22) + 1), y=rows(ld=1 << 23)) == UNSUPPORTED
    assert f(d(m=0)) == 0 and f(d(n=0)) == 0


def test_adamw_arguments(lib):
    T = _lib.RaceAdamwTensor
    d = lambda **k: _lib.RaceAdamwDesc(**{**dict(lr=1e-3, beta_one=0.9, beta_two=0.99, eps=1e-8, weight_decay=0.0,  # noqa: E731
                                                 seed=0, state_bits=32), **k})
    t = lambda **k: T(**{**dict(param=ADDR, grad=ADDR, exp_avg=ADDR, exp_avg_sq=ADDR, numel=5, first=0, dtype=0,  # noqa: E731
                                step=0), **k})
    f = lambda desc, x=None: lib.race_adamw(desc, ctypes.byref(x or t()), 1, None)  # noqa: E731
    assert f(None) == INVALID and f(d(state_bits=16)) == INVALID and f(d(beta_one=1.0)) == INVALID
    assert f(d(eps=-1.0)) == INVALID and f(d(eps=float("nan"))) == INVALID
    assert f(d(), t(numel=-1)) == INVALID and f(d(), t(param=None)) == INVALID
    assert f(d(), t(dtype=7)) == INVALID and f(d(), t(step=-1)) == INVALID and f(d(), t(first=4)) == INVALID
    assert f(d(state_bits=8)) == INVALID                      # scales are missing
    assert f(d(), t(exp_avg=ADDR + 4)) == ALIGN and f(d(), t(param=ADDR + 2)) == ALIGN
    assert lib.race_adamw(d(), None, 0, None) == 0
    assert lib.race_adamw(d(), None, 2, None) == INVALID


def test_python_refusals_on_the_host(lib):
    from race_attention_b200.fp8 import BlockFp8, fp8_matmul, quantize_fp8, rms_norm
    x = torch.ones(3, 200)
    for f in (lambda: quantize_fp8(x), lambda: rms_norm(x, torch.ones(200))):
        with pytest.raises(RuntimeError, match="CUDA"):
            f()
    with pytest.raises(ValueError, match="transposed"):
        quantize_fp8(x, transposed="yes")
    codes, scales = U.rows(x)
    b = BlockFp8(codes, scales)
    assert not b.square and b.shape == (3, 200)
    assert torch.equal(b.dequantize(), U.values(codes, scales).float())   # one product, rounded once
    with pytest.raises(ValueError, match="float8"):
        BlockFp8(x, scales)
    with pytest.raises(ValueError, match="scales"):
        BlockFp8(codes, scales[:, :1])
    with pytest.raises(ValueError, match="float32"):
        BlockFp8(codes, scales.double())
    with pytest.raises(RuntimeError, match="CUDA"):
        fp8_matmul(b, b)
    sq = BlockFp8(*U.square(torch.randn(300, 260)))
    assert sq.square and sq.dequantize().shape == (300, 260)
