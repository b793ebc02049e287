"""Addresses that the 8-bit kernels could not read or write are refused by the C
entry points, before anything runs (no GPU needed)."""
import ctypes

import pytest

from race_attention_b200 import _lib
from race_attention_b200._lib import RaceBlocks, RaceMatmulDesc, RaceNormDesc, RaceRows

ALIGN = 3
AT = 0x7000000000          # host addresses that the entry points only look at
NOROWS, NOBLOCKS = RaceRows(None, 0), RaceBlocks(None, 0, None, 0, 0)


@pytest.fixture(scope="module")
def lib():
    import os
    if not os.path.exists(_lib.LIB_PATH):
        from race_attention_b200.build import build
        build()
    return _lib.load()


def blocks(scales):
    return RaceBlocks(AT, 64, scales, 1, 64)


def test_quantize(lib):
    for pair in ((blocks(AT + 2), NOBLOCKS), (NOBLOCKS, blocks(AT + 1))):
        assert lib.race_quantize(RaceRows(AT, 64), 0, 4, 64, 0, *pair, None) == ALIGN


@pytest.mark.parametrize("dtype,odd", [(0, 2), (1, 1)])
def test_norm(lib, dtype, odd):
    d = RaceNormDesc(dtype=0, weight_dtype=dtype, rows=4, width=64, eps=1e-6)
    x = RaceRows(AT, 64)
    assert lib.race_rms_norm(d, x, NOROWS, AT + odd, x, NOBLOCKS, NOROWS, None, None) == ALIGN
    assert lib.race_rms_norm(d, x, NOROWS, AT, x, NOBLOCKS, NOROWS, AT + 2, None) == ALIGN
    assert lib.race_rms_norm(d, x, NOROWS, AT, NOROWS, blocks(AT + 2), NOROWS, None, None) == ALIGN
    back = lambda weight=AT, rstd=AT, dweight=AT, ws=AT: lib.race_rms_norm_backward(  # noqa: E731
        d, x, NOROWS, x, weight, rstd, x, dweight, ws, 1 << 30, None)
    assert back(weight=AT + odd) == ALIGN and back(rstd=AT + 2) == ALIGN
    assert back(dweight=AT + odd) == ALIGN and back(ws=AT + 8) == ALIGN


def test_product(lib):
    d = RaceMatmulDesc(out_dtype=1, b_square=1, m=4, n=8, k=64, wait_polls=0, reserved=0)
    f = lambda a=blocks(AT), b=blocks(AT), status=None, ws=None: lib.race_scaled_matmul(  # noqa: E731
        d, a, b, RaceRows(AT, 64), status, ws, 0, None)
    assert f(a=blocks(AT + 2)) == ALIGN and f(b=blocks(AT + 1)) == ALIGN
    assert f(status=AT + 2) == ALIGN and f(ws=AT + 8) == ALIGN


def test_adamw(lib):
    d = _lib.RaceAdamwDesc(lr=1e-3, beta_one=0.9, beta_two=0.99, eps=1e-8, weight_decay=0.0, seed=0, state_bits=8)
    for m, v in ((AT + 2, AT), (AT, AT + 1)):
        t = _lib.RaceAdamwTensor(param=AT, grad=AT, exp_avg=AT, exp_avg_sq=AT, exp_avg_scale=m, exp_avg_sq_scale=v,
                                 numel=5, first=0, dtype=0, step=0)
        assert lib.race_adamw(d, ctypes.byref(t), 1, None) == ALIGN
