"""Weights held in 8 bits: what is refused before anything runs, without a GPU."""
import pytest
import torch

from race_attention_b200 import _lib
from tests import fp8_util as U


@pytest.fixture(autouse=True, scope="module")
def lib():
    import os
    if not os.path.exists(_lib.LIB_PATH):
        from race_attention_b200.build import build
        build()
    return _lib.load()


def pair(n, k, device="cpu"):
    """A weight and its transpose, as quantize_fp8(w, square=True, transposed=True) returns them."""
    from race_attention_b200.fp8 import BlockFp8
    codes, scales = U.square(torch.randn(n, k, generator=torch.Generator().manual_seed(n)))
    return BlockFp8(codes, scales), BlockFp8(codes.t().contiguous(), scales.t())


@pytest.mark.parametrize("n,k", [(300, 260), (256, 256)])
def test_the_transpose_is_checked(n, k):
    from race_attention_b200.fp8 import BlockFp8, fp8_linear
    w, t = pair(n, k)
    rows = BlockFp8(*U.rows(torch.randn(k, n)))                    # a transpose with scales of rows
    narrow = BlockFp8(t.codes[:, :n - 128], t.scales[:, :-1])      # would be read past its end
    short = BlockFp8(t.codes[:k - 128], t.scales[:-1])
    x = torch.randn(5, k)
    for bad in (rows, narrow, short):
        with pytest.raises(ValueError, match="transpose"):
            fp8_linear(x, (w, bad))
    with pytest.raises(ValueError, match="transpose"):
        fp8_linear(x, (w, w))
    with pytest.raises(ValueError, match="transpose"):
        fp8_linear(x, (w, BlockFp8(w.codes, w.scales)))
    meta = BlockFp8(torch.empty(k, n, dtype=U.F8, device="meta"), torch.empty(t.scales.shape, device="meta"))
    with pytest.raises(ValueError, match="device"):
        fp8_linear(x, (w, meta))
    for odd in ((w,), (w, None), (w, t, t), (w.codes, t.codes)):
        with pytest.raises(ValueError, match="pair"):
            fp8_linear(x, odd)
    for good in ((w, t), (w, BlockFp8(w.codes.t(), w.scales.t()))):
        with pytest.raises(RuntimeError, match="CUDA"):            # past the checks of the pair
            fp8_linear(x, good)
