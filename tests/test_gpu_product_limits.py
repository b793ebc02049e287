"""Products whose bounded waits run out (needs a B200): the kernels report it, give
nothing back while copies or instructions are in flight, and the next call is whole."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from race_attention_b200 import _lib
    _lib.load()


def held(rows, cols, seed, square):
    from race_attention_b200.fp8 import quantize_fp8
    g = torch.Generator(device="cuda").manual_seed(seed)
    return quantize_fp8(torch.randn(rows, cols, generator=g, device="cuda"), square=square)


def limited(a, b, polls):
    """The product with `polls` polls a wait: the bits of its status word."""
    from race_attention_b200 import _lib
    lib = _lib.load()
    (m, k), n = a.shape, b.shape[0]
    out = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    word = torch.zeros(1, dtype=torch.int32, pin_memory=True)
    desc = _lib.RaceMatmulDesc(_lib.RACE_BF16, int(b.square), m, n, k, polls, 0)
    need = lib.race_scaled_matmul_workspace(desc)
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    blocks = lambda x: _lib.RaceBlocks(x.codes.data_ptr(), x.codes.stride(0), x.scales.data_ptr(),  # noqa: E731
                                       *x.scales.stride())
    _lib.check(lib.race_scaled_matmul(desc, blocks(a), blocks(b), _lib.RaceRows(out.data_ptr(), n), word.data_ptr(),
                                      ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    return int(word)


@pytest.mark.parametrize("polls", [1, 8, 48])
@pytest.mark.parametrize("m,n,k", [
    (1, 128, 128),       # one block: every copy is issued before any wait runs out
    (8, 640, 1280),      # clusters whose ranks issue two or three copies, fewer than there are stages
    (20, 256, 640),      # as many copies as stages
    (50, 256, 2048),     # more copies than stages
    (100, 2304, 768)])
def test_copies_land_before_the_kernel_leaves(m, n, k, polls):
    """A limit this short runs out in some wait or in none; nothing stays in flight
    either way, and the product behind it is whole."""
    from race_attention_b200 import _lib
    from race_attention_b200.fp8 import fp8_matmul
    a, b = held(m, k, 1, False), held(n, k, 2, True)
    ref = fp8_matmul(a, b)
    for _ in range(5):
        bits = limited(a, b, polls)
        assert bits in (0, _lib.RACE_DEV_TIMEOUT)
        assert bits or polls > 1             # one poll is over long before a copy has landed
        assert torch.equal(fp8_matmul(a, b), ref)


@pytest.mark.parametrize("polls", [1, 8, 48])
@pytest.mark.parametrize("square", [True, False], ids=["square", "rows"])
@pytest.mark.parametrize("m,n,k", [
    (20000, 2304, 256),      # pairs of CTAs, tiles of two blocks, fewer than there are stages
    (4096, 2304, 768),       # several tiles a pair
    (2304, 768, 20000)])     # a contraction that is cut
def test_instructions_end_before_a_pair_leaves(m, n, k, square, polls):
    from race_attention_b200 import _lib
    from race_attention_b200.fp8 import fp8_matmul
    a, b = held(m, k, 3, False), held(n, k, 4, square)
    ref = fp8_matmul(a, b)
    assert _lib.last_kernels()[0] == "mm_pair"
    for _ in range(5):
        bits = limited(a, b, polls)
        assert bits in (0, _lib.RACE_DEV_TIMEOUT)
        assert bits or polls > 1
        assert torch.equal(fp8_matmul(a, b), ref)
