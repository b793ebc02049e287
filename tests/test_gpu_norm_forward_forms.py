"""The norm's forward pass in each of its forms (needs a B200): rows that are walked or
not, by type, width and result, with more rows than the grid has places."""
import pytest
import torch

from tests import fp8_util as U

pytestmark = pytest.mark.gpu

F32 = 8 * 2.0 ** -24      # the sum's, the root's and three products' roundings, as beside the norm's other tests


@pytest.fixture(autouse=True, scope="module")
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from race_attention_b200 import _lib
    _lib.load()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("r,k", [(30001, 60), (30000, 64), (20001, 96), (9000, 100), (9001, 255), (7000, 260), (6001, 383),
                                 (6000, 385), (5000, 511), (4001, 700), (4000, 767), (3001, 768), (3000, 1001),
                                 (2001, 1024), (1300, 1601), (1001, 2500), (700, 4096), (650, 4099), (333, 5003),
                                 (301, 8192), (201, 12288), (170, 16383), (160, 16388), (155, 16390), (151, 32768),
                                 (149, 65535), (150, 65536)])
@pytest.mark.parametrize("weight", [torch.float32, torch.bfloat16], ids=["wf32", "wbf16"])
def test_results(r, k, dtype, weight):
    from race_attention_b200.fp8 import rms_norm
    g = torch.Generator(device="cuda").manual_seed(k)
    x, res = (torch.randn(r, k, generator=g, device="cuda").to(dtype) for _ in range(2))
    w = (1 + 0.2 * torch.randn(k, generator=g, device="cuda")).to(weight)
    tol = F32 if dtype == torch.float32 else 2.0 ** -9
    for second in (None, res):
        h = x.double() if second is None else x.double() + second.double()
        ref = h * (h.square().mean(1, keepdim=True) + 1e-6).rsqrt() * w.double()
        got = rms_norm(x, w, residual=second)
        y = got if second is None else got[0]
        assert U.rel_l2(y, ref) < tol
        worst = ((y.double() - ref).norm(dim=1) / ref.norm(dim=1)).max()
        assert float(worst) < 2 * tol                      # every row, the last ones too
        q = rms_norm(x, w, residual=second, quantize=True)
        if second is not None:
            assert torch.equal(got[1], (x.float() + second.float()).to(dtype)) and torch.equal(q[1], got[1])
            q = q[0]
        if dtype == torch.float32:                         # the 8-bit form of the same 32-bit result
            pad = torch.nn.functional.pad(y, (0, (-k) % 128)).view(r, -1, 128)
            s = (pad.abs().amax(2) * torch.tensor(1 / 448, dtype=torch.float32, device="cuda")).clamp_min(2.0 ** -126)
            codes = (pad * (1.0 / s)[:, :, None]).clamp(-448, 448).view(r, -1)[:, :k].to(U.F8)
            assert torch.equal(q.scales, s) and torch.equal(q.codes.float(), codes.float())
        else:
            v = q.codes.double() * q.scales.double().repeat_interleave(128, 1)[:, :k]
            s = q.scales.double().repeat_interleave(128, 1)[:, :k]
            assert bool(((v - ref).abs() <= (2.0 ** -4 + 1e-5) * ref.abs() + (2.0 ** -10 + 1e-6) * s).all())
