"""AdamW as an object that programs copy, save and watch (needs a B200)."""
import copy
import pickle

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from race_attention_b200 import _lib
    _lib.load()


def params(dtype=torch.float32):
    g = torch.Generator().manual_seed(0)
    return [torch.nn.Parameter(torch.randn(*s, generator=g).to(dtype).cuda()) for s in ((7, 30), (129,), (3,))]


def step(opt, seed):
    g = torch.Generator().manual_seed(seed)
    for group in opt.param_groups:
        for p in group["params"]:
            p.grad = torch.randn(p.shape, generator=g).to(p.dtype).cuda()
    opt.step()


def moving(opt):
    return [p.detach().clone() for g in opt.param_groups for p in g["params"]]


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("how", [copy.deepcopy, lambda o: pickle.loads(pickle.dumps(o))], ids=["deepcopy", "pickle"])
def test_a_copy_goes_on_by_itself(how, bits):
    from race_attention_b200.optim import AdamW
    ps = params()
    opt = AdamW([{"params": ps[:2]}, {"params": ps[2:], "lr": 0.1}], state_bits=bits, seed=3)
    step(opt, 1)
    twin = how(opt)
    other = [p for g in twin.param_groups for p in g["params"]]
    assert all(a is not b for a, b in zip(ps, other)) and twin.exp_avg.data_ptr() != opt.exp_avg.data_ptr()
    step(twin, 2)
    assert [int(twin.state[p]["step"]) for p in other] == [2, 2, 2]
    assert [int(opt.state[p]["step"]) for p in ps] == [1, 1, 1]
    step(opt, 2)
    assert all(torch.equal(a, b) for a, b in zip(moving(opt), moving(twin)))
    assert [twin.offsets[p] for p in other] == [opt.offsets[p] for p in ps]
    twin.add_param_group({"params": [torch.nn.Parameter(torch.ones(5, device="cuda"))]})
    step(twin, 4)
    assert int(twin.state[twin.param_groups[-1]["params"][0]]["step"]) == 1


def test_state_dict_hooks_run():
    from race_attention_b200.optim import AdamW
    ps = params()
    opt = AdamW(ps, lr=0.1, state_bits=8)
    step(opt, 1)
    seen = []
    opt.register_state_dict_pre_hook(lambda o: seen.append("before"))
    opt.register_state_dict_post_hook(lambda o, s: s | {"epoch": 7})
    opt.register_load_state_dict_pre_hook(lambda o, s: s | {"seed": s["seed"] + 1})
    opt.register_load_state_dict_post_hook(lambda o: seen.append("after"))
    saved = opt.state_dict()
    assert seen == ["before"] and saved["epoch"] == 7 and saved["seed"] == 0
    step(opt, 2)
    opt.load_state_dict(saved)
    assert seen == ["before", "after"] and opt.seed == 1 and saved["seed"] == 0
    assert [int(opt.state[p]["step"]) for p in ps] == [1, 1, 1]


@pytest.mark.parametrize("bits", [8, 32])
def test_groups_without_parameters_beside_others(bits):
    from race_attention_b200.optim import AdamW
    a, b = params(), params()
    one = AdamW([{"params": []}, {"params": a, "lr": 0.1}, {"params": []}], state_bits=bits)
    two = AdamW(b, lr=0.1, state_bits=bits)
    for s in (1, 2):
        step(one, s)
        step(two, s)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    late = AdamW([{"params": []}], state_bits=bits)
    late.add_param_group({"params": [torch.nn.Parameter(p.detach().clone()) for p in a], "lr": 0.1})
    step(late, 1)
    late.load_state_dict(late.state_dict())
