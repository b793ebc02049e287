"""Parameter groups without parameters, without a GPU."""
import os

import pytest
import torch

from race_attention_b200 import _lib


@pytest.fixture(autouse=True, scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        from race_attention_b200.build import build
        build()
    return _lib.load()


@pytest.mark.parametrize("bits", [8, 32])
def test_groups_without_parameters(bits):
    from race_attention_b200.optim import AdamW
    opt = AdamW([{"params": []}, {"params": [], "lr": 0.5}], state_bits=bits)
    assert opt.exp_avg is None and opt.step() is None and opt.step(lambda: 3) == 3
    opt.load_state_dict(opt.state_dict())
    with pytest.raises(ValueError, match="CUDA"):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.ones(3))]})
    assert len(opt.param_groups) == 2
