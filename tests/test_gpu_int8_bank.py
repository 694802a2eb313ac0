"""What an ``Int8ExpertBank`` holds is what its step reads."""
import numpy as np
import pytest
import torch

from mylocal_llm_amd import synthetic
from mylocal_llm_amd.int8_moe import Int8ExpertBank, int8_moe_step
from gpu_util import announce
from test_gpu_int8 import layer, rows

pytestmark = pytest.mark.gpu
TENSORS = ("gate_tiles", "up_tiles", "down_tiles", "gate_scales", "up_scales", "down_scales")


@pytest.mark.parametrize("t", [1, 9, 40])
@pytest.mark.parametrize("name", TENSORS)
def test_a_tensor_put_in_a_banks_place_is_read(cuda, name, t):
    """Rebound or with another storage, the step reads what the attribute holds, as ``expert()`` does."""
    announce("int8 bank", name, t)
    e, k, d, f = 8, 2, 128, 96
    first, other = (layer(e, d, f, 0, seed)[0] for seed in (3, 4))
    which, kind = name.split("_")
    at = ("gate", "up", "down").index(which)
    mixed = list(first)
    mixed[at] = (other[at][0], first[at][1]) if kind == "tiles" else (first[at][0], other[at][1])
    want_bank, bank, source = Int8ExpertBank(*mixed), Int8ExpertBank(*first), Int8ExpertBank(*other)
    x, logits = rows(t, d, 2), torch.from_numpy(synthetic.router_logits(t, e, 5)).cuda()
    want = int8_moe_step(x, want_bank, k, logits=logits)
    before = int8_moe_step(x, bank, k, logits=logits)
    assert not torch.equal(before, want)
    old = getattr(bank, name)                 # (kept: memory that the step must not read, but could)
    setattr(bank, name, getattr(source, name).clone())
    assert torch.equal(int8_moe_step(x, bank, k, logits=logits), want)
    setattr(bank, name, old)
    assert torch.equal(int8_moe_step(x, bank, k, logits=logits), before)
    view = old.view(old.shape)                # the same tensor object with another storage
    setattr(bank, name, view)
    view.data = getattr(source, name).clone()
    assert torch.equal(int8_moe_step(x, bank, k, logits=logits), want)
    assert np.isfinite(want.cpu().numpy()).all()
