"""What an ``Int8ExpertBank`` takes in a tensor's place, without a GPU."""
import copy

import pytest
import torch

from mylocal_llm_amd import _lib
from mylocal_llm_amd.int8_moe import Int8ExpertBank

E, D, F = 3, 64, 32
SHAPES = {"gate_tiles": (E * F * D,), "up_tiles": (E * F * D,), "down_tiles": (E * D * 64,), "gate_scales": (E, F), "up_scales": (E, F), "down_scales": (E, D)}


def bank():
    b = Int8ExpertBank.__new__(Int8ExpertBank)
    made = [torch.zeros(shape, dtype=torch.uint8 if "tiles" in name else torch.float32) for name, shape in SHAPES.items()]
    b._hold(tuple(made[:3]), tuple(made[3:]), E, D, F)
    return b


def addresses(b):
    args = _lib.Int8MoeArgs()
    b.fill(args)
    assert (args.n_experts, args.d_model, args.d_ff) == (E, D, F)
    return dict(zip(SHAPES, (args.gate, args.up, args.down, args.gate_scales, args.up_scales, args.down_scales)))


@pytest.mark.parametrize("name", SHAPES)
def test_a_tensor_that_fits_takes_the_place(name):
    b = bank()
    before = addresses(b)
    other = torch.ones_like(getattr(b, name))
    setattr(b, name, other)
    assert getattr(b, name) is other
    assert addresses(b) == {**before, name: other.data_ptr()}


@pytest.mark.parametrize("name", SHAPES)
def test_one_that_does_not_fit_is_refused(name):
    b = bank()
    before, old = addresses(b), getattr(b, name)
    wide = torch.zeros((*old.shape[:-1], 2 * old.shape[-1]), dtype=old.dtype)
    for bad in (None, old.numpy(), old[:1], old.double(), wide, wide[..., ::2], old.reshape(-1, 1)):
        with pytest.raises(ValueError, match=f"{name} must be contiguous"):
            setattr(b, name, bad)
    with pytest.raises(ValueError, match="same device"):
        setattr(b, name, torch.empty(old.shape, dtype=old.dtype, device="meta"))
    assert getattr(b, name) is old and addresses(b) == before


@pytest.mark.parametrize("name", SHAPES)
def test_a_tensor_resized_in_place_is_refused(name):
    b = bank()
    getattr(b, name).data = torch.zeros(4, dtype=getattr(b, name).dtype)
    with pytest.raises(ValueError, match="resized"):
        addresses(b)


def test_a_copy_reads_its_own_tensors():
    b = bank()
    other = copy.deepcopy(b)
    assert all(addresses(b)[name] != addresses(other)[name] for name in SHAPES)
