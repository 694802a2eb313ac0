"""Refusals of the 8-bit integer operators that need no GPU, and the oracle of their tests against hand-made values."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import int8_np as Q
from mylocal_llm_amd import _lib
from mylocal_llm_amd.int8_linear import Int8Weight, int8_linear, int8_quantize, int8_swiglu
from mylocal_llm_amd.int8_moe import Int8ExpertBank, int8_moe_step
from mylocal_llm_amd.quantized_linear import quantized_linear, quantized_swiglu

FAKE = 4096               # never dereferenced: every call below is refused first


def linear(lib, **kw):
    names = [("tiles", FAKE), ("scales", FAKE), ("n", 16), ("k", 64), ("x", FAKE), ("xdt", 0), ("xs", None), ("t", 1), ("y", FAKE), ("ydt", 0),
             ("ws", FAKE), ("bytes", 1 << 20), ("stream", None)]
    return lib.qmoe_int8_linear(*[kw.get(n, d) for n, d in names])


def test_linear_refuses_before_any_launch():
    lib = _lib.load()
    for name in ("tiles", "scales", "x", "y"):
        assert linear(lib, **{name: None}) == 1 and b"null" in lib.qmoe_last_error()
    assert linear(lib, n=0) == 1 and linear(lib, k=0) == 1 and linear(lib, t=-1) == 1
    assert linear(lib, k=131072) == 2 and b"int32" in lib.qmoe_last_error()
    assert linear(lib, xdt=7) == 1 and linear(lib, ydt=3) == 1
    assert linear(lib, xdt=3) == 1 and b"scales" in lib.qmoe_last_error()
    assert linear(lib, tiles=FAKE + 8) == 1 and linear(lib, x=FAKE + 2) == 1 and linear(lib, y=FAKE + 1) == 1
    assert linear(lib, t=2, ws=None) == 4 and linear(lib, t=2, ws=FAKE + 16) == 4 and linear(lib, t=2, bytes=64) == 4
    assert linear(lib, n=1 << 27) == 2 and linear(lib, t=1 << 23) == 2
    assert linear(lib, t=0) == 0


def test_swiglu_quantise_and_tiles_refuse_before_any_launch():
    lib = _lib.load()
    sw = lambda up=FAKE, us=FAKE, k=64: lib.qmoe_int8_swiglu(FAKE, FAKE, up, us, 16, k, FAKE, 0, None, 1, FAKE, 0, FAKE, 1 << 20, None)
    assert sw(up=None) == 1 and sw(us=None) == 1 and sw(k=200000) == 2
    qz = lambda x=FAKE, dt=0, rows=1, k=4, c=FAKE, s=FAKE: lib.qmoe_int8_quantize(x, dt, rows, k, c, s, None)
    assert qz(x=None) == 1 and qz(c=None) == 1 and qz(s=None) == 1 and qz(dt=3) == 1 and qz(rows=-1) == 1 and qz(k=0) == 1
    assert qz(x=FAKE + 1) == 1 and qz(s=FAKE + 2) == 1 and qz(rows=1 << 33) == 2 and qz(rows=0) == 0
    tl = lambda c=FAKE, m=1, n=4, k=4, t=FAKE: lib.qmoe_int8_tiles(c, m, n, k, t, None)
    assert tl(c=None) == 1 and tl(t=None) == 1 and tl(m=0) == 1 and tl(n=0) == 1 and tl(k=131072) == 2 and tl(t=FAKE + 4) == 1 and tl(m=1 << 30) == 2


def test_sizes():
    lib = _lib.load()
    assert lib.qmoe_int8_matrix_bytes(1, 1) == 16 * 64 and lib.qmoe_int8_matrix_bytes(17, 65) == 32 * 128 and lib.qmoe_int8_matrix_bytes(0, 4) == 0
    assert lib.qmoe_int8_matrix_bytes(70000, 65536) == 70000 * 65536
    a, b = lib.qmoe_int8_workspace_bytes(64, 100, 3, 0), lib.qmoe_int8_workspace_bytes(64, 100, 30, 2)
    assert 0 < a < b and a % 256 == b % 256 == 0 and lib.qmoe_int8_workspace_bytes(64, 100, 0, 0) == 0
    assert lib.qmoe_int8_workspace_bytes(64, 100, 1, 0) == 0 and lib.qmoe_int8_workspace_bytes(64, 100, 1, 3) == 0
    assert lib.qmoe_int8_workspace_bytes(20000, 100, 500, 3) > 0
    m = [lib.qmoe_int8_moe_workspace_bytes(t, 10, 512, 2048, 512, 2048) for t in (1, 16, 4096)]
    assert 0 < m[0] < m[1] < m[2] and lib.qmoe_int8_moe_workspace_bytes(1, 0, 4, 4, 4, 0) == 0


def moe_args(**kw):
    a = _lib.Int8MoeArgs()
    base = dict(hidden=FAKE, hidden_dtype=0, tokens=2, top_k=2, logits=FAKE, floor_value=1e-6, renormalize=1, gate=FAKE, up=FAKE, down=FAKE,
                gate_scales=FAKE, up_scales=FAKE, down_scales=FAKE, n_experts=8, d_model=64, d_ff=64, out=FAKE, out_dtype=0)
    for name, value in {**base, **kw}.items():
        setattr(a, name, value)
    return ctypes.byref(a)


def test_step_refuses_before_any_launch():
    lib = _lib.load()
    call = lambda ws=FAKE, nbytes=1 << 30, **kw: lib.qmoe_int8_moe_forward(moe_args(**kw), ws, nbytes, None)
    assert lib.qmoe_int8_moe_forward(None, FAKE, 1 << 30, None) == 1
    for name in ("hidden", "out", "gate", "up", "down", "gate_scales", "up_scales", "down_scales"):
        assert call(**{name: None}) == 1, name
    assert call(logits=None) == 1 and call(logits=None, in_weights=FAKE) == 1
    assert call(tokens=-1) == 1 and call(hidden_dtype=3) == 1 and call(out_dtype=9) == 1 and call(d_model=0) == 1 and call(d_ff=-4) == 1
    assert call(n_experts=4097) == 2 and call(top_k=0) == 2 and call(top_k=9) == 2 and call(top_k=33, n_experts=64) == 2
    assert call(d_ff=131072) == 2 and call(tokens=1 << 30, top_k=2) == 2 and call(tokens=(1 << 21) + 1, top_k=2) == 2
    assert call(d_ff_shared=16) == 1 and call(shared_gate_w=FAKE) == 1
    assert call(d_ff_shared=16, shared_gate_w=FAKE, shared_up_w=FAKE, shared_down_w=FAKE, shared_gate_scales=FAKE, shared_up_scales=FAKE) == 1
    assert call(floor_value=0.0) == 1 and call(floor_value=float("nan")) == 1
    assert call(gate=FAKE + 4) == 1 and call(residual=FAKE + 2) == 1 and call(logits=None, in_weights=FAKE, in_ids=FAKE + 4) == 1
    assert call(ws=None) == 4 and call(ws=FAKE + 16) == 4 and call(nbytes=1024) == 4
    assert call(tokens=0) == 0


def test_python_refusals():
    cpu = torch.zeros((2, 8))
    with pytest.raises(TypeError, match="CUDA"):
        int8_quantize(cpu)
    with pytest.raises(TypeError, match="CUDA"):
        int8_quantize(np.zeros((2, 8), np.float32))
    with pytest.raises(TypeError, match="CUDA torch.int8"):
        Int8Weight(torch.zeros((2, 8), dtype=torch.int8), torch.zeros(2))
    with pytest.raises(ValueError, match=r"\[N, K\]"):
        Int8Weight.quantize(torch.zeros(8))
    with pytest.raises(TypeError, match="DevicePackedGGUFWeight"):
        Int8Weight.from_packed(cpu)
    with pytest.raises(TypeError, match="Int8Weight"):
        int8_linear(cpu, cpu)
    with pytest.raises(TypeError, match="Int8Weight"):
        int8_swiglu(cpu, cpu, cpu)
    with pytest.raises(TypeError, match="Int8ExpertBank"):
        int8_moe_step(cpu, None, 2)
    with pytest.raises(TypeError, match="pair"):
        Int8ExpertBank(cpu, cpu, cpu)
    with pytest.raises(TypeError, match="DevicePackedExpertBank"):
        Int8ExpertBank.from_packed(cpu)


class Shape:
    """A matrix that was never on a device, for the checks in front of one."""

    def __new__(cls, n, k):
        w = Int8Weight.__new__(Int8Weight)
        w.tiles = w.scales = None
        w.shape, w.device = (n, k), torch.device("cuda", 0)
        return w


def test_product_refusals_of_host_activations_and_shapes():
    w = Shape(4, 8)
    for call in (lambda x: int8_linear(x, w), lambda x: int8_swiglu(x, w, w), lambda x: quantized_linear(x, w), lambda x: quantized_swiglu(x, w, w)):
        with pytest.raises(TypeError, match="CUDA"):
            call(torch.zeros((2, 8)))
    with pytest.raises(ValueError, match="share"):
        int8_swiglu(torch.zeros((2, 8)), w, Shape(5, 8))
    with pytest.raises(TypeError, match="NumPy"):
        quantized_linear(np.zeros((2, 8), np.float32), w)
    with pytest.raises(ValueError, match="block_k"):
        quantized_linear(torch.zeros((2, 8)), w, block_k=100)


def test_oracle_quantises_by_hand():
    x = np.array([[127.0, 0.5, 1.5, -0.5, -2.5, 63.49], [0, 0, 0, 0, 0, 0], [np.nan, 1, 2, 3, 4, 5], [254, 1, 3, -3, 127.5, -254]])
    q, s = Q.quantize(x)
    assert s[0] == 1 and s[1] == 0 and np.isnan(s[2]) and s[3] == 2
    assert q.tolist() == [[127, 0, 2, 0, -2, 63], [0] * 6, [0] * 6, [127, 0, 2, -2, 64, -127]]


def test_oracle_step_by_hand():
    """Two experts of one hidden unit, codes chosen so that every number is small: silu(2) * 3 = h, then down."""
    gate = (np.array([[[1, 0]], [[0, 1]]], np.int8), np.array([[1.0], [1.0]], np.float32))
    up = (np.array([[[3, 0]], [[0, 3]]], np.int8), np.array([[0.5], [0.5]], np.float32))
    down = (np.array([[[1], [2]], [[3], [4]]], np.int8), np.ones((2, 2), np.float32))
    x = np.array([[127.0, 127.0]])
    terms = Q.moe_terms(x, np.array([[0.25, 0.75]]), np.array([[1, 0]]), gate, up, down)
    h = np.float32(127.0 / (1 + np.exp(-127.0)) * 190.5)
    s = np.float32(np.float64(h) / 127)
    np.testing.assert_allclose(terms[0], [[0.25 * 127 * s * 3, 0.25 * 127 * s * 4], [0.75 * 127 * s, 0.75 * 127 * s * 2]], rtol=1e-12)
    again = Q.moe_terms(x, np.array([[0.25, 0.75]]), np.array([[1, 1]]), gate, up, down)
    assert np.array_equal(again[0, 0], terms[0, 0]) and not again[0, 1].any()
