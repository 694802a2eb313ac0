"""The 8-bit integer products take several kernels, by their sizes; a value's bits may depend on none of that.

Sizes are chosen so that the tiles of many tokens are what runs, and ``tiled`` asserts it: codes need a workspace only there.
(A pair is taken by the few-token kernel up to 256 blocks of 16 channels x 32 tokens.)
"""
import ctypes

import numpy as np
import pytest
import torch

from oracle import int8_np as Q
from mylocal_llm_amd import _lib, synthetic
from mylocal_llm_amd.int8_linear import Int8Weight, int8_linear, int8_quantize, int8_swiglu
from mylocal_llm_amd.int8_moe import Int8ExpertBank, int8_moe_step
from mylocal_llm_amd.quantized_linear import _TORCH_DTYPE_ID
from gpu_util import announce
from test_gpu_int8 import DTYPES, U, as_np, close, host, layer, matrix, rows

pytestmark = pytest.mark.gpu
INT8 = 3


def tiled(t, n, k):
    """Both a product and a pair of these sizes run on the tiles of many tokens."""
    assert _lib.load().qmoe_int8_workspace_bytes(n, k, t, INT8) > 0 and (n + 15) // 16 * ((t + 31) // 32) > 256


def pair_of(n, k, seed):
    g, u = matrix(n, k, seed), matrix(n, k, seed + 1)
    g[1].mul_(20.0 / k ** 0.5)
    return g, u


def both(gate, up, dtype):
    return [("linear", lambda x, s: int8_linear(x, gate, x_scales=s, out_dtype=dtype)),
            ("swiglu", lambda x, s: int8_swiglu(x, gate, up, x_scales=s, out_dtype=dtype))]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,n,k", [(512, 2048, 256), (300, 2000, 200), (4096, 4096, 64)])
def test_a_row_does_not_move_its_neighbours_bits(cuda, t, n, k, dtype):
    """Rows whose scale is NaN, infinite, tiny, huge or 0 between ordinary ones: the others keep every bit."""
    announce("int8 neighbours", t, n, k, dtype)
    tiled(t, n, k)
    g, u = pair_of(n, k, t + n)
    codes, scales = int8_quantize(rows(t, k, t))
    for name, call in both(Int8Weight(*g), Int8Weight(*u), dtype):
        clean = call(codes, scales)
        odd = torch.arange(7, t, 37, device=cuda)
        keep = torch.ones(t, dtype=torch.bool, device=cuda)
        keep[odd] = False
        for bad in (float("nan"), float("inf"), 1e-30, 1e30, 0.0):
            s = scales.clone()
            s[odd] = bad
            got = call(codes, s)
            assert torch.equal(got[keep], clean[keep]), (name, bad, int((got[keep] != clean[keep]).sum()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,n,k", [(512, 2048, 256), (300, 2000, 200), (4096, 4096, 64), (700, 3600, 1000), (100, 1601, 96)])
def test_a_token_alone_and_in_a_prompt_gets_the_same_bits(cuda, t, n, k, dtype):
    announce("int8 alone and in a prompt", t, n, k, dtype)
    tiled(t, n, k)
    g, u = pair_of(n, k, t + k)
    codes, scales = int8_quantize(rows(t, k, t))
    for name, call in both(Int8Weight(*g), Int8Weight(*u), dtype):
        whole = call(codes, scales)
        for lo, hi in ((0, 1), (1, 17), (t - 16, t), (t // 2, t // 2 + 5)):
            part = call(codes[lo:hi].contiguous(), scales[lo:hi].contiguous())
            assert torch.equal(part, whole[lo:hi]), (name, lo, hi, int((part != whole[lo:hi]).sum()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,n,k", [(512, 2048, 256), (300, 2000, 200), (4096, 4096, 64)])
def test_a_values_bits_do_not_depend_on_where_it_lies(cuda, t, n, k, dtype):
    """The last blocks of a narrower matrix, rows that start anywhere, an output at an odd address."""
    announce("int8 places", t, n, k, dtype)
    g, u = pair_of(n, k, t + 3)
    codes, scales = int8_quantize(rows(t, k, t))
    lib, stream = _lib.load(), torch.cuda.current_stream().cuda_stream
    work = torch.empty(lib.qmoe_int8_workspace_bytes(n, k, t, INT8), dtype=torch.uint8, device=cuda)
    gate, up = Int8Weight(*g), Int8Weight(*u)
    whole = [call(codes, scales) for _, call in both(gate, up, dtype)]
    for m in (n - 1, n - 14, n - 100, n // 2 + 602):
        tiled(t, m, k)
        parts = [Int8Weight(w[0][:m].contiguous(), w[1][:m].contiguous()) for w in (g, u)]
        for (name, call), want in zip(both(*parts, dtype), whole):
            got = call(codes, scales)
            assert torch.equal(got, want[:, :m]), (name, m, int((got != want[:, :m]).sum()))
    base = torch.full((t * n + 2,), 3.0, dtype=dtype, device=cuda)
    odt = _TORCH_DTYPE_ID[dtype]
    for pair, want in enumerate(whole):
        head = [gate.tiles.data_ptr(), gate.scales.data_ptr()] + ([up.tiles.data_ptr(), up.scales.data_ptr()] if pair else [])
        entry = lib.qmoe_int8_swiglu if pair else lib.qmoe_int8_linear
        base.fill_(3.0)
        assert entry(*head, n, k, codes.data_ptr(), INT8, scales.data_ptr(), t, base[1:].data_ptr(), odt, work.data_ptr(), work.numel(), stream) == 0
        torch.cuda.synchronize()
        assert torch.equal(base[1:-1].reshape(t, n), want) and base[0] == 3 and base[-1] == 3


@pytest.mark.parametrize("t", [1, 16, 600])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_swiglu_far_below_zero(cuda, t, dtype):
    """g from -70 to -110, where exp(-g) is beyond fp32 from -88.7 on; u is large, so that silu(g) u is a normal number.

    g and u are sums times scales in 64 bits, h is rounded to fp32 and then to its type: 1.01 * 2^-24 in front of that."""
    n, k = 2048, 64
    announce("int8 swiglu far below zero", t, dtype)
    x = torch.full((t, k), 127, dtype=torch.int8, device=cuda)
    gate = torch.zeros((n, k), dtype=torch.int8, device=cuda)
    gate[:, 0] = -127
    scale = torch.linspace(70, 110, n, device=cuda) / 127 ** 2
    up = torch.full((n, k), 100, dtype=torch.int8, device=cuda)
    wide = torch.full((n,), 1e4, device=cuda)
    one = torch.ones(t, device=cuda)
    want = Q.swish(Q.product(x.cpu().numpy(), np.ones(t), gate.cpu().numpy(), as_np(scale)), Q.product(x.cpu().numpy(), np.ones(t), up.cpu().numpy(), as_np(wide)))
    close(int8_swiglu(x, Int8Weight(gate, scale), Int8Weight(up, wide), x_scales=one, out_dtype=dtype), want, 1.01 * U)


@pytest.mark.parametrize("t,n,k", [(1, 1601, 512), (16, 2048, 300), (140, 1100, 200), (600, 3584, 256), (4096, 4096, 64)])
@pytest.mark.parametrize("reach", [0.05, 3.0, 30.0])
def test_swiglu_is_the_exact_value_rounded(cuda, t, n, k, reach):
    """From |g| far below one, where 1 + exp(-g) is near two, to hundreds; 2^-46 and the oracle's own error are in the 0.01."""
    announce("int8 swiglu, 64 bits", t, n, k, reach)
    g, u = pair_of(n, k, t + n)
    g[1].mul_(reach)
    x = rows(t, k, t)
    q, s = Q.quantize(as_np(x))
    close(int8_swiglu(x, Int8Weight(*g), Int8Weight(*u)), Q.swish(Q.product(q, s, *host(g)), Q.product(q, s, *host(u))), 1.01 * U)


def test_swiglu_of_infinite_scales(cuda):
    """silu(inf) u is inf u, silu(-inf) is NaN (inf / inf), and so is a sum of 0 times an infinite scale, on both kernels."""
    n, k = 1100, 64
    for t in (3, 140):
        codes = torch.zeros((n, k), dtype=torch.int8, device=cuda)
        codes[::3, 0], codes[1::3, 0] = 1, -1
        x, one = torch.ones((t, k), dtype=torch.int8, device=cuda), torch.ones(t, device=cuda)
        gate, up = Int8Weight(codes, torch.full((n,), float("inf"), device=cuda)), Int8Weight(torch.ones_like(codes), torch.ones(n, device=cuda))
        got = int8_swiglu(x, gate, up, x_scales=one)
        assert torch.isposinf(got[:, ::3]).all() and torch.isnan(got[:, 1::3]).all() and torch.isnan(got[:, 2::3]).all()


def test_the_longest_row(cuda):
    """2^31 - 1 columns, where the number of pieces of eight must not be counted in 32 bits."""
    k = 2 ** 31 - 1
    announce("int8 longest row")
    x = torch.zeros((1, k), dtype=torch.float16, device=cuda)
    places, values = [0, 1, 7, 2 ** 20 + 3, 2 ** 30, k - 8, k - 2, k - 1], [1.0, -0.5, 0.25, -1.0, 0.75, 0.125, -0.996, 1.0]
    x[0, places] = torch.tensor(values, dtype=torch.float16, device=cuda)
    want, scale = Q.quantize(as_np(x[:, places]))
    codes, scales = int8_quantize(x)
    del x
    np.testing.assert_array_equal(scales.cpu().numpy(), scale)
    np.testing.assert_array_equal(codes[:, places].cpu().numpy(), want)
    assert int(torch.count_nonzero(codes[0, :2 ** 30])) + int(torch.count_nonzero(codes[0, 2 ** 30:])) == len(places)
    del codes
    torch.cuda.empty_cache()


# ---- what the tiles of many tokens do at the edges ------------------------------------------------------

EDGES = [(140, 1100, 200), (141, 1101, 201), (600, 3584, 256), (1100, 4099, 130)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,n,k", EDGES)
def test_rows_that_are_not_finite_in_a_prompt(cuda, t, n, k, dtype):
    announce("int8 prompt with NaN", t, n, k, dtype)
    tiled(t, n, k)
    g, u = pair_of(n, k, n + k)
    gate, up = Int8Weight(*g), Int8Weight(*u)
    x = rows(t, k, 5, dtype)
    clean = int8_linear(x, gate), int8_swiglu(x, gate, up)
    bad = {0: float("nan"), t // 2: float("inf"), t - 1: -float("inf")}
    for row, value in bad.items():
        x[row, row % k] = value
    keep = [i for i in range(t) if i not in bad]
    for got, want in zip((int8_linear(x, gate), int8_swiglu(x, gate, up)), clean):
        assert torch.isnan(got[list(bad)]).all() and torch.equal(got[keep], want[keep])


def test_extreme_codes_fill_the_int32_sum_of_a_prompt(cuda):
    t, n, k = 140, 1100, 131071
    announce("int8 prompt, extreme codes")
    tiled(t, n, k)
    codes = torch.full((n, k), -128, dtype=torch.int8, device=cuda)
    codes[1::2] = 127
    weight = Int8Weight(codes, torch.ones(n, device=cuda))
    del codes
    x = torch.full((t, k), -128, dtype=torch.int8, device=cuda)
    got = int8_linear(x, weight, x_scales=torch.ones(t, device=cuda))
    assert got[:, ::2].eq(128.0 * 128 * k).all()
    assert got[:, 1::2].double().sub(-127.0 * 128 * k).abs().le(127.0 * 128 * k * U).all()
    x[:, -1] = 127                            # the last column is multiplied, the padding behind it is not
    got = int8_linear(x, weight, x_scales=torch.ones(t, device=cuda))
    want = 128.0 * 128 * (k - 1) - 128.0 * 127
    assert got[:, ::2].double().sub(want).abs().le(want * U).all()


def test_prompts_on_two_streams_do_not_meet(cuda):
    gate, up = (Int8Weight(*m) for m in pair_of(1100, 256, 3))
    xs = [rows(t, 256, t, dtype) for t, dtype in ((140, torch.float32), (300, torch.bfloat16), (700, torch.float16))]
    for x in xs:
        tiled(x.shape[0], 1100, 256)
    want = [(int8_linear(x, gate), int8_swiglu(x, gate, up)) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for _ in range(5):
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append((int8_linear(x, gate), int8_swiglu(x, gate, up)))
    torch.cuda.synchronize()
    for i, (a, b) in enumerate(got):
        assert torch.equal(a, want[i % 3][0]) and torch.equal(b, want[i % 3][1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_prompts_replay_from_two_graphs(cuda, dtype):
    """Rows quantised on the way, so each graph keeps a workspace of its own."""
    announce("int8 prompt graphs", dtype)
    t, n, k = 300, 1100, 256
    tiled(t, n, k)
    gate, up = (Int8Weight(*m) for m in pair_of(n, k, 3))
    x = rows(t, k, 1, dtype)
    step = lambda: (int8_linear(x, gate), int8_swiglu(x, gate, up))
    step()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    for seed in range(4):
        x.copy_(rows(t, k, seed + 2, dtype))
        eager = step()
        torch.cuda.synchronize()
        for graph, out in zip(graphs, outs):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1])


# ---- guards around every output and workspace of the C entries -----------------------------------------

GUARD = 512


class Guarded:
    """A buffer of exactly `nbytes` between two guards, at a 256-byte aligned address."""

    def __init__(self, nbytes, fill=93):
        self.nbytes, self.fill = nbytes, fill
        self.bytes = torch.full((nbytes + 2 * GUARD,), fill, dtype=torch.uint8, device="cuda")

    @property
    def at(self):
        return self.bytes.data_ptr() + GUARD

    def as_(self, dtype, *shape):
        return self.bytes[GUARD:GUARD + self.nbytes].view(dtype).reshape(shape)

    def whole(self):
        return bool(self.bytes[:GUARD].eq(self.fill).all()) and bool(self.bytes[GUARD + self.nbytes:].eq(self.fill).all())


@pytest.mark.parametrize("t,n,k", [(1, 70, 200), (5, 71, 200), (16, 70, 129), (19, 70, 200)] + EDGES[:2])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("given", [False, True])
def test_products_write_their_output_and_workspace_only(cuda, t, n, k, dtype, given):
    announce("int8 guards", t, n, k, dtype, given)
    lib, stream = _lib.load(), torch.cuda.current_stream().cuda_stream
    gate, up = (Int8Weight(*m) for m in pair_of(n, k, 2))
    x = rows(t, k, 3, dtype)
    codes, scales = int8_quantize(x)
    odt = _TORCH_DTYPE_ID[dtype]
    xdt, xat, sat = (INT8, codes.data_ptr(), scales.data_ptr()) if given else (odt, x.data_ptr(), None)
    need = lib.qmoe_int8_workspace_bytes(n, k, t, xdt)
    for pair, want in enumerate((int8_linear(x, gate), int8_swiglu(x, gate, up))):
        work, out = Guarded(need), Guarded(t * n * x.element_size())
        head = [gate.tiles.data_ptr(), gate.scales.data_ptr()] + ([up.tiles.data_ptr(), up.scales.data_ptr()] if pair else [])
        entry = lib.qmoe_int8_swiglu if pair else lib.qmoe_int8_linear
        assert entry(*head, n, k, xat, xdt, sat, t, out.at, odt, work.at if need else None, need, stream) == 0
        torch.cuda.synchronize()
        assert torch.equal(out.as_(dtype, t, n), want) and out.whole() and work.whole()


@pytest.mark.parametrize("t", [1, 4, 5, 16, 17, 60])
@pytest.mark.parametrize("e,k,d,f,fs", [(12, 4, 160, 96, 64), (7, 3, 65, 33, 17), (40, 2, 128, 64, 0)])
@pytest.mark.parametrize("routed", [False, True])
def test_step_writes_its_outputs_and_workspace_only(cuda, t, e, k, d, f, fs, routed):
    announce("int8 step guards", t, e, k, d, f, fs, routed)
    lib, stream = _lib.load(), torch.cuda.current_stream().cuda_stream
    parts, shared, vec = layer(e, d, f, fs, 3)
    bank, dshared = Int8ExpertBank(*parts), tuple(Int8Weight(*m) for m in shared) if shared else None
    x, residual, logits = rows(t, d, 1, torch.bfloat16), rows(t, d, 2), torch.from_numpy(synthetic.router_logits(t, e, 3)).cuda()
    want, w, ids = int8_moe_step(x, bank, k, logits=logits, shared=dshared, shared_gate=vec, residual=residual, return_routing=True)
    need = lib.qmoe_int8_moe_workspace_bytes(t, k, e, d, f, fs)
    work, out, out_w, out_i, status = Guarded(need), Guarded(t * d * 2), Guarded(t * k * 4), Guarded(t * k * 8), Guarded(4, 0)
    a = _lib.Int8MoeArgs()
    a.hidden, a.hidden_dtype, a.tokens, a.top_k = x.data_ptr(), _TORCH_DTYPE_ID[x.dtype], t, k
    a.floor_value, a.renormalize = 2.0 ** -14, 1
    if routed:
        a.in_weights, a.in_ids = w.data_ptr(), ids.data_ptr()
    else:
        a.logits = logits.data_ptr()
    a.gate, a.up, a.down = bank.gate_tiles.data_ptr(), bank.up_tiles.data_ptr(), bank.down_tiles.data_ptr()
    a.gate_scales, a.up_scales, a.down_scales = bank.gate_scales.data_ptr(), bank.up_scales.data_ptr(), bank.down_scales.data_ptr()
    a.n_experts, a.d_model, a.d_ff, a.d_ff_shared = e, d, f, fs
    if fs:
        a.shared_gate_w, a.shared_up_w, a.shared_down_w = (m.tiles.data_ptr() for m in dshared)
        a.shared_gate_scales, a.shared_up_scales, a.shared_down_scales = (m.scales.data_ptr() for m in dshared)
        a.shared_gate = vec.data_ptr()
    a.out, a.out_dtype, a.out_weights, a.out_ids = out.at, a.hidden_dtype, out_w.at, out_i.at
    a.residual, a.status_out = residual.data_ptr(), status.at
    assert lib.qmoe_int8_moe_forward(ctypes.byref(a), work.at, need, stream) == 0
    torch.cuda.synchronize()
    assert torch.equal(out.as_(torch.bfloat16, t, d), want) and torch.equal(out_w.as_(torch.float32, t, k), w) and torch.equal(out_i.as_(torch.int64, t, k), ids)
    assert not status.bytes.any()
    assert work.whole() and out.whole() and out_w.whole() and out_i.whole()
    assert lib.qmoe_int8_moe_forward(ctypes.byref(a), work.at, need - 1, stream) == 4      # the size above is needed whole


@pytest.mark.parametrize("big,small", [(16, 1), (16, 4), (16, 5), (17, 16), (17, 4), (40, 16), (130, 1), (130, 17)])
@pytest.mark.parametrize("fs", [0, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_tokens_step_has_the_same_bits_in_every_batch(cuda, big, small, fs, dtype):
    """Codes, sums, hidden activations and the order of additions are the same on every path."""
    announce("int8 step in batches", big, small, fs, dtype)
    e, k, d, f = 24, 4, 256, 192
    parts, shared, _ = layer(e, d, f, fs, 6)
    bank, dshared = Int8ExpertBank(*parts), tuple(Int8Weight(*m) for m in shared) if shared else None
    x, residual, logits = rows(big, d, 2), rows(big, d, 3), torch.from_numpy(synthetic.router_logits(big, e, 3)).cuda()
    whole = int8_moe_step(x, bank, k, logits=logits, shared=dshared, residual=residual, out_dtype=dtype)
    for lo in (0, big - small):
        s = slice(lo, lo + small)
        part = int8_moe_step(x[s].contiguous(), bank, k, logits=logits[s].contiguous(), shared=dshared, residual=residual[s].contiguous(),
                             out_dtype=dtype)
        assert torch.equal(whole[s], part)


@pytest.mark.parametrize("big,small,d", [(17, 16, 256), (40, 4, 300), (130, 1, 1031), (60, 5, 2048)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_the_shared_experts_admission_has_the_same_bits_in_every_batch(cuda, big, small, d, dtype):
    """The gate's dot product of fp32 is added in one order, whether a front kernel or a prompt's combine forms it."""
    announce("int8 admission in batches", big, small, d, dtype)
    e, k, f, fs = 12, 2, 64, 96
    parts, shared, vec = layer(e, d, f, fs, 6)
    bank, dshared = Int8ExpertBank(*parts), tuple(Int8Weight(*m) for m in shared)
    x, logits = rows(big, d, 2, dtype), torch.from_numpy(synthetic.router_logits(big, e, 3)).cuda()
    whole = int8_moe_step(x, bank, k, logits=logits, shared=dshared, shared_gate=vec, out_dtype=torch.float32)
    for lo in range(0, big - small + 1, small):
        s = slice(lo, lo + small)
        part = int8_moe_step(x[s].contiguous(), bank, k, logits=logits[s].contiguous(), shared=dshared, shared_gate=vec, out_dtype=torch.float32)
        assert torch.equal(whole[s], part), (lo, int((whole[s] != part).sum()))
