"""8-bit integer quantisation, linear, SwiGLU and the MoE step against their definitions in 64 bits.

Tolerances (before any run): codes and scales are equal.  A product is an exact integer times two scales in 64
bits, rounded to fp32 (2^-24) and then to its type (eps / 2, or half the smallest subnormal).  SwiGLU in fp32: g and
u carry 2^-24 each, silu'(g) g / silu(g) is at most |g| + 1, and exp, the division and two products add a few units:
(|g| + 8) 2^-24.  The step adds k weighted outputs (+ shared + residual), each rounded (k + 4 roundings of 2^-24 of the
sum of magnitudes at most), and the admission gate's fp32 dot product.  Products of many tokens scale 16-bit results in
fp32: the sum's conversion, s * c and their product round, 3 * 2^-24 instead of one, for g and u too.
"""
import numpy as np
import pytest
import torch

from oracle import int8_np as Q
from oracle import reference_np as R
from mylocal_llm_amd import synthetic
from mylocal_llm_amd.int8_linear import Int8Weight, int8_linear, int8_quantize, int8_swiglu
from mylocal_llm_amd.int8_moe import Int8ExpertBank, int8_moe_step
from mylocal_llm_amd.moe import DevicePackedExpertBank, ExpertsInference, Qwen3NextMoEInference, moe_step
from mylocal_llm_amd.quantized_linear import PackedExpertFFNInference, quantized_linear, quantized_swiglu
from gpu_util import announce, upload

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def as_np(t):
    return t.detach().to(torch.float64).cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def close(got, want, rel32, extra=0.0):
    """|got - want| within rel32 of fp32 error plus one rounding to got's type."""
    info = torch.finfo(got.dtype)
    half = info.eps / 2 if got.dtype != torch.float32 else 0.0
    got = as_np(got)
    bound = np.abs(want) * (rel32 + half) * (1 + rel32) + extra * (1 + half) + info.smallest_normal * info.eps / 2
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (int(bad.sum()), bad.size, float(np.nanmax(np.abs(got - want) / np.maximum(bound, 1e-300))))


def front(dtype):
    """Roundings of 2^-24 in front of the one to the output's type."""
    return 1.01 if dtype == torch.float32 else 3.01


def rows(t, k, seed, dtype=torch.float32, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((t, k), generator=g) * (1 + 11 * (torch.rand(k, generator=g) < 0.01))
    return x.to(dtype).to(device)


def matrix(n, k, seed, lead=(), device="cuda"):
    rng = np.random.default_rng(seed)
    codes = rng.integers(-127, 128, (*lead, n, k), dtype=np.int8)
    scales = (rng.random((*lead, n)) * 1e-3 + 1e-4).astype(np.float32)
    return torch.from_numpy(codes).to(device), torch.from_numpy(scales).to(device)


def host(pair):
    return pair[0].cpu().numpy(), pair[1].cpu().numpy()


# ---- quantisation ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,k", [(1, 1), (1, 4096), (3, 7), (5, 64), (2, 63), (4, 65), (333, 1999), (7, 2048), (6, 2056), (9, 8192),
                                 (2, 16384), (3, 14336), (1, 40000), (2, 131075), (1000, 2), (17, 516),
                                 (3, 32768), (2, 32776), (3, 65536), (2, 65544), (2, 20001), (2, 40001), (1030, 1024), (1024, 1031), (1100, 4104)])
def test_codes_and_scales_are_the_definition(cuda, dtype, t, k):
    announce("quantise", dtype, t, k)
    x = rows(t, k, 1000 * t + k, dtype)
    codes, scales = int8_quantize(x)
    q, s = Q.quantize(as_np(x))
    assert codes.dtype == torch.int8 and codes.shape == x.shape and scales.shape == (t,)
    np.testing.assert_array_equal(scales.cpu().numpy(), s)
    np.testing.assert_array_equal(codes.cpu().numpy(), q)


def test_quotients_on_and_next_to_a_half(cuda):
    """Rows whose scale is a power of two hold exact halves; their fp32 neighbours must not be drawn onto them."""
    halves = np.arange(-126, 127, dtype=np.float32) + np.float32(0.5)
    up, down = np.nextafter(halves, np.float32(200)), np.nextafter(halves, np.float32(-200))
    x = np.concatenate([[np.float32(127)], halves, up, down]).astype(np.float32)
    tricky = [x, x * np.float32(2.0 ** -100), x * np.float32(2.0 ** 90)]
    rng = np.random.default_rng(3)
    for _ in range(61):      # scales that are no power of two: the neighbours of (n + 1/2) s
        top = np.float32(rng.random() + 0.5)
        s = np.float32(np.float64(top) / 127.0)
        mid = (halves.astype(np.float64) * np.float64(s)).astype(np.float32)
        row = np.concatenate([[top], mid, np.nextafter(mid, np.float32(9)), np.nextafter(mid, np.float32(-9))])
        tricky.append(np.clip(row, -top, top))
    x = np.stack(tricky).astype(np.float32)
    codes, scales = int8_quantize(torch.from_numpy(x).cuda())
    q, s = Q.quantize(x)
    np.testing.assert_array_equal(scales.cpu().numpy(), s)
    np.testing.assert_array_equal(codes.cpu().numpy(), q)


@pytest.mark.parametrize("k", [5, 512, 4100])
def test_rows_of_zeros_tiny_huge_and_not_finite_values(cuda, k):
    x = torch.zeros((9, k))
    x[1] = 3e38
    x[2] = 1e-45
    x[3] = -1e-38
    x[4, k // 2] = float("nan")
    x[5, k - 1] = float("inf")
    x[6, 0] = -float("inf")
    x[7] = -0.0
    x[8] = torch.linspace(-1, 1, k)
    codes, scales = int8_quantize(x.cuda())
    q, s = Q.quantize(x.numpy())
    np.testing.assert_array_equal(scales.cpu().numpy(), s)
    np.testing.assert_array_equal(codes.cpu().numpy(), q)
    assert torch.isnan(scales[4:7]).all() and not codes[4:7].any()


def test_views_at_odd_addresses_and_higher_ranks(cuda):
    base = rows(1, 5000, 4, torch.bfloat16).reshape(-1)
    for lo, shape in ((1, (3, 7, 129)), (3, (2, 2048)), (5, (4, 1000))):
        x = base[lo:lo + int(np.prod(shape))].reshape(shape)
        codes, scales = int8_quantize(x)
        q, s = Q.quantize(as_np(x))
        assert codes.shape == shape and scales.shape == shape[:-1]
        np.testing.assert_array_equal(scales.cpu().numpy(), s)
        np.testing.assert_array_equal(codes.cpu().numpy(), q)
    empty = int8_quantize(torch.empty((0, 5), device=cuda))
    assert empty[0].shape == (0, 5) and empty[1].shape == (0,)


# ---- linear ----------------------------------------------------------------------------------------------

SHAPES = [(1, 1, 1), (1, 16, 64), (1, 17, 65), (1, 4096, 512), (2, 15, 63), (3, 100, 129), (5, 33, 1000), (15, 48, 4096), (16, 64, 192), (17, 250, 128),
          (31, 1, 257), (33, 129, 320), (48, 272, 511), (64, 144, 640), (65, 16, 64), (77, 1001, 1234), (100, 300, 96), (128, 256, 256),
          (129, 257, 257), (200, 64, 2048), (256, 512, 128), (300, 520, 448), (513, 130, 200), (1, 32, 14336), (1, 33, 16385), (4, 32, 20000), (40, 32, 14336), (700, 700, 320), (300, 16 * 300, 64)]


@pytest.mark.parametrize("t,n,k", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_is_the_exact_sum_rounded_once(cuda, t, n, k, dtype):
    announce("linear", t, n, k, dtype)
    x, w = rows(t, k, t + n + k, dtype), matrix(n, k, t * n + k)
    weight = Int8Weight(*w)
    q, s = Q.quantize(as_np(x))
    want = Q.product(q, s, *host(w))
    got = int8_linear(x, weight)
    assert got.dtype == dtype and got.shape == (t, n)
    close(got, want, front(dtype) * U)
    codes, scales = int8_quantize(x)
    again = int8_linear(codes, weight, x_scales=scales, out_dtype=dtype)
    assert torch.equal(again, got)           # the same integers, the same scales
    if dtype != torch.float32:
        close(int8_linear(x, weight, out_dtype=torch.float32), want, 1.01 * U)


# sizes behind each of the tiles for many tokens, whole and with rests on every side; K from one column to many chunks
TILED = [(950, 3590, 1), (960, 3584, 200), (1800, 4096, 64), (1790, 4090, 321), (4096, 4096, 72), (4001, 4085, 130), (700, 704, 1100), (690, 1000, 513),
         (500, 3600, 330), (130, 1000, 2900), (140, 1001, 1700), (150, 990, 1300), (1000, 2000, 1500)]


@pytest.mark.parametrize("t,n,k", TILED)
@pytest.mark.parametrize("dtype", DTYPES)
def test_tiles_of_many_tokens(cuda, t, n, k, dtype):
    announce("int8 tiles", t, n, k, dtype)
    x, g, u = rows(t, k, t + n, dtype), matrix(n, k, n + k), matrix(n, k, n + k + 1)
    g[1].mul_(20.0 / k ** 0.5)
    gate, up = Int8Weight(*g), Int8Weight(*u)
    q, s = Q.quantize(as_np(x))
    gv, uv = Q.product(q, s, *host(g)), Q.product(q, s, *host(u))
    got = int8_linear(x, gate)
    close(got, gv, front(dtype) * U)
    close(int8_swiglu(x, gate, up), Q.swish(gv, uv), (front(dtype) * np.abs(gv) + 12) * U)
    codes, scales = int8_quantize(x)
    assert torch.equal(int8_linear(codes, gate, x_scales=scales, out_dtype=dtype), got)
    some = torch.arange(0, t, 97, device=cuda)
    few = int8_linear(x[some].contiguous(), gate, out_dtype=torch.float32)
    assert torch.equal(int8_linear(x, gate, out_dtype=torch.float32)[some], few)      # one formula on every path


@pytest.mark.parametrize("t,n,k", [(1, 700, 200), (20, 700, 200), (100, 704, 200), (720, 704, 200), (720, 1001, 64)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scales_far_from_one(cuda, t, n, k, dtype):
    """s * c beyond fp32's normal range on either side, results inside it.  (extra: half of fp32's smallest subnormal)"""
    announce("int8 scales", t, n, k, dtype)
    x, (codes, scales) = rows(t, k, t), matrix(n, k, n)
    x = (x * torch.tensor([1e-39, 1e-30, 1e-10, 1.0, 1e10, 1e28], device=cuda)[torch.arange(t, device=cuda) % 6][:, None]).to(dtype)
    scales = scales * torch.tensor([1e-8, 1.0, 1e4], device=cuda)[torch.arange(n, device=cuda) % 3]
    scales[5::50] = 0.0
    q, s = Q.quantize(as_np(x))
    close(int8_linear(x, Int8Weight(codes, scales)), Q.product(q, s, codes.cpu().numpy(), scales.cpu().numpy()), front(dtype) * U, 2.0 ** -150)


@pytest.mark.parametrize("t", [1, 5, 16, 40, 130])
def test_a_tokens_result_does_not_depend_on_the_others(cuda, t):
    x, weight = rows(t, 1030, 9), Int8Weight(*matrix(150, 1030, 8))
    whole = int8_linear(x, weight)
    for i in range(0, t, 7):
        assert torch.equal(int8_linear(x[i:i + 1], weight), whole[i:i + 1])


@pytest.mark.parametrize("t", [1, 3, 16, 17, 140])
def test_not_finite_rows_give_nan_and_leave_the_others(cuda, t):
    x = rows(t, 200, 5)
    weight = Int8Weight(*matrix(70, 200, 6))
    clean = int8_linear(x, weight)
    x[t // 2, 77] = float("inf")
    got = int8_linear(x, weight)
    assert torch.isnan(got[t // 2]).all()
    keep = [i for i in range(t) if i != t // 2]
    assert torch.equal(got[keep], clean[keep])


def test_extreme_codes_fill_the_int32_sum(cuda):
    k = 131071
    codes = torch.full((2, k), -128, dtype=torch.int8, device=cuda)
    codes[1] = 127
    weight = Int8Weight(codes, torch.ones(2, device=cuda))
    for t in (1, 20):
        x = torch.full((t, k), -128, dtype=torch.int8, device=cuda)
        got = int8_linear(x, weight, x_scales=torch.ones(t, device=cuda))
        assert got[:, 0].eq(128.0 * 128 * k).all()
        assert got[:, 1].double().sub(-127.0 * 128 * k).abs().le(127.0 * 128 * k * U).all()


def test_matrix_beyond_four_gigabytes(cuda):
    n, k = 70000, 65536
    codes = torch.zeros((n, k), dtype=torch.int8, device=cuda)
    tail = matrix(40, k, 3)
    codes[-40:] = tail[0]
    scales = torch.ones(n, device=cuda)
    scales[-40:] = tail[1]
    weight = Int8Weight(codes, scales)
    del codes
    for t in (1, 24, 130):
        x = rows(t, k, t)
        got = int8_linear(x, weight)
        q, s = Q.quantize(as_np(x))
        close(got[:, -40:], Q.product(q, s, *host(tail)), 1.01 * U)
        assert not got[:, :-40].any()
        del got
    del weight
    torch.cuda.empty_cache()


def test_three_dimensional_input_zero_rows_and_odd_addresses(cuda):
    weight = Int8Weight(*matrix(37, 100, 2))
    x = rows(6, 100, 3).reshape(2, 3, 100)
    flat = int8_linear(x.reshape(6, 100), weight)
    assert torch.equal(int8_linear(x, weight), flat.reshape(2, 3, 37))
    assert int8_linear(x[:0], weight).shape == (0, 3, 37)
    base = rows(1, 700, 7, torch.float16).reshape(-1)
    view = base[1:601].reshape(6, 100)       # rows at 2-byte addresses
    assert torch.equal(int8_linear(view, weight), int8_linear(view.clone(), weight))
    codes, scales = int8_quantize(rows(3, 129, 8))
    wide = Int8Weight(*matrix(20, 128, 2))
    odd = codes.reshape(-1)[1:257].reshape(2, 128)
    assert torch.equal(int8_linear(odd, wide, x_scales=scales[:2]), int8_linear(odd.clone(), wide, x_scales=scales[:2]))


def test_weight_round_trip_and_from_packed(cuda):
    codes, scales = matrix(45, 130, 5)
    weight = Int8Weight(codes, scales)
    assert torch.equal(weight.codes(), codes) and weight.shape == (45, 130)
    packed = upload(synthetic.packed_weight("Q6_K", (96, 512), 7), cuda)
    made = Int8Weight.from_packed(packed)
    q, s = Q.quantize(as_np(packed.dequantize()))
    np.testing.assert_array_equal(made.codes().cpu().numpy(), q)
    np.testing.assert_array_equal(made.scales.cpu().numpy(), s)
    # 8-bit rows stand for the packed matrix to half a step of the row's scale
    assert (made.dequantize() - packed.dequantize()).abs().le(made.scales[:, None] * 0.5001).all()


# ---- SwiGLU ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("t,f,k", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_swiglu(cuda, t, f, k, dtype):
    announce("swiglu", t, f, k, dtype)
    x, g, u = rows(t, k, t + f, dtype), matrix(f, k, 1 + t + k), matrix(f, k, 2 + t + k)
    g[1].mul_(20.0 / k ** 0.5)                # keep |g| where silu is neither linear nor zero everywhere
    q, s = Q.quantize(as_np(x))
    gv, uv = Q.product(q, s, *host(g)), Q.product(q, s, *host(u))
    want = Q.swish(gv, uv)
    got = int8_swiglu(x, Int8Weight(*g), Int8Weight(*u))
    assert got.dtype == dtype
    close(got, want, (front(dtype) * np.abs(gv) + 12) * U)
    codes, scales = int8_quantize(x)
    assert torch.equal(int8_swiglu(codes, Int8Weight(*g), Int8Weight(*u), x_scales=scales, out_dtype=dtype), got)


def test_packed_operators_take_int8_weights(cuda):
    x, g, u, d = rows(5, 256, 3), matrix(96, 256, 4), matrix(96, 256, 5), matrix(256, 96, 6)
    gate, up, down = Int8Weight(*g), Int8Weight(*u), Int8Weight(*d)
    assert torch.equal(quantized_linear(x, gate), int8_linear(x, gate))
    assert torch.equal(quantized_swiglu(x, gate, up), int8_swiglu(x, gate, up))
    want = int8_linear(int8_swiglu(x, gate, up), down)
    assert torch.equal(PackedExpertFFNInference(gate, up, down).forward(x), want)


# ---- the expert step ---------------------------------------------------------------------------------------

def layer(e, d, f, fs, seed):
    bank = tuple(matrix(n, k, seed + i, (e,)) for i, (n, k) in enumerate(((f, d), (f, d), (d, f))))
    shared = tuple(matrix(n, k, seed + 3 + i) for i, (n, k) in enumerate(((fs, d), (fs, d), (d, fs)))) if fs else None
    vec = torch.from_numpy(np.random.default_rng(seed).normal(0, 0.05, d).astype(np.float32)).cuda() if fs else None
    return bank, shared, vec


def check_step(x, bank, shared, vec, weights, ids, residual, got):
    k, d = ids.shape[1], x.shape[1]
    x64, w, i = as_np(x), as_np(weights), ids.cpu().numpy()
    admit = Q.admission(x64, vec.cpu().numpy()) if shared else None
    terms = Q.moe_terms(x64, w, i, *(host(m) for m in bank), shared=tuple(host(m) for m in shared) if shared else None, admit=admit)
    total, size = terms.sum(1), np.abs(terms).sum(1)
    extra = (k + 4) * U * size
    if shared:
        dot = np.abs(x64) @ np.abs(vec.cpu().numpy().astype(np.float64))
        extra += np.abs(terms[:, -1]) * ((-(-d // 256) + 12) * U * dot + 6 * U)[:, None]
    if residual is not None:
        r = as_np(residual)
        total, extra = total + r, extra + U * (np.abs(r) + size)
    close(got, total, 1.01 * U, extra)


CASES = [  # tokens, experts, top_k, d_model, d_ff, d_shared
    (1, 4, 1, 64, 64, 0), (1, 16, 4, 256, 128, 256), (1, 512, 10, 2048, 512, 2048), (2, 8, 8, 100, 50, 30), (3, 7, 3, 65, 33, 0),
    (4, 32, 2, 192, 1536, 64), (5, 60, 4, 128, 704, 100), (9, 512, 10, 256, 64, 0), (15, 5, 5, 330, 130, 17), (16, 64, 6, 512, 256, 512),
    (16, 2, 1, 64, 2048, 0), (17, 16, 4, 256, 256, 256), (33, 9, 2, 130, 70, 0), (64, 40, 8, 256, 100, 128), (100, 3, 3, 77, 91, 13), (200, 64, 2, 320, 192, 0),
    (1, 8, 2, 4096, 300, 0), (7, 8, 2, 300, 4096, 0), (2, 4, 2, 8200, 80, 16),
    (16, 12, 2, 8128, 1500, 0), (17, 6, 2, 8128, 100, 40), (64, 8, 4, 192, 160, 96), (40, 2, 1, 64, 300, 0), (300, 3, 2, 128, 130, 50), (70, 2, 1, 200, 97, 0),
    (120, 4, 1, 130, 70, 33), (220, 6, 2, 300, 190, 100), (400, 2, 1, 260, 65, 0)]


@pytest.mark.parametrize("t,e,k,d,f,fs", CASES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_step_from_logits(cuda, t, e, k, d, f, fs, dtype):
    announce("int8 moe step", t, e, k, d, f, fs, dtype)
    bank, shared, vec = layer(e, d, f, fs, 17 * t + e)
    x, residual = rows(t, d, t + e, dtype), rows(t, d, t + e + 1) if t % 2 else None
    logits = torch.from_numpy(synthetic.router_logits(t, e, t + 5)).cuda()
    dev = Int8ExpertBank(*bank)
    dshared = tuple(Int8Weight(*m) for m in shared) if shared else None
    got, w, ids = int8_moe_step(x, dev, k, logits=logits, shared=dshared, shared_gate=vec, residual=residual, return_routing=True)
    want_w, want_ids = R.router_topk(logits.cpu().numpy(), k)
    np.testing.assert_array_equal(ids.cpu().numpy(), want_ids)
    np.testing.assert_allclose(w.cpu().numpy(), want_w, rtol=2e-6, atol=2e-7)
    assert got.dtype == dtype
    check_step(x, bank, shared, vec, w, ids, residual, got)
    # given the same routing the step is the same, bit for bit
    again, w2, ids2 = int8_moe_step(x, dev, k, weights=w, ids=ids, shared=dshared, shared_gate=vec, residual=residual, return_routing=True)
    assert torch.equal(again, got) and torch.equal(w2, w) and torch.equal(ids2, ids)


@pytest.mark.parametrize("t", [1, 3, 12, 40])
@pytest.mark.parametrize("e,k", [(3, 3), (64, 8), (512, 10), (700, 32), (1024, 1), (1500, 7), (4096, 4)])
def test_routing_order_ties_infinities_and_nan(cuda, t, e, k):
    """Rows of equal logits, of few distinct values, with infinities and NaN: ids equal the router's everywhere."""
    announce("int8 routing", t, e, k)
    d, f = 64, 16
    bank, _, _ = layer(e, d, f, 0, 1) if e <= 700 else (tuple((torch.ones((e, *s), dtype=torch.int8, device=cuda), torch.full((e, s[0]), 1e-3, device=cuda))
                                                              for s in ((f, d), (f, d), (d, f))), None, None)
    dev = Int8ExpertBank(*bank)
    rng = np.random.default_rng(e + t)
    kinds = [np.zeros((t, e)), rng.integers(0, 3, (t, e)), rng.standard_normal((t, e)), np.where(rng.random((t, e)) < 0.3, -np.inf, rng.standard_normal((t, e))),
             np.where(rng.random((t, e)) < 0.2, np.nan, rng.standard_normal((t, e))), np.full((t, e), -np.inf), -np.abs(rng.standard_normal((t, e))) * 1e-30]
    x = rows(t, d, 1)
    for z in kinds:
        z = z.astype(np.float32)
        _, w, ids = int8_moe_step(x, dev, k, logits=torch.from_numpy(z).cuda(), return_routing=True)
        with np.errstate(all="ignore"):
            want_w, want_ids = R.router_topk(z, k)
        np.testing.assert_array_equal(ids.cpu().numpy(), want_ids)
        np.testing.assert_allclose(w.cpu().numpy(), want_w, rtol=2e-6, atol=2e-7, equal_nan=True)


@pytest.mark.parametrize("t", [1, 6, 16, 50])
def test_step_with_bad_ids_repeats_and_rows(cuda, t):
    e, k, d, f = 12, 4, 160, 96
    bank, shared, vec = layer(e, d, f, 64, 3)
    dev, dshared = Int8ExpertBank(*bank), tuple(Int8Weight(*m) for m in shared)
    x = rows(t, d, 1)
    rng = np.random.default_rng(t)
    ids = torch.from_numpy(np.stack([rng.choice(e, k, replace=False) for _ in range(t)])).cuda()
    w = torch.rand((t, k), device=cuda)
    kwargs = dict(shared=dshared, shared_gate=vec)
    clean = int8_moe_step(x, dev, k, weights=w, ids=ids, check_routing=True, **kwargs)
    check_step(x, bank, shared, vec, w, ids, None, clean)
    odd = ids.clone()
    odd[0, 1] = odd[0, 3]                     # a repeat: the first slot counts
    odd[t - 1, 0] = e if t % 2 else -1        # outside the bank
    odd[t // 2, 2] = 2 ** 40
    check_step(x, bank, shared, vec, w, odd, None, int8_moe_step(x, dev, k, weights=w, ids=odd, **kwargs))
    with pytest.raises(ValueError, match="outside the bank"):
        int8_moe_step(x, dev, k, weights=w, ids=odd, check_routing=True, **kwargs)
    odd[:] = -1                               # no expert at all: only the shared one
    check_step(x, bank, shared, vec, w, odd, None, int8_moe_step(x, dev, k, weights=w, ids=odd, **kwargs))
    assert not int8_moe_step(x, dev, k, weights=w, ids=odd).any()
    x[t // 2, 3] = float("nan")
    got = int8_moe_step(x, dev, k, weights=w, ids=ids, **kwargs)
    assert torch.isnan(got[t // 2]).all()
    keep = [i for i in range(t) if i != t // 2]
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("big,small", [(40, 16), (16, 1), (7, 3), (130, 1)])
def test_a_tokens_step_does_not_depend_on_the_batch(cuda, big, small):
    """The codes of the hidden activations are the same on every path, so a token's expert outputs are; only the order of
    fp32 additions may differ between token counts."""
    e, k, d, f, fs = 24, 4, 256, 192, 128
    bank, shared, vec = layer(e, d, f, fs, 6)
    dev, dshared = Int8ExpertBank(*bank), tuple(Int8Weight(*m) for m in shared)
    x, logits = rows(big, d, 2), torch.from_numpy(synthetic.router_logits(big, e, 3)).cuda()
    whole, w, ids = int8_moe_step(x, dev, k, logits=logits, shared=dshared, shared_gate=vec, return_routing=True)
    part = int8_moe_step(x[:small].contiguous(), dev, k, logits=logits[:small].contiguous(), shared=dshared, shared_gate=vec)
    check_step(x, bank, shared, vec, w, ids, None, whole)
    check_step(x[:small], bank, shared, vec, w[:small], ids[:small], None, part)


def test_modules_and_executor_take_an_int8_bank(cuda):
    from mylocal_llm_amd.expert_executor import ResidentExpertExecutor
    e, k, d, f, fs = 16, 4, 128, 96, 64
    bank, shared, vec = layer(e, d, f, fs, 9)
    dev, dshared = Int8ExpertBank(*bank), tuple(Int8Weight(*m) for m in shared)
    x = rows(6, d, 4).reshape(2, 3, d)
    router = torch.from_numpy(np.random.default_rng(2).normal(0, 0.3, (e, d)).astype(np.float32)).cuda()
    block = Qwen3NextMoEInference(dev, k, router, dshared, vec)
    logits = block.router.logits(x.reshape(6, d))
    want = int8_moe_step(x.reshape(6, d), dev, k, logits=logits, shared=dshared, shared_gate=vec)
    assert torch.equal(block.forward(x).reshape(6, d), want)
    assert torch.equal(moe_step(x.reshape(6, d), dev, k, logits=logits, shared=dshared, shared_gate=vec), want)
    gamma = torch.rand(d, device=cuda) + 0.5
    after = block.forward_after_norm(x, gamma, 1e-6)
    from mylocal_llm_amd.moe import norm_router
    rows_, bias = block.router.rows_and_bias()
    normalized, lg = norm_router(x.reshape(6, d), gamma, 1e-6, rows_, bias)
    assert torch.equal(after.reshape(6, d), int8_moe_step(normalized, dev, k, logits=lg, shared=dshared, shared_gate=vec, residual=x.reshape(6, d)))
    w, ids = block.router.route_logits(logits)
    routed = int8_moe_step(x.reshape(6, d), dev, k, weights=w, ids=ids)
    assert torch.equal(ExpertsInference(d, f, e, expert_executor=dev).forward(x, w.reshape(2, 3, k), ids.reshape(2, 3, k)).reshape(6, d), routed)
    executor = ResidentExpertExecutor(d, f)
    executor.register_layer(0, dev)
    assert torch.equal(ExpertsInference(d, f, e, expert_executor=executor).forward(x, w.reshape(2, 3, k), ids.reshape(2, 3, k)).reshape(6, d), routed)
    one = executor.forward(0, 3, x.reshape(6, d))
    assert torch.equal(one, PackedExpertFFNInference(*dev.expert(3)).forward(x.reshape(6, d)))
    assert executor.try_forward_grouped(0, [1, 2], x.reshape(6, d)[:1], w[0, :2], [0, 1]) is None


def test_bank_from_packed(cuda):
    gate, up, down = (synthetic.packed_weight("Q8_0", s, i) for i, s in enumerate(((4, 64, 96), (4, 64, 96), (4, 96, 64))))
    packed = DevicePackedExpertBank(gate, up, down, device=cuda)
    dev = Int8ExpertBank.from_packed(packed)
    assert (dev.n_experts, dev.d_model, dev.d_ff) == (4, 96, 64)
    for i in range(4):
        for codes, w in zip(dev.codes(i), packed.expert(i)):
            q, _ = Q.quantize(as_np(w.dequantize()))
            np.testing.assert_array_equal(codes.cpu().numpy(), q)
    x, logits = rows(5, 96, 1), torch.from_numpy(synthetic.router_logits(5, 4, 1)).cuda()
    near = moe_step(x, packed, 2, logits=logits)
    got = moe_step(x, dev, 2, logits=logits)
    assert (got - near).norm() <= 0.05 * near.norm()      # two 8-bit roundings a product: per cent, not per mille


# ---- streams, graphs, workspaces ---------------------------------------------------------------------------

def sequence(x, logits, residual, gamma, block):
    """What a decoder layer's second half calls: norm, router, experts, then a projection of the result."""
    y = block.forward_after_norm(residual, gamma, 1e-6)
    return int8_linear(y.reshape(-1, y.shape[-1]), block.shared[0])


@pytest.mark.parametrize("t", [1, 12, 40])
def test_a_run_of_the_operators_replays_from_a_graph(cuda, t):
    announce("int8 graph", t)
    e, k, d, f, fs = 32, 4, 256, 128, 192
    bank, shared, vec = layer(e, d, f, fs, 12)
    router = torch.from_numpy(np.random.default_rng(2).normal(0, 0.3, (e, d)).astype(np.float32)).cuda()
    block = Qwen3NextMoEInference(Int8ExpertBank(*bank), k, router, tuple(Int8Weight(*m) for m in shared), vec)
    x, gamma = torch.zeros((1, t, d), device=cuda), torch.rand(d, device=cuda) + 0.5
    step = lambda: sequence(None, None, x, gamma, block)
    x.copy_(rows(t, d, 1).reshape(1, t, d))
    step()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):                       # two graphs over the same weights, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    for seed in range(4):
        x.copy_(rows(t, d, seed + 2).reshape(1, t, d))
        eager = step()
        torch.cuda.synchronize()
        for graph, out in zip(graphs, outs):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, eager)


@pytest.mark.parametrize("t", [1, 4, 9, 16, 60])
def test_the_same_call_gives_the_same_bits(cuda, t):
    e, k, d, f, fs = 24, 4, 320, 192, 128
    bank, shared, vec = layer(e, d, f, fs, 4)
    dev, dshared = Int8ExpertBank(*bank), tuple(Int8Weight(*m) for m in shared)
    x, logits = rows(t, d, 2), torch.from_numpy(synthetic.router_logits(t, e, 3)).cuda()
    first = int8_moe_step(x, dev, k, logits=logits, shared=dshared, shared_gate=vec)
    for _ in range(6):
        assert torch.equal(int8_moe_step(x, dev, k, logits=logits, shared=dshared, shared_gate=vec), first)
    order = torch.randperm(t)
    moved = int8_moe_step(x[order].contiguous(), dev, k, logits=logits[order].contiguous(), shared=dshared, shared_gate=vec)
    assert torch.equal(moved, first[order])          # a token's result does not depend on its place


def test_calls_on_two_streams_do_not_meet(cuda):
    e, k, d, f = 32, 4, 256, 128
    bank, _, _ = layer(e, d, f, 0, 12)
    dev, weight = Int8ExpertBank(*bank), Int8Weight(*matrix(600, 256, 3))
    xs = [rows(t, d, t) for t in (1, 9, 30, 64)]
    lg = [torch.from_numpy(synthetic.router_logits(x.shape[0], e, 3)).cuda() for x in xs]
    want = [(int8_moe_step(x, dev, k, logits=z), int8_linear(x, weight)) for x, z in zip(xs, lg)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for _ in range(5):
        for s, x, z in zip(streams, xs, lg):
            with torch.cuda.stream(s):
                got.append((int8_moe_step(x, dev, k, logits=z), int8_linear(x, weight)))
    torch.cuda.synchronize()
    for i, (a, b) in enumerate(got):
        assert torch.equal(a, want[i % 4][0]) and torch.equal(b, want[i % 4][1])


@pytest.mark.parametrize("t,n,k", [(1, 64, 128), (20, 64, 128), (150, 256, 128), (130, 128, 256)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_outputs_at_odd_addresses(cuda, t, n, k, dtype):
    """The C entry writes to any address that its element type allows; results equal the aligned ones."""
    from mylocal_llm_amd import _lib
    from mylocal_llm_amd.quantized_linear import _TORCH_DTYPE_ID
    lib = _lib.load()
    x, weight = rows(t, k, 3, dtype), Int8Weight(*matrix(n, k, 4))
    want = int8_linear(x, weight)
    base = torch.full((t * n + 2,), 3.0, dtype=dtype, device=cuda)
    work = torch.empty(lib.qmoe_int8_workspace_bytes(n, k, t, 0) + 256, dtype=torch.uint8, device=cuda)
    rc = lib.qmoe_int8_linear(weight.tiles.data_ptr(), weight.scales.data_ptr(), n, k, x.data_ptr(), _TORCH_DTYPE_ID[dtype], None, t,
                              base[1:].data_ptr(), _TORCH_DTYPE_ID[dtype], work.data_ptr(), work.numel(), torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    torch.cuda.synchronize()
    got = base[1:-1].reshape(t, n)
    if dtype == torch.float32:
        assert torch.equal(got, want)
    else:                     # (fp32 or 64-bit scaling in front of the one rounding: a neighbour at most)
        close(got, as_np(want), 4 * U)
    assert base[0] == 3 and base[-1] == 3


def test_many_short_rows_and_long_prompts_are_cut_into_launches(cuda):
    x = torch.ones((4_000_003, 1), dtype=torch.float16, device=cuda)
    x[-1] = -5.0
    codes, scales = int8_quantize(x)
    assert codes[:-1].eq(127).all() and codes[-1] == -127 and scales[-1].item() == np.float32(np.float64(5.0) / 127)
    e, k, d, f = 6, 2, 64, 32
    bank, _, _ = layer(e, d, f, 0, 2)
    dev = Int8ExpertBank(*bank)
    t = 9000                  # more than one call's worth of tokens
    x, logits = rows(t, d, 1), torch.from_numpy(synthetic.router_logits(t, e, 3)).cuda()
    got, w, ids = int8_moe_step(x, dev, k, logits=logits, return_routing=True)
    at = torch.tensor([0, 1, 4095, 4096, 8191, 8192, 8999], device=cuda)
    check_step(x[at], bank, None, None, w[at], ids[at], None, got[at])
    part = int8_moe_step(x[4096:8192].contiguous(), dev, k, logits=logits[4096:8192].contiguous())
    assert torch.equal(part, got[4096:8192])


def test_rows_behind_the_output_are_left_alone(cuda):
    """The products and the step through the C entry points with guard rows around every output and workspace."""
    import ctypes
    from mylocal_llm_amd import _lib
    lib = _lib.load()
    t, n, k = 19, 70, 200
    x, weight = rows(t, k, 3), Int8Weight(*matrix(n, k, 4))
    out = torch.full((t + 2, n), 7.0, device=cuda)
    need = lib.qmoe_int8_workspace_bytes(n, k, t, 0)
    work = torch.full((need + 512,), 123, dtype=torch.uint8, device=cuda)
    for m in (1, 5, 16, t):
        out.fill_(7.0)
        rc = lib.qmoe_int8_linear(weight.tiles.data_ptr(), weight.scales.data_ptr(), n, k, x.data_ptr(), 0, None, m, out[1].data_ptr(), 0,
                                  work[256:].data_ptr(), lib.qmoe_int8_workspace_bytes(n, k, m, 0), torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        torch.cuda.synchronize()
        assert out[0].eq(7).all() and out[1 + m:].eq(7).all() and torch.equal(out[1:1 + m], int8_linear(x[:m], weight))
        assert work[:256].eq(123).all() and work[256 + need:].eq(123).all()
