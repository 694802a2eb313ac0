"""What the 8-bit integer operators cost, case by case: row quantisation, the linear and SwiGLU products of 8-bit codes with a
scale for each token and output channel, and the mixture-of-experts step on such weights.

With ``own`` false, ``run`` computes the plain form from elementary torch operations; with ``own`` true it makes the calls a
user makes of the package.  Shapes: the 8B projections (4096 / 14336) and the 512-expert top-10 layer (2048 / 512, shared expert
2048) of the benchmark, the ranges around them, and generic odd sizes.
"""
import math

import torch

own = False

_DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_DEVICE = "cuda"
_FLOOR = 2.0 ** -14


def listed():
    return [
        # the rows of one decoded token in front of a projection: latency only
        {"name": "quantize_one_token", "op": "quantize", "tokens": 1, "k": 4096, "dtype": "float32"},
        # a prompt's hidden states
        {"name": "quantize_prompt", "op": "quantize", "tokens": 4096, "k": 4096, "dtype": "bfloat16"},
        # odd everything: a ragged batch of rows whose width is no multiple of anything
        {"name": "quantize_odd", "op": "quantize", "tokens": 333, "k": 1999, "dtype": "float16"},
        # one token through an attention projection: the smallest call of a decode step
        {"name": "linear_one_token", "op": "linear", "tokens": 1, "n": 4096, "k": 4096, "dtype": "bfloat16", "codes": False},
        # a batch of decoding sequences through the widest projection
        {"name": "linear_batch", "op": "linear", "tokens": 16, "n": 14336, "k": 4096, "dtype": "float32", "codes": False},
        # a short prompt of odd sizes whose rows come as codes already
        {"name": "linear_odd", "op": "linear", "tokens": 77, "n": 1001, "k": 1234, "dtype": "float16", "codes": True},
        # a long prompt through the widest projection: the largest product
        {"name": "linear_prompt", "op": "linear", "tokens": 4096, "n": 14336, "k": 4096, "dtype": "bfloat16", "codes": False},
        # one token through gate and up
        {"name": "swiglu_one_token", "op": "swiglu", "tokens": 1, "n": 14336, "k": 4096, "dtype": "bfloat16", "codes": False},
        # a prompt through a shared expert's gate and up
        {"name": "swiglu_prompt", "op": "swiglu", "tokens": 512, "n": 2048, "k": 2048, "dtype": "float32", "codes": False},
        # one decoded token through the whole expert layer, router and residual included
        {"name": "moe_one_token", "op": "moe", "tokens": 1, "experts": 512, "top_k": 10, "d_model": 2048, "d_ff": 512, "d_shared": 2048,
         "dtype": "float32", "out_dtype": "float32", "zipf": False, "residual": True, "routed": False},
        # sixteen decoding sequences
        {"name": "moe_batch", "op": "moe", "tokens": 16, "experts": 512, "top_k": 10, "d_model": 2048, "d_ff": 512, "d_shared": 2048,
         "dtype": "bfloat16", "out_dtype": "bfloat16", "zipf": False, "residual": False, "routed": False},
        # a prompt whose experts are not equally popular
        {"name": "moe_prompt", "op": "moe", "tokens": 512, "experts": 512, "top_k": 10, "d_model": 2048, "d_ff": 512, "d_shared": 2048,
         "dtype": "float32", "out_dtype": "float32", "zipf": True, "residual": True, "routed": False},
    ]


def _spread(rng, low, high):
    """A whole number of low..high, evenly over the logarithm; often a multiple of 64 where that is in range."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if v >= 128 and rng.random() < 0.5:
        v = v // 64 * 64
    return max(low, min(high, v))


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "swiglu", "moe", "moe"])
    dtype = rng.choice(sorted(_DTYPES))
    if op == "quantize":
        tokens, k = _spread(rng, 1, 8192), _spread(rng, 1, 16384)
        return {"op": op, "tokens": max(1, min(tokens, (1 << 24) // k)), "k": k, "dtype": dtype}
    if op in ("linear", "swiglu"):
        n, k, tokens = _spread(rng, 1, 14336), _spread(rng, 1, 14336), _spread(rng, 1, 4096)
        most = (4096 * 14336 * 4096) // (n * k * (2 if op == "swiglu" else 1))
        return {"op": op, "tokens": max(1, min(tokens, most)), "n": n, "k": k, "dtype": dtype, "codes": rng.random() < 0.3}
    experts = _spread(rng, 4, 512)
    d_model, d_ff = _spread(rng, 64, 2048), _spread(rng, 32, 1536)
    while experts * d_model * d_ff > 512 * 2048 * 512:
        experts //= 2
    return {"op": op, "tokens": _spread(rng, 1, 512), "experts": experts, "top_k": rng.randint(1, min(10, experts)), "d_model": d_model, "d_ff": d_ff,
            "d_shared": rng.choice([0, 0, d_ff, _spread(rng, 32, 2048)]), "dtype": dtype, "out_dtype": rng.choice([dtype, "float32"]),
            "zipf": rng.random() < 0.5, "residual": rng.random() < 0.5, "routed": rng.random() < 0.4}


# ---- inputs ------------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device=_DEVICE).manual_seed(int(seed))


def _rows(gen, tokens, k, dtype):
    """Hidden states: N(0, 1) with a few channels that are larger everywhere, as trained models have them."""
    x = torch.randn((tokens, k), generator=gen, device=_DEVICE)
    loud = torch.rand(k, generator=gen, device=_DEVICE) < 0.004
    return torch.where(loud, x * 12.0, x).to(_DTYPES[dtype])


def _matrix(gen, *shape):
    """Codes and channel scales of weights N(0, 0.02): a row's largest of some thousand values lies near four sigma."""
    codes = torch.empty(shape, dtype=torch.int8, device=_DEVICE)
    flat = codes.reshape(-1)
    step = 1 << 27
    for lo in range(0, flat.numel(), step):
        part = flat[lo:lo + step]
        part.copy_((torch.randn(part.shape, generator=gen, device=_DEVICE) * 32.0).round_().clamp_(-127, 127))
    scales = (0.02 / 32.0) * (1.0 + 0.1 * torch.randn(shape[:-1], generator=gen, device=_DEVICE)).clamp(0.5, 1.5)
    return codes, scales


def _logits(gen, tokens, experts, zipf):
    if not zipf:
        return torch.randn((tokens, experts), generator=gen, device=_DEVICE)
    rank = (torch.randperm(experts, generator=gen, device=_DEVICE) + 1).double()
    u = torch.rand((tokens, experts), generator=gen, device=_DEVICE, dtype=torch.float64).clamp_min(1e-12)
    return (-1.1 * rank.log()[None, :] - (-u.log()).log()).float()


def _inputs(case, seed):
    gen = _generator(seed)
    op, tokens = case["op"], case["tokens"]
    s = {"op": op}
    if op == "quantize":
        s["x"] = _rows(gen, tokens, case["k"], case["dtype"])
        return s
    if op in ("linear", "swiglu"):
        n, k = case["n"], case["k"]
        x = _rows(gen, tokens, k, case["dtype"])
        s["out_dtype"] = _DTYPES[case["dtype"]]
        if case["codes"]:
            s["x"], s["x_scales"] = _plain_quantize(x)
        else:
            s["x"], s["x_scales"] = x, None
        s["w"] = _matrix(gen, n, k)
        if op == "swiglu":
            s["w2"] = _matrix(gen, n, k)
        return s
    e, d, f, fs, k = case["experts"], case["d_model"], case["d_ff"], case["d_shared"], case["top_k"]
    s["top_k"], s["out_dtype"] = k, _DTYPES[case["out_dtype"]]
    s["x"] = _rows(gen, tokens, d, case["dtype"])
    s["gate"], s["up"], s["down"] = _matrix(gen, e, f, d), _matrix(gen, e, f, d), _matrix(gen, e, d, f)
    s["shared"] = (_matrix(gen, fs, d), _matrix(gen, fs, d), _matrix(gen, d, fs)) if fs else None
    s["shared_gate"] = 0.02 * torch.randn(d, generator=gen, device=_DEVICE) if fs else None
    s["residual"] = torch.randn((tokens, d), generator=gen, device=_DEVICE) if case["residual"] else None
    logits = _logits(gen, tokens, e, case["zipf"])
    if case["routed"]:     # routing decided elsewhere: weights and ids are the inputs
        ids = torch.sort(logits, dim=-1, descending=True, stable=True)[1][:, :k].contiguous()
        w = torch.rand((tokens, k), generator=gen, device=_DEVICE) + 0.05
        s["logits"], s["weights"], s["ids"] = None, w / w.sum(-1, keepdim=True), ids
    else:
        s["logits"], s["weights"], s["ids"] = logits, None, None
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and s["op"] != "quantize":
        from mylocal_llm_amd.int8_linear import Int8Weight
        if s["op"] == "moe":
            from mylocal_llm_amd.int8_moe import Int8ExpertBank
            s["own_bank"] = Int8ExpertBank(s.pop("gate"), s.pop("up"), s.pop("down"))
            shared = s.pop("shared")
            s["own_shared"] = tuple(Int8Weight(*m) for m in shared) if shared is not None else None
        else:
            s["own_w"] = Int8Weight(*s.pop("w"))
            if s["op"] == "swiglu":
                s["own_w2"] = Int8Weight(*s.pop("w2"))
    return s


# ---- the framework's operators ------------------------------------------------------------------------

def _run_own(s):
    op = s["op"]
    if op == "quantize":
        from mylocal_llm_amd.int8_linear import int8_quantize
        return int8_quantize(s["x"])
    if op == "linear":
        from mylocal_llm_amd.int8_linear import int8_linear
        return int8_linear(s["x"], s["own_w"], x_scales=s["x_scales"], out_dtype=s["out_dtype"])
    if op == "swiglu":
        from mylocal_llm_amd.int8_linear import int8_swiglu
        return int8_swiglu(s["x"], s["own_w"], s["own_w2"], x_scales=s["x_scales"], out_dtype=s["out_dtype"])
    from mylocal_llm_amd.int8_moe import int8_moe_step
    return int8_moe_step(s["x"], s["own_bank"], s["top_k"], logits=s["logits"], weights=s["weights"], ids=s["ids"], shared=s["own_shared"],
                         shared_gate=s["shared_gate"], floor=_FLOOR, residual=s["residual"], out_dtype=s["out_dtype"], return_routing=True)


# ---- the plain forms ----------------------------------------------------------------------------------

def _plain_quantize(x):
    """Codes and scales of rows: s = max|x| / 127, q = x / s to the nearest whole number, halves to even (in 64 bits: a quotient
    next to a half must not be moved onto it).  A row that is not finite has the scale NaN and codes of zero."""
    x = x.float()
    top = x.abs().amax(-1)
    scale = (top.double() / 127.0).float()
    good = torch.isfinite(top)
    scale = torch.where(good, scale, torch.full_like(scale, math.nan))
    safe = torch.where(good & (scale > 0), scale, torch.full_like(scale, math.inf)).double()
    q = torch.where(good[..., None], x, torch.zeros_like(x)).double() / safe[..., None]
    return q.round().clamp(-127, 127).to(torch.int8), scale


def _plain_rows(s):
    if s.get("x_scales") is not None:
        return s["x"], s["x_scales"]
    return _plain_quantize(s["x"])


def _plain_product(q, qs, w, ws):
    return (q.float() @ w.float().t()) * qs[:, None] * ws[None, :]


def _silu_product(g, u):
    return g / (1.0 + torch.exp(-g)) * u


def _hidden(q, qs, gate, up):
    """The stored activation of an expert for its rows, in 64 bits and rounded to 32 once: it is cut into codes next."""
    q, qs = q.double(), qs.double()[:, None]
    g = (q @ gate[0].double().t()) * qs * gate[1].double()
    u = (q @ up[0].double().t()) * qs * up[1].double()
    return _silu_product(g, u).float()


def _plain_moe(s):
    x, k = s["x"], s["top_k"]
    tokens, d = x.shape
    if s["logits"] is not None:
        z = s["logits"]
        p = torch.exp(z - z.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        ids = torch.sort(z, dim=-1, descending=True, stable=True)[1][:, :k].contiguous()
        w = torch.gather(p, 1, ids)
        w = w / w.sum(-1, keepdim=True).clamp_min(_FLOOR)
    else:
        w, ids = s["weights"], s["ids"]
    q, qs = _plain_quantize(x)
    (gc, gs), (uc, us), (dc, ds) = s["gate"], s["up"], s["down"]
    f = gc.shape[1]
    out = torch.zeros((tokens, d), device=x.device)
    step = max(1, min(16, (1 << 26) // (f * d)))        # tokens whose experts' matrices are gathered at a time
    for lo in range(0, tokens, step):
        hi = min(tokens, lo + step)
        rows, scale = q[lo:hi, :, None].double(), qs[lo:hi, None].double()
        for j in range(k):
            e = ids[lo:hi, j]
            g = torch.bmm(gc[e].double(), rows)[..., 0] * scale * gs[e].double()
            u = torch.bmm(uc[e].double(), rows)[..., 0] * scale * us[e].double()
            hq, hs = _plain_quantize(_silu_product(g, u).float())
            y = torch.bmm(dc[e].float(), hq[:, :, None].float())[..., 0] * hs[:, None] * ds[e]
            out[lo:hi] += y * w[lo:hi, j, None]
    if s["shared"] is not None:
        gate, up, down = s["shared"]
        hq, hs = _plain_quantize(_hidden(q, qs, gate, up))
        admit = torch.sigmoid((x.float() * s["shared_gate"]).sum(-1))
        out = out + _plain_product(hq, hs, *down) * admit[:, None]
    if s["residual"] is not None:
        out = s["residual"] + out
    return out.to(s["out_dtype"]), w, ids


def _run_plain(s):
    op = s["op"]
    if op == "quantize":
        return _plain_quantize(s["x"])
    if op == "linear":
        return _plain_product(*_plain_rows(s), *s["w"]).to(s["out_dtype"])
    if op == "swiglu":
        q, qs = _plain_rows(s)
        return _silu_product(_plain_product(q, qs, *s["w"]), _plain_product(q, qs, *s["w2"])).to(s["out_dtype"])
    return _plain_moe(s)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without ----------------------------------------------------------------------

def _size(name):
    return 4 if name == "float32" else 2


def work(case):
    op, t = case["op"], case["tokens"]
    if op == "quantize":
        return {"bytes": t * case["k"] * (_size(case["dtype"]) + 1) + 4 * t, "flops": 3 * t * case["k"]}
    if op in ("linear", "swiglu"):
        n, k, pair = case["n"], case["k"], 2 if op == "swiglu" else 1
        x = t * (k + 4) if case["codes"] else t * k * _size(case["dtype"])
        return {"bytes": pair * n * (k + 4) + x + t * n * _size(case["dtype"]), "flops": 2 * pair * t * n * k}
    e, d, f, fs, k = case["experts"], case["d_model"], case["d_ff"], case["d_shared"], case["top_k"]
    if case["zipf"]:       # expected number of distinct experts: draws without replacement, popularity rank ** -1.1
        p = [r ** -1.1 for r in range(1, e + 1)]
        low, high = 0.0, 1e9
        for _ in range(60):    # the rate at which a token holds k experts on average
            mid = (low + high) / 2
            low, high = (mid, high) if sum(1 - math.exp(-mid * v) for v in p) < k else (low, mid)
        distinct = sum(1 - math.exp(-low * v * t) for v in p)
    else:
        distinct = e * (1 - (1 - k / e) ** t)
    weights = distinct * (3 * d * f + 4 * (2 * f + d)) + (3 * d * fs + 4 * (2 * fs + d))
    rows = t * d * (_size(case["dtype"]) + _size(case["out_dtype"]) + (4 if case["residual"] else 0))
    routing = t * k * 12 * (2 if case["routed"] else 1) + (0 if case["routed"] else t * e * 4)
    return {"bytes": int(weights + rows + routing), "flops": int(6 * t * d * (k * f + fs))}


# ---- the definitions, in 64 bits --------------------------------------------------------------------------

def _codes64(rows):
    """(whole numbers as doubles, scale as stored in 32 bits) of finite rows."""
    rows = rows.to(torch.float64)
    scale = (rows.abs().max(dim=-1).values / 127).to(torch.float32).to(torch.float64)
    divisor = torch.where(scale == 0, torch.ones_like(scale), scale)
    whole = torch.round(rows / divisor.unsqueeze(-1))
    whole = torch.where((scale == 0).unsqueeze(-1), torch.zeros_like(whole), whole)
    return whole.clamp(min=-127, max=127), scale


def _dot64(rows, scale, matrix, channel):
    """Sum over columns of whole numbers (exact), then the two scales; the channels in parts, to bound the temporary."""
    parts = []
    for lo in range(0, matrix.shape[0], 4096):
        parts.append(torch.mm(rows, matrix[lo:lo + 4096].to(torch.float64).transpose(0, 1).contiguous()))
    return torch.cat(parts, 1) * scale.unsqueeze(1) * channel.to(torch.float64).unsqueeze(0)


def _swish64(a, b):
    return a * b / (torch.exp(-a) + 1)


def _expert64(rows, scale, gate, up, down):
    stored = _swish64(_dot64(rows, scale, *gate), _dot64(rows, scale, *up)).to(torch.float32)
    return _dot64(*_codes64(stored), *down)


def exact(case, seed):
    s = _inputs(case, seed)
    op = s["op"]
    if op == "quantize":
        whole, scale = _codes64(s["x"])
        return whole.to(torch.int8), scale
    if op in ("linear", "swiglu"):
        rows, scale = (s["x"].to(torch.float64), s["x_scales"].to(torch.float64)) if case["codes"] else _codes64(s["x"])
        y = _dot64(rows, scale, *s["w"])
        return _swish64(y, _dot64(rows, scale, *s["w2"])) if op == "swiglu" else y
    x = s["x"].to(torch.float64)
    tokens, k, e = case["tokens"], case["top_k"], case["experts"]
    if s["logits"] is not None:
        z = s["logits"].to(torch.float64)
        order = sorted_ids = torch.argsort(-z, dim=1, stable=True)[:, :k]
        share = torch.softmax(z, dim=1).gather(1, order)
        share = share / torch.clamp(share.sum(1, keepdim=True), min=_FLOOR)
    else:
        share, sorted_ids = s["weights"].to(torch.float64), s["ids"]
    rows, scale = _codes64(s["x"])
    total = torch.zeros_like(x)
    host = sorted_ids.cpu()
    for expert in range(e):
        at = (host == expert).nonzero()
        if not len(at):
            continue
        who, slot = at[:, 0].to(x.device), at[:, 1].to(x.device)
        part = [(m[0][expert], m[1][expert]) for m in (s["gate"], s["up"], s["down"])]
        total.index_add_(0, who, _expert64(rows[who], scale[who], *part) * share[who, slot].unsqueeze(1))
    if s["shared"] is not None:
        admit = 1 / (1 + torch.exp(-torch.mv(x, s["shared_gate"].to(torch.float64))))
        total = total + _expert64(rows, scale, *s["shared"]) * admit.unsqueeze(1)
    if s["residual"] is not None:
        total = total + s["residual"].to(torch.float64)
    return total, share, sorted_ids
