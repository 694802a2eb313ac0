"""Test infrastructure: the 8-bit integer operators in 64-bit NumPy, element definitions only."""
import numpy as np


def quantize(x):
    """(codes as int64, scales fp32) of rows: s = fl32(max|x| / 127), q = x / s to nearest, halves to even."""
    x = np.asarray(x, np.float64)
    top = np.max(np.abs(x), axis=-1)
    finite = np.isfinite(top)
    s = np.where(finite, np.where(finite, top, 0.0) / 127.0, np.nan).astype(np.float32)
    s64 = s.astype(np.float64)
    live = finite & (s64 > 0)
    q = np.where(live[..., None], x, 0.0) / np.where(live, s64, 1.0)[..., None]
    return np.clip(np.rint(q), -127, 127).astype(np.int64), s


def product(q, s, w, c):
    """sum_k q w (exact) * s * c in 64 bits; q [T, K], w [N, K] whole numbers."""
    acc = np.asarray(q, np.float64) @ np.asarray(w, np.float64).T        # (whole numbers below 2^53: exact in any order)
    return acc * (np.asarray(s, np.float64)[:, None] * np.asarray(c, np.float64)[None, :])


def swish(g, u):
    with np.errstate(over="ignore"):
        return g / (1.0 + np.exp(-g)) * u


def expert(q, s, gate, up, down):
    """One expert's output rows in 64 bits: hidden rounded to fp32, then quantised."""
    h = swish(product(q, s, *gate), product(q, s, *up)).astype(np.float32)
    return product(*quantize(h), *down)


def moe_terms(x, weights, ids, gate, up, down, shared=None, admit=None):
    """[T, slots (+1 with a shared expert), D] weighted outputs in 64 bits, before any sum; ids outside the bank and
    repeats within a token contribute nothing."""
    q, s = quantize(x)
    t, k = ids.shape
    n = k + (shared is not None)
    out = np.zeros((t, n, x.shape[1]))
    for e in range(gate[0].shape[0]):
        at = [(i, j) for i in range(t) for j in range(k) if ids[i, j] == e and e not in ids[i, :j]]
        if not at:
            continue
        rows = [i for i, _ in at]
        y = expert(q[rows], s[rows], *((m[0][e], m[1][e]) for m in (gate, up, down)))
        for r, (i, j) in enumerate(at):
            out[i, j] = y[r] * np.float64(weights[i, j])
    if shared is not None:
        out[:, k] = expert(q, s, *shared) * admit[:, None]
    return out


def admission(x, vector):
    a = np.asarray(x, np.float64) @ np.asarray(vector, np.float64)
    return 1.0 / (1.0 + np.exp(-a))
