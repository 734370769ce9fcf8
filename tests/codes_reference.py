"""Embedding lookup, its gradient and counter-based dropout from their definitions, in numpy and float64, and the bounds
that fp32 arithmetic with one rounding to the output's type keeps to."""
import numpy as np
import torch

# half a step of each type, relative to the value, and half its smallest step (below the normal numbers)
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
U32 = 2.0 ** -24


def philox_words(first, count, seed, offset):
    """Words 4 first .. 4 (first + count) of the stream: Philox4x32-10 (Salmon et al., SC'11) in Python's integers' width
    (uint64 products of 32-bit halves)."""
    m = np.uint64(0xFFFFFFFF)
    s = np.uint64(32)
    i = np.arange(first, first + count, dtype=np.uint64)
    c = [i & m, i >> s, np.full_like(i, offset & 0xFFFFFFFF), np.full_like(i, (offset >> 32) & 0xFFFFFFFF)]
    k = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> s) ^ c[1] ^ np.uint64(k[0]), b & m, (a >> s) ^ c[3] ^ np.uint64(k[1]), a & m]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, 1).reshape(-1)


def keep_mask(n, p, seed, offset):
    t = int(np.floor(p * 4294967296.0 + 0.5))
    if n == 0:
        return np.zeros(0, bool)
    return philox_words(0, (n + 3) // 4, seed, offset & 0xFFFFFFFFFFFFFFFF)[:n] >= np.uint64(t)


def f64(t):
    return t.detach().cpu().double().numpy()


def factor(scale, p):
    return 0.0 if np.floor(p * 4294967296.0 + 0.5) >= 4294967296.0 else scale / (1.0 - p)


def dropout(x, p, rng):
    """(values, bound)"""
    v = f64(x)
    keep = keep_mask(v.size, p, *rng).reshape(v.shape)
    y = np.where(keep, v * factor(1.0, p), 0.0)
    # the factor and the product are rounded to fp32, then once to the type
    return y, np.abs(y) * (HALF[x.dtype] + 3 * U32) + TINY[x.dtype]


def lookup(table, ids, out_dtype, scale=1.0, p=0.0, rng=(0, 0)):
    t, i = f64(table), ids.cpu().numpy().astype(np.int64)
    V, D = t.shape
    ok = (i >= 0) & (i < V)
    y = np.where(ok[..., None], t[np.where(ok, i, 0)] * factor(scale, p), 0.0)
    if p > 0.0:
        y = np.where(keep_mask(y.size, p, *rng).reshape(y.shape), y, 0.0)
    return y, np.abs(y) * (HALF[out_dtype] + 3 * U32) + TINY[out_dtype]


def table_gradient(g, ids, V, dtype, scale=1.0, p=0.0, rng=(0, 0), pad=-1):
    D = g.shape[-1]
    v, i = f64(g).reshape(-1, D), ids.cpu().numpy().astype(np.int64).reshape(-1)
    if p > 0.0:
        v = np.where(keep_mask(v.size, p, *rng).reshape(v.shape), v, 0.0)
    ok = (i >= 0) & (i < V) & (i != pad)
    v, i = v[ok], i[ok]
    total, size, count = np.zeros((V, D)), np.zeros((V, D)), np.zeros(V)
    np.add.at(total, i, v)
    np.add.at(size, i, np.abs(v))
    np.add.at(count, i, 1.0)
    f = factor(scale, p)
    y = total * f
    # n terms added in fp32 in any order: n - 1 roundings, each at most 2^-24 of the sum of magnitudes (to first order;
    # the factor 1.01 covers the rest for the counts here); then the factor, the product, and the type
    err = 1.01 * count[:, None] * U32 * size * abs(f)
    return y, err + (np.abs(y) + err) * (HALF[dtype] + 3 * U32) + TINY[dtype]


def assert_within(got, want, bound, what=""):
    got = f64(got)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~(np.abs(got - want) <= bound)
    if bad.any():
        at = tuple(int(k) for k in np.argwhere(bad)[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.size} outside the bound, first at {at}: got {got[at]!r}, "
                             f"want {want[at]!r} +- {bound[at]!r}")
