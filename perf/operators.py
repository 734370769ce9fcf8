"""Workloads of the learned-code operators: embedding lookup with scaling (and fused dropout), its gradient by sorted
ids, and dropout whose mask is a function of a Philox counter.

A case is a dict of plain values; `prepare` makes what a program holds before the call, `run` is one call (the plain
torch form, or this package's kernels when `own` is true), `exact` the same outputs in 64 bits.

  lookup   out[n, :] = f * table[ids[n], :] * keep(n, :)                    f = scale / (1 - p)
  train    the lookup and  grad[v, :] = f * sum over n with ids[n] == v of keep(n, :) * g[n, :]   (0 for padding_idx)
  dropout  y[e] = x[e] * keep(e) / (1 - p),  and its gradient g[e] * keep(e) / (1 - p) when `train`

keep(e) of element e (in the contiguous order of the output) is 1 where word e % 4 of
Philox4x32-10(key = seed, counter = (e / 4, offset)) is >= round(p * 2^32), else 0: the mask is never stored.
"""
import math

import numpy as np
import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one training step of a conditional scene: one image, its code out of a table of one code per Lego image
        dict(name="code_step", op="train", n=1, rows=100, dim=32, dtype="fp32", ids="uniform", idx="int64", scale=1.0,
             p=0.0, pad=-1),
        # 4096 rays of a step, each with the code of the image it came from, codes dropped out in training
        dict(name="codes_per_ray", op="train", n=4096, rows=100, dim=48, dtype="fp32", ids="uniform", idx="int64",
             scale=1.0, p=0.1, pad=-1),
        # a code per point of a Fern batch (1024 rays x 128 points, 17 images): a few very long rows of the gradient
        dict(name="codes_per_point", op="train", n=131072, rows=17, dim=64, dtype="bf16", ids="uniform", idx="int32",
             scale=1.0, p=0.0, pad=-1),
        # odd everything: rows that no vector load fits, a padding id, few terms a row
        dict(name="ragged", op="train", n=10007, rows=777, dim=37, dtype="fp16", ids="zipf", idx="int64", scale=0.5,
             p=0.25, pad=3),
        # a word table under a text-conditioned scene: long rows, word frequencies, sqrt(dim) scaling, dropout
        dict(name="words", op="train", n=16384, rows=50000, dim=1024, dtype="bf16", ids="zipf", idx="int64",
             scale=32.0, p=0.1, pad=0),
        # a dense feature grid of 80^3 vertices, the 8 corners around each of a step's 4096 x 192 fine points
        dict(name="grid_corners", op="train", n=6291456, rows=512000, dim=2, dtype="fp32", ids="grid", idx="int32",
             scale=1.0, p=0.0, pad=-1),
        # serving one word: a single long row
        dict(name="one_word", op="lookup", n=1, rows=50000, dim=4096, dtype="bf16", ids="zipf", idx="int64",
             scale=64.0, p=0.0, pad=-1),
        # an 800 x 800 evaluation image with a code per pixel
        dict(name="image_codes", op="lookup", n=640000, rows=1024, dim=16, dtype="bf16", ids="uniform", idx="int64",
             scale=1.0, p=0.0, pad=-1),
        # dropout of the codes of 4096 rays
        dict(name="drop_codes", op="dropout", n=4096, dim=48, dtype="fp32", p=0.1, train=True),
        # an odd number of elements
        dict(name="drop_odd", op="dropout", n=1000003, dim=1, dtype="fp16", p=0.5, train=True),
        # inference-time dropout (an uncertainty estimate) over the 128-wide colour layer of the coarse points
        dict(name="drop_colour", op="dropout", n=262144, dim=128, dtype="fp32", p=0.25, train=False),
        # a 256-wide hidden layer over a step's 4096 x 192 fine points
        dict(name="drop_hidden", op="dropout", n=786432, dim=256, dtype="bf16", p=0.1, train=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["train", "train", "lookup", "dropout"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    p = rng.choice([0.0, 0.1, 0.25, 0.5, rng.uniform(0.01, 0.99)])
    if op == "dropout":
        dim = _log_int(rng, 1, 512)
        n = _log_int(rng, 1, 40_000_000 // dim)
        return dict(op=op, n=n, dim=dim, dtype=dtype, p=p or 0.1, train=rng.random() < 0.7)
    dim = _log_int(rng, 1, 4096)
    n = _log_int(rng, 1, min(4_000_000, 16_000_000 // dim))
    rows = _log_int(rng, 1, min(500_000, 50_000_000 // dim))
    pad = rng.choice([-1, -1, rng.randrange(rows)])
    return dict(op=op, n=n, rows=rows, dim=dim, dtype=dtype, ids=rng.choice(["uniform", "zipf"]),
                idx=rng.choice(["int64", "int32"]), scale=rng.choice([1.0, 0.5, math.sqrt(dim)]), p=p, pad=pad)


# ------------------------------------------------------------------------------------------------- inputs
def _ids(case, gen, dev):
    n, rows = case["n"], case["rows"]
    if case["ids"] == "uniform":
        ids = torch.randint(0, rows, (n,), generator=gen, device=dev)
    elif case["ids"] == "zipf":  # P(id) proportional to log((id + 2) / (id + 1)), about 1 / rank
        u = torch.rand(n, generator=gen, device=dev, dtype=torch.float64)
        ids = (torch.exp(u * math.log(rows + 1.0)) - 1.0).long().clamp_(0, rows - 1)
    else:  # the 8 vertices around points on rays through a cube of res^3 vertices
        res = round(rows ** (1.0 / 3.0))
        pts = 192
        rays = n // (8 * pts)
        a, b = (torch.rand(rays, 1, 3, generator=gen, device=dev) for _ in range(2))
        t = torch.linspace(0, 1, pts, device=dev).view(1, pts, 1)
        cell = ((a + (b - a) * t) * (res - 1)).long().clamp_(0, res - 2).view(-1, 1, 3)
        corner = torch.tensor([[i >> 2 & 1, i >> 1 & 1, i & 1] for i in range(8)], device=dev)
        xyz = cell + corner
        ids = ((xyz[..., 0] * res + xyz[..., 1]) * res + xyz[..., 2]).reshape(-1)
    return ids.to(torch.int32 if case["idx"] == "int32" else torch.int64)


def _inputs(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32).to(dt)

    s = dict(rng=(seed * 7919 + 12345, (seed * 104729 + 17) << 3))
    if case["op"] == "dropout":
        s["x"] = normal(case["n"], case["dim"])
        if case["train"]:
            s["g"] = normal(case["n"], case["dim"])
        return s
    s["ids"] = _ids(case, gen, dev)
    s["table"] = normal(case["rows"], case["dim"])
    if case["op"] == "train":
        s["g"] = normal(case["n"], case["dim"])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    leaf = "x" if case["op"] == "dropout" else "table"
    if "g" in s:
        s[leaf].requires_grad_(True)
    if own:
        import yanerf_boot  # noqa: F401
        from yanerf_amd import ops
        s["ops"] = ops
    return s


# ------------------------------------------------------------------------------------------------- the plain form
def _mul_hi_lo(m, c):
    prod = c * m  # modulo 2^64, whose bits are the product's
    return (prod >> 32) & 0xFFFFFFFF, prod & 0xFFFFFFFF


def _keep(numel, p, rng, dev):
    """The mask of `numel` elements as a flat truth tensor."""
    seed, offset = rng
    k0, k1 = seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF
    e = torch.arange((numel + 3) // 4, device=dev, dtype=torch.int64)
    c0, c1 = e & 0xFFFFFFFF, e >> 32
    c2 = torch.full_like(e, offset & 0xFFFFFFFF)
    c3 = torch.full_like(e, (offset >> 32) & 0xFFFFFFFF)
    for _ in range(10):
        h0, l0 = _mul_hi_lo(0xD2511F53, c0)
        h1, l1 = _mul_hi_lo(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    words = torch.stack([c0, c1, c2, c3], dim=1).reshape(-1)[:numel]
    return words >= int(p * 4294967296.0 + 0.5)


def _plain(state):
    case = state["case"]
    p = case["p"]
    if case["op"] == "dropout":
        x = state["x"].detach()
        keep = _keep(x.numel(), p, state["rng"], x.device).view(x.shape)
        f = 1.0 / (1.0 - p)
        out = [torch.where(keep, x.float() * f, 0.0).to(x.dtype)]
        if case["train"]:
            out.append(torch.where(keep, state["g"].float() * f, 0.0).to(x.dtype))
        return out
    table = state["table"].detach()
    ids = state["ids"].long()
    f = case["scale"] / (1.0 - p)
    val = table[ids].float() * f
    keep = _keep(val.numel(), p, state["rng"], val.device).view(val.shape) if p > 0.0 else None
    if keep is not None:
        val = torch.where(keep, val, 0.0)
    out = [val.to(table.dtype)]
    if case["op"] == "train":
        g = state["g"]
        if keep is not None:
            g = torch.where(keep, g, 0.0)
        acc = torch.zeros(table.shape, dtype=torch.float64, device=table.device)  # a row may sum 10^5 terms and more
        acc.index_add_(0, ids, g.double())
        if case["pad"] >= 0:
            acc[case["pad"]] = 0.0
        out.append((acc * f).to(table.dtype))
    return out


# ------------------------------------------------------------------------------------------------- the kernels
def _own(state):
    case, ops = state["case"], state["ops"]
    if case["op"] == "dropout":
        y = ops.dropout(state["x"], case["p"], rng=state["rng"])
        if not case["train"]:
            return [y]
        (gx,) = torch.autograd.grad(y, state["x"], state["g"])
        return [y.detach(), gx]
    # check=False: ids that the program drew itself need no read-back of the out-of-range flag in every step
    out = ops.embedding(state["table"], state["ids"], scale=case["scale"], dropout=case["p"], rng=state["rng"],
                        padding_idx=case["pad"] if case["pad"] >= 0 else None, check=False)
    if case["op"] == "lookup":
        return [out]
    (gt,) = torch.autograd.grad(out, state["table"], state["g"])
    return [out.detach(), gt]


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------- work
def _distinct(case):
    """Expected number of different ids among n."""
    n, rows = case["n"], case["rows"]
    if case["ids"] == "uniform":
        return rows * -math.expm1(n * math.log1p(-1.0 / rows)) if rows > 1 else 1.0
    if case["ids"] == "zipf":
        i = np.arange(rows, dtype=np.float64)
        pr = np.log((i + 2.0) / (i + 1.0)) / math.log(rows + 1.0)
        return float(-np.expm1(n * np.log1p(-np.minimum(pr, 1.0 - 1e-12))).sum())
    return float(min(n, rows))


def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    n, d = case["n"], case["dim"]
    if case["op"] == "dropout":
        k = 4 if case["train"] else 2
        return {"bytes": k * n * d * es, "flops": n * d * (k // 2)}
    b = n * (4 if case["idx"] == "int32" else 8) + _distinct(case) * d * es + n * d * es
    fl = n * d
    if case["op"] == "train":
        b += n * d * es + case["rows"] * d * es
        fl += n * d + case["rows"] * d
    return {"bytes": int(b), "flops": fl}


# ------------------------------------------------------------------------------------------------- 64 bits
def _exact_keep(numel, p, rng):
    """The mask on the host, 2^15 counters at a time (uint64 products of 32-bit halves)."""
    seed, offset = rng
    m32 = np.uint64(0xFFFFFFFF)
    s32 = np.uint64(32)
    out = np.empty(((numel + 3) // 4, 4), dtype=bool)
    thr = np.uint64(min(int(p * 4294967296.0 + 0.5), 1 << 32))
    for a in range(0, out.shape[0], 1 << 15):
        i = np.arange(a, min(a + (1 << 15), out.shape[0]), dtype=np.uint64)
        ctr = [i & m32, i >> s32, np.full_like(i, offset & 0xFFFFFFFF), np.full_like(i, (offset >> 32) & 0xFFFFFFFF)]
        key = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
        for _ in range(10):
            pa, pb = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
            ctr = [(pb >> s32) ^ ctr[1] ^ np.uint64(key[0]), pb & m32, (pa >> s32) ^ ctr[3] ^ np.uint64(key[1]), pa & m32]
            key = [(key[0] + 0x9E3779B9) & 0xFFFFFFFF, (key[1] + 0xBB67AE85) & 0xFFFFFFFF]
        for w in range(4):
            out[a:a + i.size, w] = ctr[w] >= thr
    return out.reshape(-1)[:numel]


def _host64(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def exact(case, seed):
    s = _inputs(case, seed)
    p = case["p"]
    if case["op"] == "dropout":
        keep = _exact_keep(case["n"] * case["dim"], p, s["rng"]).reshape(case["n"], case["dim"])
        res = []
        for k in ("x", "g") if case["train"] else ("x",):
            v = _host64(s[k])
            v /= 1.0 - p
            v[~keep] = 0.0
            res.append(torch.from_numpy(v))
        return res
    f = case["scale"] / (1.0 - p)
    ids = s["ids"].cpu().numpy().astype(np.int64)
    val = _host64(s["table"])[ids] * f
    keep = _exact_keep(val.size, p, s["rng"]).reshape(val.shape) if p > 0.0 else None
    if keep is not None:
        val[~keep] = 0.0
    res = [torch.from_numpy(val)]
    if case["op"] == "train":
        g = _host64(s["g"])
        if keep is not None:
            g[~keep] = 0.0
        order = np.argsort(ids, kind="stable")
        srt = ids[order]
        first = np.flatnonzero(np.concatenate([[True], srt[1:] != srt[:-1]]))
        grad = np.zeros((case["rows"], case["dim"]))
        grad[srt[first]] = np.add.reduceat(g[order], first, axis=0) * f
        if case["pad"] >= 0:
            grad[case["pad"]] = 0.0
        res.append(torch.from_numpy(grad))
    return res
