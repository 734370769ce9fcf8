"""Gradients of the embedding lookup where every sum is exact: g holds small integers, so that any order of fp32 additions
gives the integer sum, and a missing or doubled term shows whatever the run's length is. What remains is the formula's one
product with f = scale / (1 - p) and one rounding, so the result has to be the float64 product's, bit for bit, halves of a
step that go to the even neighbour among them."""
import numpy as np
import pytest
import torch

import codes_reference as R
import yanerf_boot  # noqa: F401
from test_gpu_codes import BF16, DEV, F16, F32, NAME, TYPES, some_ids

pytestmark = pytest.mark.gpu


def integers(n, d, dtype, most, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-most, most + 1, (n, d), generator=g).to(dtype).to(DEV)


def expected(g, ids, v, dtype, scale, p, rng, pad=-1):
    """float64 sums and product, rounded to fp32 and to the type (both to nearest even)."""
    d = g.shape[-1]
    x, i = R.f64(g).reshape(-1, d), ids.cpu().numpy().astype(np.int64).reshape(-1)
    if p > 0.0:
        x = np.where(R.keep_mask(x.size, p, *rng).reshape(x.shape), x, 0.0)
    total, size = np.zeros((v, d)), np.zeros((v, d))
    use = (i >= 0) & (i < v) & (i != pad)
    order = np.argsort(i[use], kind="stable")
    if order.size:
        rows, xs = i[use][order], x[use][order]
        first = np.flatnonzero(np.concatenate([[True], rows[1:] != rows[:-1]]))
        total[rows[first]] = np.add.reduceat(xs, first, axis=0)
        size[rows[first]] = np.add.reduceat(np.abs(xs), first, axis=0)
    assert size.max(initial=0.0) <= 2.0 ** 24  # every partial sum, in any order, is an integer that fp32 holds
    return torch.from_numpy(total * (scale / (1.0 - p))).float().to(dtype)


def check_exact(n, v, d, *, dtype=F32, out=None, kind="uniform", idt=torch.int64, scale=1.0, p=0.0, pad=None, most=8, seed=0):
    from yanerf_amd import ops
    out = out or dtype
    ids = some_ids(n, v, kind, seed + 1, idt)
    g = integers(n, d, out, most, seed + 2)
    rng = (seed * 1000003 + 5, 1 << (seed % 50))
    table = torch.zeros(v, d, dtype=dtype, device=DEV, requires_grad=True)
    y = ops.embedding(table, ids, scale=scale, padding_idx=pad, dropout=p, out_dtype=out, rng=rng)
    (got,) = torch.autograd.grad(y, table, g)
    want = expected(g, ids, v, dtype, scale, p, rng, -1 if pad is None else pad % v)
    got = got.cpu()
    bad = got != want
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} differ, first at {bad.nonzero()[0].tolist()}: "
                           f"got {got[bad][0].item()!r}, want {want[bad][0].item()!r}")


# scale / (1 - p) = 320 / 9, 2 / 3 and 25 / 9: sums that are multiples of 9 or 3 give whole products, a half of a step of
# bf16 and fp16 among them, which a factor rounded to fp32 would push off the half
@pytest.mark.parametrize("scale,p", [(32.0, 0.1), (0.5, 0.25), (2.5, 0.1)])
@pytest.mark.parametrize("n,v,d", [(3000, 200, 20), (4096, 900, 48),   # one launch
                                   (9000, 17, 64), (9000, 32, 3),      # a table a lane
                                   (9000, 3000, 33), (16384, 700, 24),  # ranks
                                   (40000, 9000, 2), (40000, 5, 1000),  # buckets; a table a lane, wide rows
                                   (40000, 9000, 40)])                 # radix sort
@pytest.mark.parametrize("dtype", TYPES, ids=NAME.get)
def test_halves_go_to_even(n, v, d, scale, p, dtype):
    check_exact(n, v, d, dtype=dtype, scale=scale, p=p, kind="zipf", most=128, seed=n % 89)
