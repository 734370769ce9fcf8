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


# the sizes, tables, types and orders of ids of the bounded tests, whose bound a long run's missing part can stay under
@pytest.mark.parametrize("d", [1, 2, 3, 4, 5, 8, 12, 16, 31, 32, 37, 64, 100, 128, 257, 512, 1000, 1024, 2056])
@pytest.mark.parametrize("dtype", TYPES, ids=NAME.get)
def test_dims(d, dtype):
    check_exact(301, 77, d, dtype=dtype, scale=0.75, p=0.25, seed=d)
    check_exact(301, 77, d, dtype=dtype, kind="zipf", seed=d + 1)
    check_exact(5001, 77, d, dtype=dtype, kind="zipf", p=0.5, seed=d + 2)
    check_exact(17001, 77, d, dtype=dtype, kind="one", seed=d + 3)


@pytest.mark.parametrize("n", [1, 2, 3, 63, 64, 65, 255, 256, 257, 1000, 4095, 4096, 4097, 16383, 16384, 16385, 20000, 70001])
@pytest.mark.parametrize("kind", ["uniform", "zipf", "one", "sorted", "ends"])
def test_counts(n, kind):
    check_exact(n, 300, 6, kind=kind, seed=n % 97)
    check_exact(n, 300, 40, dtype=BF16, kind=kind, p=0.1, seed=n % 97)
    check_exact(n, 300, 3, dtype=F16, kind=kind, p=0.5, seed=n % 97, most=1)
    check_exact(n, 30, 7, kind=kind, seed=n % 97)


@pytest.mark.parametrize("v", [1, 2, 3, 17, 32, 33, 100, 127, 128, 255, 256, 257, 511, 512, 513, 1024, 32767, 32768, 65535, 65536, 300000])
@pytest.mark.parametrize("n", [1, 700, 9001, 40000])
def test_tables(v, n):
    check_exact(n, v, 4, seed=v % 89)
    check_exact(n, v, 3, kind="zipf", idt=torch.int32, pad=v // 2, seed=v % 89)
    check_exact(n, v, 24, dtype=F16, kind="uniform", p=0.5, pad=-1, seed=v % 89, most=2)


def test_ranks_of_wide_keys():
    for v in ((1 << 18) - 1, 1 << 18, 5000000):
        for kind in ("uniform", "zipf", "one"):
            check_exact(16384, v, 5, kind=kind, seed=v % 13)
    for v in (40, 1000, 60000):
        check_exact(16384, v, 20, kind="one", seed=v % 13)
        check_exact(16383, v, 20, kind="ends", p=0.1, seed=v % 13)


def test_tables_around_the_path_limits():
    for v in (16383, 16384, 16385):
        check_exact(3000, v, 512, kind="zipf", seed=v % 7)
        check_exact(3000, v, 1024, dtype=BF16, kind="one", p=0.1, seed=v % 7)
    for n in (16384, 16385):
        for d in (4, 5):
            for kind in ("uniform", "one"):
                check_exact(n, 900, d, kind=kind, seed=d)


def test_long_runs():
    """Runs over many workgroups, tiles and joins: all ids in one row, nearly all, or dealt out."""
    for kind in ("one", "ends", "zipf", "uniform"):
        check_exact(500000, 100000, 2, kind=kind, seed=7)
        check_exact(500000, 100000, 2, kind=kind, p=0.3, dtype=BF16, seed=8)
        check_exact(600000, 17, 16, kind=kind, idt=torch.int32, seed=6)
        check_exact(300001, 5000, 40, kind=kind, seed=9)
        check_exact(300001, 5000, 5, kind=kind, dtype=BF16, out=F32, p=0.5, seed=10)
        check_exact(30000, 50000, 256, dtype=BF16, kind=kind, seed=4)
        check_exact(5000, 20000, 1024, dtype=BF16, kind=kind, scale=32.0, p=0.1, pad=0, seed=3)


@pytest.mark.parametrize("d", [1, 2, 3, 4, 5, 6, 7, 8])
@pytest.mark.parametrize("dtype", TYPES, ids=NAME.get)
def test_short_rows_and_long_lists(d, dtype):
    check_exact(20000, 3000, d, dtype=dtype, seed=d)
    check_exact(70001, 200000, d, dtype=dtype, kind="zipf", p=0.3, pad=1, idt=torch.int32, seed=d + 1)
    check_exact(50000, 9000, d, dtype=dtype, kind="one", p=0.3, seed=d + 2, most=2)
    check_exact(50000, 7, d, dtype=dtype, kind="sorted", seed=d + 3)
    check_exact(100001, 2050, d, dtype=dtype, kind="ends", seed=d + 4, most=2)


@pytest.mark.parametrize("out", TYPES, ids=NAME.get)
@pytest.mark.parametrize("dtype", TYPES, ids=NAME.get)
def test_type_pairs(dtype, out):
    for d in (2, 7, 48, 320):
        for n in (500, 6000, 18000):
            check_exact(n, 600, d, dtype=dtype, out=out, scale=1.5, p=0.2, seed=d)
            check_exact(n, 600, d, dtype=dtype, out=out, kind="one", scale=0.5, p=0.5, seed=d, most=2)


def test_unaligned_gradients():
    """Gradients of the output that start off a 16-byte boundary."""
    from yanerf_amd import ops
    for dtype in TYPES:
        for shift in (1, 2, 3, 5):
            for n in (200, 6000, 20000):
                ids, rng = some_ids(n, 50, "zipf", seed=shift), (9, shift)
                table = torch.zeros(50, 64, dtype=dtype, device=DEV, requires_grad=True)
                y = ops.embedding(table, ids, dropout=0.4, rng=rng)
                g = integers(n * 64 + 8, 1, dtype, 4, shift).view(-1)[shift:shift + n * 64].view(n, 64)
                (got,) = torch.autograd.grad(y, table, g)
                assert torch.equal(got.cpu(), expected(g, ids, 50, dtype, 1.0, 0.4, rng)), (dtype, shift, n)
