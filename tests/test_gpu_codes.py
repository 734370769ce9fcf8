"""Learned codes on the GPU: embedding lookup, its gradient by sorted ids and counter-based dropout against their
definitions in float64 (codes_reference), at the sizes, types, strides and ids where they can go wrong; and CodeTable in the
pipeline."""
import numpy as np
import pytest
import torch

import codes_reference as R
import yanerf_boot  # noqa: F401

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]
NAME = {F32: "fp32", BF16: "bf16", F16: "fp16"}


@pytest.fixture(scope="module")
def ops():
    from yanerf_amd import ops as o
    return o


def rand(*shape, dtype=F32, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=F32).to(dtype).to(DEV)


def some_ids(n, v, kind="uniform", seed=0, dtype=torch.int64):
    g = torch.Generator().manual_seed(seed)
    if kind == "uniform":
        i = torch.randint(0, v, (n,), generator=g)
    elif kind == "zipf":
        i = (torch.exp(torch.rand(n, generator=g, dtype=torch.float64) * np.log(v + 1.0)) - 1).long().clamp(0, v - 1)
    elif kind == "one":
        i = torch.full((n,), v - 1)
    elif kind == "sorted":
        i = torch.arange(n) * v // max(n, 1)
    else:  # a run of the first row, then one id of the last
        i = torch.zeros(n, dtype=torch.int64)
        i[-1:] = v - 1
    return i.to(dtype).to(DEV)


def check_train(ops, n, v, d, *, dtype=F32, out=None, kind="uniform", idt=torch.int64, scale=1.0, p=0.0, pad=None, seed=0):
    out = out or dtype
    table = rand(v, d, dtype=dtype, seed=seed).requires_grad_()
    ids = some_ids(n, v, kind, seed + 1, idt)
    g = rand(n, d, dtype=out, seed=seed + 2)
    rng = (seed * 1000003 + 5, 1 << (seed % 50))
    y = ops.embedding(table, ids, scale=scale, padding_idx=pad, dropout=p, out_dtype=out, rng=rng)
    assert y.shape == (n, d) and y.dtype == out
    R.assert_within(y, *R.lookup(table, ids, out, scale, p, rng), what="lookup")
    (gt,) = torch.autograd.grad(y, table, g)
    assert gt.dtype == dtype and gt.shape == (v, d)
    want = R.table_gradient(g, ids, v, dtype, scale, p, rng, -1 if pad is None else pad % v)
    R.assert_within(gt, *want, what="gradient")
    y2 = ops.embedding(table, ids, scale=scale, padding_idx=pad, dropout=p, out_dtype=out, rng=rng)
    (gt2,) = torch.autograd.grad(y2, table, g)
    assert torch.equal(y2, y) and torch.equal(gt2, gt)  # the same bits on every run
    return y, gt


# ------------------------------------------------------------------------------------------- lookup and gradient
@pytest.mark.parametrize("d", [1, 2, 3, 4, 5, 8, 12, 16, 31, 32, 37, 64, 100, 128, 257, 512, 1000, 1024, 2056])
@pytest.mark.parametrize("dtype", TYPES, ids=NAME.get)
def test_dims(ops, d, dtype):
    check_train(ops, 301, 77, d, dtype=dtype, scale=0.75, p=0.25, seed=d)
    check_train(ops, 301, 77, d, dtype=dtype, kind="zipf", seed=d + 1)


@pytest.mark.parametrize("n", [1, 2, 3, 63, 64, 65, 255, 256, 257, 1000, 4095, 4096, 4097, 16383, 16384, 16385, 20000, 70001])
@pytest.mark.parametrize("kind", ["uniform", "zipf", "one", "sorted", "ends"])
def test_counts(ops, n, kind):
    check_train(ops, n, 300, 6, kind=kind, seed=n % 97)
    check_train(ops, n, 300, 40, dtype=BF16, kind=kind, p=0.1, seed=n % 97)


@pytest.mark.parametrize("v", [1, 2, 3, 17, 32, 33, 100, 127, 128, 255, 256, 257, 511, 512, 513, 1024, 32767, 32768, 65535, 65536, 300000])
@pytest.mark.parametrize("n", [1, 700, 9001, 40000])
def test_tables(ops, v, n):
    check_train(ops, n, v, 4, seed=v % 89)
    check_train(ops, n, v, 3, kind="zipf", idt=torch.int32, pad=v // 2, seed=v % 89)
    check_train(ops, n, v, 24, dtype=F16, kind="uniform", p=0.5, pad=-1, seed=v % 89)


def test_ranks_of_wide_keys(ops):
    """Up to 16384 ids are ranked in LDS: ids beyond 2^18 need 64-bit pairs, and all ids in one row fill one bin."""
    for v in ((1 << 18) - 1, 1 << 18, 5000000):
        for kind in ("uniform", "zipf", "one"):
            check_train(ops, 16384, v, 5, kind=kind, seed=v % 13)
    for v in (40, 1000, 60000):
        check_train(ops, 16384, v, 20, kind="one", seed=v % 13)
        check_train(ops, 16383, v, 20, kind="ends", p=0.1, seed=v % 13)


def test_tables_around_the_path_limits(ops):
    """Gradients around 32 MB, where short id lists leave the one-launch path, and row sizes around 16 bytes."""
    for v in (16383, 16384, 16385):
        check_train(ops, 3000, v, 512, kind="zipf", seed=v % 7)
        check_train(ops, 3000, v, 1024, dtype=BF16, kind="uniform", p=0.1, seed=v % 7)
    for n in (16384, 16385):
        for d in (4, 5):
            check_train(ops, n, 900, d, seed=d)


def test_wide_rows_and_many_ids(ops):
    check_train(ops, 5000, 20000, 1024, dtype=BF16, kind="zipf", scale=32.0, p=0.1, pad=0, seed=3)
    check_train(ops, 30000, 50000, 256, dtype=BF16, kind="zipf", seed=4)
    check_train(ops, 200000, 40000, 8, kind="uniform", seed=5)
    check_train(ops, 600000, 17, 16, dtype=F32, kind="uniform", idt=torch.int32, seed=6)
    check_train(ops, 500000, 100000, 2, kind="one", seed=7)
    check_train(ops, 500000, 100000, 2, kind="zipf", p=0.3, seed=8)


@pytest.mark.parametrize("d", [1, 2, 3, 4, 5, 6, 7, 8])
@pytest.mark.parametrize("dtype", TYPES, ids=NAME.get)
def test_short_rows_and_long_lists(ops, d, dtype):
    """Rows of up to 16 bytes by more than 16384 ids: buckets of one tile and of many, empty ones, one that holds all."""
    check_train(ops, 20000, 3000, d, dtype=dtype, seed=d)
    check_train(ops, 70001, 200000, d, dtype=dtype, kind="zipf", p=0.3, pad=1, idt=torch.int32, seed=d + 1)
    check_train(ops, 50000, 9000, d, dtype=dtype, kind="one", p=0.3, seed=d + 2)
    check_train(ops, 50000, 7, d, dtype=dtype, kind="sorted", seed=d + 3)
    check_train(ops, 100001, 2050, d, dtype=dtype, kind="ends", seed=d + 4)


@pytest.mark.parametrize("out", TYPES, ids=NAME.get)
@pytest.mark.parametrize("dtype", TYPES, ids=NAME.get)
def test_type_pairs(ops, dtype, out):
    for d in (2, 7, 48, 320):
        check_train(ops, 500, 60, d, dtype=dtype, out=out, scale=1.5, p=0.2, seed=d)
        check_train(ops, 6000, 600, d, dtype=dtype, out=out, scale=1.5, p=0.2, seed=d)
        check_train(ops, 18000, 600, d, dtype=dtype, out=out, scale=1.5, p=0.2, seed=d)


@pytest.mark.parametrize("p", [0.0, 1e-9, 1e-4, 0.5, 0.999, 1.0 - 1e-12, 1.0])
def test_probabilities(ops, p):
    check_train(ops, 400, 50, 20, p=p, seed=11)


def test_empty_and_degenerate(ops):
    table = rand(5, 4).requires_grad_()
    y = ops.embedding(table, torch.zeros(0, dtype=torch.int64, device=DEV), dropout=0.5)
    assert y.shape == (0, 4)
    (g,) = torch.autograd.grad(y, table, torch.zeros_like(y))
    assert not g.any()
    y = ops.embedding(table, torch.zeros(2, 0, 3, dtype=torch.int64, device=DEV))
    assert y.shape == (2, 0, 3, 4)
    y = ops.embedding(table, torch.tensor(3, device=DEV))
    assert y.shape == (4,) and torch.equal(y, table[3])
    thin = torch.zeros(5, 0, device=DEV, requires_grad=True)
    y = ops.embedding(thin, torch.tensor([1, 2], device=DEV))
    assert y.shape == (2, 0) and torch.autograd.grad(y.sum(), thin)[0].shape == (5, 0)
    with pytest.raises(IndexError):
        ops.embedding(torch.zeros(0, 4, device=DEV), torch.tensor([0], device=DEV))
    assert ops.embedding(torch.zeros(0, 4, device=DEV), torch.zeros(0, dtype=torch.int64, device=DEV)).shape == (0, 4)
    assert ops.dropout(torch.zeros(0, 3, device=DEV), 0.5).shape == (0, 3)


@pytest.mark.parametrize("dtype", TYPES, ids=NAME.get)
def test_strides_and_shapes(ops, dtype):
    big = rand(40, 100, dtype=dtype)
    ids = some_ids(60, 40).view(3, 20)
    for table in (big[:, :64], big[:, 1:33], big[:, 3:40], big[::2][:, 8:72], big[:, ::2], big.t()[:40, :36],
                  big[:1].expand(40, 100)):
        leaf = table.detach().requires_grad_()
        v, d = leaf.shape
        i = ids % v
        y = ops.embedding(leaf, i, scale=2.0, dropout=0.3, rng=(3, 4))
        R.assert_within(y, *R.lookup(leaf, i, dtype, 2.0, 0.3, (3, 4)))
        g = rand(3, 20, d, dtype=dtype, seed=2)
        gn = rand(d, 20, 3, dtype=dtype, seed=3).permute(2, 1, 0)  # not contiguous
        ge = rand(d, dtype=dtype, seed=4).expand(3, 20, d)         # broadcast
        for gg in (g, gn, ge):
            (gt,) = torch.autograd.grad(y, leaf, gg, retain_graph=True)
            R.assert_within(gt, *R.table_gradient(gg, i, v, dtype, 2.0, 0.3, (3, 4)))
    it = some_ids(120, 40).view(20, 6).t()[:, ::2]  # strided ids
    y = ops.embedding(big, it)
    assert torch.equal(y, big[it])


def test_unaligned_storage(ops):
    """Tables, outputs' gradients and dropout inputs that start off a 16-byte boundary."""
    for dtype in TYPES:
        for shift in (1, 2, 3, 5):
            table = rand(50 * 64 + 8, dtype=dtype)[shift:shift + 50 * 64].view(50, 64).detach().requires_grad_()
            ids = some_ids(200, 50, seed=shift)
            y = ops.embedding(table, ids, dropout=0.4, rng=(9, shift))
            R.assert_within(y, *R.lookup(table, ids, dtype, 1.0, 0.4, (9, shift)))
            g = rand(200 * 64 + 8, dtype=dtype, seed=shift)[shift:shift + 200 * 64].view(200, 64)
            (gt,) = torch.autograd.grad(y, table, g)
            R.assert_within(gt, *R.table_gradient(g, ids, 50, dtype, 1.0, 0.4, (9, shift)))
            i32 = some_ids(201, 50, seed=shift, dtype=torch.int32)[1:]
            assert torch.equal(ops.embedding(table, i32), table[i32.long()])
            x = rand(5000, dtype=dtype)[shift:]
            R.assert_within(ops.dropout(x, 0.4, rng=(9, shift)), *R.dropout(x, 0.4, (9, shift)))


def test_ids_outside_the_table(ops):
    table = rand(10, 16).requires_grad_()
    for bad in (-1, 10, 2 ** 40, -2 ** 63, 2 ** 63 - 1):
        ids = torch.tensor([3, bad, 3, 9], device=DEV)
        with pytest.raises(IndexError):
            ops.embedding(table, ids)
        y = ops.embedding(table, ids, check=False)
        assert not y[1].any() and torch.equal(y[0], table[3]) and torch.equal(y[3], table[9])
        (gt,) = torch.autograd.grad(y, table, torch.ones_like(y))
        assert gt[3].eq(2).all() and gt[9].eq(1).all() and gt.sum() == 3 * 16
        with pytest.raises(IndexError):
            ops.check_embedding_ids(DEV)
        ops.check_embedding_ids("cuda")  # reported once
    for n in (5000, 40000):
        ids = some_ids(n, 10)
        ids[::7] = 10
        ids[1::7] = -5
        y = ops.embedding(table, ids, check=False)
        g = rand(n, 16)
        (gt,) = torch.autograd.grad(y, table, g)
        R.assert_within(y, *R.lookup(table, ids, F32))
        R.assert_within(gt, *R.table_gradient(g, ids, 10, F32))
    with pytest.raises(IndexError):
        ops.check_embedding_ids(DEV)


def test_refusals(ops):
    t, i = rand(6, 4), some_ids(3, 6)
    for call, exc in [(lambda: ops.embedding(t[0], i), ValueError), (lambda: ops.embedding(t.double(), i), TypeError),
                      (lambda: ops.embedding(t, i.short()), TypeError), (lambda: ops.embedding(t, i.float()), TypeError),
                      (lambda: ops.embedding(t, i, out_dtype=torch.float64), TypeError),
                      (lambda: ops.embedding(t, i, padding_idx=6), ValueError),
                      (lambda: ops.embedding(t, i, padding_idx=-7), ValueError),
                      (lambda: ops.embedding(t, i, scale=float("nan")), ValueError),
                      (lambda: ops.embedding(t, i, dropout=-0.1), ValueError),
                      (lambda: ops.embedding(t, i.cpu()), RuntimeError),
                      (lambda: ops.embedding(t, i, dropout=0.5, rng_base=t), ValueError),
                      (lambda: ops.dropout(t, 2.0), ValueError), (lambda: ops.dropout(i, 0.5), TypeError),
                      (lambda: ops.dropout(t, 0.5, rng_base=torch.zeros(2, dtype=torch.int64, device=DEV)), ValueError)]:
        with pytest.raises(exc):
            call()


@pytest.mark.parametrize("n", [50, 30000])
def test_values_that_are_not_numbers(ops, n):
    """Infinities and NaN reach the rows they belong to and no other: dropped elements are 0 whatever they held, and the
    padding row's gradient stays 0."""
    v, d, p, rng = 40, 12, 0.5, (21, 22)
    table = rand(v, d)
    table[5] = float("nan")
    table[6] = float("inf")
    table.requires_grad_()
    ids = some_ids(n, v)
    y = ops.embedding(table, ids, dropout=p, rng=rng, padding_idx=8)
    keep = torch.from_numpy(R.keep_mask(n * d, p, *rng).reshape(n, d)).to(DEV)
    assert (y[~keep] == 0).all()
    assert torch.equal(torch.isnan(y), keep & (ids == 5)[:, None]) and torch.equal(torch.isinf(y), keep & (ids == 6)[:, None])
    g = rand(n, d)
    g[~keep] = float("nan")
    g[ids == 8] = float("inf")
    one = int((ids == 9).nonzero()[0])
    g[one] = float("inf")
    (gt,) = torch.autograd.grad(y, table, g)
    assert not gt[8].any()
    bad = ~torch.isfinite(gt)
    assert torch.equal(bad.any(1).nonzero().flatten(), torch.tensor([9], device=DEV))
    assert torch.equal(bad[9], keep[one])


def test_gradient_against_differences(ops):
    """The lookup is linear in the table, so a central difference of a fixed linear functional of it is its gradient up to
    fp32 rounding of the two lookups (2^-22 of sums of 30 products of size about 1)."""
    table, ids, w = rand(6, 5).requires_grad_(), some_ids(30, 6), rand(30, 5, seed=3)
    f = lambda t: (ops.embedding(t, ids, scale=1.3, dropout=0.2, rng=(1, 2)).double() * w.double()).sum()
    (gt,) = torch.autograd.grad(f(table), table)
    with torch.no_grad():
        for v in range(6):
            for d in range(5):
                e = torch.zeros_like(table)
                e[v, d] = 0.5
                diff = (f(table + e) - f(table - e)).item()
                assert abs(diff - gt[v, d].item()) < 30 * 8 * 2.0 ** -22


def test_double_backward_is_refused(ops):
    x, t, i = rand(8).requires_grad_(), rand(5, 8).requires_grad_(), some_ids(8, 5)
    for y, leaf in ((ops.dropout(x, 0.5), x), (ops.embedding(t, i), t)):
        g = torch.randn_like(y, requires_grad=True)
        with pytest.raises(RuntimeError, match="create_graph"):
            torch.autograd.grad(y, leaf, g, create_graph=True)
        (once,) = torch.autograd.grad(y, leaf, g.detach(), create_graph=True)  # nothing to differentiate again
        assert not once.requires_grad


def test_graph_is_freed_and_versions_are_checked(ops):
    """A second backward through a freed graph and ids changed in place between forward and backward are errors, as for any
    torch operation; retain_graph allows the first."""
    t, i = rand(5, 8).requires_grad_(), some_ids(8, 5)
    y = ops.embedding(t, i)
    y.sum().backward(retain_graph=True)
    first = t.grad.clone()
    y.sum().backward()
    assert torch.equal(t.grad, 2 * first)
    with pytest.raises(RuntimeError):
        y.sum().backward()
    y = ops.embedding(t, i)
    i.fill_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()
    with torch.no_grad():
        assert not ops.embedding(t, i).requires_grad and not ops.dropout(t, 0.5).requires_grad
    z = ops.dropout(ops.embedding(t, i), 0.0)
    z.sum().backward()
    assert "Yanerf" in type(z.grad_fn).__name__ or "Yanerf" in z.grad_fn.name()


def test_threads(ops):
    """Lookups and backwards from several Python threads at once."""
    import threading
    t, i, g = rand(100, 16).requires_grad_(), some_ids(6000, 100), rand(6000, 16)
    want = torch.autograd.grad(ops.embedding(t, i, dropout=0.1, rng=(1, 2)), t, g)[0]
    out = [None] * 4

    def work(k):
        for _ in range(20):
            out[k] = torch.autograd.grad(ops.embedding(t, i, dropout=0.1, rng=(1, 2), check=False), t, g)[0]
        torch.cuda.synchronize()

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for x in threads:
        x.start()
    for x in threads:
        x.join()
    for o in out:
        assert torch.equal(o, want)


@pytest.mark.parametrize("small_rows", [11, 40])
def test_past_32_bits(ops, small_rows):
    """A table and an output of more than 2^32 elements: rows behind that line are read, written and (the mask's counter)
    drawn at their own place."""
    v, d = 70000, 65536
    table = torch.empty(v, d, dtype=BF16, device=DEV)
    table[-3:] = rand(3, d, dtype=BF16)
    table[:2] = rand(2, d, dtype=BF16, seed=1)
    ids = torch.tensor([v - 1, 0, v - 3, v - 2, 1], device=DEV)
    assert torch.equal(ops.embedding(table, ids), table[ids])
    del table
    small = rand(small_rows, d, dtype=BF16)
    ids = some_ids(v, small_rows)
    y = ops.embedding(small, ids, dropout=0.5, rng=(5, 6), scale=0.5)
    for n in (0, 65535, 65536, v - 1):
        keep = R.philox_words(n * d // 4, d // 4, 5, 6) >= np.uint64(1 << 31)
        want = torch.where(torch.from_numpy(keep).to(DEV), small[ids[n]], torch.zeros((), dtype=BF16, device=DEV))
        assert torch.equal(y[n], want), n
    x = y.view(-1)
    z = ops.dropout(x, 0.5, rng=(7, 8))
    for n in (0, 65536, v - 1):
        keep = R.philox_words(n * d // 4, d // 4, 7, 8) >= np.uint64(1 << 31)
        want = torch.where(torch.from_numpy(keep).to(DEV), 2 * y[n], torch.zeros((), dtype=BF16, device=DEV))
        assert torch.equal(z[n * d:(n + 1) * d], want), n
    del z
    leaf = small.clone().requires_grad_()
    out = ops.embedding(leaf, ids)
    (gt,) = torch.autograd.grad(out, leaf, y)
    want = torch.zeros(small_rows, d, dtype=torch.float64, device=DEV)
    size = torch.zeros(small_rows, d, dtype=torch.float64, device=DEV)
    for k in range(small_rows):
        sel = (ids == k).nonzero().flatten()
        for part in sel.split(1024):
            want[k] += y[part].double().sum(0)
            size[k] += y[part].double().abs().sum(0)
    bound = 1.01 * (ids.bincount(minlength=small_rows)[:, None].double() * 2.0 ** -24) * size
    assert ((gt.double() - want).abs() <= bound + (want.abs() + bound) * (2.0 ** -8 + 2.0 ** -22)).all()


# ------------------------------------------------------------------------------------------- dropout
@pytest.mark.parametrize("dtype", TYPES, ids=NAME.get)
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 7, 8, 9, 255, 1023, 1024, 1025, 4099, 100003])
def test_dropout(ops, n, dtype):
    x = rand(n, dtype=dtype, seed=n).requires_grad_()
    for p, rng in ((0.1, (n, 5)), (0.5, (2 ** 64 - 1, 2 ** 64 - 1)), (0.0, (1, 1)), (1.0, (1, 1))):
        y = ops.dropout(x, p, rng=rng)
        R.assert_within(y, *R.dropout(x, p, rng))
        g = rand(n, dtype=dtype, seed=n + 1)
        (gx,) = torch.autograd.grad(y, x, g)
        R.assert_within(gx, *R.dropout(g, p, rng))


def test_dropout_shapes_and_stream(ops):
    x = rand(6, 5, 9).permute(2, 0, 1)  # not contiguous: the mask follows the logical order
    R.assert_within(ops.dropout(x, 0.3, rng=(1, 2)), *R.dropout(x, 0.3, (1, 2)))
    xe = rand(9).expand(6, 9)
    R.assert_within(ops.dropout(xe, 0.3, rng=(1, 2)), *R.dropout(xe, 0.3, (1, 2)))
    x = rand(5000)
    torch.manual_seed(123)
    a, b = ops.dropout(x, 0.5), ops.dropout(x, 0.5)
    torch.manual_seed(124)
    torch.randn(1)
    c = ops.dropout(x, 0.5)
    ops.RNG.set_state((None, 0))
    torch.manual_seed(123)
    a2 = ops.dropout(x, 0.5)
    assert torch.equal(a, a2) and not torch.equal(a, b) and not torch.equal(a, c)
    # two draws of the module stream are independent: the share of elements that both keep
    both = ((a != 0) & (b != 0)).float().mean().item()
    assert abs(both - 0.25) < 5 * (0.1875 / 5000) ** 0.5
    x = rand(16).requires_grad_()
    y = ops.dropout(ops.dropout(x, 0.5, rng=(1, 1)), 0.5, rng=(1, 2))
    y.sum().backward()
    assert torch.equal(x.grad != 0, y != 0)


def test_dropped_values_are_zero(ops):
    for dtype in TYPES:
        x = torch.full((4097,), float("nan"), device=DEV, dtype=dtype)
        x[::2] = float("inf")
        y = ops.dropout(x, 0.5, rng=(3, 3))
        keep = torch.from_numpy(R.keep_mask(4097, 0.5, 3, 3)).to(DEV)
        assert (y[~keep] == 0).all() and not torch.isfinite(y[keep]).any()
        assert (ops.dropout(x, 1.0) == 0).all()


def test_embedding_dropout_is_dropout_of_embedding(ops):
    """The fused mask is the mask of dropout() over the result: equal where no rounding differs (p = 0.5, fp32)."""
    for n, d in ((33, 7), (64, 48), (1000, 5)):
        t, i = rand(20, d), some_ids(n, 20)
        assert torch.equal(ops.embedding(t, i, dropout=0.5, rng=(4, 9)), ops.dropout(ops.embedding(t, i), 0.5, rng=(4, 9)))


# ------------------------------------------------------------------------------------------- streams and graphs
def test_other_streams(ops):
    table, ids, g = rand(100, 48).requires_grad_(), some_ids(20000, 100), rand(20000, 48)
    y0 = ops.embedding(table, ids, dropout=0.2, rng=(1, 2))
    (g0,) = torch.autograd.grad(y0, table, g)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    res = []
    for s in streams:
        with torch.cuda.stream(s):
            y = ops.embedding(table, ids, dropout=0.2, rng=(1, 2), check=False)
            res.append((y, torch.autograd.grad(y, table, g)[0]))
    torch.cuda.synchronize()
    for y, gt in res:
        assert torch.equal(y, y0) and torch.equal(gt, g0)


@pytest.mark.parametrize("n,v,d,dtype", [(1, 100, 32, F32), (4096, 100, 48, F32), (20000, 3000, 8, F32),
                                         (40000, 17, 64, BF16), (3000, 5000, 1024, BF16)])
def test_graph_replays(ops, n, v, d, dtype):
    """Lookup, dropout and both backwards captured once and replayed with new ids, values and masks (rng_base advanced
    between replays, as yanerf_step_advance does), with eager work between: every replay equals the eager result."""
    table, ids = rand(v, d, dtype=dtype).requires_grad_(), some_ids(n, v)
    g, base = rand(n, d, dtype=dtype), torch.zeros(1, dtype=torch.int64, device=DEV)

    def step():
        y = ops.embedding(table, ids, scale=0.5, dropout=0.25, rng=(7, 100), rng_base=base, check=False)
        z = ops.dropout(y, 0.5, rng=(7, 1 << 40), rng_base=base)
        (gt,) = torch.autograd.grad(z, table, g)
        return y.detach(), z.detach(), gt

    def eager(b):
        y = ops.embedding(table, ids, scale=0.5, dropout=0.25, rng=(7, 100 + b))
        z = ops.dropout(y, 0.5, rng=(7, (1 << 40) + b))
        (gt,) = torch.autograd.grad(z, table, g)
        return y.detach(), z.detach(), gt

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for r in range(4):
        with torch.no_grad():
            ids.copy_(some_ids(n, v, ["uniform", "zipf", "one", "ends"][r], seed=r))
            table.copy_(rand(v, d, dtype=dtype, seed=r))
            g.copy_(rand(n, d, dtype=dtype, seed=10 + r))
            base.fill_(1000 * r)
        want = eager(1000 * r)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b), r
    del graph


def test_two_graphs_do_not_share_workspaces(ops):
    """Two captured gradients replayed side by side on two streams."""
    s = [(rand(50, 16, seed=k).requires_grad_(), some_ids(20000, 50, seed=k), rand(20000, 16, seed=k)) for k in range(2)]
    f = lambda t, i, g: torch.autograd.grad(ops.embedding(t, i, dropout=0.1, rng=(1, 1), check=False), t, g)[0]
    want = [f(*a) for a in s]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for a in s:
            f(*a)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for a in s:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(f(*a))
        graphs.append(gr)
    st = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for gr, x in zip(graphs, st):
            with torch.cuda.stream(x):
                gr.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


def test_backward_mask_survives_an_advanced_base(ops):
    """The step state moves on between a forward and its backward: the backward still draws the forward's mask."""
    x, base = rand(3000).requires_grad_(), torch.full((1,), 77, dtype=torch.int64, device=DEV)
    y = ops.dropout(x, 0.5, rng=(1, 2), rng_base=base)
    table, ids = rand(30, 8).requires_grad_(), some_ids(500, 30)
    e = ops.embedding(table, ids, dropout=0.5, rng=(1, 3), rng_base=base)
    base.fill_(12345)
    g = rand(3000, seed=1)
    R.assert_within(torch.autograd.grad(y, x, g)[0], *R.dropout(g, 0.5, (1, 79)))
    ge = rand(500, 8, seed=2)
    R.assert_within(torch.autograd.grad(e, table, ge)[0], *R.table_gradient(ge, ids, 30, F32, 1.0, 0.5, (1, 80)))


# ------------------------------------------------------------------------------------------- in the pipeline
def conditional_pipeline(extractor):
    from yanerf_amd.pipelines.builder import PIPELINES
    return PIPELINES.build(dict(
        type="NeRFPipeline",
        model=dict(type="NeRFMLP", n_layers=8, input_skips=[5], n_harmonic_functions_xyz=10,
                   harmonic_functions_xyz_append_intput=True, n_hidden_neurons_xyz=256, n_harmonic_functions_dir=4,
                   harmonic_functions_dir_append_intput=True, n_hidden_neurons_dir=128, latent_dim=4, input_xyz=True,
                   color_dim=3),
        ray_sampler=dict(type="RaySampler", image_width=10, image_height=6, n_rays_per_image_sampled_from_mask=4,
                         min_depth=0.5, max_depth=1.0, scene_extent=0.0, n_pts_per_ray_training=5,
                         n_pts_per_ray_evaluation=5, stratified_point_sampling_training=True,
                         stratified_point_sampling_evaluation=False),
        renderer=dict(type="MultipassEmissionAbsorpsionRenderer", n_pts_per_ray_fine_training=5,
                      n_pts_per_ray_fine_evaluation=5, append_coarse_samples_to_fine=True, density_noise_std_train=0.0,
                      bg_color=[0.0, 0.0, 0.0], blend_output=True),
        chunk_size_grid=30, num_passes=2, loss_weights={"loss_rgb_mse": 1.0, "loss_prev_stage_rgb_mse": 1.0},
        output_rasterized_mc=False, feature_extractor=extractor)).to(DEV)


def test_code_table_in_the_pipeline(ops):
    """The conditional pipeline with learned codes: its render equals the render of the same codes passed through an
    IdentityMapper bit for bit, and a training step's code gradient is the table's gradient formula applied to the gradient
    of the codes."""
    from yanerf_amd.pipelines.utils import EvaluationMode as EM
    torch.manual_seed(0)
    learned = conditional_pipeline(dict(type="CodeTable", num_codes=7, latent_dim=4, scale=2.0, dropout=0.25, init_std=1.0))
    plain = conditional_pipeline(dict(type="IdentityMapper"))
    plain.load_state_dict(learned.state_dict(), strict=False)
    ce = learned.feature_extractors[0]
    B = 3
    poses, focal = torch.randn(B, 3, 4, device=DEV), torch.ones(B, device=DEV) * 500
    image = torch.rand(B, 6, 10, 3, device=DEV)
    ids = torch.tensor([5, 2, 5])

    learned.eval()
    with torch.no_grad():
        a = learned(poses=poses, focal_lengths=focal, image_rgb=image, evaluation_mode=EM.EVALUATION, image_ids=ids)
        b = plain(poses=poses, focal_lengths=focal, image_rgb=image, evaluation_mode=EM.EVALUATION,
                  global_codes=2.0 * ce.table[ids])
    assert torch.equal(a["rendered_images"], b["rendered_images"])

    learned.train()
    ops.RNG.set_state((torch.initial_seed(), 1 << 20))
    preds = learned(poses=poses, focal_lengths=focal, image_rgb=image, evaluation_mode=EM.TRAINING, image_ids=ids)
    preds["objective"].mean().backward()
    grad = ce.table.grad
    assert grad[[0, 1, 3, 4, 6]].abs().sum() == 0 and torch.isfinite(grad).all() and grad[[2, 5]].abs().sum() > 0
    # the same draws with the codes passed in: raygen takes the first draws, the lookup the next
    ops.RNG.set_state((torch.initial_seed(), 1 << 20))
    mask = R.keep_mask(B * 4, 0.25, torch.initial_seed(), (1 << 20) + B * 4 * 5)
    codes = (2.0 / 0.75 * ce.table.detach()[ids] * torch.from_numpy(mask.reshape(B, 4)).to(DEV)).requires_grad_()
    ops_next = ops.RNG.next

    def skip_lookup(n=1, state={"calls": 0}):
        state["calls"] += 1
        r = ops_next(n)
        if state["calls"] == 1:
            ops_next(B * 4)  # the lookup's draw
        return r

    ops.RNG.next = skip_lookup
    try:
        p2 = plain(poses=poses, focal_lengths=focal, image_rgb=image, evaluation_mode=EM.TRAINING, global_codes=codes)
    finally:
        del ops.RNG.next
    assert abs(p2["objective"].mean().item() - preds["objective"].mean().item()) <= 1e-5 * abs(p2["objective"].mean().item())
    p2["objective"].mean().backward()
    gc = codes.grad.double() * torch.from_numpy(mask.reshape(B, 4)).to(DEV) * (2.0 / 0.75)
    want = torch.zeros(7, 4, dtype=torch.float64, device=DEV).index_add_(0, ids.to(DEV), gc)
    assert (grad.double() - want).abs().max() <= 1e-4 * want.abs().max()


def test_code_table_learns(ops):
    """Codes and MLPs train together through Adam for a few steps; only the rows that were looked up move, and the padding
    row stays."""
    from yanerf_amd.pipelines.utils import EvaluationMode as EM
    torch.manual_seed(1)
    pipe = conditional_pipeline(dict(type="CodeTable", num_codes=6, latent_dim=4, dropout=0.1, padding_idx=3))
    start = pipe.feature_extractors[0].table.detach().clone()
    opt = torch.optim.Adam(pipe.parameters(), lr=1e-3)
    poses, focal = torch.randn(3, 3, 4, device=DEV), torch.ones(3, device=DEV) * 500
    image = torch.rand(3, 6, 10, 3, device=DEV)
    for _ in range(3):
        opt.zero_grad()
        p = pipe(poses=poses, focal_lengths=focal, image_rgb=image, evaluation_mode=EM.TRAINING,
                 image_ids=torch.tensor([0, 3, 4], device=DEV))
        p["objective"].mean().backward()
        opt.step()
    now = pipe.feature_extractors[0].table.detach()
    moved = (now != start).any(1).tolist()
    assert moved == [True, False, False, False, True, False]
    assert torch.isfinite(now).all()
