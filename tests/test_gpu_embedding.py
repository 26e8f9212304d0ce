"""Embedding lookup, its gradient by sorted tokens and dropout on the GPU, against their definitions in 64 bits.

Tolerances are sums of roundings, U = 2^-24 being half a step of fp32 and `half(t)` half a step of the result's type:
a looked-up or dropped element is weight x factor (the factor rounded once, the product once) rounded to the type; a sum of k such
elements in fp32 is off by at most (k + 2) U times the sum of their sizes, whatever the order."""

import ctypes
import math

import numpy as np
import pytest
import torch

from tests import token_oracle as T

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = 2.0**-24


def half(dtype):
    return torch.finfo(dtype).eps / 2


def smallest_half(dtype):
    """Half the distance between the smallest values of a type: what rounding a subnormal result may cost."""
    return {torch.float32: 2.0**-150, torch.bfloat16: 2.0**-134, torch.float16: 2.0**-25}[dtype]


def f64(t):
    return t.detach().to(torch.float64).cpu().numpy()


def element_close(got, want, dtype, terms=2):
    """`terms` roundings in fp32 and one to the result's type."""
    got = f64(got)
    assert got.shape == want.shape
    assert np.array_equal(np.isnan(got), np.isnan(want))
    bound = np.abs(want) * (terms * U + half(dtype)) * (1 + 2.0**-6) + smallest_half(dtype)
    bad = ~np.isnan(want) & ~(np.abs(got - want) <= bound)
    assert not bad.any(), (int(bad.sum()), got[bad][:4], want[bad][:4])


def rand(shape, dtype, seed, std=1.0, nonzero=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * std
    if nonzero:
        x = torch.where(x.abs() < 0.01 * std, torch.full_like(x, std), x)
    return x.to(dtype).cuda()


# ---- dropout ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [0, 1, 7, 8, 9, 1000, 8192 * 3 + 5, 1_000_003])
@pytest.mark.parametrize("p", [0.0, 0.1, 1 / 3, 0.999, 1.0])
def test_dropout_elements(dtype, n, p):
    import flashoptim_jax_b200 as fo

    dt, seed, offset = DTYPES[dtype], 2**63 + 12345, 2**40 + n
    x = rand((n,), dt, n, nonzero=True)
    y = fo.dropout(x, p, seed, offset)
    assert y.dtype == dt and y.shape == x.shape
    want = T.dropout(f64(x), p, seed, offset)
    assert np.array_equal(f64(y) != 0, want != 0)  # the same elements, all of them
    element_close(y, want, dt)
    if p == 0.0:
        assert torch.equal(x, y)
    r = rand((n,), dt, n + 1)
    z = f64(fo.dropout(x, p, seed, offset, residual=r))
    want = want + f64(r)
    # factor, product and sum in fp32: relative to the parts, not to what is left of them
    bound = (np.abs(want - f64(r)) * 2 * U + np.abs(want) * (U + half(dt))) * (1 + 2.0**-6) + smallest_half(dt)
    assert (np.abs(z - want) <= bound).all()


def test_ties_of_the_upper_half_are_settled_by_the_lower():
    """p = (h + 1/2) / 2^16: of the elements whose upper 16 bits are h, half stay.  A million elements have some sixteen of them."""
    import flashoptim_jax_b200 as fo

    n, p = 4_000_000, (20000 + 0.5) / 65536
    u = T.uniform32(n, 5, 6)
    ties = (u >> np.uint64(16)) == 20000
    kept = f64(fo.dropout(torch.ones(n, device="cuda"), p, 5, 6)) != 0
    assert np.array_equal(kept, T.keep(n, p, 5, 6))
    assert kept[ties].any() and not kept[ties].all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_dropped_elements_are_zero_whatever_they_held(dtype):
    import flashoptim_jax_b200 as fo

    dt, n = DTYPES[dtype], 10007
    for bad in (math.inf, -math.inf, math.nan):
        y = f64(fo.dropout(torch.full((n,), bad, dtype=dt, device="cuda"), 0.5, 1, 2))
        k = T.keep(n, 0.5, 1, 2)
        assert (y[~k] == 0).all() and np.array_equal(np.isnan(y[k]), np.full(k.sum(), math.isnan(bad)))


@pytest.mark.parametrize("dtype", DTYPES)
def test_dropout_of_views(dtype):
    import flashoptim_jax_b200 as fo

    dt = DTYPES[dtype]
    base = rand((4 * 1031 + 3,), dt, 3, nonzero=True)
    for x in (base[1:], base[3:1004], base[: 4 * 1031].view(4, 1031).t(), base[::2], base[5:6].expand(77)):
        r = rand(tuple(x.shape), dt, 4)
        want = T.dropout(f64(x), 0.3, 9, 1)
        element_close(fo.dropout(x, 0.3, 9, 1), want, dt)
        one = fo.dropout(x.contiguous().clone(), 0.3, 9, 1, residual=r)
        assert torch.equal(one, fo.dropout(x, 0.3, 9, 1, residual=r))
        assert torch.equal(one, fo.dropout(x, 0.3, 9, 1, residual=torch.cat([r.reshape(-1)[:1], r.reshape(-1)])[1:].view(x.shape)))


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_an_offset_on_the_device(dtype):
    import flashoptim_jax_b200 as fo

    x = rand((5000,), torch.bfloat16, 1)
    table, ids = rand((50, 16), torch.float32, 2), torch.arange(40, device="cuda")
    dy = rand((40, 16), torch.float32, 3)
    for value in (0, 7, -1, 2**31 - 1) + ((2**40 + 5,) if dtype == torch.int64 else ()):
        at = torch.full((), value, dtype=dtype, device="cuda")
        assert torch.equal(fo.dropout(x, 0.5, 3, at), fo.dropout(x, 0.5, 3, value))
        assert torch.equal(fo.embed(table, ids, p=0.5, seed=3, offset=at), fo.embed(table, ids, p=0.5, seed=3, offset=value))
        assert torch.equal(fo.embed_grad(dy, ids, 50, p=0.5, seed=3, offset=at), fo.embed_grad(dy, ids, 50, p=0.5, seed=3, offset=value))
    assert not torch.equal(fo.dropout(x, 0.5, 3, 1), fo.dropout(x, 0.5, 3, 2))


def test_dropout_in_place_through_the_library():
    from flashoptim_jax_b200 import _lib
    import flashoptim_jax_b200 as fo

    for n in (1005, 300_001):
        for shift in (0, 1):
            x, r = rand((n + shift,), torch.float16, 1)[shift:], rand((n + shift,), torch.float16, 2)[shift:]
            want = fo.dropout(x, 0.25, 11, 12, residual=r)
            f = _lib.FoDropout(p=0.25, seed=11, offset=12)
            for into in (x.clone(), r.clone()):
                a, b = (into, r) if torch.equal(into, x) else (x, into)
                _lib.check(_lib.lib().fo_dropout(a.data_ptr(), b.data_ptr(), into.data_ptr(), _lib.FO_F16, n, ctypes.byref(f), torch.cuda.current_stream().cuda_stream))
                assert torch.equal(into, want)


# ---- lookup ----------------------------------------------------------------------------------------------------------
def some_ids(shape, rows, seed, dtype=torch.int64, odd=True):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, max(1, rows), shape, generator=g)
    if odd and ids.numel() > 4:
        flat = ids.reshape(-1)
        flat[::7] = -1
        flat[3] = rows - 1
        flat[2] = 0
    return ids.to(dtype).cuda()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [1, 3, 8, 33, 64, 768, 1001])
@pytest.mark.parametrize("shape", [(0,), (), (1,), (3, 5), (701,)])
def test_embed_rows(dtype, dim, shape):
    import flashoptim_jax_b200 as fo

    dt, rows = DTYPES[dtype], 53
    table = rand((rows, dim), dt, dim)
    ids = some_ids(shape, rows, dim, torch.int32 if dim % 2 else torch.int64)
    at, w = ids.cpu().numpy(), f64(table)
    y = fo.embed(table, ids)
    assert y.dtype == dt and y.shape == (*shape, dim)
    assert np.array_equal(f64(y), T.embed(w, at))  # nothing to round
    y = fo.embed(table, ids, dtype=torch.float32)
    assert y.dtype == torch.float32 and np.array_equal(f64(y), T.embed(w, at))
    element_close(fo.embed(table, ids, scale=math.sqrt(dim)), T.embed(w, at, math.sqrt(dim)), dt)
    y = fo.embed(table, ids, scale=-1.7, p=0.3, seed=4, offset=dim)
    element_close(y, T.embed(w, at, -1.7, 0.3, 4, dim), dt)
    # the lookup's dropout is dropout's
    assert torch.equal(fo.embed(table, ids, p=0.3, seed=4, offset=5), fo.dropout(fo.embed(table, ids), 0.3, 4, 5))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("bits", [24, 32])
@pytest.mark.parametrize("dim", [5, 64, 1001])
def test_embed_of_master_weights(dtype, bits, dim):
    import flashoptim_jax_b200 as fo

    dt = DTYPES[dtype]
    theta = rand((91, dim), torch.float32, dim, std=0.02)
    theta[3] = 0.0
    theta[4, 0], theta[5] = 1e-39, 1e-6
    lp, ecc = fo.split_leaf(theta, dt, bits)
    ids = some_ids((211,), 91, 1)
    master = fo.reconstruct_leaf(lp, ecc)
    y = fo.embed(lp, ids, ecc=ecc)
    assert y.dtype == torch.float32
    some = ids >= 0
    assert torch.equal(y[some], master[ids[some]]) and not y[~some].any()
    element_close(fo.embed(lp, ids, ecc=ecc, dtype=dt), T.embed(f64(master), ids.cpu().numpy()), dt)
    element_close(fo.embed(lp, ids, ecc=ecc, scale=3.3, p=0.2, seed=1), T.embed(f64(master), ids.cpu().numpy(), 3.3, 0.2, 1), torch.float32)
    # the marker of a leaf without codes
    assert torch.equal(fo.embed(lp, ids, ecc=torch.zeros((), dtype=torch.int32, device="cuda")), fo.embed(lp, ids))


@pytest.mark.parametrize("dtype", DTYPES)
def test_ids_outside_the_table_read_nothing(dtype):
    import flashoptim_jax_b200 as fo

    for dim in (7, 64):
        table = rand((10, dim), DTYPES[dtype], 1)
        ids = torch.tensor([0, 9, 10, -1, 2**31 - 1, -(2**31), 2**62, -(2**62), 5], device="cuda")
        y = fo.embed(table, ids)
        assert np.array_equal(f64(y), T.embed(f64(table), ids.cpu().numpy()), equal_nan=True)
        assert torch.isnan(y[[2, 4, 6]]).all()
        g = fo.embed_grad(torch.ones(9, dim, device="cuda"), ids, 10)
        assert np.array_equal(f64(g)[:, 0], [1, 0, 0, 0, 0, 1, 0, 0, 0, 1])
        empty = fo.embed(table[:0], ids)
        assert torch.isnan(empty[ids >= 0]).all() and not empty[ids < 0].any()


def test_embed_of_strided_tables():
    import flashoptim_jax_b200 as fo

    wide = rand((40, 100), torch.bfloat16, 1)
    ids = some_ids((33,), 40, 2)
    for table in (wide[:, :64], wide[:, 8:72], wide[:, 3:67], wide[::3][:14, :64], wide.t()[:40], wide[:1].expand(40, 100), wide[:, :1], wide[:, ::2]):
        at = ids % table.shape[0]
        assert torch.equal(fo.embed(table, at), fo.embed(table.contiguous(), at))
    codes = torch.randint(-127, 128, (40, 100), device="cuda", dtype=torch.int8)
    for lo in (0, 8, 4, 3):
        got = fo.embed(wide[:, lo:lo + 64], ids, ecc=codes[:, lo:lo + 64])
        assert torch.equal(got, fo.embed(wide[:, lo:lo + 64].contiguous(), ids, ecc=codes[:, lo:lo + 64].contiguous()))
    two = ids.reshape(3, 11).t()
    assert torch.equal(fo.embed(wide, two), fo.embed(wide, two.contiguous()))


# ---- gradient --------------------------------------------------------------------------------------------------------
def check_grad(got, dy, ids, rows, dtype, scale=1.0, p=0.0, seed=0, offset=0, before=None):
    total, size, count = T.embed_grad(f64(dy), ids.cpu().numpy(), rows, scale, p, seed, offset)
    got = f64(got)
    old = 0.0 if before is None else f64(before)
    want = total + old
    k = count[:, None] + (0 if before is None else 1)
    bound = ((k + 2) * U * (size + np.abs(old)) + np.abs(want) * half(dtype)) * (1 + 2.0**-6) + smallest_half(dtype)
    if before is not None:  # rows without a token are as they were
        assert np.array_equal(got[count == 0], old[count == 0])
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4], got[bad][:4], want[bad][:4])


def ids_of(kind, n, rows, seed):
    g = torch.Generator().manual_seed(seed)
    if kind == "uniform":
        ids = torch.randint(0, rows, (n,), generator=g)
    elif kind == "text":  # 1 / rank
        ids = (torch.rand(n, generator=g, dtype=torch.float64) * math.log(rows + 1)).exp().long() - 1
    elif kind == "one":
        ids = torch.full((n,), rows // 2)
    elif kind == "none":
        ids = torch.full((n,), -1)
    else:  # most of one id, some of none, some behind the table
        ids = torch.randint(0, rows, (n,), generator=g)
        u = torch.rand(n, generator=g)
        ids[u < 0.5] = 1
        ids[u > 0.9] = -5
        ids[u > 0.95] = rows
    return ids.clamp(max=rows).cuda()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["uniform", "text", "one", "none", "mixed"])
@pytest.mark.parametrize("n,rows,dim", [(0, 5, 8), (1, 1, 1), (2, 300, 33), (33, 700, 256), (64, 9000, 5), (65, 40, 520), (257, 64, 1001), (1000, 50, 24), (4099, 5000, 264), (9001, 129, 72)])
def test_embed_grad_rows(dtype, kind, n, rows, dim):
    import flashoptim_jax_b200 as fo

    dt = DTYPES[dtype]
    ids = ids_of(kind, n, rows, n + rows)
    if n % 2:
        ids = ids.int()
    dy = rand((n, dim), dt, n + dim)
    got = fo.embed_grad(dy, ids, rows)
    assert got.dtype == dt and got.shape == (rows, dim)
    check_grad(got, dy, ids, rows, dt)
    assert torch.equal(got, fo.embed_grad(dy, ids, rows))  # same inputs, same bits
    other = torch.bfloat16 if dt == torch.float32 else torch.float32
    check_grad(fo.embed_grad(dy, ids, rows, dtype=other, scale=2.7, p=0.4, seed=8, offset=n), dy, ids, rows, other, 2.7, 0.4, 8, n)
    before = rand((rows, dim), dt, 5)
    out = before.clone()
    assert fo.embed_grad(dy, ids, rows, out=out, accumulate=True) is out
    check_grad(out, dy, ids, rows, dt, before=before)
    out.fill_(math.nan)
    assert torch.equal(fo.embed_grad(dy, ids, rows, out=out), got)


@pytest.mark.parametrize("kind", ["uniform", "text", "one", "mixed"])
@pytest.mark.parametrize("n,rows,dim", [(65536, 1000, 8), (65537, 1000, 8), (70001, 300_000, 16), (200_003, 30, 9)])
def test_embed_grad_of_many_tokens(kind, n, rows, dim):
    import flashoptim_jax_b200 as fo

    ids, dy = ids_of(kind, n, rows, 1), rand((n, dim), torch.bfloat16, 2)
    got = fo.embed_grad(dy, ids, rows, dtype=torch.float32)
    check_grad(got, dy, ids, rows, torch.float32)
    assert torch.equal(got, fo.embed_grad(dy, ids, rows, dtype=torch.float32))
    before = rand((rows, dim), torch.float32, 3)
    check_grad(fo.embed_grad(dy, ids, rows, out=before.clone(), accumulate=True, p=0.25, seed=2), dy, ids, rows, torch.float32, p=0.25, seed=2, before=before)


@pytest.mark.parametrize("n,rows,dim", [(8192, 262_143, 8), (8193, 262_143, 8), (100, 262_144, 8), (8193, 262_144, 8), (30_000, 3, 300), (5000, 127, 16), (5000, 129, 16),
                                        (20_000, 1, 520), (65, 70_000, 3), (2048, 2048, 2048), (65_537, 212_991, 8), (65_537, 212_992, 8), (1_048_577, 500, 8)])
def test_embed_grad_where_the_ways_to_sort_meet(n, rows, dim):
    import flashoptim_jax_b200 as fo

    for kind in ("uniform", "text", "mixed"):
        ids, dy = ids_of(kind, n, rows, 7), rand((n, dim), torch.float16, 8)
        got = fo.embed_grad(dy, ids, rows, scale=0.5)
        check_grad(got, dy, ids, rows, torch.float16, scale=0.5)
        assert torch.equal(got, fo.embed_grad(dy, ids, rows, scale=0.5))


@pytest.mark.parametrize("seed", range(24))
def test_random_sizes(seed):
    """Sizes spread over three orders of magnitude, odd and even widths, every type, dropout, views into larger buffers."""
    import random

    import flashoptim_jax_b200 as fo

    rng = random.Random(seed)

    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    dt = rng.choice(list(DTYPES.values()))
    dim = rng.choice([8 * log(1, 100), log(1, 900)])
    rows, n = log(1, 20_000), log(1, min(30_000, 6_000_000 // dim))
    p, scale, offset = rng.choice([0.0, 0.1, 0.77]), rng.choice([1.0, -3.7]), rng.randrange(2**40)
    pad = rng.choice([0, 0, 1, 5])
    ids = ids_of(rng.choice(["uniform", "text", "mixed"]), n, rows, seed)
    dy = rand((n, dim + pad), dt, seed)[:, pad // 2:pad // 2 + dim]
    check_grad(fo.embed_grad(dy, ids, rows, scale=scale, p=p, seed=seed, offset=offset), dy, ids, rows, dt, scale, p, seed, offset)
    before = rand((rows, dim), torch.float32, seed + 1)
    got = fo.embed_grad(dy, ids, rows, scale=scale, p=p, seed=seed, offset=offset, out=before.clone(), accumulate=True)
    check_grad(got, dy, ids, rows, torch.float32, scale, p, seed, offset, before=before)
    table = rand((rows, dim + pad), dt, seed + 2)[:, pad // 2:pad // 2 + dim]
    y = fo.embed(table, ids, scale=scale, p=p, seed=seed, offset=offset)
    element_close(y, T.embed(f64(table), ids.cpu().numpy(), scale, p, seed, offset), dt)
    element_close(fo.dropout(dy, p, seed, offset), T.dropout(f64(dy), p, seed, offset), dt)


@pytest.mark.parametrize("n", [5, 3000, 80_000])
def test_untouched_rows_keep_their_bits(n):
    import flashoptim_jax_b200 as fo

    rows, dim = 4000, 40
    ids = torch.randint(0, 100, (n,), device="cuda") * 2
    out = torch.full((rows, dim), math.nan, dtype=torch.bfloat16, device="cuda")
    out[0:200:2] = 0
    fo.embed_grad(torch.ones(n, dim, dtype=torch.bfloat16, device="cuda"), ids, rows, out=out, accumulate=True)
    assert torch.isnan(out[1:200:2]).all() and torch.isnan(out[200:]).all()
    assert torch.equal(out[0:200:2, 0].float(), torch.bincount(ids, minlength=200)[0:200:2].bfloat16().float())


def test_embed_grad_of_views():
    import flashoptim_jax_b200 as fo

    wide = rand((301, 200), torch.bfloat16, 1)
    ids = some_ids((301,), 40, 2)
    for dy in (wide[:, :128], wide[:, 8:136], wide[:, 5:133], wide[:1, :64].expand(301, 64), wide[:, ::2], rand((64, 301), torch.bfloat16, 3).t()):
        assert torch.equal(fo.embed_grad(dy, ids, 40, p=0.1, seed=1), fo.embed_grad(dy.contiguous(), ids, 40, p=0.1, seed=1))
    flat = torch.zeros(40 * 64 + 9, dtype=torch.bfloat16, device="cuda")
    for at in (0, 1, 8):  # a leaf of a flat gradient buffer
        flat.fill_(7.0)
        leaf = flat[at:at + 40 * 64].view(40, 64)
        want = fo.embed_grad(wide[:, :64], ids, 40)
        fo.embed_grad(wide[:, :64], ids, 40, out=leaf)
        assert torch.equal(leaf, want) and (flat[:at] == 7).all() and (flat[at + 40 * 64:] == 7).all()
    three = wide[:300, :64].reshape(3, 100, 64)
    assert torch.equal(fo.embed_grad(three, ids[:300].reshape(3, 100), 40), fo.embed_grad(wide[:300, :64], ids[:300], 40))
    assert torch.equal(fo.embed_grad(wide[0, :64], ids[1], 40), fo.embed_grad(wide[:1, :64], ids[1:2], 40))


def test_tables_and_rows_behind_the_reach_of_32_bits():
    import flashoptim_jax_b200 as fo

    rows, dim = 540_000, 4104  # 2.2e9 elements, 4.4 GB
    table = torch.zeros((rows, dim), dtype=torch.bfloat16, device="cuda")
    at = [0, 1, 523_000, 523_265, 539_998, 539_999]
    table[at] = rand((6, dim), torch.bfloat16, 1)
    ids = torch.tensor([*at, *at[::-1]], device="cuda")
    y = fo.embed(table, ids)
    assert torch.equal(y, table[ids])
    table.fill_(9.0)
    fo.embed_grad(y, ids, rows, out=table)
    assert torch.equal(table[at], (2 * y[:6].float()).bfloat16())
    assert table.count_nonzero(1).nonzero()[:, 0].tolist() == at
    fo.embed_grad(y, ids, rows, out=table, accumulate=True)
    assert torch.equal(table[at], (4 * y[:6].float()).bfloat16())
    del table
    big = torch.zeros((rows, dim), dtype=torch.bfloat16, device="cuda")  # as activations
    big[at] = rand((6, dim), torch.bfloat16, 1)
    ids = torch.full((rows,), -1, device="cuda")
    ids[at] = torch.tensor([3, 1, 2, 2, 0, 3], device="cuda")
    grad = fo.embed_grad(big, ids, 4, dtype=torch.float32)
    x = big[at].float()
    assert torch.equal(grad, torch.stack([x[4], x[1], x[2] + x[3], x[0] + x[5]]))
    z = fo.dropout(big, 0.5, 1, 2)
    assert z.count_nonzero(1).nonzero()[:, 0].tolist() == at


# ---- gradients, graphs, streams --------------------------------------------------------------------------------------
def test_autograd_gives_the_gradients_by_hand():
    import flashoptim_jax_b200 as fo

    for dt in DTYPES.values():
        table = rand((60, 40), dt, 1).requires_grad_()
        ids, dy, r = some_ids((9, 11), 60, 2), rand((9, 11, 40), dt, 3), rand((9, 11, 40), dt, 4).requires_grad_()
        x = fo.embed(table, ids, scale=1.5, p=0.2, seed=7, offset=8)
        y = fo.dropout(x, 0.3, 9, 10, residual=r)
        g_table, g_r = torch.autograd.grad(y, (table, r), dy)
        assert torch.equal(g_r, dy)
        dx = fo.dropout(dy, 0.3, 9, 10)
        assert torch.equal(g_table, fo.embed_grad(dx, ids, 60, scale=1.5, p=0.2, seed=7, offset=8)) and g_table.dtype == dt
    with torch.no_grad():
        assert not fo.embed(table, ids).requires_grad
    # gradients that are no plain matrix: broadcast by a sum, transposed by what comes behind
    (g,) = torch.autograd.grad(fo.embed(table, ids).sum(), table)
    assert torch.equal(g, fo.embed_grad(torch.ones(9, 11, 40, dtype=dt, device="cuda"), ids, 60))
    (g,) = torch.autograd.grad(fo.embed(table, ids[0]).t().contiguous(), table, dy[0].t().contiguous())
    assert torch.equal(g, fo.embed_grad(dy[0], ids[0], 60))
    # master weights: the gradient is the weights', in the parameters' type
    lp = rand((60, 40), torch.bfloat16, 5).requires_grad_()
    out = fo.embed(lp, ids, ecc=torch.zeros((60, 40), dtype=torch.int8, device="cuda"))
    (g,) = torch.autograd.grad(out, lp, dy.float())
    assert out.dtype == torch.float32 and g.dtype == torch.bfloat16
    with pytest.raises(RuntimeError):  # once differentiable
        x = fo.dropout(r, 0.5, 1)
        (g,) = torch.autograd.grad((x * x).sum(), r, create_graph=True)
        torch.autograd.grad(g.sum(), r)


def test_gradients_against_differences():
    """The loss is linear in table and residual, so the difference quotient is the gradient but for the roundings of both losses."""
    import flashoptim_jax_b200 as fo

    table, ids = rand((30, 24), torch.float32, 1).requires_grad_(), some_ids((50,), 30, 2)
    weight, r = rand((50, 24), torch.float32, 3), rand((50, 24), torch.float32, 4).requires_grad_()

    def loss(t, s):
        return (fo.dropout(fo.embed(t, ids, scale=2.0, p=0.25, seed=1), 0.5, 2, residual=s).double() * weight.double()).sum()

    grads = torch.autograd.grad(loss(table, r), (table, r))
    step = 2.0**-3
    for k, (x, g) in enumerate(zip((table, r), grads)):
        d = torch.sign(rand(tuple(x.shape), torch.float32, 5 + k, nonzero=True))
        with torch.no_grad():
            moved = [x + step * d if j == k else y for j, y in enumerate((table, r))]
            slope = (loss(*moved) - loss(table, r)) / step
        want = (g.double() * d.double()).sum()
        # each output: |x| + step <= 8, times 2 / 0.75 / 0.5, plus a residual of at most 8; some six roundings in each loss, and in the
        # gradient's elements sums of at most 50 terms
        size = float(weight.abs().double().sum()) * (8 * 2 / 0.75 / 0.5 + 8)
        assert abs(float(slope - want)) <= 6 * 2 * U * size / step + 60 * U * size


def test_a_captured_run_of_lookup_dropout_and_gradient():
    import flashoptim_jax_b200 as fo

    for n in (64, 2000, 70_000):
        table, ids = rand((500, 64), torch.bfloat16, 1), some_ids((n,), 500, 2)
        dy, head = rand((n, 64), torch.bfloat16, 3), rand((500, 64), torch.bfloat16, 4)
        at = torch.zeros((), dtype=torch.int64, device="cuda")
        tied = torch.empty_like(head)

        def run(offset):
            y = fo.dropout(fo.embed(table, ids, p=0.1, seed=1, offset=offset), 0.2, 2, offset)
            g = fo.embed_grad(fo.dropout(dy, 0.2, 2, offset), ids, 500, p=0.1, seed=1, offset=offset)
            tied.copy_(head)
            fo.embed_grad(dy, ids, 500, out=tied, accumulate=True)
            return y, g

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(at)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = run(at)
        other = torch.cuda.CUDAGraph()
        with torch.cuda.graph(other):
            more = run(at)
        for k in (3, 5):
            ids.copy_(some_ids((n,), 500, k))
            dy.copy_(rand((n, 64), torch.bfloat16, k))
            at.fill_(k)
            graph.replay()
            other.replay()
            graph.replay()
            y, g, t = [x.clone() for x in (*got, tied)]
            want = run(k)
            assert torch.equal(y, want[0]) and torch.equal(g, want[1]) and torch.equal(t, tied)
            assert torch.equal(more[0], y) and torch.equal(more[1], g)


def test_calls_on_two_streams_do_not_meet():
    import flashoptim_jax_b200 as fo

    cases = [(rand((n, 256), torch.bfloat16, n), ids_of("text", n, 3000, n)) for n in (3000, 5000, 66_000)]
    want = [fo.embed_grad(dy, ids, 3000) for dy, ids in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for _ in range(5):
        for (dy, ids), s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(fo.embed_grad(dy, ids, 3000))
    torch.cuda.synchronize()
    for k, g in enumerate(got):
        assert torch.equal(g, want[k % len(cases)])


def test_two_threads_at_once():
    import threading

    import flashoptim_jax_b200 as fo

    cases = [(rand((n, 264), torch.float32, n), ids_of("mixed", n, 900, n)) for n in (40, 3000, 20_000)]

    def work(dy, ids):
        y = fo.dropout(dy, 0.2, 1, 2)
        g = fo.embed_grad(y, ids, 900)
        return g, fo.embed(g, ids.clamp(max=899), p=0.1, seed=3)

    want = [work(*c) for c in cases]
    torch.cuda.synchronize()
    got, errors = {}, []

    def run(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[k] = work(*cases[k])
            torch.cuda.synchronize()
        except Exception as e:  # noqa: BLE001 (reported below)
            errors.append(e)

    threads = [threading.Thread(target=run, args=(k,)) for k in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for k, w in enumerate(want):
        assert all(torch.equal(x, y) for x, y in zip(got[k], w))


def test_dependent_calls_see_each_other():
    """Each call's input is what the one in front of it has just written, without a wait between them."""
    import flashoptim_jax_b200 as fo

    ids = ids_of("text", 4000, 2000, 1)

    def chain(pause):
        x = rand((2000, 128), torch.float32, 2, std=0.1)
        for k in range(6):
            y = fo.embed(x, ids, p=0.1, seed=k)
            pause()
            y = fo.dropout(y, 0.1, k, residual=y)
            pause()
            g = fo.embed_grad(y, ids, 2000, scale=0.01)
            pause()
            x = x - g
            pause()
            fo.embed_grad(y, ids, 2000, out=x, accumulate=True, scale=0.01, p=0.5, seed=k)
            pause()
        return x

    assert torch.equal(chain(lambda: None), chain(torch.cuda.synchronize))


# ---- with the optimizers ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("name", ["flash_adamw", "flash_lion", "flash_sgdw"])
@pytest.mark.parametrize("how", ["donated", "copied", "clipped", "captured"])
def test_a_step_on_token_gradients(name, how):
    """A step whose embedding leaf comes as tokens is, bit for bit, the step on the gradient that embed_grad makes; and the tree trains on:
    lookup on master weights, dropout, gradients, step."""
    import flashoptim_jax_b200 as fo
    from flashoptim_jax_b200 import clipping

    def tree():
        return {"wte": rand((300, 64), torch.bfloat16, 1, std=0.02), "head": {"w": rand((64, 32), torch.bfloat16, 2, std=0.02), "b": torch.zeros(32, device="cuda")}}

    def run(tokens):
        tx = getattr(fo, name)(learning_rate=1e-2, donate=how != "copied", capturable=how == "captured")
        if how == "clipped":
            tx = clipping.clip_by_global_norm(tx, 0.5)
        p = tree()
        s = tx.init(p)
        for k in range(4):
            ids = some_ids((7, 30), 300, k)
            ecc = (s["opt"] if how == "clipped" else s).ecc["wte"]
            x = fo.embed(p["wte"], ids, ecc=ecc, scale=8.0, p=0.1, seed=1, offset=k)
            dlogits = rand((7, 30, 32), torch.float32, k, std=0.1)
            grads = {"wte": fo.TokenGradient((dlogits @ p["head"]["w"].float().t()).bfloat16(), ids, scale=8.0, p=0.1, seed=1, offset=k),
                     "head": {"w": torch.einsum("btd,btv->dv", x, dlogits).bfloat16(), "b": dlogits.sum((0, 1))}}
            if not tokens:
                t = grads["wte"]
                grads["wte"] = fo.embed_grad(t.dy, t.ids, 300, scale=8.0, p=0.1, seed=1, offset=k)
            p, s = tx.step(p, s, grads)
        return p, s

    from flashoptim_jax_b200 import tree as pytree

    a, b = pytree.tree_leaves(run(True)), pytree.tree_leaves(run(False))
    assert len(a) == len(b)
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def test_a_sharded_step_on_token_gradients():
    """Zero1Optimizer on one rank: a TokenGradient goes straight into the flat gradient buffer."""
    import flashoptim_jax_b200 as fo
    from flashoptim_jax_b200 import tree as pytree
    from flashoptim_jax_b200.zero1 import Zero1Optimizer

    def params():
        return {"a": torch.ones(33, device="cuda"), "wte": rand((500, 70), torch.bfloat16, 1, std=0.02), "z": rand((11, 7), torch.bfloat16, 2)}

    one, two = (Zero1Optimizer("adamw", params(), learning_rate=1e-3, weight_decay=1e-2, master_weight_bits=32) for _ in range(2))
    for k in range(3):
        ids, dy = ids_of("mixed", 700, 500, k), rand((700, 70), torch.bfloat16, k)
        rest = {"a": rand((33,), torch.float32, k), "z": rand((11, 7), torch.bfloat16, k)}
        one.step({**rest, "wte": fo.TokenGradient(dy, ids, scale=2.0)})
        two.step({**rest, "wte": fo.embed_grad(dy, ids, 500, scale=2.0)})
    for x, y in zip(pytree.tree_leaves(one.params), pytree.tree_leaves(two.params)):
        assert torch.equal(x, y)
    with pytest.raises(TypeError, match="narrowed"):  # as for any other gradient
        one.step({**rest, "wte": fo.TokenGradient(dy.float(), ids)})


def test_a_token_gradient_for_the_wrong_leaf_is_refused():
    import flashoptim_jax_b200 as fo

    tx = fo.flash_adamw()
    p = {"a": rand((30, 8), torch.bfloat16, 1), "b": rand((8,), torch.bfloat16, 1)}
    s = tx.init(p)
    tokens = fo.TokenGradient(rand((4, 8), torch.bfloat16, 1), torch.arange(4, device="cuda"))
    with pytest.raises(ValueError, match="does not belong"):
        tx.step(p, s, {"a": p["a"], "b": tokens})
    with pytest.raises(ValueError, match="must match"):
        tx.step(p, s, {"a": tokens})


# ---- refusals --------------------------------------------------------------------------------------------------------
def test_refusals():
    import flashoptim_jax_b200 as fo

    t, ids = rand((10, 8), torch.bfloat16, 1), torch.arange(4, device="cuda")
    dy = rand((4, 8), torch.bfloat16, 2)
    with pytest.raises(ValueError, match="matrix"):
        fo.embed(t[0], ids)
    with pytest.raises(ValueError, match="matrix"):
        fo.embed(t.double(), ids)
    with pytest.raises(ValueError, match="int32 or int64"):
        fo.embed(t, ids.float())
    with pytest.raises(ValueError, match="int32 or int64"):
        fo.embed_grad(dy, ids.to(torch.uint8), 10)
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        fo.embed(t, ids.cpu())
    for ecc in (torch.zeros((10, 8), device="cuda"), torch.zeros((10, 7), dtype=torch.int8, device="cuda"), torch.zeros((10, 8), dtype=torch.int8)):
        with pytest.raises(ValueError, match="does not belong"):
            fo.embed(t, ids, ecc=ecc)
    with pytest.raises(ValueError, match="does not belong"):
        fo.embed(t.float(), ids, ecc=torch.zeros((10, 8), dtype=torch.int8, device="cuda"))
    with pytest.raises(ValueError, match="dtype"):
        fo.embed(t, ids, dtype=torch.float16)
    for p in (-0.1, 1.1, math.nan):
        with pytest.raises(ValueError, match="between 0 and 1"):
            fo.embed(t, ids, p=p)
        with pytest.raises(ValueError, match="between 0 and 1"):
            fo.embed_grad(dy, ids, 10, p=p)
        with pytest.raises(ValueError, match="between 0 and 1"):
            fo.dropout(t, p, 1)
    for scale in (math.inf, math.nan):
        with pytest.raises(ValueError, match="finite"):
            fo.embed(t, ids, scale=scale)
    for offset in (torch.zeros(2, dtype=torch.int64, device="cuda"), torch.zeros(1, device="cuda"), torch.zeros(1, dtype=torch.int64)):
        with pytest.raises(ValueError, match="offset"):
            fo.dropout(t, 0.5, 1, offset)
    with pytest.raises(ValueError, match="does not belong"):
        fo.embed_grad(dy[:3], ids, 10)
    with pytest.raises(ValueError, match="does not belong"):
        fo.embed_grad(dy, ids.view(2, 2), 10)
    with pytest.raises(ValueError, match="negative"):
        fo.embed_grad(dy, ids, -1)
    with pytest.raises(ValueError, match="accumulate"):
        fo.embed_grad(dy, ids, 10, accumulate=True)
    for out in (torch.zeros(10, 7, device="cuda"), torch.zeros(10, 8, device="cuda", dtype=torch.float64), torch.zeros(10, 8)):
        with pytest.raises((ValueError, RuntimeError)):
            fo.embed_grad(dy, ids, 10, out=out)
    with pytest.raises(ValueError, match="contiguous"):
        fo.embed_grad(dy, ids, 10, out=torch.zeros(8, 10, device="cuda").t())
    with pytest.raises(ValueError, match="not a gradient"):
        fo.embed_grad(dy, ids, 10, out=torch.zeros(10, 8, device="cuda"), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        fo.embed_grad(dy, ids, 10, dtype=torch.float64)
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        fo.dropout(ids, 0.5, 1)
    for r in (t[:5], t.float(), t.cpu()):
        with pytest.raises((ValueError, RuntimeError)):
            fo.dropout(t, 0.5, 1, residual=r)
    with pytest.raises(ValueError, match="rows"):
        fo.embed_grad(dy, ids, 2**31)
