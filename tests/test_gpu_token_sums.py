"""Sums that can be told exactly: whole numbers, which fp32 adds up without rounding below 2^24, against sums in 64-bit whole numbers; and what is
dropped at either end of the thresholds."""

import functools

import pytest
import torch

from tests import token_oracle as T

pytestmark = pytest.mark.gpu


def whole(shape, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-8, 9, shape, generator=g).to(dtype).cuda()


def ids_of(kind, n, rows, seed):
    g = torch.Generator().manual_seed(seed)
    if kind == "one":
        ids = torch.full((n,), rows // 2)
    elif kind == "two":  # of one block of the sort each, in runs
        ids = (torch.arange(n) // 1000 % 2) * (rows - 1)
    else:  # half of one id, a tenth no token or behind the table, the others spread
        ids = torch.randint(0, rows, (n,), generator=g)
        u = torch.rand(n, generator=g)
        ids[u < 0.5] = 1
        ids[u > 0.9] = -5
        ids[u > 0.95] = rows
    return ids.cuda()


def exact(dy, ids, rows):
    """dy: whole numbers in 64 bits."""
    good = (ids >= 0) & (ids < rows)
    return torch.zeros((rows, dy.shape[1]), dtype=torch.int64, device="cuda").index_add_(0, ids[good], dy[good])


@functools.lru_cache(maxsize=4)
def kept(n, p, seed, offset):
    return torch.from_numpy(T.keep(n, p, seed, offset)).cuda()


@pytest.mark.parametrize("kind", ["one", "two", "mixed"])
@pytest.mark.parametrize("p", [0.0, 0.5])
@pytest.mark.parametrize("n,rows,dims", [(64, 30, (8, 9)), (65, 30, (8, 521)), (9001, 129, (72, 73)), (20_000, 30, (264, 33)), (65_536, 300, (40, 33)), (65_537, 30, (40, 33)), (200_003, 30, (16, 9)),
                                         (1_048_577, 500, (8, 9)), (9001, 300_000, (8, 9))])
def test_whole_numbers_are_added_up_exactly(n, rows, dims, p, kind):
    """At most 2^20 + 1 terms of at most 8, or half as many (and some) of 16: every partial sum is a whole number below 2^24."""
    import flashoptim_jax_b200 as fo

    ids = ids_of(kind, n, rows, n)
    for dim in dims:
        dy, old = whole((n, dim), n + dim), whole((rows, dim), dim)
        seen = dy.long()
        if p:
            seen = torch.where(kept(n * dim, p, 5, 6).view(n, dim), 2 * seen, 0)
        size = exact(seen.abs(), ids, rows)
        assert int(size.max()) + 8 < 2**24
        want = exact(seen, ids, rows)
        assert torch.equal(fo.embed_grad(dy, ids, rows, p=p, seed=5, offset=6).long(), want)
        out = old.clone()
        fo.embed_grad(dy, ids, rows, p=p, seed=5, offset=6, out=out, accumulate=True)
        assert torch.equal(out.long(), want + old.long())
        # 16-bit gradients hold them as well; the sums stay in fp32
        assert torch.equal(fo.embed_grad(dy.bfloat16(), ids.int(), rows, p=p, seed=5, offset=6, dtype=torch.float32).long(), want)


@pytest.mark.parametrize("p", [1e-5, 2.0**-32, 2.0**-33, 2.0**-16, 65535 / 65536, 65535.5 / 65536, 1 - 2.0**-32, 1 - 2.0**-33, 1 - 2.0**-20])
def test_what_is_dropped_at_the_ends_of_the_thresholds(p):
    """Upper halves of the threshold that are all zeros or all ones, where ties decide most or all, and thresholds of one and of all but one."""
    import flashoptim_jax_b200 as fo

    n, seed, offset = 1 << 22, 11, 12
    want = kept(n, p, seed, offset)
    ones = torch.ones(n, device="cuda")
    assert torch.equal(fo.dropout(ones, p, seed, offset) != 0, want)
    assert torch.equal(fo.dropout(ones.half()[1:], p, seed, offset) != 0 if p < 0.99 else fo.dropout(ones[1:], p, seed, offset) != 0, want[:-1])  # not aligned
    for rows, dim in ((64, 1 << 16), (65, 64_520), (64, 65_533), (65, 64_523), (8192, 512), (8191, 511)):
        count = rows * dim
        mask = want[:count].view(rows, dim)
        ids = torch.randperm(rows, generator=torch.Generator().manual_seed(rows)).cuda()
        table = torch.ones((rows, dim), device="cuda")
        assert torch.equal(fo.embed(table, ids, p=p, seed=seed, offset=offset) != 0, mask)
        got = fo.embed_grad(table, ids, rows, p=p, seed=seed, offset=offset)
        assert torch.equal(got[ids] != 0, mask)


def test_a_captured_step_on_token_gradients():
    """tx.step with tokens in a CUDA graph, replayed with other ids, rows and offsets, against the same steps without a graph."""
    import flashoptim_jax_b200 as fo
    from flashoptim_jax_b200 import tree as pytree

    n, rows, dim = 300, 500, 72

    def start():
        g = torch.Generator().manual_seed(1)
        p = {"head": (torch.randn((dim, 16), generator=g) * 0.02).bfloat16().cuda(), "wte": (torch.randn((rows, dim), generator=g) * 0.02).bfloat16().cuda()}
        tx = fo.flash_adamw(learning_rate=1e-2, capturable=True, donate=True)
        return tx, p, tx.init(p)

    def inputs(k):
        g = torch.Generator().manual_seed(100 + k)
        return (torch.randint(-1, rows, (n,), generator=g).cuda(), torch.randn((n, dim), generator=g).bfloat16().cuda(), torch.randn((dim, 16), generator=g).bfloat16().cuda())

    tx, p, s = start()
    eager = []
    for k in range(5):
        ids, dy, head = inputs(k)
        p, s = tx.step(p, s, {"head": head, "wte": fo.TokenGradient(dy, ids, scale=2.0, p=0.25, seed=3, offset=k)})
        eager.append([x.clone() for x in pytree.tree_leaves((p, s))])

    tx, p, s = start()
    ids, dy, head = inputs(0)
    at = torch.zeros((), dtype=torch.int64, device="cuda")
    grads = {"head": head, "wte": fo.TokenGradient(dy, ids, scale=2.0, p=0.25, seed=3, offset=at)}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        p, s = tx.step(p, s, grads)  # the first step, eagerly
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(pytree.tree_leaves((p, s)), eager[0]):
        assert torch.equal(x, y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p2, s2 = tx.step(p, s, grads)
    for x, y in zip(pytree.tree_leaves(p), pytree.tree_leaves(p2)):
        assert x.data_ptr() == y.data_ptr()  # in place
    for k in range(1, 5):
        for mine, theirs in zip((ids, dy, head), inputs(k)):
            mine.copy_(theirs)
        at.fill_(k)
        graph.replay()
        for x, y in zip(pytree.tree_leaves((p2, s2)), eager[k]):
            assert torch.equal(x, y), k


@pytest.mark.parametrize("p", [0.0, 0.5])
@pytest.mark.parametrize("n", [64, 65, 9000])
def test_rows_are_cleared_behind_the_reach_of_32_bits(n, p):
    """A gradient of 2.2e9 elements, 4.4 GB: every row without a token is cleared, every other one written, wherever it lies."""
    import flashoptim_jax_b200 as fo

    rows, dim = 540_000, 4104
    ids = torch.linspace(0, rows - 1, n, dtype=torch.float64).round().long().cuda()
    dy = (whole((n, 1), n) + 20.0).expand(n, dim).bfloat16()  # no zeros
    out = torch.full((rows, dim), 9.0, dtype=torch.bfloat16, device="cuda")
    fo.embed_grad(dy, ids, rows, p=p, seed=1, out=out)
    want = fo.dropout(dy, p, 1)
    assert torch.equal(out[ids], want)
    out[ids] = 0
    assert not out.any()
