"""Embedding lookup, its gradient and dropout in 64 bits on the CPU, from their definitions (include/flashoptim_b200.h)."""

import numpy as np

M32 = np.uint64(0xFFFFFFFF)


def philox4x32(counter, key, rounds=10):
    """Philox of Salmon et al. (2011): counter is four, key two uint64 arrays or numbers holding 32 bits each."""
    c = [np.asarray(x, dtype=np.uint64) for x in counter]
    k = [int(x) for x in key]
    for _ in range(rounds):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & M32, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & M32]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def uniform32(n, seed, offset):
    """The 32-bit number of each of n elements."""
    e = np.arange(n, dtype=np.uint64)
    block, j = e >> np.uint64(3), (e & np.uint64(7)).astype(np.int64)
    seed, offset = seed % 2**64, offset % 2**64
    halves = []
    for top in (0, 1 << 31):
        blocks = np.arange(int(block[-1]) + 1 if n else 0, dtype=np.uint64)
        w = philox4x32([blocks & M32, (blocks >> np.uint64(32)) | np.uint64(top), np.full_like(blocks, offset & 0xFFFFFFFF), np.full_like(blocks, offset >> 32)],
                       (seed & 0xFFFFFFFF, seed >> 32))
        w = np.stack(w, 1) if n else np.zeros((0, 4), np.uint64)
        word = w[block.astype(np.int64), j // 2]
        halves.append((word >> np.uint64(16) * (j % 2).astype(np.uint64)) & np.uint64(0xFFFF))
    return (halves[0] << np.uint64(16)) | halves[1]


def keep(n, p, seed, offset):
    return uniform32(n, seed, offset) >= np.uint64(int(p * 2.0**32 + 0.5))


def factor(p):
    return 1.0 / (1.0 - p) if p < 1.0 else 0.0


def dropout(x, p, seed, offset):
    """x: float64."""
    k = keep(x.size, p, seed, offset).reshape(x.shape)
    with np.errstate(invalid="ignore"):
        return np.where(k, x * factor(p), 0.0)


def embed(table, ids, scale=1.0, p=0.0, seed=0, offset=0):
    """table: float64 (rows, dim); NaN rows for ids behind the table, zeros for negative ones."""
    rows, dim = table.shape
    flat = np.asarray(ids).reshape(-1)
    y = np.zeros((flat.size, dim))
    good = (flat >= 0) & (flat < rows)
    y[good] = table[flat[good]] * scale
    y[flat >= rows] = np.nan
    return dropout(y, p, seed, offset).reshape(*np.shape(ids), dim)


def embed_grad(dy, ids, rows, scale=1.0, p=0.0, seed=0, offset=0):
    """(sum, sum of absolute values, number of tokens of each row): the gradient and what its rounding is measured by."""
    flat = np.asarray(ids).reshape(-1)
    dim = dy.shape[-1]
    dy = dropout(dy.reshape(flat.size, dim) * scale, p, seed, offset)
    total, size, count = np.zeros((rows, dim)), np.zeros((rows, dim)), np.zeros(rows, np.int64)
    good = np.nonzero((flat >= 0) & (flat < rows))[0]
    np.add.at(total, flat[good], dy[good])
    np.add.at(size, flat[good], np.abs(dy[good]))
    np.add.at(count, flat[good], 1)
    return total, size, count
